// Beam search's selection: log-probabilities of every beam over the vocabulary and, per prompt, the best candidates of all its beams.
//
// Reference: none (davidjoyme/mini-inference engine/core/sampler.py:3-11 knows argmax and a draw).  With logits x[r, v] and running scores s[r]
//     lse[r] = log sum_v e^x[r, v],   candidate (r, v) has the value (s[r] - lse[r]) + x[r, v],
// and a group of rows gives its `num` largest: by value, then the lower row, then the larger logit, then the lower token.  A row whose logits hold
// NaN or +inf or no finite number, or whose score is not finite, offers nothing, nor does a logit of -inf; places that stay empty hold (-inf, -1, -1).
//
// The order of two candidates is a whole number, so values are compared in float64 and the sum of exponentials is kept to about 1e-9: float32's 1e-7
// would swap two neighbours that lie 0.05 apart once in some hundred thousand pairs, a step of 64 beams has a thousand.  Within a row the logits
// themselves decide, exactly.
//
// Two launches.  beam_slice_kernel: a block takes a slice of one row into registers once, and leaves the slice's maximum, its sum of exponentials and
// its `num` largest logits in order.  The num-th largest of the threads' own maxima is a bound that at least num logits reach; what reaches it (a few
// more than num) goes to shared memory and every entry counts those before it.  Where more reach it than fit (many equal logits) the block picks num
// times the next one.  beam_merge_kernel: a block per group joins the slices' sums, and chooses among their candidates the same way.
#include "common.cuh"
#include <math.h>

using namespace mi;

namespace {

constexpr int NT = 256, CAP = 1024;                 // threads of a block (at least MAX_NUM); candidates that fit in shared memory
constexpr int MAX_NUM = 128;
typedef unsigned long long u64;

struct __align__(16) SliceSum { double sum; float top; int count; };

// larger logit first, then the lower token; 0 is below every candidate's key
__device__ __forceinline__ u64 logit_key(float v, int token) {
    uint32_t u = __float_as_uint(v);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((u64)u << 32) | (0xffffffffu - (uint32_t)token);
}
__device__ __forceinline__ float key_logit(u64 key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ int key_token(u64 key) { return (int)(0xffffffffu - (uint32_t)key); }

template <typename T> __device__ __forceinline__ T block_max(T v, T* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { const T w = __shfl_xor_sync(0xffffffffu, v, o); v = w > v ? w : v; }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int w = 0; w < NT / 32; ++w) v = scratch[w] > v ? scratch[w] : v;
    return v;
}
__device__ __forceinline__ double block_sum(double v, double* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.;
    for (int w = 0; w < NT / 32; ++w) v += scratch[w];
    return v;
}

// The num-th largest of the threads' values (num <= NT): at least num of what the threads hold reach it
template <typename T> __device__ __forceinline__ T threshold(T mine, int num, T* all, T* answer) {
    __syncthreads();
    all[threadIdx.x] = mine;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < NT; ++i) { const T o = all[i]; before += o > mine || (o == mine && i < threadIdx.x); }
    if (before == num - 1) *answer = mine;
    __syncthreads();
    return *answer;
}

// EPT logits a thread, four neighbours at a time
template <int EPT>
__global__ void __launch_bounds__(NT) beam_slice_kernel(const float* __restrict__ logits, long long ld, int vocab, int num, SliceSum* __restrict__ sums,
                                                        u64* __restrict__ keys) {
    __shared__ union { double d[NT / 32]; float f[NT / 32]; u64 u[NT / 32]; } scratch;
    __shared__ float maxima[NT], bound;
    __shared__ u64 found[CAP];
    __shared__ int count;
    pdl_trigger();
    pdl_wait(logits);
    const int r = blockIdx.y, slice = blockIdx.x, slices = gridDim.x, base = slice * NT * EPT;
    const float* row = logits + (long long)r * ld;
    const bool vec = ((uintptr_t)row & 15) == 0;
    float x[EPT];
#pragma unroll
    for (int k = 0; k < EPT / 4; ++k) {
        const int i = base + (k * NT + threadIdx.x) * 4;
        if (vec && i + 3 < vocab) {
            load16(row + i, x + 4 * k);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * k + e] = i + e < vocab ? row[i + e] : -INFINITY;
        }
    }
    float top = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
        bad |= !(x[e] < INFINITY);
        x[e] += 0.f;                                 // -0 is 0
        top = fmaxf(top, x[e]);
    }
    if (threadIdx.x == 0) count = 0;
    const float m = block_max(top, scratch.f);
    bad = __syncthreads_or(bad);
    SliceSum* out = sums + (size_t)r * slices + slice;
    if (bad || m == -INFINITY) {
        if (threadIdx.x == 0) *out = SliceSum{bad ? (double)NAN : 0., m, 0};
        return;
    }
    double sum = 0.;
#pragma unroll
    for (int e = 0; e < EPT; ++e) sum += exp((double)x[e] - (double)m);
    sum = block_sum(sum, scratch.d);

    const float least = threshold(top, num, maxima, &bound);
#pragma unroll
    for (int e = 0; e < EPT; ++e)
        if (x[e] >= least && x[e] > -INFINITY) {
            const int at = atomicAdd(&count, 1);
            if (at < CAP) found[at] = logit_key(x[e], base + ((e >> 2) * NT + threadIdx.x) * 4 + (e & 3));
        }
    __syncthreads();
    const int n = count;
    u64* best = keys + ((size_t)r * slices + slice) * num;
    if (n <= CAP) {
        for (int i = threadIdx.x; i < n; i += NT) {
            const u64 mine = found[i];
            int before = 0;
            for (int o = 0; o < n; ++o) before += found[o] > mine;
            if (before < num) best[before] = mine;
        }
    } else {
        u64 last = ~0ull;
        for (int k = 0; k < num; ++k) {
            u64 next = 0;
#pragma unroll
            for (int e = 0; e < EPT; ++e) {
                const u64 key = x[e] > -INFINITY ? logit_key(x[e], base + ((e >> 2) * NT + threadIdx.x) * 4 + (e & 3)) : 0;
                if (key < last && key > next) next = key;
            }
            last = block_max(next, scratch.u);
            if (threadIdx.x == 0) best[k] = last;
        }
    }
    if (threadIdx.x == 0) *out = SliceSum{sum, m, min(n, num)};
}

struct Candidate { double value; int row; u64 key; };
__device__ __forceinline__ bool goes_before(const Candidate& a, const Candidate& b) {
    return a.value != b.value ? a.value > b.value : a.row != b.row ? a.row < b.row : a.key > b.key;
}

__global__ void __launch_bounds__(NT) beam_merge_kernel(const SliceSum* sums, const u64* keys, int slices, int num, const float* __restrict__ scores, int rows,
                                                        const int* __restrict__ group_start, double* base, float* __restrict__ values, int* __restrict__ out_rows,
                                                        int* __restrict__ out_tokens) {
    __shared__ double maxima[NT], bound;
    __shared__ Candidate found[CAP];
    __shared__ Candidate warp_best[NT / 32];
    __shared__ int count;
    pdl_trigger();
    pdl_wait(scores, group_start);
    const int g = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int a = max(0, min(group_start[g], rows)), b = max(a, min(group_start[g + 1], rows));
    // s[r] - lse[r], a warp per row
    for (int r = a + warp; r < b; r += NT / 32) {
        const SliceSum* mine = sums + (size_t)r * slices;
        float m = -INFINITY;
        for (int i = lane; i < slices; i += 32) m = fmaxf(m, mine[i].top);
        m = warp_max(m);
        double sum = 0.;
        for (int i = lane; i < slices; i += 32) sum += mine[i].sum * (mine[i].top == -INFINITY ? 1. : exp((double)mine[i].top - (double)m));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const double v = (double)scores[r] - ((double)m + log(sum));
        if (lane == 0) base[r] = isfinite(v) ? v : -(double)INFINITY;
    }
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    // candidate i: row, slice, place in the slice's list
    const long long n = (long long)(b - a) * slices * num;
    auto at = [&](long long i) {
        const int list = (int)(i / num), k = (int)(i % num), r = a + list / slices;
        const size_t where = (size_t)r * slices + list % slices;
        Candidate c{-(double)INFINITY, r, 0};
        const double from = base[r];
        if (k < sums[where].count && from != -(double)INFINITY) {
            c.key = keys[where * num + k];
            c.value = from + (double)key_logit(c.key);
        }
        return c;
    };
    double top = -(double)INFINITY;
    for (long long i = threadIdx.x; i < n; i += NT) top = fmax(top, at(i).value);
    const double least = threshold(top, num, maxima, &bound);
    for (long long i = threadIdx.x; i < n; i += NT) {
        const Candidate c = at(i);
        if (c.value >= least && c.value > -(double)INFINITY) {
            const int p = atomicAdd(&count, 1);
            if (p < CAP) found[p] = c;
        }
    }
    __syncthreads();
    const int have = count;
    auto write = [&](int place, const Candidate& c) {
        const size_t o = (size_t)g * num + place;
        values[o] = (float)c.value; out_rows[o] = c.row; out_tokens[o] = key_token(c.key);
    };
    if (have <= CAP) {
        for (int i = threadIdx.x; i < have; i += NT) {
            const Candidate mine = found[i];
            int before = 0;
            for (int o = 0; o < have; ++o) before += goes_before(found[o], mine);
            if (before < num) write(before, mine);
        }
    } else {
        Candidate last{(double)INFINITY, -1, 0};
        for (int k = 0; k < num; ++k) {              // the first of those behind the last one
            Candidate next{-(double)INFINITY, 0x7fffffff, 0};
            for (long long i = threadIdx.x; i < n; i += NT) {
                const Candidate c = at(i);
                if (c.value >= least && c.value > -(double)INFINITY && goes_before(last, c) && goes_before(c, next)) next = c;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const Candidate w{__shfl_xor_sync(0xffffffffu, next.value, o), __shfl_xor_sync(0xffffffffu, next.row, o), __shfl_xor_sync(0xffffffffu, next.key, o)};
                if (goes_before(w, next)) next = w;
            }
            __syncthreads();
            if (lane == 0) warp_best[warp] = next;
            __syncthreads();
            last = warp_best[0];
            for (int w = 1; w < NT / 32; ++w) if (goes_before(warp_best[w], last)) last = warp_best[w];
            if (threadIdx.x == 0) write(k, last);
        }
    }
    for (int k = have + threadIdx.x; k < num; k += NT) {
        const size_t o = (size_t)g * num + k;
        values[o] = -INFINITY; out_rows[o] = -1; out_tokens[o] = -1;
    }
}

int slice_size(int rows, int vocab) {
    // enough blocks for two an SM where the logits allow it
    for (int ept : {32, 16})
        if ((long long)rows * ((vocab + NT * ept - 1) / (NT * ept)) >= 2ll * device_sms()) return ept;
    return 8;
}

}  // namespace

// Bytes of the work space of a call.
MI_EXPORT long long mi_beam_select_bytes(int rows, int vocab, int num) {
    if (rows < 0 || vocab < 1 || num < 1 || num > MAX_NUM) return -2;
    const int ept = slice_size(rows, vocab);
    const long long slices = (vocab + (long long)NT * ept - 1) / (NT * ept);
    return rows * (slices * (long long)(sizeof(SliceSum) + num * sizeof(u64)) + (long long)sizeof(double));
}

// logits float32 [rows, vocab], rows ld apart; scores float32 [rows]; group_start int32 [groups + 1]; values float32, out_rows and out_tokens int32 [groups, num].
// work: mi_beam_select_bytes of it, on 16 bytes.
MI_EXPORT int mi_beam_select(const float* logits, long long ld, int rows, int vocab, const float* scores, const int* group_start, int groups, int num,
                             float* values, int* out_rows, int* out_tokens, void* work, cudaStream_t stream) {
    if (groups == 0) return 0;
    if (rows < 0 || groups < 0 || vocab < 1 || vocab > 0x7fffffff - NT * 32 || num < 1 || num > MAX_NUM || (rows && ld < vocab) || rows > 65535 || ((uintptr_t)work % 16)) return -2;
    const int ept = slice_size(rows, vocab), slices = (vocab + NT * ept - 1) / (NT * ept);
    SliceSum* sums = (SliceSum*)work;
    u64* keys = (u64*)(sums + (size_t)rows * slices);
    double* base = (double*)(keys + (size_t)rows * slices * num);
    if (rows) {
        cudaError_t e;
        const dim3 grid(slices, rows);
        if (ept == 32) e = launch_pdl(beam_slice_kernel<32>, grid, dim3(NT), 0, stream, logits, ld, vocab, num, sums, keys);
        else if (ept == 16) e = launch_pdl(beam_slice_kernel<16>, grid, dim3(NT), 0, stream, logits, ld, vocab, num, sums, keys);
        else e = launch_pdl(beam_slice_kernel<8>, grid, dim3(NT), 0, stream, logits, ld, vocab, num, sums, keys);
        if (e != cudaSuccess) return (int)e;
    }
    return (int)launch_pdl(beam_merge_kernel, dim3(groups), dim3(NT), 0, stream, sums, keys, slices, num, scores, rows, group_start, base, values, out_rows, out_tokens);
}

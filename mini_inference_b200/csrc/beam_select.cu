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
// its `num` largest logits in order.  The num / 8-th largest of each warp's 32 threads' maxima, the least of the eight, is a bound that at least num
// logits reach; what reaches it (a few more than num) goes to shared memory and every entry counts those before it.  Where more reach it than fit (many
// equal logits) the num-th of those that found room is the next bound: all candidates differ in their order, so each turn has at least CAP - num fewer.  beam_merge_kernel: a block per group joins the slices' sums, and chooses among their sorted lists the
// same way: a bound from the lists' heads, then a thread per list follows its list down to the bound.
#include "common.cuh"
#include <math.h>

using namespace mi;

namespace {

constexpr int NT = 256, CAP = 1024, BASES = 128;                 // threads of a block (at least MAX_NUM); candidates that fit in shared memory
constexpr int MAX_NUM = 128, WARPS = NT / 32;
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

template <typename T> __device__ __forceinline__ T warp_largest(T v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { const T w = __shfl_xor_sync(0xffffffffu, v, o); v = w > v ? w : v; }
    return v;
}
// The `turn`-th largest of a warp's values (lowest: below all of them), and the largest
template <typename T> __device__ __forceinline__ T warp_nth(T mine, int turn, T lowest, T& largest) {
    T best = largest = warp_largest(mine);
    for (int k = 1; k < turn; ++k) {                 // once more without the lane that had it
        const uint32_t who = __ballot_sync(0xffffffffu, mine == best);
        if ((threadIdx.x & 31) == __ffs(who) - 1) mine = lowest;
        best = warp_largest(mine);
    }
    return best;
}
// A bound that at least num (<= NT) of the threads' values reach: the least over the warps of their num / 8-th largest
__device__ __forceinline__ int turns(int num) { return (num + WARPS - 1) / WARPS; }
__device__ __forceinline__ double threshold(double mine, int num, double* scratch) {
    double largest;
    double best = warp_nth(mine, turns(num), -(double)INFINITY, largest);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) best = fmin(best, scratch[w]);
    return best;
}

// e^(x - m) for logits x <= m, |m| <= 1024, with errors of about 5e-10 of it, as a leading and a small part: 2^t, t = n + j / 32 + r, is 2^n times a table's 2^(j / 32)
// times a polynomial in r, |r| <= 1/64 (table-driven, after Tang).  m log2(e) is split into a multiple of 2^-12, to which j / 32 is added without
// rounding, and the rest, so that r is off by 2^-31 or so.  The table is spread over a warp's lanes.
constexpr float LOG2E_HI = 0x1.715476p+0f, LOG2E_LO = 0x1.4ae0cp-26f;
__device__ const float2 POWERS[32] = {        // 2^(j / 32) and what its rounding left
    {1.f, 0.f}, {1.0218971967697144f, -4.81155986e-08f}, {1.0442737340927124f, 4.83347016e-08f}, {1.0671404600143433f, -5.93375198e-08f},
    {1.0905077457427979f, -1.30775399e-08f}, {1.114386796951294f, -5.43554002e-08f}, {1.1387885808944702f, 5.38622231e-08f}, {1.1637248992919922f, -4.05144149e-08f},
    {1.1892070770263672f, 3.79763527e-08f}, {1.215247392654419f, -3.26739489e-08f}, {1.2418577671051025f, 4.4968381e-08f}, {1.2690509557724f, 1.41933332e-09f},
    {1.2968395948410034f, -4.01899953e-08f}, {1.3252366781234741f, -3.49637332e-08f}, {1.3542555570602417f, -1.01233493e-08f}, {1.3839099407196045f, -5.87557736e-08f},
    {1.4142135381698608f, 2.4203235e-08f}, {1.4451807737350464f, 3.32419994e-08f}, {1.4768261909484863f, -4.50089885e-08f}, {1.5091644525527954f, -2.49593732e-08f},
    {1.5422108173370361f, 8.07090483e-09f}, {1.5759809017181396f, -5.66102543e-08f}, {1.610490322113037f, 9.83621717e-09f}, {1.6457555294036865f, -5.12497209e-08f},
    {1.6817928552627563f, -2.47553267e-08f}, {1.7186193466186523f, -4.8496176e-08f}, {1.7562521696090698f, -9.23577037e-09f}, {1.7947090864181519f, -1.14150449e-08f},
    {1.8340080976486206f, -1.1239278e-08f}, {1.8741676807403564f, -4.66300563e-08f}, {1.9152065515518188f, 9.84532811e-09f}, {1.9571441411972046f, -1.70218044e-08f}};
struct Exponential {
    float2 power;                                    // of this lane
    float m_hi, m_lo, m_32, least;
    __device__ __forceinline__ Exponential(float m, const float2& power_) : power(power_) {
        const double y = (double)m * 1.4426950408889634074;
        m_hi = (float)(rint(y * 4096.) * (1. / 4096.));
        m_lo = (float)(y - (double)m_hi);
        m_32 = -32.f * m_hi;
        least = m - 44.f;                            // e^-44 = 2^-63: logits below it (-inf among them) count as that
    }
    // of two logits at once: adds their leading parts to sum and the rest to rest
    __device__ __forceinline__ void operator()(float x0, float x1, double& sum, float& rest) const {
        const float2 x = make_float2(fmaxf(x0, least), fmaxf(x1, least)), magic = make_float2(12582912.f, 12582912.f);
        const float2 z = __fadd2_rn(__ffma2_rn(x, make_float2(32.f * LOG2E_HI, 32.f * LOG2E_HI), make_float2(m_32, m_32)), magic);      // its last bits: 32 t rounded to a whole number
        const float2 k = __fadd2_rn(z, make_float2(-12582912.f, -12582912.f));
        const float2 c = __ffma2_rn(k, make_float2(-1.f / 32.f, -1.f / 32.f), make_float2(-m_hi, -m_hi));
        const float2 r = __fadd2_rn(__ffma2_rn(x, make_float2(LOG2E_LO, LOG2E_LO), __ffma2_rn(x, make_float2(LOG2E_HI, LOG2E_HI), c)), make_float2(-m_lo, -m_lo));
        float2 p = __ffma2_rn(r, make_float2(0x1.3b2ab6p-7f, 0x1.3b2ab6p-7f), make_float2(0x1.c6b08ep-5f, 0x1.c6b08ep-5f));                // ln(2)^i / i!
        p = __ffma2_rn(r, p, make_float2(0x1.ebfbep-3f, 0x1.ebfbep-3f));
        p = __fmul2_rn(r, __ffma2_rn(r, p, make_float2(0x1.62e43p-1f, 0x1.62e43p-1f)));
        const int k0 = __float_as_int(z.x), k1 = __float_as_int(z.y);      // the magic number's own last bits are 0
        const float2 hi = make_float2(__shfl_sync(0xffffffffu, power.x, k0), __shfl_sync(0xffffffffu, power.x, k1));
        const float2 lo = make_float2(__shfl_sync(0xffffffffu, power.y, k0), __shfl_sync(0xffffffffu, power.y, k1));
        // 2^floor(k / 32): bits 5 and up of k (mod 2^8) into the exponent
        const float2 scale = make_float2(__int_as_float(((k0 >> 5) + 127) << 23), __int_as_float(((k1 >> 5) + 127) << 23));
        const float2 lead = __fmul2_rn(hi, scale), small = __fmul2_rn(__ffma2_rn(hi, p, lo), scale);
        sum += (double)lead.x;
        sum += (double)lead.y;
        rest += small.x + small.y;
    }
};

// EPT logits a thread, four neighbours at a time
template <int EPT>
__global__ void __launch_bounds__(NT, 4) beam_slice_kernel(const float* __restrict__ logits, long long ld, int vocab, int num, SliceSum* __restrict__ sums,
                                                           u64* __restrict__ keys) {
    __shared__ float tops[WARPS], bounds[WARPS];
    __shared__ double parts[WARPS];
    __shared__ u64 found[CAP], floor_of;
    __shared__ int count;
    pdl_trigger();
    const float2 power = POWERS[threadIdx.x & 31];
    pdl_wait(logits);
    const int r = blockIdx.y, slice = blockIdx.x, slices = gridDim.x, base = slice * NT * EPT, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* row = logits + (long long)r * ld;
    const bool vec = ((uintptr_t)row & 15) == 0;
    const auto index = [&](int e) { return base + ((e >> 2) * NT + (int)threadIdx.x) * 4 + (e & 3); };
    float x[EPT];
#pragma unroll
    for (int k = 0; k < EPT / 4; ++k) {
        const int i = index(4 * k);
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
        top = fmaxf(top, x[e]);
    }
    if (bad) top = INFINITY;
    float largest;
    const float nth = warp_nth(top, turns(num), -INFINITY, largest);
    if (threadIdx.x == 0) count = 0;
    if (lane == 0) { tops[warp] = largest; bounds[warp] = nth; }
    __syncthreads();
    float m = tops[0], least = bounds[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) { m = fmaxf(m, tops[w]); least = fminf(least, bounds[w]); }
    SliceSum* out = sums + (size_t)r * slices + slice;
    u64* best = keys + ((size_t)r * slices + slice) * num;
    if (!(fabsf(m) < INFINITY)) {                    // NaN or +inf (the row offers nothing), or nothing above -inf
        if (threadIdx.x == 0) *out = SliceSum{m == -INFINITY ? 0. : (double)NAN, m, 0};
        for (int k = threadIdx.x; k < num; k += NT) best[k] = 0;
        return;
    }
    double sum = 0.;
    if (fabsf(m) <= 1024.f) {
        const Exponential exponential(m, power);
        float rest = 0.f;
#pragma unroll
        for (int e = 0; e < EPT; e += 2) exponential(x[e], x[e + 1], sum, rest);
        sum += (double)rest;
    } else {
#pragma unroll
        for (int e = 0; e < EPT; ++e) sum += exp((double)x[e] - (double)m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) parts[warp] = sum;
    uint32_t hits = 0;                               // few of a thread's logits reach the bound: those are read once more
#pragma unroll
    for (int e = 0; e < EPT; ++e) hits |= (x[e] >= least && x[e] > -INFINITY ? 1u : 0u) << e;
    int n;
    for (u64 floor_key = 0;;) {
        for (uint32_t left = hits; left; left &= left - 1) {
            const int i = index(__ffs(left) - 1);
            const u64 key = logit_key(row[i] + 0.f, i);      // -0 is 0
            if (key >= floor_key) {
                const int at = atomicAdd(&count, 1);
                if (at < CAP) found[at] = key;
            }
        }
        __syncthreads();
        n = count;
        if (n <= CAP) break;
        for (int i = threadIdx.x; i < CAP; i += NT) {
            const u64 mine = found[i];
            int before = 0;
            for (int o = 0; o < CAP; ++o) before += found[o] > mine;
            if (before == num - 1) floor_of = mine;
        }
        __syncthreads();
        floor_key = floor_of;
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
    }
    for (int i = threadIdx.x; i < n; i += NT) {
        const u64 mine = found[i];
        int before = 0;
#pragma unroll 8
        for (int o = 0; o < n; ++o) before += found[o] > mine;
        if (before < num) best[before] = mine;
    }
    for (int k = n + threadIdx.x; k < num; k += NT) best[k] = 0;
    if (threadIdx.x == 0) {
        for (int w = 1; w < WARPS; ++w) sum += parts[w];
        *out = SliceSum{sum, m, min(n, num)};
    }
}

struct Candidate { double value; int row; u64 key; };
__device__ __forceinline__ bool goes_before(const Candidate& a, const Candidate& b) {
    return a.value != b.value ? a.value > b.value : a.row != b.row ? a.row < b.row : a.key > b.key;
}
struct Found {                                       // candidates in shared memory
    double value[CAP]; u64 key[CAP]; int row[CAP];
    __device__ __forceinline__ Candidate get(int i) const { return Candidate{value[i], row[i], key[i]}; }
    __device__ __forceinline__ void put(int i, const Candidate& c) { value[i] = c.value; key[i] = c.key; row[i] = c.row; }
    __device__ __forceinline__ int before(const Candidate& c, int n) const {       // how many of the first n go before c, which is one of them
        int before = 0, same = 0;
#pragma unroll 8
        for (int o = 0; o < n; ++o) { const double v = value[o]; before += v > c.value; same += v == c.value; }
        if (same > 1)
            for (int o = 0; o < n; ++o) before += value[o] == c.value && (row[o] != c.row ? row[o] < c.row : key[o] > c.key);
        return before;
    }
};

__global__ void __launch_bounds__(NT) beam_merge_kernel(const SliceSum* sums, const u64* keys, int slices, int num, const float* __restrict__ scores, int rows,
                                                        const int* __restrict__ group_start, double* base, float* __restrict__ values, int* __restrict__ out_rows,
                                                        int* __restrict__ out_tokens) {
    __shared__ double scratch[WARPS], near_base[BASES];
    __shared__ Found found;
    __shared__ Candidate bound;
    __shared__ int count;
    pdl_trigger();
    pdl_wait(scores, group_start);
    const int g = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int a = max(0, min(group_start[g], rows)), b = max(a, min(group_start[g + 1], rows));
    // s[r] - lse[r], a warp per row
    for (int r = a + warp; r < b; r += WARPS) {
        const SliceSum* mine = sums + (size_t)r * slices;
        float m = -INFINITY;
        for (int i = lane; i < slices; i += 32) m = fmaxf(m, mine[i].top);
        m = warp_max(m);
        double sum = 0.;
        for (int i = lane; i < slices; i += 32) sum += mine[i].sum * (mine[i].top == -INFINITY ? 1. : exp((double)mine[i].top - (double)m));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const double v = (double)scores[r] - ((double)m + log(sum));
        if (lane == 0) { base[r] = isfinite(v) ? v : -(double)INFINITY; if (r - a < BASES) near_base[r - a] = base[r]; }
    }
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    // list i: row, slice; candidate k of it
    const int lists = (b - a) * slices;
    const auto at = [&](int list, int k) {
        const int r = a + list / slices;
        const size_t where = (size_t)r * slices + list % slices;
        Candidate c{-(double)INFINITY, r, 0};
        const double from = r - a < BASES ? near_base[r - a] : base[r];
        if (k < num) c.key = keys[where * num + k];
        if (c.key) c.value = from + (double)key_logit(c.key);
        return c;
    };
    // A value that at least num candidates reach: from the heads where every warp has enough lists (list i belongs to warp i % 8), else the least of
    // the depth-th candidates, depth the number of lists in num.
    const int first = lane * WARPS + warp;
    double least;
    if (lists / WARPS >= turns(num)) {
        double top = -(double)INFINITY;
        for (int i = first; i < lists; i += NT) top = fmax(top, at(i, 0).value);
        least = threshold(top, num, scratch);
    } else {
        const int depth = lists ? (num + lists - 1) / lists : 1;
        double low = (double)INFINITY;
        for (int i = first; i < lists; i += NT) low = fmin(low, at(i, depth - 1).value);
        low = -warp_largest(-low);
        if (lane == 0) scratch[warp] = low;
        __syncthreads();
        least = scratch[0];
        for (int w = 1; w < WARPS; ++w) least = fmin(least, scratch[w]);
    }
    int have;
    for (bool bounded = false;; bounded = true) {
        for (int i = first; i < lists; i += NT)
            for (int k = 0; k < num; ++k) {
                const Candidate c = at(i, k);
                if (!(c.value >= least && c.value > -(double)INFINITY) || (bounded && goes_before(bound, c))) break;      // lists are in order
                const int p = atomicAdd(&count, 1);
                if (p < CAP) found.put(p, c);
            }
        __syncthreads();
        have = count;
        if (have <= CAP) break;
        for (int i = threadIdx.x; i < CAP; i += NT) {
            const Candidate mine = found.get(i);
            if (found.before(mine, CAP) == num - 1) bound = mine;
        }
        __syncthreads();
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
    }
    // many more than num reach the bound: a better one, from the candidates themselves, while it leaves a good part of them out
    while (have > num + NT / 4) {
        constexpr int MINE = CAP / NT;
        Candidate mine[MINE];
        double top = -(double)INFINITY;
#pragma unroll
        for (int e = 0; e < MINE; ++e) {
            const int i = threadIdx.x + e * NT;
            mine[e] = i < have ? found.get(i) : Candidate{-(double)INFINITY, 0, 0};
            top = fmax(top, mine[e].value);
        }
        least = threshold(top, num, scratch);      // (its barriers stand between the reads and the writes)
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < MINE; ++e)
            if (mine[e].value >= least && mine[e].value > -(double)INFINITY) found.put(atomicAdd(&count, 1), mine[e]);
        __syncthreads();
        const int left = count;
        const bool enough = left > have - have / 4;
        have = left;
        __syncthreads();
        if (enough) break;
    }
    for (int i = threadIdx.x; i < have; i += NT) {
        const Candidate mine = found.get(i);
        const int before = found.before(mine, have);
        if (before < num) {
            const size_t o = (size_t)g * num + before;
            values[o] = (float)mine.value; out_rows[o] = mine.row; out_tokens[o] = key_token(mine.key);
        }
    }
    for (int k = have + threadIdx.x; k < num; k += NT) {
        const size_t o = (size_t)g * num + k;
        values[o] = -INFINITY; out_rows[o] = -1; out_tokens[o] = -1;
    }
}

int slice_size(int rows, int vocab) {
    // enough blocks for two an SM where the logits allow it
    return (long long)rows * ((vocab + NT * 16 - 1) / (NT * 16)) >= 2ll * device_sms() ? 16 : 8;
}

}  // namespace

// Bytes of the work space of a call.
MI_EXPORT long long mi_beam_select_bytes(int rows, int vocab, int num) {
    if (rows < 0 || vocab < 1 || num < 1 || num > MAX_NUM) return -2;
    const int ept = slice_size(rows, vocab);
    const long long slices = (vocab + (long long)NT * ept - 1) / (NT * ept);
    return rows * (slices * (long long)(sizeof(SliceSum) + num * sizeof(u64)) + (long long)sizeof(double));
}

// logits float32 [rows, vocab], rows ld apart; scores float32 [rows]; group_start int32 [groups + 1]; values float32 [groups, num], chosen int32 [2, groups, num]: rows, then tokens.
// work: mi_beam_select_bytes of it, on 16 bytes.
MI_EXPORT int mi_beam_select(const float* logits, long long ld, int rows, int vocab, const float* scores, const int* group_start, int groups, int num,
                             float* values, int* chosen, void* work, cudaStream_t stream) {
    if (groups == 0) return 0;
    if (rows < 0 || groups < 0 || vocab < 1 || vocab > 0x7fffffff - NT * 32 || num < 1 || num > MAX_NUM || (rows && ld < vocab) || rows > 65535 || ((uintptr_t)work % 16)) return -2;
    const int ept = slice_size(rows, vocab), slices = (vocab + NT * ept - 1) / (NT * ept);
    SliceSum* sums = (SliceSum*)work;
    u64* keys = (u64*)(sums + (size_t)rows * slices);
    double* base = (double*)(keys + (size_t)rows * slices * num);
    if (rows) {
        cudaError_t e;
        const dim3 grid(slices, rows);
        if (ept == 16) e = launch_pdl(beam_slice_kernel<16>, grid, dim3(NT), 0, stream, logits, ld, vocab, num, sums, keys);
        else e = launch_pdl(beam_slice_kernel<8>, grid, dim3(NT), 0, stream, logits, ld, vocab, num, sums, keys);
        if (e != cudaSuccess) return (int)e;
    }
    return (int)launch_pdl(beam_merge_kernel, dim3(groups), dim3(NT), 0, stream, sums, keys, slices, num, scores, rows, group_start, base, values, chosen,
                           chosen + (size_t)groups * num);
}

// Beam search's selection: log-probabilities of every beam over the vocabulary and, per prompt, the best candidates of all its beams.
//
// Reference: none (davidjoyme/mini-inference engine/core/sampler.py:3-11 knows argmax and a draw).  With logits x[r, v] and running scores s[r]
//     lse[r] = log sum_v e^x[r, v],   candidate (r, v) has the value (s[r] - lse[r]) + x[r, v],
// and a group of rows gives its `num` largest: by value, then the lower row, then the larger logit, then the lower token.  A row whose logits hold
// NaN or +inf or no finite number, or whose score is not finite, offers nothing, nor does a logit of -inf; places that stay empty hold (-inf, -1, -1).
//
// The order of two candidates is a whole number, so values are compared in float64 and the sum of exponentials is kept to about 1e-9: float32's 1e-7
// would swap two neighbours that lie 0.05 apart once in some hundred thousand pairs, a step of 64 beams has a thousand.  Within a row the logits
// themselves decide, exactly.  Scores come in float32, so a caller with long sums gives what each row is behind its group's best one (as engine/beam.py does): a
// number common to all rows of a group changes no order, and -800 in float32 is off by 3e-5.
//
// Two launches.  beam_slice_kernel: a block streams a slice of one row once (asynchronous copies, up to three tiles in front) and keeps its sum of exponentials and, per
// thread, the largest logit.  The num / 8-th largest of each warp's 32 threads, the least of the eight, is a bound that num threads reach; the num-th of those that do is a
// better one, and only the logits of threads whose largest reaches that are read again (from the L2 cache, 1 / 16 of the slice for num = 16) and put in order by counting.
// Keeping candidates while streaming cost three instructions a logit and ten for each that a bound from the first tiles lets through: 24 us instead of 19 at 64 x 151,936.
// Where more reach the bound than fit (many equal logits) the num-th of those that found room is the next bound: all candidates differ in their order, so
// each turn has at least CAP - num fewer.
// beam_merge_kernel: a block per group joins the slices' sums, finds a bound from the first, second, fourth, ... candidates of their sorted lists, and follows each list down to it.
// Bounds from the first ones alone let every list of a beam far ahead of the others through: 16 us instead of 8 for 16 beams with scores some units apart.
// Time at 64 rows x 151,936, num 16: 24 us (38.9 MB: 6 us); 38 instructions a logit, 18 of them the exponential, keep two of three issue slots busy.
// 4 x 32,768: 8 us, two launches with everything cold.
#include "common.cuh"
#include <algorithm>
#include <float.h>
#include <math.h>

using namespace mi;

namespace {

constexpr int NT = 256, EPT = 8, TILE = NT * EPT;                // threads of a block (at least MAX_NUM), logits of a thread and of all at a time
constexpr int AHEAD = 4, BLOCKS = 4;                              // tiles in shared memory; blocks an SM
constexpr int CAP = 1024, BASES = 128;                           // candidates that fit in shared memory; rows of a group whose base does
constexpr int MAX_NUM = 128, WARPS = NT / 32;
typedef unsigned long long u64;

__device__ __forceinline__ float max_or_nan(float a, float b, float c) { float d; asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }
// A sum of exponentials in units of 2^at (at a whole number: units are changed without rounding) or, where logits are large, e^at.
// at NaN: the row offers nothing; -inf: no logit above -inf
struct __align__(16) SliceSum { double sum; float at; int binary; };
__device__ __forceinline__ double log_unit(const SliceSum& s) { return s.binary ? (double)s.at * 0.6931471805599453 : (double)s.at; }
__device__ __forceinline__ double in_units(const SliceSum& s, const SliceSum& of) {      // of is the larger unit
    if (s.at == -INFINITY) return 0.;
    if (s.binary && of.binary) return s.sum * __hiloint2double((1023 + max((int)(s.at - of.at), -1000)) << 20, 0);
    return s.sum * exp(log_unit(s) - log_unit(of));
}
__device__ __forceinline__ SliceSum larger_unit(const SliceSum& a, const SliceSum& b) {  // sum aside; NaN is the largest
    if (a.binary && b.binary) return SliceSum{0., max_or_nan(a.at, b.at, -INFINITY), 1};
    return isnan(a.at) || isnan(b.at) ? SliceSum{0., NAN, 1} : log_unit(a) >= log_unit(b) ? a : b;
}

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

__device__ __forceinline__ float warp_largest(float v) { float d; asm("redux.sync.max.f32 %0, %1, 0xffffffff;\n" : "=f"(d) : "f"(v)); return d; }
__device__ __forceinline__ float warp_least(float v) { float d; asm("redux.sync.min.f32 %0, %1, 0xffffffff;\n" : "=f"(d) : "f"(v)); return d; }
__device__ __forceinline__ double warp_largest(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { const double w = __shfl_xor_sync(0xffffffffu, v, o); v = w > v ? w : v; }
    return v;
}
// The n-th largest of a warp's values
__device__ __forceinline__ float warp_nth(float mine, int n) {
    if (n == 1) return warp_largest(mine);
    const int lane = threadIdx.x & 31;
    int before = 0;
#pragma unroll 8
    for (int o = 1; o < 32; ++o) {
        const float other = __shfl_xor_sync(0xffffffffu, mine, o);
        before += (other > mine) | ((other == mine) & ((lane ^ o) < lane));
    }
    return __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, before == n - 1)) - 1);
}
__device__ __forceinline__ double warp_nth(double mine, int n) {
    for (int k = 1;; ++k) {
        const double best = warp_largest(mine);
        if (k == n) return best;
        const uint32_t who = __ballot_sync(0xffffffffu, mine == best);      // once more without the lane that had it
        if ((threadIdx.x & 31) == __ffs(who) - 1) mine = -(double)INFINITY;
    }
}
// A bound that at least num (<= NT) of the threads' values reach: the least over the warps of their num / 8-th largest
__device__ __forceinline__ int turns(int num) { return (num + WARPS - 1) / WARPS; }
__device__ __forceinline__ double threshold(double mine, int num, double* scratch) {
    double best = warp_nth(mine, turns(num));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) best = fmin(best, scratch[w]);
    return best;
}

// e^x for logits |x| <= 1024 up to a largest one, in units of 2^at, with errors of about 5e-10 of it, as a leading and a small part: 2^t, t = x log2(e) - at = n + j / 32 + r,
// is 2^n times a table's 2^(j / 32) times a polynomial in r, |r| <= 1/64 (table-driven, after Tang).  at is a whole number, so that taking it and
// n + j / 32 away leaves nothing to round but r itself, 2^-31 or so.  The table is spread over a warp's lanes.
constexpr float LOG2E_HI = 0x1.715476p+0f, LOG2E_LO = 0x1.4ae0cp-26f;
__device__ const float2 POWERS[32] = {        // 2^(j / 32) and what its rounding left (not 0, 2^-40: its exponent is added to)
    {1.f, 1e-12f}, {1.0218971967697144f, -4.81155986e-08f}, {1.0442737340927124f, 4.83347016e-08f}, {1.0671404600143433f, -5.93375198e-08f},
    {1.0905077457427979f, -1.30775399e-08f}, {1.114386796951294f, -5.43554002e-08f}, {1.1387885808944702f, 5.38622231e-08f}, {1.1637248992919922f, -4.05144149e-08f},
    {1.1892070770263672f, 3.79763527e-08f}, {1.215247392654419f, -3.26739489e-08f}, {1.2418577671051025f, 4.4968381e-08f}, {1.2690509557724f, 1.41933332e-09f},
    {1.2968395948410034f, -4.01899953e-08f}, {1.3252366781234741f, -3.49637332e-08f}, {1.3542555570602417f, -1.01233493e-08f}, {1.3839099407196045f, -5.87557736e-08f},
    {1.4142135381698608f, 2.4203235e-08f}, {1.4451807737350464f, 3.32419994e-08f}, {1.4768261909484863f, -4.50089885e-08f}, {1.5091644525527954f, -2.49593732e-08f},
    {1.5422108173370361f, 8.07090483e-09f}, {1.5759809017181396f, -5.66102543e-08f}, {1.610490322113037f, 9.83621717e-09f}, {1.6457555294036865f, -5.12497209e-08f},
    {1.6817928552627563f, -2.47553267e-08f}, {1.7186193466186523f, -4.8496176e-08f}, {1.7562521696090698f, -9.23577037e-09f}, {1.7947090864181519f, -1.14150449e-08f},
    {1.8340080976486206f, -1.1239278e-08f}, {1.8741676807403564f, -4.66300563e-08f}, {1.9152065515518188f, 9.84532811e-09f}, {1.9571441411972046f, -1.70218044e-08f}};
struct Exponential {
    float2 power;                                    // of this lane
    float at, least;
    __device__ __forceinline__ Exponential(float m, const float2& power_) : power(power_) {
        at = rintf(m * LOG2E_HI);
        least = m - 44.f;                            // e^-44 = 2^-63: logits below it (-inf among them) count as that
    }
    // of two logits at once: adds their leading parts to sum and the rest to rest
    __device__ __forceinline__ void operator()(float x0, float x1, double& sum, float& rest) const {
        constexpr float MAGIC = 12582912.f;          // its last bit is 1, so adding it rounds to a whole number
        const float start = fmaf(-32.f, at, MAGIC), back = MAGIC / 32.f - at;      // both exact
        const float2 x = make_float2(fmaxf(x0, least), fmaxf(x1, least));
        const float2 z = __ffma2_rn(x, make_float2(32.f * LOG2E_HI, 32.f * LOG2E_HI), make_float2(start, start));      // its last bits: 32 t rounded to a whole number
        const float2 c = __ffma2_rn(z, make_float2(-1.f / 32.f, -1.f / 32.f), make_float2(back, back));                 // -(at + that / 32), exact
        const float2 r = __ffma2_rn(x, make_float2(LOG2E_LO, LOG2E_LO), __ffma2_rn(x, make_float2(LOG2E_HI, LOG2E_HI), c));
        float2 p = __ffma2_rn(r, make_float2(0x1.c6b08ep-5f, 0x1.c6b08ep-5f), make_float2(SQUARE, SQUARE));             // ln(2)^i / i!
        p = __fmul2_rn(r, __ffma2_rn(r, p, make_float2(0x1.62e43p-1f, 0x1.62e43p-1f)));
        const int k0 = __float_as_int(z.x), k1 = __float_as_int(z.y);      // the magic number's own last bits are 0
        const auto times = [](float v, int k) { return __int_as_float(__float_as_int(v) + ((k & ~31) << 18)); };      // 2^floor(k / 32) v: bits 5 and up of k added to the exponent
        const float2 hi = make_float2(times(__shfl_sync(0xffffffffu, power.x, k0), k0), times(__shfl_sync(0xffffffffu, power.x, k1), k1));
        const float2 lo = make_float2(times(__shfl_sync(0xffffffffu, power.y, k0), k0), times(__shfl_sync(0xffffffffu, power.y, k1), k1));
        const float2 small = __ffma2_rn(hi, p, lo);
        sum += (double)hi.x;
        sum += (double)hi.y;
        rest += small.x + small.y;
    }
    // r^4 ln(2)^4 / 24 over |r| <= 1/64 is r^2 ln(2)^4 / (24 64^2) to 1.5e-10
    static constexpr float SQUARE = (float)(0.24022650695910072 + 0.23083509858308343 / (24. * 4096.));
};


__device__ __forceinline__ void cp_async16(float* to, const float* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" :: "r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" :: "n"(N) : "memory"); }

// The best num of the first n (<= CAP) of found, to its front and in order.  Returns how many.
__device__ __forceinline__ int keep_best(u64* found, int n, int num) {
    constexpr int MINE = CAP / NT;
    u64 mine[MINE];
    int before[MINE];
#pragma unroll
    for (int e = 0; e < MINE; ++e) {
        const int i = threadIdx.x + e * NT;
        before[e] = num;
        if (i < n) {
            mine[e] = found[i];
            before[e] = 0;
#pragma unroll 8
            for (int o = 0; o < n; ++o) before[e] += found[o] > mine[e];
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < MINE; ++e)
        if (before[e] < num) found[before[e]] = mine[e];
    __syncthreads();
    return min(n, num);
}

// A block takes `per` logits of a row, TILE at a time; AHEAD tiles are on their way to shared memory meanwhile, each thread reading what it asked for itself.
// Each warp has its own sum, in units of its own; nothing else is kept but each thread's largest.
__global__ void __launch_bounds__(NT, BLOCKS) beam_slice_kernel(const float* __restrict__ logits, long long ld, int vocab, int per, int num, SliceSum* __restrict__ sums,
                                                           u64* __restrict__ keys) {
    extern __shared__ __align__(16) float ring[];    // [AHEAD][EPT / 4][NT][4]; then candidates
    __shared__ float bounds[WARPS];
    __shared__ SliceSum parts[WARPS];
    __shared__ int count, lists;
    __shared__ float2 hits[NT];                      // a thread's largest logit, and the thread
    __shared__ float better;
    pdl_trigger();
    const float2 power = POWERS[threadIdx.x & 31];
    if (threadIdx.x == 0) count = lists = 0;
    pdl_wait(logits);
    const int r = blockIdx.y, slice = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // the row from a 16-byte boundary on, up to three numbers in front of it
    const int off = (int)((uintptr_t)(logits + (long long)r * ld) >> 2 & 3);
    const float* row = logits + (long long)r * ld - off;
    const int begin = max(off, slice * per), end = min((slice + 1) * per, vocab + off), tiles = max(1, (end - slice * per + TILE - 1) / TILE);
    const auto fetch = [&](int tile) {
        if (tile < tiles) {
            float* to = ring + (tile % AHEAD * TILE + (int)threadIdx.x * 4);
            const int i0 = slice * per + tile * TILE + (int)threadIdx.x * 4;
#pragma unroll
            for (int k = 0; k < EPT / 4; ++k) {
                const int i = i0 + k * NT * 4;
                if (i >= begin && i + 3 < end) {
                    cp_async16(to + k * NT * 4, row + i);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) to[k * NT * 4 + e] = i + e >= begin && i + e < end ? row[i + e] : -INFINITY;
                }
            }
        }
        cp_async_commit();
    };
    for (int tile = 0; tile < AHEAD - 1; ++tile) fetch(tile);
    Exponential exponential(0.f, power);
    float near = -INFINITY, mine = -INFINITY;        // what the warp's units are for (the largest logit when they were taken); this thread's largest
    SliceSum all{0., -INFINITY, 1};
    for (int tile = 0; tile < tiles; ++tile) {
        cp_async_wait<AHEAD - 2>();
        float x[EPT];
#pragma unroll
        for (int k = 0; k < EPT / 4; ++k) load16(ring + (tile % AHEAD * TILE + (k * NT + (int)threadIdx.x) * 4), x + 4 * k);
        fetch(tile + AHEAD - 1);
        float top = x[0];
#pragma unroll
        for (int e = 1; e + 1 < EPT; e += 2) top = max_or_nan(top, x[e], x[e + 1]);
        top = max_or_nan(top, x[EPT - 1], -INFINITY);
        if (!(top < INFINITY)) top = INFINITY;       // NaN too: the row offers nothing
        mine = fmaxf(mine, top);
        if (__any_sync(0xffffffffu, top > near + 20.f)) {      // other units: not often
            near = warp_largest(top);
            if (near < INFINITY) {
                SliceSum now{0., near, 0};
                if (fabsf(near) <= 1000.f) {
                    exponential = Exponential(near, power);
                    now = SliceSum{0., exponential.at, 1};
                }
                now.sum = in_units(all, now);
                all = now;
            }
        }
        if (fabsf(near) <= 1000.f) {
            float rest = 0.f;
#pragma unroll
            for (int e = 0; e < EPT; e += 2) exponential(x[e], x[e + 1], all.sum, rest);
            all.sum += (double)rest;
        } else if (fabsf(near) < INFINITY) {
#pragma unroll 1
            for (int k = 0; k < EPT; ++k) {
                float v = x[0];
#pragma unroll
                for (int e = 1; e < EPT; ++e) v = k == e ? x[e] : v;
                all.sum += exp((double)v - (double)near);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all.sum += __shfl_xor_sync(0xffffffffu, all.sum, o);
    const float largest = warp_largest(mine), nth = warp_nth(mine, turns(num));
    if (lane == 0) {
        if (largest == INFINITY) all = SliceSum{0., NAN, 1};
        parts[warp] = all;
        bounds[warp] = nth;
    }
    __syncthreads();
    SliceSum whole = parts[lane % WARPS];
    const bool bad = __any_sync(0xffffffffu, isnan(whole.at)), none = !__any_sync(0xffffffffu, whole.at > -INFINITY);
    SliceSum* out = sums + (size_t)r * gridDim.x + slice;
    const size_t list = (size_t)r * gridDim.x + slice, all_lists = (size_t)gridDim.y * gridDim.x;      // a list's k-th candidate is keys[k all_lists + list]
    if (bad || none) {
        if (threadIdx.x == 0) *out = SliceSum{0., bad ? NAN : -INFINITY, 1};
        for (int k = threadIdx.x; k < num; k += NT) keys[k * all_lists + list] = 0;
        return;
    }
    // num threads' largest reach the bound.  The num-th of those that do is a better one; the logits of the threads that reach that are looked at once more.
    float least = fmaxf(warp_least(bounds[lane % WARPS]), -FLT_MAX);
    if (mine >= least) hits[atomicAdd(&lists, 1)] = make_float2(mine, __int_as_float((int)threadIdx.x));
    __syncthreads();
    const int reach = lists, quads = tiles * (EPT / 4);
    if (reach >= num && reach * quads > NT) {        // (fewer than num: a row with few logits above -inf)
        if ((int)threadIdx.x < reach) {
            const float2 me = hits[threadIdx.x];
            int before = 0;
#pragma unroll 4
            for (int o = 0; o < reach; ++o) { const float2 other = hits[o]; before += (other.x > me.x) | ((other.x == me.x) & (o < (int)threadIdx.x)); }
            if (before == num - 1) better = me.x;
        }
        __syncthreads();
        least = better;
    }
    u64* found = reinterpret_cast<u64*>(ring);       // nothing is on its way any more
    u64 floor_key = 0;
    for (;;) {
        for (int q = threadIdx.x; q < reach * quads; q += NT) {      // a quad a thread
            const float2 hit = hits[q / quads];
            if (hit.x < least) continue;
            const int i = slice * per + (q % quads * NT + __float_as_int(hit.y)) * 4;
            float x[4];
            if (i >= begin && i + 3 < end) {
                load16(row + i, x);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = i + e >= begin && i + e < end ? row[i + e] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (x[e] >= least) {
                    const u64 key = logit_key(x[e] + 0.f, i + e - off);      // -0 is 0
                    if (key < floor_key) continue;
                    const int p = atomicAdd(&count, 1);
                    if (p < CAP) found[p] = key;
                }
        }
        __syncthreads();
        const int n = keep_best(found, min(count, CAP), num);
        if (count <= CAP) {
            for (int k = threadIdx.x; k < num; k += NT) keys[k * all_lists + list] = k < n ? found[k] : 0;
            break;
        }
        floor_key = found[num - 1];                  // many equal logits: once more, from the num-th of those that found room on
        __syncthreads();
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
    }
    if (warp == 0) {
        SliceSum unit = whole;
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1)
            unit = larger_unit(unit, SliceSum{0., __shfl_xor_sync(0xffffffffu, unit.at, o), __shfl_xor_sync(0xffffffffu, unit.binary, o)});
        unit.sum = in_units(whole, unit);
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) unit.sum += __shfl_xor_sync(0xffffffffu, unit.sum, o);
        if (lane == 0) *out = unit;
    }
}

static_assert(AHEAD * TILE * 4 >= CAP * (int)sizeof(u64) && AHEAD * TILE * 4 <= 40 * 1024, "");

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
    __shared__ float bounds[WARPS];
    __shared__ Found found;
    __shared__ Candidate bound;
    __shared__ int count;
    pdl_trigger();
    pdl_wait(scores, group_start);
    const int g = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int a = max(0, min(group_start[g], rows)), b = max(a, min(group_start[g + 1], rows));
    // list i: slice i % slices of row a + i / slices, in order
    const int lists = (b - a) * slices;
    const float per_slice = 1.f / (float)slices;
    const u64* mine = keys + (size_t)a * slices;     // (the lists' first candidates, then all second ones, ...)
    const size_t all_lists = (size_t)rows * slices;
    const int d = 1 << warp, n = (num + d - 1) / d;  // (see below) this warp's d
    const bool looks = d <= num && n <= 32 && lists > 0;
    constexpr int EARLY = 4;
    u64 ahead[EARLY];                                // asked for before the rows' sums
#pragma unroll
    for (int e = 0; e < EARLY; ++e) ahead[e] = 0;
    const u64* depth = mine + (d - 1) * all_lists;
    const auto ask = [&](int i0) {                   // (a list twice behind the last one: no branch)
#pragma unroll
        for (int e = 0; e < EARLY; ++e) ahead[e] = depth[min(i0 + 32 * e, lists - 1)];
    };
    if (looks) ask(lane);
    // s[r] - lse[r]: a warp per row, or a quarter of one
    const int width = b - a > WARPS ? 8 : 32, part = threadIdx.x % width;
    for (int r0 = a; r0 < b; r0 += NT / width) {
        const int r = r0 + threadIdx.x / width;
        const SliceSum* own = sums + (size_t)r * slices;
        SliceSum all{0., -INFINITY, 1};
        for (int i = part; i < slices && r < b; i += width) all = larger_unit(all, own[i]);
        for (int o = width / 2; o > 0; o >>= 1) {
            const SliceSum other{0., __shfl_xor_sync(0xffffffffu, all.at, o), __shfl_xor_sync(0xffffffffu, all.binary, o)};
            all = larger_unit(all, other);
        }
        double sum = 0.;
        if (all.at > -INFINITY)
            for (int i = part; i < slices && r < b; i += width) sum += in_units(own[i], all);
        for (int o = width / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (part == 0 && r < b) {
            const double v = all.at > -INFINITY ? (double)scores[r] - (log_unit(all) + log(sum)) : NAN;
            base[r] = isfinite(v) ? v : -(double)INFINITY;
            if (r - a < BASES) near_base[r - a] = base[r];
        }
    }
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    const auto candidate = [&](int list, u64 key) {
        const int r = a + (int)(((float)list + 0.5f) * per_slice);      // list / slices: at most 65,535 lists, no rounding reaches the next whole number
        const double from = r - a < BASES ? near_base[r - a] : base[r];
        return Candidate{key ? from + (double)key_logit(key) : -(double)INFINITY, r, key};
    };
    const auto at = [&](int list, int k) { return candidate(list, k < num ? mine[k * all_lists + list] : 0); };
    // A value that at least num candidates reach: where n lists' d-th candidates reach it, n d candidates do.  Each warp takes another d, and of its 32 lanes (a lane
    // has many lists) the ceil(num / d)-th best d-th candidate.  d = 1 is the good one where rows are alike, a large one where a row is far ahead.
    {
        float top = -INFINITY, nth = -INFINITY;
        if (looks) {
            for (int i = lane;;) {
#pragma unroll
                for (int e = 0; e < EARLY; ++e) {
                    const int list = i + 32 * e;
                    top = fmaxf(top, list < lists ? __double2float_rd(candidate(min(list, lists - 1), ahead[e]).value) : -INFINITY);
                }
                i += 32 * EARLY;
                if (i - lane >= lists) break;
                ask(i);
            }
            nth = warp_nth(top, n);
        }
        if (lane == 0) bounds[warp] = nth;
    }
    __syncthreads();
    double least = (double)bounds[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) least = fmax(least, (double)bounds[w]);
    // several threads to a list where there are few lists, four candidates at a time
    const int step = lists ? max(1, NT / lists) : 1, skip = lists > NT ? NT : lists;
    const int from = (int)threadIdx.x < step * skip ? threadIdx.x % skip : lists, k0 = skip ? threadIdx.x / skip : 0;
    int have;
    for (bool bounded = false;; bounded = true) {
        for (int i = from; i < lists; i += NT)
            for (int k = k0, on = 1; k < num && on; k += 4 * step) {
                Candidate c[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) c[e] = at(i, k + e * step);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    on = on && c[e].value >= least && c[e].value > -(double)INFINITY;      // lists are in order
                    if (!on || (bounded && goes_before(bound, c[e]))) continue;
                    const int p = atomicAdd(&count, 1);
                    if (p < CAP) found.put(p, c[e]);
                }
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

// Slices of a row: as many as give each block of a grid that fills the GPU once a share, of whole tiles.  shift: numbers between the row and the 16-byte boundary
// in front of it, at most
int slices_of(int rows, int vocab, int shift) {
    const long long tiles = (vocab + (long long)shift + TILE - 1) / TILE, blocks = (long long)BLOCKS * device_sms() / (rows > 0 ? rows : 1), each = blocks > 0 ? (tiles + blocks - 1) / blocks : tiles;
    return (int)((tiles + each - 1) / each);
}

}  // namespace

// Bytes of the work space of a call.
MI_EXPORT long long mi_beam_select_bytes(int rows, int vocab, int num) {
    if (rows < 0 || vocab < 1 || num < 1 || num > MAX_NUM) return -2;
    const long long slices = std::max(slices_of(rows, vocab, 0), slices_of(rows, vocab, 3));
    return rows * (slices * (long long)(sizeof(SliceSum) + num * sizeof(u64)) + (long long)sizeof(double));
}

// logits float32 [rows, vocab], rows ld apart; scores float32 [rows]; group_start int32 [groups + 1]; values float32, chosen_rows and chosen_tokens int32 [groups, num].
// work: mi_beam_select_bytes of it, on 16 bytes.
MI_EXPORT int mi_beam_select(const float* logits, long long ld, int rows, int vocab, const float* scores, const int* group_start, int groups, int num,
                             float* values, int* chosen_rows, int* chosen_tokens, void* work, cudaStream_t stream) {
    if (groups == 0) return 0;
    if (rows < 0 || groups < 0 || vocab < 1 || vocab > 0x7fffffff - NT * 32 || num < 1 || num > MAX_NUM || (rows && ld < vocab) || rows > 65535 || ((uintptr_t)work % 16)) return -2;
    const int shift = ((uintptr_t)logits | (uintptr_t)(ld * 4)) % 16 ? 3 : 0, slices = slices_of(rows, vocab, shift);
    const int per = (int)(((long long)vocab + shift + slices - 1) / slices + 3) / 4 * 4;
    SliceSum* sums = (SliceSum*)work;
    u64* keys = (u64*)(sums + (size_t)rows * slices);
    double* base = (double*)(keys + (size_t)rows * slices * num);
    if (rows) {
        const cudaError_t e = launch_pdl(beam_slice_kernel, dim3(slices, rows), dim3(NT), AHEAD * TILE * 4, stream, logits, ld, vocab, per, num, sums, keys);
        if (e != cudaSuccess) return (int)e;
    }
    return (int)launch_pdl(beam_merge_kernel, dim3(groups), dim3(NT), 0, stream, sums, keys, slices, num, scores, rows, group_start, base, values, chosen_rows,
                           chosen_tokens);
}

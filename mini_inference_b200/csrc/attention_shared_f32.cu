// Decode attention over a shared prefix in true float32, head size 64 or 128 (what the work is and how it is cut: attention_shared.cuh).
//
// A tile of rows is up to 32 (row, query head) pairs of one key head, a tile of keys 32.  Keys and values come by cp.async into two stages, a tile ahead, over the
// ends of pieces too; what lies outside the visible keys comes as zeros.  Scores: a thread has two rows and two keys (padded rows in shared memory, so that
// 16 keys' pieces lie in different banks); softmax: eight threads a row, float32, base 2; weighted sums: a warp has four rows, a lane D / 32
// neighbouring columns in registers.  Bound by shared-memory reads (six wavefronts for sixteen multiply-adds of a warp); a tail's few rows leave most warps
// out, and there it is bound by the bytes.  13 rows in two groups on 1,504 and 976 shared and 100 own keys (32 heads over 8 of 128): 37 us with the merge (row by
// row, as calls of that size run, 29); its
// multiply-adds would take 4.  A block has three to five tiles then, and each piece's queries, page numbers and first keys come one behind the other.  Scores in
// 4 x 4 squares over quarters of the head, and a warp per four keys for tails, took 36 us there and 8 % less at 8 x 2,048 keys, 8 % more for tails alone.
#include "attention_shared.cuh"
#include <math.h>

using namespace mi;
using namespace mi::shared_attention;

namespace {

constexpr int KT = 32, M = 32, THREADS = 256;

template <int D> struct Tiles {                      // floats in shared memory
    static constexpr int QS = D + 4, KS = D + 4, PS = KT + 4;
    static constexpr int Q = 0, K = Q + M * QS, V = K + 2 * KT * KS, P = V + 2 * KT * D, ALPHA = P + M * PS, END = ALPHA + M;
};

__device__ __forceinline__ void fetch16(float* to, const float* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" :: "r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
}

template <int D>
__global__ void __launch_bounds__(THREADS, 2) attn_shared_f32_kernel(const __grid_constant__ Args a, const float* __restrict__ q, long long q_stride,
                                                                     const float* __restrict__ k_cache, const float* __restrict__ v_cache, float scale_log2) {
    using T = Tiles<D>;
    constexpr int PIECES = D / 4, C = D / 32;        // 16-byte pieces of a row; columns of a lane
    extern __shared__ __align__(16) float smem[];
    const Plan plan(reinterpret_cast<int*>(smem + T::END), a.G, a.R);
    pdl_trigger();
    pdl_wait(q, k_cache, v_cache);
    make_plan<KT>(a, plan);
    __syncthreads();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, Hg = a.H / a.KV;

    Walk<KT> ahead(a, plan), walk(a, plan);
    int ahead_tile = 0, ahead_tiles = 0;
    const int* table = nullptr;
    auto load_next = [&](int stage) {                // the line's next tile, if there is one
        if (ahead_tile == ahead_tiles) {
            ahead_tile = ahead_tiles = 0;
            if (ahead.next()) { ahead_tiles = ahead.tiles; table = a.block_table + (size_t)ahead.table_row() * a.table_stride; }
        }
        if (ahead_tile < ahead_tiles) {
            const int key = ahead.key0 + ahead_tile++ * KT;
            for (int id = tid; id < KT * PIECES; id += THREADS) {
                const int j = id / PIECES, c = id % PIECES * 4, at = key + j;
                const bool there = at >= ahead.lo && at < ahead.hi;
                const long long off = there ? ((long long)((long long)table[at / a.ps] * a.KV + ahead.kvh) * a.ps + at % a.ps) * D + c : 0;
                fetch16(smem + T::K + (stage * KT + j) * T::KS + c, k_cache + off, there);
                fetch16(smem + T::V + (stage * KT + j) * D + c, v_cache + off, there);
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };

    load_next(0);
    int n = 0;
    while (walk.next()) {
        const int rows = walk.rows * Hg;
        for (int id = tid; id < rows * PIECES; id += THREADS) {
            const int row = id / PIECES, c = id % PIECES * 4, r = walk.row0 + row / Hg, h = walk.kvh * Hg + row % Hg;
            *reinterpret_cast<float4*>(smem + T::Q + row * T::QS + c) =
                *reinterpret_cast<const float4*>(q + (size_t)plan.token[r] * q_stride + (size_t)h * D + c);
        }
        const int my_row = tid >> 3;                 // softmax: eight threads a row
        const int hi = my_row < rows ? walk.end_of(my_row / Hg) : 0;
        float m = -INFINITY, l = 0.f, acc[4][C];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c) acc[i][c] = 0.f;
        for (int i = 0; i < walk.tiles; ++i, ++n) {
            const int s = n & 1, key = walk.key0 + i * KT;
            load_next(s ^ 1);
            asm volatile("cp.async.wait_group 1;\n" ::: "memory");
            __syncthreads();
            const int ty = tid >> 4, tx = tid & 15;
            if (2 * ty < rows) {
                float sc[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
                const float *q0 = smem + T::Q + 2 * ty * T::QS, *k0 = smem + T::K + (s * KT + tx) * T::KS;
#pragma unroll 8
                for (int c = 0; c < D; c += 4) {
                    const float4 qa = *reinterpret_cast<const float4*>(q0 + c), qb = *reinterpret_cast<const float4*>(q0 + T::QS + c);
                    const float4 ka = *reinterpret_cast<const float4*>(k0 + c), kb = *reinterpret_cast<const float4*>(k0 + 16 * T::KS + c);
                    sc[0][0] = fmaf(qa.w, ka.w, fmaf(qa.z, ka.z, fmaf(qa.y, ka.y, fmaf(qa.x, ka.x, sc[0][0]))));
                    sc[0][1] = fmaf(qa.w, kb.w, fmaf(qa.z, kb.z, fmaf(qa.y, kb.y, fmaf(qa.x, kb.x, sc[0][1]))));
                    sc[1][0] = fmaf(qb.w, ka.w, fmaf(qb.z, ka.z, fmaf(qb.y, ka.y, fmaf(qb.x, ka.x, sc[1][0]))));
                    sc[1][1] = fmaf(qb.w, kb.w, fmaf(qb.z, kb.z, fmaf(qb.y, kb.y, fmaf(qb.x, kb.x, sc[1][1]))));
                }
                float* p = smem + T::P + 2 * ty * T::PS + tx;
                p[0] = sc[0][0]; p[16] = sc[0][1]; p[T::PS] = sc[1][0]; p[T::PS + 16] = sc[1][1];
            }
            __syncthreads();
            if (my_row < (rows + 3) / 4 * 4) {       // whole warps: four rows
                float* p = smem + T::P + my_row * T::PS + (tid & 7) * 4;
                float sc[4], top = -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = key + (tid & 7) * 4 + e;
                    sc[e] = at >= walk.lo && at < hi ? p[e] * scale_log2 : -INFINITY;
                    top = fmaxf(top, sc[e]);
                }
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const float now = fmaxf(m, top), off = now == -INFINITY ? 0.f : now, alpha = exp2f(m - off);
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) { sc[e] = exp2f(sc[e] - off); sum += sc[e]; }
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                l = l * alpha + sum;
                m = now;
                *reinterpret_cast<float4*>(p) = make_float4(sc[0], sc[1], sc[2], sc[3]);
                if ((tid & 7) == 0) smem[T::ALPHA + my_row] = alpha;
                __syncwarp();
                // weighted sums: this warp's four rows are the ones whose weights it just made
                const float *pw = smem + T::P + 4 * warp * T::PS, *v = smem + T::V + s * KT * D + C * lane;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float f = smem[T::ALPHA + 4 * warp + r];
#pragma unroll
                    for (int c = 0; c < C; ++c) acc[r][c] *= f;
                }
#pragma unroll 2
                for (int j = 0; j < KT; j += 4) {
                    float w[4][4], x[4][C];
#pragma unroll
                    for (int r = 0; r < 4; ++r) load16(pw + r * T::PS + j, w[r]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (C == 4) load16(v + (j + e) * D, x[e]);
                        else load2(v + (j + e) * D, x[e][0], x[e][1]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int c = 0; c < C; ++c) acc[r][c] = fmaf(w[r][e], x[e][c], acc[r][c]);
                }
            }
            __syncthreads();                         // the stage, the scores and (behind the last tile) the queries are free
        }
        const size_t at = (size_t)walk.place();
        float* o = (walk.prefix ? a.o_prefix : a.o_tail) + at * D + (C * lane / 4 * rows + 4 * warp) * 4 + C * lane % 4;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (4 * warp + r < rows) {
                store2(o + 4 * r, acc[r][0], acc[r][1]);
                if constexpr (C == 4) store2(o + 4 * r + 2, acc[r][2], acc[r][3]);
            }
        if (my_row < rows && (tid & 7) == 0) (walk.prefix ? a.ml_prefix : a.ml_tail)[at + my_row] = make_float2(m, l);
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
}

bool fits(int R, int G, int H, int KV, int D, int ps) {
    return R > 0 && G >= 0 && R + G <= MAX_ENTITIES && KV > 0 && KV <= 65535 && H % KV == 0 && H / KV <= M && (D == 64 || D == 128) && ps > 0;
}
int tile_rows_of(int H, int KV) { return M / (H / KV); }
int slot_rows_of(int H, int KV, int most) { const int t = tile_rows_of(H, KV); return (most < t ? (most > 1 ? most : 1) : t) * (H / KV); }
// a call's sizes, without its pointers
Args sizes(int R, int G, int entries, int most, int table_stride, int H, int KV, int ps) {
    Args a = {};
    a.R = R; a.G = G; a.entries = entries; a.most = most > R ? R : most > 1 ? most : 1; a.table_stride = table_stride; a.H = H; a.KV = KV; a.ps = ps;
    a.tile_rows = tile_rows_of(H, KV); a.copies = 0; a.slot_rows = slot_rows_of(H, KV, a.most); a.tail_rows = H / KV;
    return a;
}

}  // namespace

// Bytes of the work space of a call; -2: sizes that this kernel does not take.  most: rows of the largest group.
MI_EXPORT long long mi_attn_shared_f32_bytes(int R, int G, int most, int H, int KV, int D, int ps) {
    if (!fits(R, G, H, KV, D, ps)) return -2;
    return scratch(sizes(R, G, 1, most, 0, H, KV, ps), D, 2 * device_sms()).bytes;
}

// As mi_attn_shared_tc, in float32.
MI_EXPORT int mi_attn_shared_f32(const float* q, int q_stride, const float* k_cache, const float* v_cache, float* out, const int* decode_segs, int R,
                                 const int* seg_q_start, const int* seg_kv_len, int entries, const int* block_table, const int* table_rows, int table_stride,
                                 const int* shared_start, const int* shared_len, int G, int most, int H, int KV, int D, int ps, float scale, void* work,
                                 cudaStream_t stream) {
    if (R == 0) return 0;
    if (!fits(R, G, H, KV, D, ps) || entries < 1 || q_stride % 4 || (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)work) % 16)) return -2;
    const int blocks = 2 * device_sms();
    Args a = sizes(R, G, entries, most, table_stride, H, KV, ps);
    a.decode_segs = decode_segs; a.seg_q_start = seg_q_start; a.seg_kv_len = seg_kv_len; a.block_table = block_table; a.table_rows = table_rows;
    a.shared_start = shared_start; a.shared_len = shared_len;
    const Scratch s = scratch(a, D, blocks);
    if (s.bytes < 0) return -2;
    place_scratch(a, s, work);
    const float scale_log2 = scale * 1.4426950408889634f;
#define LAUNCH(DD) do { \
        const size_t smem = (size_t)Tiles<DD>::END * 4, plan = (size_t)plan_ints(G, R) * 4; \
        static std::atomic<unsigned long long> done{0}; \
        cudaError_t e = allow_shared(attn_shared_f32_kernel<DD>, (int)(smem + (6 * MAX_ENTITIES + 1) * 4), done); \
        if (e == cudaSuccess) e = launch_pdl(attn_shared_f32_kernel<DD>, dim3(blocks), dim3(THREADS), smem + plan, stream, a, q, (long long)q_stride, k_cache, v_cache, \
                                             scale_log2); \
        if (e == cudaSuccess) e = merge<float, DD>(a, out, stream); \
        return (int)e; \
    } while (0)
    if (D == 128) LAUNCH(128);
    LAUNCH(64);
#undef LAUNCH
}

// Decode attention over a shared prefix on the 5th-generation tensor cores (tcgen05 + tensor memory + TMA), bfloat16, head size 64 or 128.
//
// Reference: none; davidjoyme/mini-inference (kernels/paged_attention/decode_triton.py:6-100) reads a common prefix once per request and query head.
// What the work is and how it is cut: attention_shared.cuh.  Here a tile of rows is the M side of the products: up to 128 (row, query head) pairs
// of one key head, 128 / (H / KV) rows; a tail has the H / KV heads of its row.  Lanes beyond them hold whatever was there and write nothing.
//
// One block is seven warps, two blocks an SM; a block walks its tiles of 64 keys through all its pieces without a stop:
//   warp 0, 6  TMA: key and value tiles, box by box of the page table's rows, into rings of two tiles (128-byte swizzle).  They run ahead over
//              the end of a piece.  A tile with values in front of a piece's first or behind its last key arrives on a barrier of its own, is cleared
//              there (what lies in a page's unused part may be anything, and 0 * inf is no 0) and handed on.
//   warp 1     one thread issues S = Q K^T (scores in one of two 64-column buffers of tensor memory) a tile ahead, and O += P V
//   warps 2-5  a matrix row a thread: mask, running maximum and sum (float32, base 2; the exponent's offset is kept until the maximum has grown by 2^8),
//              weights as bfloat16 back to tensor memory; values that no row sees are cleared in shared memory.  With the last tile's weights handed over they bring the next piece's queries, then write
//              this one's O, maximum and sum.  A warp whose 32 rows are all beyond the piece only keeps step.
// Weights are rounded to bfloat16 for P V (2^-9 of each, of random sign over the keys; the sums take them unrounded), as the engine's other decode and prompt attention does.
// Two launches: this one, and the merge.  Every mbarrier wait is bounded.
#include "attention_shared.cuh"
#include "sm100.cuh"
#include <map>
#include <mutex>
#include <tuple>
#include <math.h>

using namespace mi;
using namespace mi::sm100;
using namespace mi::shared_attention;

namespace {

constexpr int BQ = 128, KT = 64, THREADS = 224;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float max3(float a, float b, float c) {      // one instruction on this architecture
    float d;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {       // tmem_st32 for 16 columns
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
                 :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                    "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}

template <int D>
__global__ void __launch_bounds__(THREADS, 2)
attn_shared_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Args a,
                      const __nv_bfloat16* __restrict__ q, long long q_stride, float scale_log2, int* __restrict__ error_word) {
    constexpr int HALVES = D / 64, Q_BYTES = BQ * D * 2, KV_BYTES = KT * D * 2;
    constexpr int TMEM_COLS = 256;                       // S0: 64, S1: 64 (P takes the first 32 columns of its S), O: D
    constexpr uint32_t S_COL = 0, O_COL = 128;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    // [Q][K0][K1][V0][V1][barriers][plan]
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + Q_BYTES + 4 * KV_BYTES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);
    const Plan plan(reinterpret_cast<int*>(bars + 16), a.G, a.R);
    const uint32_t sQ = smem_u32(base), sK = sQ + Q_BYTES, sV = sK + 2 * KV_BYTES;
    const uint32_t q_full = smem_u32(bars), k_full = smem_u32(bars + 1), k_empty = smem_u32(bars + 3), s_full = smem_u32(bars + 5),
                   p_ready = smem_u32(bars + 7), pv_done = smem_u32(bars + 8), v_full = smem_u32(bars + 9), v_empty = smem_u32(bars + 11),
                   o_free = smem_u32(bars + 13);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int Hg = a.H / a.KV;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 128);
        mbar_init(k_full, 1); mbar_init(k_full + 8, 1); mbar_init(k_empty, 1); mbar_init(k_empty + 8, 1);
        mbar_init(v_full, 1); mbar_init(v_full + 8, 1); mbar_init(v_empty, 1); mbar_init(v_empty + 8, 1);
        mbar_init(s_full, 1); mbar_init(s_full + 8, 1); mbar_init(p_ready, 128); mbar_init(pv_done, 1); mbar_init(o_free, 128);
        mbar_init_fence();
        tma_prefetch_desc(&kmap); tma_prefetch_desc(&vmap);
    }
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();                                       // behind the allocation: a kernel that starts early may want tensor memory too
    pdl_wait(q);
    make_plan<KT>(a, plan);
    __syncthreads();
    const uint32_t tmem = *tmem_slot;
    Walk<KT> walk(a, plan);

    if (warp == 0 || warp == 6) {
        // ---------------- loads.  Lane 0 owns the barriers; the boxes of a tile are issued by one lane each.
        const bool is_v = warp == 6;
        const int box = min(a.ps, KT), ops_per_tile = KT / box * HALVES;
        const uint32_t full = is_v ? v_full : k_full, empty = is_v ? v_empty : k_empty, dst0 = is_v ? sV : sK;
        const CUtensorMap* map = is_v ? &vmap : &kmap;
        bool ok = true;
        int n = 0;                                           // tiles so far
        while (ok && walk.next()) {
            const int* table = walk.table();
            for (int i = 0; i < walk.tiles && ok; ++i, ++n) {
                const int s = n & 1, key = walk.key0 + i * KT;
                if (lane == 0) {
                    if (n >= 2 && !mbar_wait(empty + 8 * s, ((n >> 1) - 1) & 1)) { atomicExch(error_word, 61); ok = false; }
                    if (ok) mbar_expect_tx(full + 8 * s, KV_BYTES);
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;
                for (int op = lane; op < ops_per_tile; op += 32) {
                    const int b = op / HALVES, hb = op % HALVES, j = key + b * box;
                    const int page = j < walk.hi ? table[j / a.ps] : 0;                        // behind the last key: the null page
                    tma_load_2d(dst0 + s * KV_BYTES + hb * (KT * 128) + b * box * 128, map, hb * 64, (page * a.KV + walk.kvh) * a.ps + j % a.ps, full + 8 * s);
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issue
        if (lane == 0) {
            const uint32_t idesc_s = umma_idesc_bf16(BQ, KT, false);      // S[128 x 64]  = Q (K-major) * K^T (K-major)
            const uint32_t idesc_o = umma_idesc_bf16(BQ, D, true);        // O[128 x D]  += P (tensor memory) * V (MN-major)
            bool ok = true;
            int n = 0, pieces = 0;
            auto issue_qk = [&](int m) {
                const int s = m & 1;
                if (!mbar_wait(k_full + 8 * s, (m >> 1) & 1)) { atomicExch(error_word, 63); ok = false; return; }
                tc_fence_after();
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint32_t qa = sQ + (ks / 4) * (BQ * 128) + (ks % 4) * 32, kb = sK + s * KV_BYTES + (ks / 4) * (KT * 128) + (ks % 4) * 32;
                    umma_ss(tmem + S_COL + 64 * s, umma_desc_sw128(qa, 16, 1024), umma_desc_sw128(kb, 16, 1024), idesc_s, ks != 0);
                }
                umma_commit(k_empty + 8 * s);                  // the keys of this stage are free once these finish
                umma_commit(s_full + 8 * s);
            };
            while (ok && walk.next()) {
                if (!mbar_wait(q_full, pieces & 1)) { atomicExch(error_word, 64); break; }
                issue_qk(n);
                for (int i = 0; i < walk.tiles && ok; ++i, ++n) {
                    const int s = n & 1;
                    if (i + 1 < walk.tiles) issue_qk(n + 1);       // a tile ahead of the softmax, within a piece
                    if (!ok) break;
                    if (!mbar_wait(p_ready, n & 1)) { atomicExch(error_word, 65); ok = false; break; }
                    if (!mbar_wait(v_full + 8 * s, (n >> 1) & 1)) { atomicExch(error_word, 66); ok = false; break; }
                    if (i == 0 && pieces > 0 && !mbar_wait(o_free, (pieces - 1) & 1)) { atomicExch(error_word, 67); ok = false; break; }
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < KT / 16; ++kk)
                        umma_ts(tmem + O_COL, tmem + S_COL + 64 * s + kk * 8, umma_desc_sw128(sV + s * KV_BYTES + kk * (16 * 128), KT * 128, 1024), idesc_o, (i | kk) != 0);
                    umma_commit(v_empty + 8 * s);
                    umma_commit(pv_done);
                }
                ++pieces;
            }
        }
    } else {
        // ---------------- softmax: thread <-> (row, head) <-> tensor-memory lane
        const int lg = warp & 3, mine = lg * 32 + lane, tid = threadIdx.x - 64;
        const uint32_t lane_addr = tmem + ((uint32_t)(lg * 32) << 16);
        auto bring_queries = [&](const Walk<KT>& w) {          // the piece's queries into swizzled rows of shared memory, eight pieces of 16 bytes of a thread in flight
            constexpr int C = D / 8, STEP = 128 / C;
            const int c = tid % C, first = tid / C, n = w.rows * Hg;
            for (int row0 = first; row0 < n; row0 += 8 * STEP) {
                uint4 v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int row = row0 + k * STEP;
                    if (row < n) v[k] = *reinterpret_cast<const uint4*>(q + (size_t)plan.token[w.row0 + row / Hg] * q_stride + (size_t)(w.kvh * Hg + row % Hg) * D + c * 8);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int row = row0 + k * STEP;
                    if (row < n) *reinterpret_cast<uint4*>(base + (c / 8) * (BQ * 128) + row * 128 + (((c % 8) ^ (row & 7)) << 4)) = v[k];
                }
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            mbar_arrive(q_full);
        };
        bool ok = true, more = walk.next();
        int n = 0;
        if (more) bring_queries(walk);
        while (more && ok) {
            const int rows = walk.rows * Hg, tiles = walk.tiles, key0 = walk.key0, lo = walk.lo, place = walk.place();
            const bool prefix = walk.prefix, active = lg * 32 < rows;
            const int hi = walk.hi;
            // a prefix's rows see no further than their own length; lanes beyond the rows hold anything
            const int mine_hi = mine < rows ? min(hi, plan.keys[walk.row0 + mine / Hg]) : hi;
            float m_ref = -INFINITY, l = 0.f;
            for (int i = 0; i < tiles && ok; ++i, ++n) {
                const int s = n & 1, key = key0 + i * KT;
                const uint32_t s_addr = lane_addr + S_COL + 64 * s;
                if (!mbar_wait(s_full + 8 * s, (n >> 1) & 1)) { atomicExch(error_word, 68); ok = false; break; }
                tc_fence_after();
                float alpha = 1.f;
                bool rescale = false;
                if (active) {
                    // The scores in two halves of 32, read twice: for the maximum, and for the weights (few registers, little code)
                    const bool whole = __all_sync(0xffffffffu, key >= lo && key + KT <= mine_hi);
                    const uint32_t from = (uint32_t)(key - lo), span = (uint32_t)max(mine_hi - lo, 0);      // a key in front of lo wraps around
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    uint32_t r[32];
#pragma unroll 1
                    for (int half = 1; half >= 0; --half) {
                        tmem_ld32(s_addr + 32 * half, r);
                        tmem_wait_ld();
                        if (!whole) {
#pragma unroll
                            for (int c = 0; c < 32; ++c) r[c] = from + (half * 32 + c) < span ? r[c] : 0xff800000u;       // -inf
                        }
#pragma unroll
                        for (int c = 0; c < 32; c += 8)
#pragma unroll
                            for (int e = 0; e < 4; ++e) mx4[e] = max3(mx4[e], __uint_as_float(r[c + 2 * e]), __uint_as_float(r[c + 2 * e + 1]));
                    }
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale_log2;      // scale > 0
                    if (mx > m_ref + 8.f) {
                        alpha = m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - mx);
                        rescale = i > 0 && m_ref != -INFINITY;
                        m_ref = mx;
                        l *= alpha;
                    }
                    const float off = m_ref == -INFINITY ? 0.f : m_ref;
                    const float2 scale2 = make_float2(scale_log2, scale_log2), noff2 = make_float2(-off, -off);
                    float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {             // r holds the first half
                        if (half) {
                            tmem_ld32(s_addr + 32, r);
                            tmem_wait_ld();
                            if (!whole) {
#pragma unroll
                                for (int c = 0; c < 32; ++c) r[c] = from + (32 + c) < span ? r[c] : 0xff800000u;
                            }
                        }
                        uint32_t pk[16];
#pragma unroll
                        for (int c = 0; c < 16; ++c) {
                            const float2 arg = __ffma2_rn(make_float2(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1])), scale2, noff2);
                            const float2 p = make_float2(fast_exp2(arg.x), fast_exp2(arg.y));
                            sums[c & 1] = __fadd2_rn(sums[c & 1], p);
                            pk[c] = pack_bf16(p.x, p.y);
                        }
                        tmem_st16(s_addr + 16 * half, pk);             // P takes the place of the first scores
                    }
                    const float2 s01 = __fadd2_rn(sums[0], sums[1]);
                    l += s01.x + s01.y;
                }
                if (key < lo || key + KT > hi) {
                    // Values in front of the piece's first or behind its last key may be anything (a page's unused part), and 0 * inf is no 0
                    if (!mbar_wait(v_full + 8 * s, (n >> 1) & 1)) { atomicExch(error_word, 62); ok = false; break; }
                    unsigned char* v = base + Q_BYTES + 2 * KV_BYTES + s * KV_BYTES;
                    for (int id = tid; id < KT * HALVES * 8; id += 128) {
                        const int chunk = id % 8, hb = id / 8 % HALVES, vr = id / (8 * HALVES);
                        if (key + vr < lo || key + vr >= hi) *reinterpret_cast<uint4*>(v + hb * (KT * 128) + vr * 128 + chunk * 16) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                }
                // every thread follows pv_done phase by phase; O holds the tile before this one completely after it
                if (n > 0 && !mbar_wait(pv_done, (n - 1) & 1)) { atomicExch(error_word, 69); ok = false; }
                if (__any_sync(0xffffffffu, rescale)) {
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(lane_addr + O_COL + c * 32, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st32(lane_addr + O_COL + c * 32, o);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(p_ready);
            }
            if (!ok) break;
            // the last tile's scores are there, so nothing reads this piece's queries any more
            more = walk.next();
            if (more) bring_queries(walk);
            if (!mbar_wait(pv_done, (n - 1) & 1)) { atomicExch(error_word, 70); break; }
            tc_fence_after();
            if (active) {
                const int rows_of = prefix ? a.slot_rows : Hg;
                float4* to = reinterpret_cast<float4*>(prefix ? a.o_prefix : a.o_tail) + (size_t)place * (D / 4) * rows_of + mine;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(lane_addr + O_COL + c * 32, o);
                    tmem_wait_ld();
                    if (mine < rows) {
#pragma unroll
                        for (int v4 = 0; v4 < 8; ++v4)
                            to[(size_t)(c * 8 + v4) * rows_of] = make_float4(__uint_as_float(o[4 * v4]), __uint_as_float(o[4 * v4 + 1]), __uint_as_float(o[4 * v4 + 2]), __uint_as_float(o[4 * v4 + 3]));
                    }
                }
                if (mine < rows) (prefix ? a.ml_prefix : a.ml_tail)[(size_t)place * rows_of + mine] = make_float2(m_ref, l);
            }
            tc_fence_before();
            mbar_arrive(o_free);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
}

std::mutex map_mutex;
std::map<std::tuple<const void*, long long, int, int>, CUtensorMap> maps;

bool cache_map(const void* cache, long long rows, int D, int box, CUtensorMap* out) {
    std::lock_guard<std::mutex> lock(map_mutex);
    const auto key = std::make_tuple(cache, rows, D, box);
    auto it = maps.find(key);
    if (it == maps.end()) {
        CUtensorMap m;
        if (!sm100_host::make_map_bf16(&m, cache, (uint64_t)rows, D, D, box, 64)) return false;
        it = maps.emplace(key, m).first;
    }
    *out = it->second;
    return true;
}

bool fits(int R, int G, int H, int KV, int D, int ps) {
    return R > 0 && G >= 0 && R + G <= MAX_ENTITIES && KV > 0 && H % KV == 0 && H / KV <= BQ && (D == 64 || D == 128) && ps % 8 == 0 &&
           (ps <= KT ? KT % ps == 0 : ps % KT == 0) && KV <= 65535;
}
int tile_rows_of(int H, int KV) { return BQ / (H / KV); }
int row_tiles_of(int H, int KV, int most) { const int t = tile_rows_of(H, KV); return most > 1 ? (most + t - 1) / t : 1; }
int slot_rows_of(int H, int KV, int most) { const int t = tile_rows_of(H, KV); return (most < t ? (most > 1 ? most : 1) : t) * (H / KV); }

}  // namespace

// Bytes of the work space of a call; -2: sizes that this kernel does not take.  most: rows of the largest group.
MI_EXPORT long long mi_attn_shared_tc_bytes(int R, int G, int most, int H, int KV, int D, int ps) {
    if (!fits(R, G, H, KV, D, ps)) return -2;
    return scratch(R, G, H, KV, D, row_tiles_of(H, KV, most), slot_rows_of(H, KV, most), 2 * device_sms()).bytes;
}

// q, out bfloat16 ([tokens, H D], rows of q q_stride apart); caches [pages, KV, ps, D] with cache_rows = pages KV ps; decode_segs int32 [R] (the entries, one token
// each), shared_start int32 [G + 1] over them, shared_len int32 [G]; block_table rows table_stride apart (entry i reads row table_rows[i], or i).
MI_EXPORT int mi_attn_shared_tc(const void* q, int q_stride, const void* k_cache, const void* v_cache, long long cache_rows, void* out, const int* decode_segs, int R,
                                const int* seg_q_start, const int* seg_kv_len, const int* block_table, const int* table_rows, int table_stride,
                                const int* shared_start, const int* shared_len, int G, int most, int H, int KV, int D, int ps, float scale, void* work,
                                int* error_word, cudaStream_t stream) {
    if (R == 0) return 0;
    if (!fits(R, G, H, KV, D, ps) || q_stride % 8 || cache_rows > 0x7fffffff || (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)work) % 16)) return -2;
    CUtensorMap kmap, vmap;
    if (!cache_map(k_cache, cache_rows, D, ps < KT ? ps : KT, &kmap) || !cache_map(v_cache, cache_rows, D, ps < KT ? ps : KT, &vmap)) return -5;
    const int blocks = 2 * device_sms();
    Args a{decode_segs, seg_q_start, seg_kv_len, block_table, table_rows, shared_start, shared_len, R, G, most > 1 ? most : 1, table_stride, H, KV, ps,
           row_tiles_of(H, KV, most), tile_rows_of(H, KV), slot_rows_of(H, KV, most)};
    place_scratch(a, scratch(R, G, H, KV, D, a.row_tiles, a.slot_rows, blocks), work);
    const auto bytes = [&](int ints) { return (size_t)BQ * D * 2 + 4 * (size_t)KT * D * 2 + 16 * 8 + (size_t)ints * 4 + 1024; };
    const size_t smem = bytes(plan_ints(G, R)), most_smem = bytes(6 * MAX_ENTITIES + 1);
    const float scale_log2 = scale * LOG2E;
#define LAUNCH(DD) do { \
        cudaError_t e = cudaFuncSetAttribute(attn_shared_tc_kernel<DD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most_smem); \
        if (e == cudaSuccess) e = launch_pdl(attn_shared_tc_kernel<DD>, dim3(blocks), dim3(THREADS), smem, stream, kmap, vmap, a, (const __nv_bfloat16*)q, \
                                             (long long)q_stride, scale_log2, error_word); \
        if (e == cudaSuccess) e = launch_pdl(merge_kernel<__nv_bfloat16, DD>, dim3(R, KV), dim3(128 * MERGE_PARTS), 0, stream, a, (__nv_bfloat16*)out); \
        return (int)e; \
    } while (0)
    if (D == 128) LAUNCH(128);
    LAUNCH(64);
#undef LAUNCH
}

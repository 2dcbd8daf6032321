// Decode attention over a shared prefix on the 5th-generation tensor cores (tcgen05 + tensor memory + TMA), bfloat16, head size 64 or 128.
//
// Reference: none; davidjoyme/mini-inference (kernels/paged_attention/decode_triton.py:6-100) reads a common prefix once per request and query head.
// What the work is and how it is cut: attention_shared.cuh.  Here a tile of rows is the M side of the products: up to 128 (row, query head) pairs
// of one key head, 128 / (H / KV) rows; a tail has the H / KV heads of its row.  Lanes beyond them hold whatever was there and write nothing.
//
// One block is seven warps, two blocks an SM; a block walks its tiles of 64 keys through all its pieces without a stop:
//   warp 0     finds the block's pieces and writes them down for the others; key tiles (TMA, box by box of the page table's rows) into a ring of two, 128-byte
//              swizzle, and each piece's queries (a box of heads per row); runs ahead over the end of a piece, and asks the page table for a tile while the one
//              before waits for its place
//   warp 6     value tiles, the same way
//   warp 1     one thread issues S = Q K^T (scores in one of two 64-column buffers of tensor memory) up to a tile ahead, over the end of a piece too, and
//              O += P V, whichever has its operands first
//   warps 2-5  a matrix row a thread: mask, running maximum and sum (float32, base 2; the exponent's offset is kept until the maximum has grown by 2^8),
//              weights as bfloat16 back to tensor memory; values that no row sees are cleared in shared memory (what lies in a page's unused part may be
//              anything, and 0 * inf is no 0; whole boxes behind the last key come as zeros).  At the end of a piece they write its O, maximum and sum.
// A warp reaches 32 rows of tensor memory, so with few rows one warp would make all weights while three wait (64 exponentials a thread are 512 clocks).
// Up to 32 rows therefore stand in the tile four times, up to 64 twice, and each copy's warps take their own part of the 64 columns, the others' weights
// being 0: a copy is a piece of its own with its own maximum and sum, so the warps need not agree on anything, and the merge adds copies like pieces.
// Pieces of up to 16 rows use the two halves of their 32 rows in turn, so the next one's queries come while this one's products run.
// Weights are rounded to bfloat16 for P V (2^-9 of each, of random sign over the keys; the sums take them unrounded), as the engine's other decode and prompt attention does.
// Two launches: this one, and the merge.  Every mbarrier wait is bounded.
//
// Measured (32 query heads over 8 key heads of 128, pages of 16): 8 groups of 8 rows on 4,096 shared and 256 own keys 48 us with the merge, 159 MB of keys and values (24 us at the
// copy rate); 16 rows of 40 heads on 32,000 + 500 keys 47 us (22 us); 64 rows on 8,192 + 1,000 keys 53 us (25 us); 4 rows on 512 + 48 keys 15 us
// (calls that read so little run row by row instead, in 8: ops.CudaOps.SHARED_BYTES).  With heads of 64 the first takes 36 us (79 MB: 12 us), 64 rows 46, 16 rows of 32 heads 33:
// a tile's softmax is the same, and its keys half as long.
// Every block spends 4 us before its first tile (the lists, then the page table, then keys: three trips to memory one behind the other) and the merge is 6 to 9 us;
// between them a tile takes an SM 1,850 clocks, memory alone would take 1,400: scores, softmax and weighted sum of a tile wait for one another, and two
// blocks an SM (all that 102 KB of shared memory leave room for) do not quite hide it.  The tensor pipe is busy for 24 % of the time, DRAM for 50 %.
// Without copies of few rows, and with queries by threads' loads instead of TMA, the first of these took 57 us where this form took 54 (both with a slower merge).
// Tails of several rows in the same tiles (boxes of a page that only their own row sees) make the line of tiles shorter and its tables longer: 52, 53, 60 and 18 us
// instead of 49, 47, 56 and 15; it was taken out again.
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

constexpr int BQ = 128, KT = 64, THREADS = 224, PIECES = 8;
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

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n"
                 :: "r"(dst), "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n"
                 :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
template <int W> __device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[W]) { if constexpr (W == 32) tmem_ld32(taddr, r); else tmem_ld16(taddr, r); }
template <int W> __device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[W]) { if constexpr (W == 16) tmem_st16(taddr, r); else tmem_st8(taddr, r); }

// A matrix row's scores of one tile, its columns col .. col + W parts - 1, to weights; the other columns' weights become 0
struct Row { float m, l; };                          // the exponent's offset (base 2) and the sum of weights
template <int W>
__device__ __forceinline__ bool weights(uint32_t s_addr, int col, int parts, bool whole, uint32_t from, uint32_t span, float scale_log2, bool first, Row& row, float& alpha) {
    uint32_t r[W];
    const auto scores = [&](int part) {
        tmem_ld<W>(s_addr + col + W * part, r);
        tmem_wait_ld();
        if (!whole) {
#pragma unroll
            for (int c = 0; c < W; ++c) r[c] = from + (part * W + c) < span ? r[c] : 0xff800000u;       // -inf
        }
    };
    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
    for (int part = parts - 1; part >= 0; --part) {
        scores(part);
#pragma unroll
        for (int c = 0; c < W; c += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx4[e] = max3(mx4[e], __uint_as_float(r[c + 2 * e]), __uint_as_float(r[c + 2 * e + 1]));
    }
    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale_log2;      // scale > 0
    bool rescale = false;
    alpha = 1.f;
    if (mx > row.m + 8.f) {
        alpha = row.m == -INFINITY ? 0.f : fast_exp2(row.m - mx);
        rescale = !first && row.m != -INFINITY;
        row.m = mx;
        row.l *= alpha;
    }
    const float off = row.m == -INFINITY ? 0.f : row.m;
    const float2 scale2 = make_float2(scale_log2, scale_log2), noff2 = make_float2(-off, -off);
    float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
    for (int part = 0; part < parts; ++part) {       // r holds the first part
        if (part) scores(part);
        uint32_t pk[W / 2];
#pragma unroll
        for (int c = 0; c < W / 2; ++c) {
            const float2 arg = __ffma2_rn(make_float2(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1])), scale2, noff2);
            const float2 p = make_float2(fast_exp2(arg.x), fast_exp2(arg.y));
            sums[c & 1] = __fadd2_rn(sums[c & 1], p);
            pk[c] = pack_bf16(p.x, p.y);
        }
        tmem_st<W / 2>(s_addr + (col + W * part) / 2, pk);             // weights take the place of the first scores
    }
    const float2 s01 = __fadd2_rn(sums[0], sums[1]);
    row.l += s01.x + s01.y;
    uint32_t none[W / 2];
#pragma unroll
    for (int c = 0; c < W / 2; ++c) none[c] = 0u;
    if (W * parts < KT) {
#pragma unroll 1
        for (int c = 0; c < KT; c += W)
            if (c != col) tmem_st<W / 2>(s_addr + c / 2, none);
    }
    return rescale;
}

template <int D>
__global__ void __launch_bounds__(THREADS, 2)
attn_shared_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                      const __grid_constant__ Args a, float scale_log2, int* __restrict__ error_word) {
    constexpr int HALVES = D / 64, Q_BYTES = BQ * D * 2, KV_BYTES = KT * D * 2;
    constexpr int TMEM_COLS = 256;                       // S0: 64, S1: 64 (P takes the first 32 columns of its S), O: D
    constexpr uint32_t S_COL = 0, O_COL = 128;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    // [Q][K0][K1][V0][V1][barriers][plan]
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + Q_BYTES + 4 * KV_BYTES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 25);
    Piece* pieces = reinterpret_cast<Piece*>(bars + 26);                // the last PIECES pieces
    const Plan plan(reinterpret_cast<int*>(pieces + PIECES), a.G, a.R);
    const uint32_t sQ = smem_u32(base), sK = sQ + Q_BYTES, sV = sK + 2 * KV_BYTES;
    // pairs: of tiles or pieces in turn
    const uint32_t q_full = smem_u32(bars), q_done = smem_u32(bars + 2), k_full = smem_u32(bars + 4), k_empty = smem_u32(bars + 6), s_full = smem_u32(bars + 8),
                   v_full = smem_u32(bars + 10), v_empty = smem_u32(bars + 12), p_ready = smem_u32(bars + 14), pv_done = smem_u32(bars + 15), o_free = smem_u32(bars + 16),
                   found = smem_u32(bars + 17);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int Hg = a.H / a.KV;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 14; ++i) mbar_init(smem_u32(bars + i), 1);
        mbar_init(p_ready, 128); mbar_init(pv_done, 1); mbar_init(o_free, 128);
        for (int i = 0; i < PIECES; ++i) mbar_init(found + 8 * i, 1);
        mbar_init_fence();
        tma_prefetch_desc(&qmap); tma_prefetch_desc(&kmap); tma_prefetch_desc(&vmap);
    }
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();                                       // behind the allocation: a kernel that starts early may want tensor memory too
    pdl_wait();
    make_plan<KT>(a, plan);
    __syncthreads();
    const uint32_t tmem = *tmem_slot;
    // Piece i, once it is found; false behind the last one (or with a wait that ran out).  Warp 0 is at most four pieces in front of all who read them: it waits
    // for the queries' rows of the piece before last, whose scores wait for the weights of the tile before last.
    const auto piece_at = [&](int i, Piece& piece) {
        if (!mbar_wait(found + 8 * (i % PIECES), (i / PIECES) & 1)) { atomicExch(error_word, 101); return false; }
        const int4* from = reinterpret_cast<const int4*>(pieces + i % PIECES);
        int4* to = reinterpret_cast<int4*>(&piece);
        to[0] = from[0]; to[1] = from[1]; to[2] = from[2];
        return piece.tiles > 0;
    };
    Piece at;

    if (warp == 0 || warp == 6) {
        // ---------------- loads.  Lane 0 owns the barriers; the boxes of a tile are issued by one lane each.
        const bool is_v = warp == 6;
        const int box = min(a.ps, KT), ops_per_tile = KT / box * HALVES, b = lane / HALVES, hb = lane % HALVES;       // this lane's box (at most 8) and half
        const uint32_t full = is_v ? v_full : k_full, empty = is_v ? v_empty : k_empty, dst0 = is_v ? sV : sK;
        const CUtensorMap* map = is_v ? &vmap : &kmap;
        Walk<KT> walk(a, plan);
        const auto next = [&](int piece) {
            if (is_v) return piece_at(piece, at);
            const bool more = walk.next();
            if (more) {
                at.prefix = walk.prefix; at.who = walk.who; at.kvh = walk.kvh; at.row0 = walk.row0; at.rows = walk.rows; at.tiles = walk.tiles; at.lo = walk.lo; at.hi = walk.hi;
                at.key0 = walk.key0; at.place = walk.place(); at.table = walk.table_row();
            } else at.tiles = 0;
            if (lane == 0) {
                pieces[piece % PIECES] = at;
                mbar_arrive(found + 8 * (piece % PIECES));
            }
            return more;
        };
        bool ok = true, more = next(0);
        int i = 0, page = 0, before = BQ;                    // the piece's tile; matrix rows of the piece in front
        const int* table = nullptr;
        const auto ask = [&]() {                             // for the next tile's page; behind the last key: none
            const int j = at.key0 + i * KT + b * box;
            page = lane < ops_per_tile && j < at.hi ? table[j / a.ps] : -1;
        };
        if (more) { table = a.block_table + (size_t)at.table * a.table_stride; ask(); }
        for (int n = 0, piece = 0; more; ++n) {
            const int s = n & 1;
            if (lane == 0) {
                if (n >= 2 && !mbar_wait(empty + 8 * s, ((n >> 1) - 1) & 1)) { atomicExch(error_word, 103); ok = false; }
                if (ok) mbar_expect_tx(full + 8 * s, KV_BYTES);
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            if (lane < ops_per_tile) {
                // no page: a row in front of the first one, which comes as zeros
                const int y = page < 0 ? -box : (page * a.KV + at.kvh) * a.ps + (at.key0 + i * KT + b * box) % a.ps;
                tma_load_2d(dst0 + s * KV_BYTES + hb * (KT * 128) + b * box * 128, map, hb * 64, y, full + 8 * s);
            }
            if (!is_v && i == 0) {                           // the piece's queries, once the rows that they take are done with
                const int rows = at.rows * Hg, copies = copies_of(1, rows), apart = BQ / copies, off = rows <= 16 && piece & 1 ? 16 : 0;
                if (piece >= 2) ok = mbar_wait(q_done + 8 * (piece & 1), ((piece >> 1) - 1) & 1);
                if (ok && piece && (rows > 16 || before > 16)) ok = mbar_wait(q_done + 8 * ((piece - 1) & 1), ((piece - 1) >> 1) & 1);
                if (!__all_sync(0xffffffffu, ok)) { if (lane == 0) atomicExch(error_word, 102); break; }
                before = rows;
                if (lane == 0) mbar_expect_tx(q_full + 8 * (piece & 1), rows * copies * D * 2);
                __syncwarp();
                for (int op = lane; op < at.rows * copies * HALVES; op += 32) {
                    const int half = op % HALVES, set = op / HALVES & (copies - 1), r = op / HALVES / copies;
                    tma_load_3d(sQ + half * (BQ * 128) + (set * apart + off + r * Hg) * 128, &qmap, half * 64, at.kvh * Hg, plan.token[at.row0 + r], q_full + 8 * (piece & 1));
                }
            }
            if (++i == at.tiles) {
                i = 0;
                ++piece;
                __syncwarp();                                // lane 0 has written this piece down
                more = next(piece);
                if (more) table = a.block_table + (size_t)at.table * a.table_stride;
            }
            if (more) ask();
        }
    } else if (warp == 1) {
        // ---------------- MMA issue
        if (lane == 0) {
            const uint32_t idesc_s = umma_idesc_bf16(BQ, KT, false);      // S[128 x 64]  = Q (K-major) * K^T (K-major)
            const uint32_t idesc_o = umma_idesc_bf16(BQ, D, true);        // O[128 x D]  += P (tensor memory) * V (MN-major)
            int m = 0, tile_s = 0, piece_s = 0;              // the next scores (up to a tile in front): tile, tile of their piece, piece
            int n = 0, tile_o = 0, piece_o = 0;              // the next weighted sum
            bool more_s = piece_at(0, at), more_o = more_s;
            int tiles_s = at.tiles, tiles_o = at.tiles;
            for (uint32_t spins = 0; more_o; ++spins) {
                if (spins == SPIN_LIMIT << 4) { atomicExch(error_word, 105); break; }
                if (more_s && tiles_s == 0 && mbar_test(found + 8 * (piece_s % PIECES), (piece_s / PIECES) & 1)) {
                    tiles_s = pieces[piece_s % PIECES].tiles;
                    more_s = tiles_s > 0;
                }
                // scores go to the buffer whose weights the sum before last used
                if (more_s && tiles_s && m <= n + 1 && mbar_test(k_full + 8 * (m & 1), (m >> 1) & 1) && (tile_s || mbar_test(q_full + 8 * (piece_s & 1), (piece_s >> 1) & 1))) {
                    const int s = m & 1;
                    tc_fence_after();
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        const uint32_t qa = sQ + (ks / 4) * (BQ * 128) + (ks % 4) * 32, kb = sK + s * KV_BYTES + (ks / 4) * (KT * 128) + (ks % 4) * 32;
                        umma_ss(tmem + S_COL + 64 * s, umma_desc_sw128(qa, 16, 1024), umma_desc_sw128(kb, 16, 1024), idesc_s, ks != 0);
                    }
                    umma_commit(k_empty + 8 * s);              // the keys of this stage are free once these finish
                    umma_commit(s_full + 8 * s);
                    ++m;
                    if (++tile_s == tiles_s) {
                        umma_commit(q_done + 8 * (piece_s & 1));
                        tile_s = tiles_s = 0;                  // the next piece's number of tiles is asked for when it is found
                        ++piece_s;
                    }
                    spins = 0;
                }
                if (n < m && mbar_test(p_ready, n & 1) && mbar_test(v_full + 8 * (n & 1), (n >> 1) & 1) && (tile_o || !piece_o || mbar_test(o_free, (piece_o - 1) & 1))) {
                    const int s = n & 1;
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < KT / 16; ++kk)
                        umma_ts(tmem + O_COL, tmem + S_COL + 64 * s + kk * 8, umma_desc_sw128(sV + s * KV_BYTES + kk * (16 * 128), KT * 128, 1024), idesc_o, (tile_o | kk) != 0);
                    umma_commit(v_empty + 8 * s);
                    umma_commit(pv_done);
                    ++n;
                    if (++tile_o == tiles_o) {
                        tile_o = 0;
                        ++piece_o;
                        more_o = piece_at(piece_o, at);
                        tiles_o = at.tiles;
                    }
                    spins = 0;
                }
            }
        }
    } else {
        // ---------------- softmax: thread <-> (row, head) <-> tensor-memory lane
        const int lg = warp & 3, tid = threadIdx.x - 64;
        const uint32_t lane_addr = tmem + ((uint32_t)(lg * 32) << 16);
        bool ok = true;
        int n = 0;
        for (int piece = 0; ok && piece_at(piece, at); ++piece) {
            const int rows = at.rows * Hg, tiles = at.tiles, lo = at.lo, hi = at.hi;
            const int copies = copies_of(1, rows), warps = 4 / copies, copy = lg / warps, col = copy * (KT / copies);
            const int mine = lg % warps * 32 + lane - (rows <= 16 && piece & 1 ? 16 : 0);      // the row
            const bool there = mine >= 0 && mine < rows, active = __any_sync(0xffffffffu, there);
            // as Walk::end_of; lanes beyond the rows hold anything
            const int mine_hi = there && at.prefix ? min(hi, plan.first[at.row0 + mine / Hg]) : hi;
            Row row{-INFINITY, 0.f};
            for (int i = 0; i < tiles && ok; ++i, ++n) {
                const int s = n & 1, key = at.key0 + i * KT;
                const uint32_t s_addr = lane_addr + S_COL + 64 * s;
                if (!mbar_wait(s_full + 8 * s, (n >> 1) & 1)) { atomicExch(error_word, 106); ok = false; break; }
                tc_fence_after();
                float alpha = 1.f;
                bool rescale = false;
                if (active) {
                    const bool whole = __all_sync(0xffffffffu, key + col >= lo && key + col + KT / copies <= mine_hi);
                    const uint32_t from = (uint32_t)(key + col - lo), span = (uint32_t)max(mine_hi - lo, 0);      // a key in front of lo wraps around
                    if (copies == 4) rescale = weights<16>(s_addr, col, 1, whole, from, span, scale_log2, i == 0, row, alpha);
                    else rescale = weights<32>(s_addr, col, 2 / copies, whole, from, span, scale_log2, i == 0, row, alpha);
                }
                if (key < lo || key + KT > hi) {
                    // Values in front of the piece's first or behind its last key may be anything (a page's unused part), and 0 * inf is no 0
                    if (!mbar_wait(v_full + 8 * s, (n >> 1) & 1)) { atomicExch(error_word, 104); ok = false; break; }
                    unsigned char* v = base + Q_BYTES + 2 * KV_BYTES + s * KV_BYTES;
                    const int box = min(a.ps, KT), first = max(0, lo - key), last = min(KT, hi - key), end = min(KT, (last + box - 1) / box * box);
                    for (int id = tid; id < (first + end - last) * HALVES * 8; id += 128) {
                        const int row = id / (8 * HALVES), vr = row < first ? row : row - first + last, chunk = id % (8 * HALVES);
                        *reinterpret_cast<uint4*>(v + chunk / 8 * (KT * 128) + vr * 128 + chunk % 8 * 16) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                }
                // every thread follows pv_done phase by phase; O holds the tile before this one completely after it
                if (n > 0 && !mbar_wait(pv_done, (n - 1) & 1)) { atomicExch(error_word, 107); ok = false; }
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
            if (!mbar_wait(pv_done, (n - 1) & 1)) { atomicExch(error_word, 108); break; }
            tc_fence_after();
            if (active) {
                const int rows_of = copies * rows, line = copy * rows + mine;
                float4* to = reinterpret_cast<float4*>(at.prefix ? a.o_prefix : a.o_tail) + (size_t)at.place * (D / 4) + line;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(lane_addr + O_COL + c * 32, o);
                    tmem_wait_ld();
                    if (there) {
#pragma unroll
                        for (int v4 = 0; v4 < 8; ++v4)
                            to[(size_t)(c * 8 + v4) * rows_of] = make_float4(__uint_as_float(o[4 * v4]), __uint_as_float(o[4 * v4 + 1]), __uint_as_float(o[4 * v4 + 2]), __uint_as_float(o[4 * v4 + 3]));
                    }
                }
                if (there) (at.prefix ? a.ml_prefix : a.ml_tail)[(size_t)at.place + line] = make_float2(row.m, row.l);
            }
            tc_fence_before();
            mbar_arrive(o_free);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
}

// Maps of the caches that calls came with: addresses and shapes.  An engine has a few; a program that makes caches over and over begins again from none.
constexpr size_t MAPS = 1024;
std::mutex map_mutex;
std::map<std::tuple<const void*, long long, int, int>, CUtensorMap> maps;

bool cache_map(const void* cache, long long rows, int D, int box, CUtensorMap* out) {
    std::lock_guard<std::mutex> lock(map_mutex);
    const auto key = std::make_tuple(cache, rows, D, box);
    auto it = maps.find(key);
    if (it == maps.end()) {
        CUtensorMap m;
        if (!sm100_host::make_map_bf16(&m, cache, (uint64_t)rows, D, D, box, 64)) return false;
        if (maps.size() >= MAPS) maps.clear();
        it = maps.emplace(key, m).first;
    }
    *out = it->second;
    return true;
}

// The queries [tokens, heads, D], tokens `stride` elements apart (whole heads), in boxes of a key head's query heads x 64 columns
bool query_map(const void* q, int tokens, int H, int D, long long stride, int heads, CUtensorMap* out) {
    auto fn = sm100_host::encoder();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)tokens}, strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)heads, 1}, one[3] = {1, 1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool fits(int R, int G, int H, int KV, int D, int ps) {
    return R > 0 && G >= 0 && R + G <= MAX_ENTITIES && KV > 0 && H % KV == 0 && H / KV <= BQ && (D == 64 || D == 128) && ps % 8 == 0 &&
           (ps <= KT ? KT % ps == 0 : ps % KT == 0) && KV <= 65535;
}
int tile_rows_of(int H, int KV) { return BQ / (H / KV); }
int slot_rows_of(int H, int KV, int most) {          // with the copies of any number of rows up to the largest tile's
    const int t = tile_rows_of(H, KV), rows = (most < t ? (most > 1 ? most : 1) : t) * (H / KV);
    return rows <= BQ / 4 ? 4 * rows : BQ;
}
int tail_rows_of(int H, int KV) { return copies_of(1, H / KV) * (H / KV); }
// a call's sizes, without its pointers
Args sizes(int R, int G, int entries, int most, int table_stride, int H, int KV, int ps) {
    Args a = {};
    a.R = R; a.G = G; a.entries = entries; a.most = most > R ? R : most > 1 ? most : 1; a.table_stride = table_stride; a.H = H; a.KV = KV; a.ps = ps;
    a.tile_rows = tile_rows_of(H, KV); a.copies = 1; a.slot_rows = slot_rows_of(H, KV, a.most); a.tail_rows = tail_rows_of(H, KV);
    return a;
}

}  // namespace

// Bytes of the work space of a call; -2: sizes that this kernel does not take.  most: rows of the largest group.
MI_EXPORT long long mi_attn_shared_tc_bytes(int R, int G, int most, int H, int KV, int D, int ps) {
    if (!fits(R, G, H, KV, D, ps)) return -2;
    return scratch(sizes(R, G, 1, most, 0, H, KV, ps), D, 2 * device_sms()).bytes;
}

// q, out bfloat16 ([tokens, H D], rows of q q_stride apart); caches [pages, KV, ps, D] with cache_rows = pages KV ps; decode_segs int32 [R] (which of the `entries` feed one token
// each), shared_start int32 [G + 1] over them, shared_len int32 [G]; block_table rows table_stride apart (entry i reads row table_rows[i], or i).
MI_EXPORT int mi_attn_shared_tc(const void* q, int q_stride, int tokens, const void* k_cache, const void* v_cache, long long cache_rows, void* out, const int* decode_segs, int R,
                                const int* seg_q_start, const int* seg_kv_len, int entries, const int* block_table, const int* table_rows, int table_stride,
                                const int* shared_start, const int* shared_len, int G, int most, int H, int KV, int D, int ps, float scale, void* work,
                                int* error_word, cudaStream_t stream) {
    if (R == 0) return 0;
    if (!fits(R, G, H, KV, D, ps) || entries < 1 || tokens < 1 || q_stride % D || cache_rows > 0x7fffffff || (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)work) % 16)) return -2;
    CUtensorMap qmap, kmap, vmap;
    if (!query_map(q, tokens, H, D, q_stride, H / KV, &qmap)) return -5;
    if (!cache_map(k_cache, cache_rows, D, ps < KT ? ps : KT, &kmap) || !cache_map(v_cache, cache_rows, D, ps < KT ? ps : KT, &vmap)) return -5;
    const int blocks = 2 * device_sms();
    Args a = sizes(R, G, entries, most, table_stride, H, KV, ps);
    a.decode_segs = decode_segs; a.seg_q_start = seg_q_start; a.seg_kv_len = seg_kv_len; a.block_table = block_table; a.table_rows = table_rows;
    a.shared_start = shared_start; a.shared_len = shared_len;
    const Scratch s = scratch(a, D, blocks);
    if (s.bytes < 0) return -2;
    place_scratch(a, s, work);
    const auto bytes = [&](int ints) { return (size_t)BQ * D * 2 + 4 * (size_t)KT * D * 2 + 26 * 8 + PIECES * sizeof(Piece) + (size_t)ints * 4 + 1024; };
    const size_t smem = bytes(plan_ints(G, R)), most_smem = bytes(6 * MAX_ENTITIES + 1);
    const float scale_log2 = scale * LOG2E;
#define LAUNCH(DD) do { \
        static std::atomic<unsigned long long> done{0}; \
        cudaError_t e = allow_shared(attn_shared_tc_kernel<DD>, (int)most_smem, done); \
        if (e == cudaSuccess) e = launch_pdl(attn_shared_tc_kernel<DD>, dim3(blocks), dim3(THREADS), smem, stream, qmap, kmap, vmap, a, scale_log2, error_word); \
        if (e == cudaSuccess) e = merge<__nv_bfloat16, DD>(a, (__nv_bfloat16*)out, stream); \
        return (int)e; \
    } while (0)
    if (D == 128) LAUNCH(128);
    LAUNCH(64);
#undef LAUNCH
}

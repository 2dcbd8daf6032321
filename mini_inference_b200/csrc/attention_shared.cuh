// Decode attention over a shared prefix: the work that attention_shared_tc.cu (bfloat16, tensor cores) and attention_shared_f32.cu share.
//
// Rows (one fed token each) come in groups; group g's rows all begin with the same shared_len[g] keys, which are read by the pages of the first row that holds
// them all, once for all rows and query heads of the group, and every row has a tail of its own.  The softmax over both is joined from running maxima and sums:
//     o = sum_i e^(m_i - M) o_i / sum_i e^(m_i - M) l_i   over the pieces i that a row's keys were cut into, M = max_i m_i.
//
// Items of work, in this order: (group, key head, tile of the group's rows) over the prefix, then (row, key head) over the tail, each a number of tiles of KT
// keys.  All tiles of all items stand in one line, and block c of a grid that fills the GPU once takes tiles [c per, (c + 1) per): every block has the same
// number of tiles whatever the lengths are, long prefixes are cut over many blocks and short tails put together in one.  A block's share of one item is a
// piece; it is kept at place item + c (items and blocks both grow along the line, so no two pieces share a place).  How many tiles each group and row has
// is known on the device alone; every block adds them up for itself (a few hundred numbers), block 0 leaves the sums for the merge.
// A group of one row has no prefix part: its whole length is its tail.
#pragma once
#include "common.cuh"

namespace mi {
namespace shared_attention {

constexpr int MAX_ENTITIES = 4096;                   // groups + rows of a call

struct Args {
    const int *decode_segs, *seg_q_start, *seg_kv_len, *block_table, *table_rows, *shared_start, *shared_len;
    int R, G, most, table_stride, H, KV, ps;           // most: rows of the largest group; rows beyond it have no prefix part
    int row_tiles, tile_rows;                        // tiles of rows of the largest group; rows of a tile (x H / KV heads = its matrix rows)
    int slot_rows;                                   // matrix rows of a prefix piece's place
    float *o_prefix, *o_tail;                        // [places][slot_rows or H / KV][D], not divided by the sums
    float2 *ml_prefix, *ml_tail;                     // [places][slot_rows or H / KV]: maximum (base 2) and sum
    int* plan;                                       // what block 0 leaves: tiles of a block, sums [G + R + 1], first tail key [R], group [R]
};

inline __host__ __device__ int plan_ints(int G, int R) { return 1 + G + R + 1 + 2 * R; }

// in shared memory: sums of tiles [G + R + 1], first tail key [R], group [R], row whose pages hold the prefix [G]
struct Plan {
    int *sums, *first, *group, *source;
    __device__ __forceinline__ Plan(int* mem, int G, int R) : sums(mem), first(mem + G + R + 1), group(first + R), source(group + R) {}
};
inline __host__ __device__ int shared_plan_ints(int G, int R) { return 2 * G + 3 * R + 1; }

__device__ __forceinline__ int group_rows(const Args& a, int g, int& start) {
    start = max(0, min(a.shared_start[g], a.R));
    return min(max(0, min(a.shared_start[g + 1], a.R) - start), a.most);
}
__device__ __forceinline__ int prefix_keys(const Args& a, int g, int rows) {
    return rows > 1 ? max(0, min(a.shared_len[g], a.table_stride * a.ps)) : 0;
}
__device__ __forceinline__ int row_keys(const Args& a, int r) { return min(a.seg_kv_len[a.decode_segs[r]], a.table_stride * a.ps); }
// a tail's tiles begin where a box of page rows does
__device__ __forceinline__ int tail_base(const Args& a, int first, int KT) { const int u = min(a.ps, KT); return first / u * u; }
__device__ __forceinline__ const int* table_of(const Args& a, int r) {
    const int seg = a.decode_segs[r];
    return a.block_table + (size_t)(a.table_rows ? a.table_rows[seg] : seg) * a.table_stride;
}

// Called by all threads of a block; afterwards (and a barrier) the sums stand in shared memory.
template <int KT>
__device__ __forceinline__ void make_plan(const Args& a, const Plan& p) {
    const int E = a.G + a.R;
    for (int r = threadIdx.x; r < a.R; r += blockDim.x) { p.first[r] = 0; p.group[r] = -1; }
    __syncthreads();
    for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
        int start;
        const int n = group_rows(a, g, start), keys = prefix_keys(a, g, n);
        for (int r = start; r < start + n; ++r) { p.first[r] = keys; p.group[r] = g; }
        p.source[g] = a.R;
        p.sums[g + 1] = a.KV * ((n + a.tile_rows - 1) / a.tile_rows) * ((keys + KT - 1) / KT);
    }
    __syncthreads();
    for (int r = threadIdx.x; r < a.R; r += blockDim.x) {
        const int len = row_keys(a, r), first = p.first[r];
        if (first > 0 && len >= first) atomicMin(&p.source[p.group[r]], r);
        p.sums[a.G + r + 1] = len > first ? a.KV * ((len - tail_base(a, first, KT) + KT - 1) / KT) : 0;
    }
    if (threadIdx.x == 0) p.sums[0] = 0;
    __syncthreads();
    if (threadIdx.x < 32) {                          // running sums, a stretch of entries a lane
        const int lane = threadIdx.x, each = (E + 31) / 32, from = min(1 + lane * each, E + 1), to = min(from + each, E + 1);
        int sum = 0;
        for (int i = from; i < to; ++i) sum += p.sums[i];
        int before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += v; }
        before -= sum;
        for (int i = from; i < to; ++i) { before += p.sums[i]; p.sums[i] = before; }
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) a.plan[0] = max(1, (p.sums[E] + (int)gridDim.x - 1) / (int)gridDim.x);
        for (int i = threadIdx.x; i <= E; i += blockDim.x) a.plan[1 + i] = p.sums[i];
        for (int r = threadIdx.x; r < a.R; r += blockDim.x) { a.plan[2 + E + r] = p.first[r]; a.plan[2 + E + a.R + r] = p.group[r]; }
    }
}

// A block's way along its tiles, piece by piece.  Every role of a block walks it for itself.
template <int KT>
struct Walk {
    const Args& a;
    const Plan& p;
    int t, end, e;                                   // next tile of the line, the block's end, group or row (G + r)
    // the piece
    bool prefix;
    int who, kvh, row_tile, rows, row0;              // group or row; its first row of the tile and how many
    int tiles, lo, hi, key0;                         // tiles; visible keys [lo, hi); key of the first tile's first column
    __device__ __forceinline__ Walk(const Args& a_, const Plan& p_) : a(a_), p(p_) {
        const int E = a.G + a.R, total = p.sums[E], per = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);
        t = min((int)blockIdx.x * per, total);
        end = min(t + per, total);
        int left = 0, right = E;                     // the entry that holds tile t: the last with sums[e] <= t that has tiles
        while (right - left > 1) { const int mid = (left + right) / 2; if (p.sums[mid] <= t) left = mid; else right = mid; }
        e = left;
    }
    __device__ __forceinline__ bool next() {
        if (t >= end) return false;
        while (p.sums[e + 1] <= t) ++e;
        const int off = t - p.sums[e];
        prefix = e < a.G;
        int all;
        if (prefix) {
            who = e;
            int start;
            const int n = group_rows(a, e, start), tm = (n + a.tile_rows - 1) / a.tile_rows;
            lo = 0; hi = prefix_keys(a, e, n);
            all = (hi + KT - 1) / KT;
            const int item = off / all;
            kvh = item / tm; row_tile = item % tm;
            row0 = start + row_tile * a.tile_rows;
            rows = min(a.tile_rows, start + n - row0);
            key0 = off % all * KT;
        } else {
            who = row0 = e - a.G; rows = 1; row_tile = 0;
            lo = p.first[who]; hi = row_keys(a, who);
            const int base = tail_base(a, lo, KT);
            all = (hi - base + KT - 1) / KT;
            kvh = off / all;
            key0 = base + off % all * KT;
        }
        tiles = min(all - off % all, end - t);
        t += tiles;
        return true;
    }
    __device__ __forceinline__ const int* table() const {
        const int holds = prefix ? p.source[who] : who;
        return table_of(a, holds < a.R ? holds : row0 - row_tile * a.tile_rows);
    }
    __device__ __forceinline__ int place() const { return (prefix ? (who * a.KV + kvh) * a.row_tiles + row_tile : who * a.KV + kvh) + (int)blockIdx.x; }
};

// out[token of row r, heads of key head] from the row's pieces: a block per (row, key head)
template <typename T, int D, int KT>
__global__ void __launch_bounds__(128) merge_kernel(const __grid_constant__ Args a, T* __restrict__ out) {
    pdl_trigger();
    pdl_wait(out);
    const int r = blockIdx.x, kvh = blockIdx.y, Hg = a.H / a.KV, E = a.G + a.R;
    const int per = a.plan[0], first = a.plan[2 + E + r], g = a.plan[2 + E + a.R + r];
    const int *sums = a.plan + 1;
    // pieces of the prefix, then of the tail: blocks from .. from + n - 1, places follow on one another
    int n_p = 0, n_t = 0, row_p = 0;
    size_t at_p = 0, at_t = 0;
    int start = 0;
    const int n = g >= 0 && first > 0 ? group_rows(a, g, start) : 0;
    if (r >= start && r < start + n) {
        const int tm = (n + a.tile_rows - 1) / a.tile_rows, all = (prefix_keys(a, g, n) + KT - 1) / KT;
        const int mt = (r - start) / a.tile_rows, t0 = sums[g] + (kvh * tm + mt) * all;
        row_p = (r - start) % a.tile_rows * Hg;
        n_p = (t0 + all - 1) / per - t0 / per + 1;
        at_p = (size_t)(g * a.KV + kvh) * a.row_tiles + mt + t0 / per;
    }
    const int tail = (sums[a.G + r + 1] - sums[a.G + r]) / a.KV;
    if (tail > 0) {
        const int t0 = sums[a.G + r] + kvh * tail;
        n_t = (t0 + tail - 1) / per - t0 / per + 1;
        at_t = (size_t)r * a.KV + kvh + t0 / per;
    }
    T* orow = out + ((size_t)a.seg_q_start[a.decode_segs[r]] * a.H + (size_t)kvh * Hg) * D;
    for (int id = threadIdx.x; id < Hg * (D / 4); id += 128) {
        const int h = id / (D / 4), d = id % (D / 4) * 4;
        float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < n_p + n_t; ++i) {
            const size_t row = i < n_p ? (at_p + i) * a.slot_rows + row_p + h : (at_t + (i - n_p)) * Hg + h;
            const float2 ml = (i < n_p ? a.ml_prefix : a.ml_tail)[row];
            if (ml.x == -INFINITY) continue;         // none of its keys is visible to this row
            float v[4];
            load16((i < n_p ? a.o_prefix : a.o_tail) + row * D + d, v);
            const float top = fmaxf(m, ml.x), old = exp2f(m - top), now = exp2f(ml.x - top);
            m = top;
            l = l * old + ml.y * now;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = o[e] * old + v[e] * now;
        }
        const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;      // no key at all: 0; NaN stays
        store2(orow + h * D + d, o[0] * inv, o[1] * inv);
        store2(orow + h * D + d + 2, o[2] * inv, o[3] * inv);
    }
}

// Scratch of a call: floats of o_prefix, o_tail, then float2 of both, then the plan
struct Scratch { long long o_prefix, o_tail, ml_prefix, ml_tail, plan, bytes; };
inline Scratch scratch(int R, int G, int H, int KV, int D, int row_tiles, int slot_rows, int blocks) {
    const long long places_p = (long long)G * KV * row_tiles + blocks, places_t = (long long)R * KV + blocks, Hg = H / KV;
    const auto up = [](long long v) { return (v + 255) / 256 * 256; };
    Scratch s;
    s.o_prefix = 0;
    s.o_tail = s.o_prefix + up(places_p * slot_rows * D * 4);
    s.ml_prefix = s.o_tail + up(places_t * Hg * D * 4);
    s.ml_tail = s.ml_prefix + up(places_p * slot_rows * 8);
    s.plan = s.ml_tail + up(places_t * Hg * 8);
    s.bytes = s.plan + up(plan_ints(G, R) * 4);
    return s;
}
inline void place_scratch(Args& a, const Scratch& s, void* work) {
    char* w = (char*)work;
    a.o_prefix = (float*)(w + s.o_prefix); a.o_tail = (float*)(w + s.o_tail);
    a.ml_prefix = (float2*)(w + s.ml_prefix); a.ml_tail = (float2*)(w + s.ml_tail);
    a.plan = (int*)(w + s.plan);
}

}  // namespace shared_attention
}  // namespace mi

// Decode attention over a shared prefix: the work that attention_shared_tc.cu (bfloat16, tensor cores) and attention_shared_f32.cu share.
//
// Rows (one fed token each) come in groups; group g's rows all begin with the same shared_len[g] keys, which are read by the pages of the first row that holds
// them all, once for all rows and query heads of the group, and every row has a tail of its own.  The softmax over both is joined from running maxima and sums:
//     o = sum_i e^(m_i - M) o_i / sum_i e^(m_i - M) l_i   over the pieces i that a row's keys were cut into, M = max_i m_i.
//
// Items of work, in this order: (group, key head, tile of the group's rows) over the prefix, then (row, key head) over the tail, each a number of tiles of KT
// keys.  All tiles of all items stand in one line, PAD empty ones in front of each item's (what beginning and ending an item costs), and block c of a grid that
// fills the GPU once takes tiles [c per, (c + 1) per): every block has the same work whatever the lengths are, long prefixes are cut over many blocks
// and short tails put together in one.  A block's share of one item is a
// piece; it is kept at place item + c (items and blocks both grow along the line, so no two pieces share a place).  How many tiles each group and row has
// is known on the device alone; every block adds them up for itself (a few hundred numbers), block 0 leaves the sums for the merge.
// A group of one row has no prefix part: its whole length is its tail.
#pragma once
#include "common.cuh"

namespace mi {
namespace shared_attention {

constexpr int PAD = 3;
constexpr int MAX_ENTITIES = 4096;                   // groups + rows of a call

struct Args {
    const int *decode_segs, *seg_q_start, *seg_kv_len, *block_table, *table_rows, *shared_start, *shared_len;
    int R, G, most, table_stride, H, KV, ps;           // most: rows of the largest group; rows beyond it have no prefix part
    int row_tiles, tile_rows;                        // tiles of rows of the largest group; rows of a tile (x H / KV heads = its matrix rows)
    int slot_rows;                                   // matrix rows of a prefix piece's place
    float *o_prefix, *o_tail;                        // [places][D / 4][slot_rows or H / KV][4], not divided by the sums: neighbouring rows' 16 bytes side by side
    float2 *ml_prefix, *ml_tail;                     // [places][slot_rows or H / KV]: maximum (base 2) and sum
    int* plan;                                       // what block 0 leaves for the merge: tiles of a block, and a Record per row
};

struct __align__(16) Record {                        // where a row's pieces are: its token; the prefix item of key head 0 (first tile, tiles to the next key head's,
    int token, prefix_at, prefix_step, prefix_tiles; // tiles, place, first matrix row) and the tail's (first tile, tiles)
    int prefix_place, prefix_row, tail_at, tail_tiles;
};

// in shared memory: sums of tiles [G + R + 1]; a row's first tail key, group (-1: none), keys, token and row of the block table [R] each; a group's first row, rows,
// shared keys and the row whose pages hold them [G] each
struct Plan {
    int *sums, *first, *group, *keys, *token, *table, *start, *rows, *shared, *source;
    __device__ __forceinline__ Plan(int* mem, int G, int R)
        : sums(mem), first(mem + G + R + 1), group(first + R), keys(group + R), token(keys + R), table(token + R), start(table + R), rows(start + G), shared(rows + G),
          source(shared + G) {}
};
inline __host__ __device__ int plan_ints(int G, int R) { return 5 * G + 6 * R + 1; }

// a tail's tiles begin where a box of page rows does
__device__ __forceinline__ int tail_base(const Args& a, int first, int KT) { const int u = min(a.ps, KT); return first / u * u; }
// tiles of an item in the line
__device__ __forceinline__ int with_pad(int tiles) { return tiles > 0 ? tiles + PAD : 0; }
__device__ __forceinline__ int tiles_of_a_block(int total) { return max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x); }

// Called by all threads of a block; afterwards (and a barrier) the sums stand in shared memory.
template <int KT>
__device__ __forceinline__ void make_plan(const Args& a, const Plan& p) {
    const int E = a.G + a.R;
    for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
        const int start = max(0, min(a.shared_start[g], a.R)), n = min(max(0, min(a.shared_start[g + 1], a.R) - start), a.most);
        const int keys = n > 1 ? max(0, min(a.shared_len[g], a.table_stride * a.ps)) : 0;
        p.start[g] = start; p.rows[g] = n; p.shared[g] = keys; p.source[g] = start + n;
        p.sums[g + 1] = a.KV * ((n + a.tile_rows - 1) / a.tile_rows) * with_pad((keys + KT - 1) / KT);
    }
    for (int r = threadIdx.x; r < a.R; r += blockDim.x) {
        const int seg = a.decode_segs[r];
        p.keys[r] = min(a.seg_kv_len[seg], a.table_stride * a.ps);
        p.token[r] = a.seg_q_start[seg];
        p.table[r] = a.table_rows ? a.table_rows[seg] : seg;
    }
    __syncthreads();
    for (int r = threadIdx.x; r < a.R; r += blockDim.x) {
        int g = 0, right = a.G;                      // the last group that starts at or in front of row r
        while (right - g > 1) { const int mid = (g + right) / 2; if (p.start[mid] <= r) g = mid; else right = mid; }
        const bool in = a.G > 0 && r >= p.start[g] && r < p.start[g] + p.rows[g];
        const int len = p.keys[r], first = in ? p.shared[g] : 0;
        p.group[r] = in ? g : -1;
        p.first[r] = first;
        if (first > 0 && len >= first) atomicMin(&p.source[g], r);
        p.sums[a.G + r + 1] = len > first ? a.KV * with_pad((len - tail_base(a, first, KT) + KT - 1) / KT) : 0;
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
        if (threadIdx.x == 0) a.plan[0] = tiles_of_a_block(p.sums[E]);
        Record* records = reinterpret_cast<Record*>(a.plan + 4);
        for (int r = threadIdx.x; r < a.R; r += blockDim.x) {
            const int g = p.group[r], at = p.sums[a.G + r];
            Record rec{p.token[r], 0, 0, 0, 0, 0, at, (p.sums[a.G + r + 1] - at) / a.KV};
            if (g >= 0) {
                const int start = p.start[g], tm = (p.rows[g] + a.tile_rows - 1) / a.tile_rows, mt = (r - start) / a.tile_rows;
                rec.prefix_tiles = with_pad((p.shared[g] + KT - 1) / KT);
                rec.prefix_at = p.sums[g] + mt * rec.prefix_tiles;
                rec.prefix_step = tm * rec.prefix_tiles;
                rec.prefix_place = g * a.KV * a.row_tiles + mt;
                rec.prefix_row = (r - start) % a.tile_rows * (a.H / a.KV);
            }
            records[r] = rec;
        }
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
        const int E = a.G + a.R, total = p.sums[E], per = tiles_of_a_block(total);
        t = min((int)blockIdx.x * per, total);
        end = min(t + per, total);
        int left = 0, right = E;                     // the entry that holds tile t: the last with sums[e] <= t that has tiles
        while (right - left > 1) { const int mid = (left + right) / 2; if (p.sums[mid] <= t) left = mid; else right = mid; }
        e = left;
    }
    __device__ __forceinline__ bool next() {
        for (;;) {
            if (t >= end) return false;
            while (p.sums[e + 1] <= t) ++e;
            const int off = t - p.sums[e];
            prefix = e < a.G;
            int all;                                 // tiles of the item in the line
            if (prefix) {
                who = e;
                const int n = p.rows[e], tm = (n + a.tile_rows - 1) / a.tile_rows;
                lo = 0; hi = p.shared[e]; key0 = 0;
                all = with_pad((hi + KT - 1) / KT);
                const int item = off / all;
                kvh = item / tm; row_tile = item % tm;
                row0 = p.start[e] + row_tile * a.tile_rows;
                rows = min(a.tile_rows, n - row_tile * a.tile_rows);
            } else {
                who = row0 = e - a.G; rows = 1; row_tile = 0;
                lo = p.first[who]; hi = p.keys[who]; key0 = tail_base(a, lo, KT);
                all = with_pad((hi - key0 + KT - 1) / KT);
                kvh = off / all;
            }
            const int at = off % all, upto = min(all, at + end - t);      // of the item's tiles
            t += upto - at;
            tiles = upto - max(at, PAD);
            key0 += (max(at, PAD) - PAD) * KT;
            if (tiles > 0) return true;
        }
    }
    __device__ __forceinline__ const int* table() const {
        int holds = who;
        if (prefix) { holds = p.source[who]; if (holds >= p.start[who] + p.rows[who]) holds = p.start[who]; }      // nobody has them all
        return a.block_table + (size_t)p.table[holds] * a.table_stride;
    }
    __device__ __forceinline__ int place() const { return (prefix ? (who * a.KV + kvh) * a.row_tiles + row_tile : who * a.KV + kvh) + (int)blockIdx.x; }
};

// out[token of row r, heads of key head] from the row's pieces: a block per (row, key head), as many heads at a time as fill 128 threads with four columns each
// (neighbouring heads in neighbouring threads).  A warp per head makes the weights of all pieces, then MERGE_PARTS groups of 128 threads take every
// MERGE_PARTS-th piece, their rows read without waiting for one another, and are added up in the groups' order.
constexpr int MERGE_PARTS = 4, MERGE_PIECES = 1280;  // pieces of a row at most: one a block for its prefix, one for its tail
template <typename T, int D>
__global__ void __launch_bounds__(128 * MERGE_PARTS) merge_kernel(const __grid_constant__ Args a, T* __restrict__ out) {
    constexpr int HEADS = 512 / D;
    __shared__ float weight[MERGE_PIECES * HEADS], inverse[HEADS];
    __shared__ float4 parts[MERGE_PARTS - 1][128];
    pdl_trigger();
    pdl_wait(out);
    const int r = blockIdx.x, kvh = blockIdx.y, Hg = a.H / a.KV, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = a.plan[0];
    const Record rec = reinterpret_cast<const Record*>(a.plan + 4)[r];
    int n_p = 0, n_t = 0;                            // pieces of the prefix, then of the tail; their places follow on one another
    size_t at_p = 0, at_t = 0;
    if (rec.prefix_tiles > 0) {
        const int t0 = rec.prefix_at + kvh * rec.prefix_step;
        n_p = (t0 + rec.prefix_tiles - 1) / per - (t0 + PAD) / per + 1;
        at_p = (size_t)rec.prefix_place + (size_t)kvh * a.row_tiles + (t0 + PAD) / per;
    }
    if (rec.tail_tiles > 0) {
        const int t0 = rec.tail_at + kvh * rec.tail_tiles;
        n_t = (t0 + rec.tail_tiles - 1) / per - (t0 + PAD) / per + 1;
        at_t = (size_t)r * a.KV + kvh + (t0 + PAD) / per;
    }
    n_p = min(n_p, MERGE_PIECES / 2);
    const int n = n_p + min(n_t, MERGE_PIECES / 2);
    for (int h0 = 0; h0 < Hg; h0 += HEADS) {
        const int heads = min(HEADS, Hg - h0);
        if (warp < heads) {
            const float2 *p = a.ml_prefix + at_p * a.slot_rows + rec.prefix_row + h0 + warp, *q = a.ml_tail + at_t * Hg + h0 + warp;
            const auto piece = [&](int i) { return i < n_p ? p[(size_t)i * a.slot_rows] : q[(size_t)(i - n_p) * Hg]; };
            const float2 first = lane < n ? piece(lane) : make_float2(-INFINITY, 0.f);
            float m = first.x, l = 0.f;
            for (int i = lane + 32; i < n; i += 32) m = fmaxf(m, piece(i).x);
            m = warp_max(m);
            const float off = m == -INFINITY ? 0.f : m;               // -inf: none of a piece's keys is visible to this row
            for (int i = lane; i < n; i += 32) {
                const float2 ml = i < 32 ? first : piece(i);
                const float w = exp2f(ml.x - off);
                weight[i * HEADS + warp] = w;
                if (w != 0.f) l = fmaf(ml.y, w, l);
            }
            l = warp_sum(l);
            if (lane == 0) inverse[warp] = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;      // no key at all: 0; NaN stays
        }
        __syncthreads();
        const int id = threadIdx.x & 127, part = threadIdx.x >> 7, h = id % heads, c = id / heads;
        const bool mine = c < D / 4;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        const auto add = [&](const float4& v, float w) {              // a weight of 0: what a piece without visible keys holds counts for nothing
            o.x = w == 0.f ? o.x : fmaf(v.x, w, o.x); o.y = w == 0.f ? o.y : fmaf(v.y, w, o.y);
            o.z = w == 0.f ? o.z : fmaf(v.z, w, o.z); o.w = w == 0.f ? o.w : fmaf(v.w, w, o.w);
        };
        if (mine) {
            const float4* p = reinterpret_cast<const float4*>(a.o_prefix) + (at_p * (D / 4) + c) * a.slot_rows + rec.prefix_row + h0 + h;
            const float4* q = reinterpret_cast<const float4*>(a.o_tail) + (at_t * (D / 4) + c) * Hg + h0 + h;
            const size_t step_p = (size_t)(D / 4) * a.slot_rows, step_q = (size_t)(D / 4) * Hg;
            int i = part;
#pragma unroll 4
            for (; i < n_p; i += MERGE_PARTS) add(p[i * step_p], weight[i * HEADS + h]);
#pragma unroll 2
            for (; i < n; i += MERGE_PARTS) add(q[(i - n_p) * step_q], weight[i * HEADS + h]);
        }
        if (part) parts[part - 1][id] = o;
        __syncthreads();
        if (part == 0 && mine) {
#pragma unroll
            for (int k = 0; k < MERGE_PARTS - 1; ++k) { const float4 v = parts[k][id]; o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w; }
            const float inv = inverse[h];
            T* to = out + ((size_t)rec.token * a.H + (size_t)kvh * Hg + h0 + h) * D + 4 * c;
            store2(to, o.x * inv, o.y * inv);
            store2(to + 2, o.z * inv, o.w * inv);
        }
        __syncthreads();
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
    s.bytes = s.plan + up(16 + (long long)R * sizeof(Record));
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

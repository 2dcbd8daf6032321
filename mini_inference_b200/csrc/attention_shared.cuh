// Decode attention over a shared prefix: the work that attention_shared_tc.cu (bfloat16, tensor cores) and attention_shared_f32.cu share.
//
// Rows (one fed token each) come in groups; group g's rows all begin with the same shared_len[g] keys, which are read by the pages of the first row that holds
// them all, once for all rows and query heads of the group that hold them all, and every row has a tail of its own.  A row that ends in front of shared_len[g] has
// all its keys in its tail: in a prefix's tile its weights behind its end would be 0, and 0 times an infinite value that another row sees is no 0.  Where every
// row ends there the group has no prefix part.  The softmax over both is joined from running maxima and sums:
//     o = sum_i e^(m_i - M) o_i / sum_i e^(m_i - M) l_i   over the pieces i that a row's keys were cut into, M = max_i m_i.
//
// Items of work, in this order: (group, key head, tile of the group's rows) over the prefix, then (row, key head) over the tail, each a number of tiles of KT
// keys.  All tiles of all items stand in one line, PAD empty ones in front of each item's (what beginning and ending an item costs), and block c of a grid that
// fills the GPU once takes tiles [c per, (c + 1) per): every block has the same work whatever the lengths are, long prefixes are cut over many blocks
// and short tails put together in one.  A block's share of one item is a
// piece.  Its rows are kept from row at(item) + c places of the largest piece on, where at leaves each item the room of its own rows: items and blocks both grow
// along the line, so no two pieces share a row, and all prefixes together take what their groups' rows take, however unlike the groups are.  How many tiles each
// group and row has is known on the device alone; every block adds them up for itself (a few hundred numbers), block 0 leaves the sums for the merge.
// A group of one row has no prefix part: its whole length is its tail.
#pragma once
#include "common.cuh"
#include <atomic>

namespace mi {
namespace shared_attention {

// 8 x 8 rows on 4,096 + 256 keys, 64 rows on 8,192 + 1,000, 21 ragged ones, us: 1: 48.9 52.6 16.7, 2: 48.3 53.8 16.9, 3: 49.0 55.5 15.8, 4: 50.2 57.3 16.0; 64 tails alone 38.5, 35.6, 36.5
constexpr int PAD = 2;
constexpr int MAX_ENTITIES = 4096;                   // groups + rows of a call

struct Args {
    const int *decode_segs, *seg_q_start, *seg_kv_len, *block_table, *table_rows, *shared_start, *shared_len;
    int R, G, entries, most, table_stride, H, KV, ps;  // most: rows of the largest group; rows beyond it have no prefix part
    int tile_rows;                                   // rows of a tile (x H / KV heads = its matrix rows)
    int copies;                                      // 1: a piece's keys may be shared out over up to 4 copies of its rows (see copies_of)
    int slot_rows, tail_rows;                        // matrix rows of the largest prefix piece and of a tail's, copies among them
    float *o_prefix, *o_tail;                        // [rows] D numbers, a piece's as [D / 4][its rows][4]: not divided by the sums, neighbouring rows' 16 bytes side by side
    float2 *ml_prefix, *ml_tail;                     // [rows]: maximum (base 2) and sum
    int* plan;                                       // what block 0 leaves for the merge: tiles of a block, and a Record per row
};

struct __align__(16) Record {                        // where a row's pieces are: its token; the prefix item of key head 0 (first tile, tiles to the next key head's,
    int token, prefix_at, prefix_step, prefix_tiles; // tiles, where its pieces' rows begin, rows to the next key head's, first matrix row) and the tail's (first tile, tiles)
    int prefix_place, prefix_head, prefix_row, tail_at, tail_tiles;      // prefix_row: the tile's rows in the upper half
};

// How often a piece of so many rows has each of them: the copies' keys are different columns of a tile, so each is a piece of its own to the merge.
// Copy s of row i is row s rows + i of the piece.
__host__ __device__ __forceinline__ int copies_of(int copies, int rows) { return !copies || rows > 64 ? 1 : rows > 32 ? 2 : 4; }
// Rows that a batch row's heads may take in a prefix piece: group g's items have this many from row room start[g] KV on (groups do not overlap)
__host__ __device__ __forceinline__ int room_of(int copies, int H, int KV) { return (copies ? 4 : 1) * (H / KV); }

// in shared memory: sums of tiles [G + R + 1]; a row's first tail key (0: it takes no part in a prefix), group (-1: none), keys, token and row of the block table [R]
// each; a group's first row, rows, shared keys and the row whose pages hold them [G] each
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

// where the rows of a group's pieces begin, by key head and tile of rows
__device__ __forceinline__ int prefix_at(const Args& a, const Plan& p, int g, int kvh, int row_tile) {
    return room_of(a.copies, a.H, a.KV) * (p.start[g] * a.KV + kvh * p.rows[g] + row_tile * a.tile_rows);
}

// Called by all threads of a block; afterwards (and a barrier) the sums stand in shared memory.
template <int KT>
__device__ __forceinline__ void make_plan(const Args& a, const Plan& p) {
    const int E = a.G + a.R;
    for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
        const int start = max(0, min(a.shared_start[g], a.R)), n = min(max(0, min(a.shared_start[g + 1], a.R) - start), a.most);
        const int keys = n > 1 ? max(0, min(a.shared_len[g], a.table_stride * a.ps)) : 0;
        p.start[g] = start; p.rows[g] = n; p.shared[g] = keys; p.source[g] = start + n;
    }
    for (int r = threadIdx.x; r < a.R; r += blockDim.x) {
        // entry r is most often entry decode_segs[r]: its numbers are asked for beside it, not behind it
        const int guess = min(r, a.entries - 1), seg = a.decode_segs[r];
        int keys = a.seg_kv_len[guess], token = a.seg_q_start[guess], row = a.table_rows ? a.table_rows[guess] : guess;
        if (seg != guess) { keys = a.seg_kv_len[seg]; token = a.seg_q_start[seg]; row = a.table_rows ? a.table_rows[seg] : seg; }
        p.keys[r] = min(keys, a.table_stride * a.ps);
        p.token[r] = token;
        p.table[r] = row;
    }
    __syncthreads();
    for (int r = threadIdx.x; r < a.R; r += blockDim.x) {
        int g = 0, right = a.G;                      // the last group that starts at or in front of row r
        while (right - g > 1) { const int mid = (g + right) / 2; if (p.start[mid] <= r) g = mid; else right = mid; }
        const bool in = a.G > 0 && r >= p.start[g] && r < p.start[g] + p.rows[g];
        const int len = p.keys[r], shared = in ? p.shared[g] : 0, first = len >= shared ? shared : 0;
        p.group[r] = in ? g : -1;
        p.first[r] = first;
        if (first > 0) atomicMin(&p.source[g], r);
        p.sums[a.G + r + 1] = len > first ? a.KV * with_pad((len - tail_base(a, first, KT) + KT - 1) / KT) : 0;
    }
    __syncthreads();
    for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
        const int n = p.rows[g];
        if (p.source[g] == p.start[g] + n) p.shared[g] = 0;      // nobody has them all
        p.sums[g + 1] = a.KV * ((n + a.tile_rows - 1) / a.tile_rows) * with_pad((p.shared[g] + KT - 1) / KT);
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
            Record rec{p.token[r], 0, 0, 0, 0, 0, 0, at, (p.sums[a.G + r + 1] - at) / a.KV};
            if (p.first[r] > 0) {
                const int start = p.start[g], tm = (p.rows[g] + a.tile_rows - 1) / a.tile_rows, mt = (r - start) / a.tile_rows;
                rec.prefix_tiles = with_pad((p.shared[g] + KT - 1) / KT);
                rec.prefix_at = p.sums[g] + mt * rec.prefix_tiles;
                rec.prefix_step = tm * rec.prefix_tiles;
                rec.prefix_place = prefix_at(a, p, g, 0, mt);
                rec.prefix_head = room_of(a.copies, a.H, a.KV) * p.rows[g];
                rec.prefix_row = (r - start) % a.tile_rows * (a.H / a.KV) | min(a.tile_rows, p.rows[g] - mt * a.tile_rows) * (a.H / a.KV) << 16;
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
    __device__ __forceinline__ int table_row() const { return p.table[prefix ? p.source[who] : who]; }
    // row r of the piece sees its keys below this: a row that is no part of a prefix none
    __device__ __forceinline__ int end_of(int r) const { return prefix ? min(hi, p.first[row0 + r]) : hi; }
    __device__ __forceinline__ int place() const {   // the piece's first row
        return prefix ? prefix_at(a, p, who, kvh, row_tile) + (int)blockIdx.x * a.slot_rows : (who * a.KV + kvh + (int)blockIdx.x) * a.tail_rows;
    }
};

// A piece as one warp of a block writes it down for the others (finding it costs a thousand clocks)
struct __align__(16) Piece { int prefix, who, kvh, row0, rows, tiles, lo, hi, key0, place, table, spare; };

// out[token of row r, heads of key head] from the row's pieces: a block per (row, key head), as many heads at a time as fill 128 threads with four columns each
// (neighbouring heads in neighbouring threads).  A warp per head makes the weights of all pieces, then PARTS groups of 128 threads take every
// PARTS-th piece, their rows read without waiting for one another, and are added up in the groups' order.
constexpr int MERGE_PIECES = 512;                      // pieces whose weights are made at a time
template <typename T, int D, int PARTS>
__global__ void __launch_bounds__(128 * PARTS, PARTS == 2 ? 4 : 1) merge_kernel(const __grid_constant__ Args a, T* __restrict__ out) {
    constexpr int HEADS = 512 / D;
    __shared__ float weight[MERGE_PIECES * HEADS], keep[HEADS], total[HEADS];
    __shared__ float4 parts[PARTS - 1][128];
    pdl_trigger();
    pdl_wait(out);
    const int r = blockIdx.x, kvh = blockIdx.y, Hg = a.H / a.KV, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = a.plan[0];
    const Record rec = reinterpret_cast<const Record*>(a.plan + 4)[r];
    // pieces of the prefix, then of the tail, every copy of the row one of them; a part's pieces lie slot_rows or tail_rows apart
    const int rows_p = rec.prefix_row >> 16, copies_p = copies_of(a.copies, rows_p), copies_t = copies_of(a.copies, Hg);
    const int shift_p = copies_p >> 1, shift_t = copies_t >> 1;        // log2 of 1, 2, 4
    int n_p = 0, n_t = 0;
    size_t at_p = 0, at_t = 0;
    if (rec.prefix_tiles > 0) {
        const int t0 = rec.prefix_at + kvh * rec.prefix_step;
        n_p = ((t0 + rec.prefix_tiles - 1) / per - (t0 + PAD) / per + 1) << shift_p;
        at_p = (size_t)rec.prefix_place + (size_t)kvh * rec.prefix_head + (size_t)((t0 + PAD) / per) * a.slot_rows;
    }
    if (rec.tail_tiles > 0) {
        const int t0 = rec.tail_at + kvh * rec.tail_tiles;
        n_t = ((t0 + rec.tail_tiles - 1) / per - (t0 + PAD) / per + 1) << shift_t;
        at_t = ((size_t)r * a.KV + kvh + (t0 + PAD) / per) * a.tail_rows;
    }
    const int n = n_p + n_t;
    for (int h0 = 0; h0 < Hg; h0 += HEADS) {
        const int heads = min(HEADS, Hg - h0), id = threadIdx.x & 127, part = threadIdx.x >> 7, h = id % heads, c = id / heads;
        const bool mine = c < D / 4;
        const int row_p = (rec.prefix_row & 0xffff) + h0, row_t = h0;
        float m = -INFINITY, l = 0.f;                // of this warp's head
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        const auto rows_of = [&](int i) {            // this thread's columns of piece i
            if (i < n_p) return reinterpret_cast<const float4*>(a.o_prefix) + (at_p + (i >> shift_p) * a.slot_rows) * (D / 4) + (c << shift_p) * rows_p + (i & (copies_p - 1)) * rows_p + row_p + h;
            i -= n_p;
            return reinterpret_cast<const float4*>(a.o_tail) + (at_t + (i >> shift_t) * a.tail_rows) * (D / 4) + c * a.tail_rows + (i & (copies_t - 1)) * Hg + row_t + h;
        };
        constexpr int EARLY = 5;                     // pieces of a thread that are asked for before their weights are there
        float4 early[EARLY];
#pragma unroll
        for (int k = 0; k < EARLY; ++k)
            if (mine && part + k * PARTS < n) early[k] = *rows_of(part + k * PARTS);
        for (int i0 = 0; i0 < max(n, 1); i0 += MERGE_PIECES) {
            const int now = min(MERGE_PIECES, n - i0);
            if (warp < heads) {
                const auto piece = [&](int i) {
                    i += i0;
                    if (i < n_p) return a.ml_prefix[at_p + (i >> shift_p) * a.slot_rows + (i & (copies_p - 1)) * rows_p + row_p + warp];
                    i -= n_p;
                    return a.ml_tail[at_t + (i >> shift_t) * a.tail_rows + (i & (copies_t - 1)) * Hg + row_t + warp];
                };
                const float2 first = lane < now ? piece(lane) : make_float2(-INFINITY, 0.f);
                float top = fmaxf(m, first.x);
                for (int i = lane + 32; i < now; i += 32) top = fmaxf(top, piece(i).x);
                top = warp_max(top);
                const float off = top == -INFINITY ? 0.f : top, old = exp2f(m - off);      // -inf: none of a piece's keys is visible to this row
                float sum = 0.f;
                for (int i = lane; i < now; i += 32) {
                    const float2 ml = i < 32 ? first : piece(i);
                    const float w = isnan(ml.y) ? ml.y : exp2f(ml.x - off);      // maxima pass NaN scores over, sums do not: the row is NaN
                    weight[i * HEADS + warp] = w;
                    if (w != 0.f) sum = fmaf(ml.y, w, sum);
                }
                m = top;
                l = l * old + warp_sum(sum);
                if (lane == 0) { keep[warp] = old; total[warp] = l; }
            }
            __syncthreads();
            if (mine) {
                const float old = keep[h];
                o.x *= old; o.y *= old; o.z *= old; o.w *= old;
                const auto add = [&](const float4& v, float w) {      // a weight of 0: what a piece without visible keys holds counts for nothing
                    o.x = w == 0.f ? o.x : fmaf(v.x, w, o.x); o.y = w == 0.f ? o.y : fmaf(v.y, w, o.y);
                    o.z = w == 0.f ? o.z : fmaf(v.z, w, o.z); o.w = w == 0.f ? o.w : fmaf(v.w, w, o.w);
                };
                int i = i0 + part;
                const int end = i0 + now;
                if (i0 == 0) {
#pragma unroll
                    for (int k = 0; k < EARLY; ++k)
                        if (part + k * PARTS < now) add(early[k], weight[(part + k * PARTS) * HEADS + h]);
                    i += EARLY * PARTS;
                }
#pragma unroll 4
                for (; i < end; i += PARTS) add(*rows_of(i), weight[(i - i0) * HEADS + h]);
            }
            __syncthreads();
        }
        if (part) parts[part - 1][id] = o;
        __syncthreads();
        if (part == 0 && mine) {
#pragma unroll
            for (int k = 0; k < PARTS - 1; ++k) { const float4 v = parts[k][id]; o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w; }
            const float sum = total[h], inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;      // no key at all: 0; NaN stays
            T* to = out + ((size_t)rec.token * a.H + (size_t)kvh * Hg + h0 + h) * D + 4 * c;
            store2(to, o.x * inv, o.y * inv);
            store2(to + 2, o.z * inv, o.w * inv);
        }
        __syncthreads();
    }
}
// Few rows leave SMs empty, and there eight groups of threads a row are the faster ones (16 rows of 8 key heads, 80 pieces each: 47 us for the
// whole operator, with two groups 58); many rows want four blocks an SM (8 x 8 rows on 4,096 keys: two groups 48 us, eight 56; 64 on 8,192: 53 and 61).
template <typename T, int D> inline cudaError_t merge(const Args& a, T* out, cudaStream_t stream) {
    if ((long long)a.R * a.KV <= device_sms()) return launch_pdl(merge_kernel<T, D, 8>, dim3(a.R, a.KV), dim3(1024), 0, stream, a, out);
    return launch_pdl(merge_kernel<T, D, 2>, dim3(a.R, a.KV), dim3(256), 0, stream, a, out);
}

// Lets a kernel have `bytes` of shared memory, once a device (asking again costs a call about 2 us).  Calls of several host threads may meet here.
template <typename Kernel> inline cudaError_t allow_shared(Kernel kernel, int bytes, std::atomic<unsigned long long>& devices_done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && devices_done.load() >> dev & 1)) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) devices_done.fetch_or(1ull << dev);
    return e;
}

// Scratch of a call: floats of o_prefix, o_tail, then float2 of both, then the plan.  bytes -2: rows that do not fit an int
struct Scratch { long long o_prefix, o_tail, ml_prefix, ml_tail, plan, bytes; };
inline Scratch scratch(const Args& a, int D, int blocks) {
    const long long rows_p = (long long)room_of(a.copies, a.H, a.KV) * a.R * a.KV + (long long)blocks * a.slot_rows, rows_t = ((long long)a.R * a.KV + blocks) * a.tail_rows;
    const auto up = [](long long v) { return (v + 255) / 256 * 256; };
    Scratch s;
    s.o_prefix = 0;
    s.o_tail = s.o_prefix + up(rows_p * D * 4);
    s.ml_prefix = s.o_tail + up(rows_t * D * 4);
    s.ml_tail = s.ml_prefix + up(rows_p * 8);
    s.plan = s.ml_tail + up(rows_t * 8);
    s.bytes = rows_p > 0x7fffffff || rows_t > 0x7fffffff ? -2 : s.plan + up(16 + (long long)a.R * sizeof(Record));
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

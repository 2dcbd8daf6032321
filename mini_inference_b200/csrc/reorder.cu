// Rows of tensors take over other rows' contents, in place: t[rows[i]] <- old t[rows[parents[i]]] for every i of a group, in any number of tensors at once.
//
// Beam search's survivors take their parents' last, partly filled pages (keys and values of every layer) and recurrent states.  A group is closed
// (parents lie in it) and holds cycles and shared parents, so a copy row by row would read what was overwritten.  But columns do not depend on one another: a
// thread takes one 16-byte column of a group's rows, brings what any other row wants of it into shared memory (cp.async, all in flight at once) and
// writes the rows that have another parent; its own part of shared memory is read by nobody else, so nothing waits for other threads.  Every row that
// another one wants is read once, every row with another parent written once: no buffer of the whole, no second pass.
// Bound by memory: 170 MB (72 tensors' pages, 8 groups of 8 rows) in 31 us, 336 MB (24 tensors' states, 8 groups of 4) in 67 us, 84 and 77 % of the copy rate; two rows'
// pages of 4 beams 4 us, which is the launch.  A block has 2,048 bytes of a row (128 threads); columns that do not lie on 16 bytes (small integer states, odd rows) go in 4-, 2-
// or 1-byte pieces the same way.
#include "common.cuh"

using namespace mi;

namespace {

constexpr int CHUNK = 2048, THREADS = 128, MOST_TENSORS = 32;
constexpr int MOST_ROWS = 100;                       // rows of a group: their columns of a block fit in shared memory (200 KB)

struct RowTensor { char* base; long long lead_stride, row_stride, row_bytes, rows, first_chunk; };
struct RowTensors { int n; RowTensor t[MOST_TENSORS]; };

template <int W> __device__ __forceinline__ void fetch(void* to, const void* from) {
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
    if constexpr (W == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" :: "r"(dst), "l"(from) : "memory");
    else if constexpr (W == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" :: "r"(dst), "l"(from) : "memory");
    else if constexpr (W == 2) *(uint16_t*)to = *(const uint16_t*)from;
    else *(uint8_t*)to = *(const uint8_t*)from;
}
template <int W> __device__ __forceinline__ void store(void* to, const void* from) {
    if constexpr (W == 16) *(uint4*)to = *(const uint4*)from;
    else if constexpr (W == 4) *(uint32_t*)to = *(const uint32_t*)from;
    else if constexpr (W == 2) *(uint16_t*)to = *(const uint16_t*)from;
    else *(uint8_t*)to = *(const uint8_t*)from;
}

template <int W>
__device__ __forceinline__ void move_columns(char* at, const RowTensor& t, int bytes, int n, const int* row, const int* parent, const int* wanted, unsigned char* stage) {
    for (int c = threadIdx.x * W; c < bytes; c += THREADS * W)
        for (int j = 0; j < n; ++j)
            if (wanted[j]) fetch<W>(stage + j * CHUNK + c, at + row[j] * t.row_stride + c);
    if (W == 16 || W == 4) asm volatile("cp.async.wait_all;\n" ::: "memory");
    for (int c = threadIdx.x * W; c < bytes; c += THREADS * W)
        for (int i = 0; i < n; ++i)
            if (parent[i] != i) store<W>(at + row[i] * t.row_stride + c, stage + parent[i] * CHUNK + c);
}

__global__ void __launch_bounds__(THREADS) reorder_kernel(const __grid_constant__ RowTensors all, const int* __restrict__ rows, const int* __restrict__ parents,
                                                          const int* __restrict__ group_start, int num_rows, int most) {
    extern __shared__ __align__(16) unsigned char stage[];
    __shared__ int row[MOST_ROWS], parent[MOST_ROWS], wanted[MOST_ROWS];
    pdl_trigger();
    pdl_wait(rows, parents, group_start);
    const int g = blockIdx.y;
    const int a = max(0, min(group_start[g], num_rows)), n = min(max(0, min(group_start[g + 1], num_rows) - a), most);
    int k = 0;
    while (k + 1 < all.n && blockIdx.x >= all.t[k + 1].first_chunk) ++k;
    const RowTensor& t = all.t[k];
    if (threadIdx.x < n) {
        const int i = threadIdx.x, p = parents[a + i] - a, r = rows[a + i];
        row[i] = r;
        parent[i] = p >= 0 && p < n ? p : i;         // what points out of its group stays as it is
        wanted[i] = 0;
    }
    __syncthreads();
    if (threadIdx.x < n) {                           // a row outside the tensor neither gives nor takes
        const int i = threadIdx.x, p = parent[i];
        if (p != i && ((unsigned)row[i] >= (unsigned long long)t.rows || (unsigned)row[p] >= (unsigned long long)t.rows)) parent[i] = i;
        else if (p != i) wanted[p] = 1;
    }
    __syncthreads();
    const long long chunk = blockIdx.x - t.first_chunk, per_row = (t.row_bytes + CHUNK - 1) / CHUNK;
    const long long off = chunk % per_row * CHUNK;
    const int bytes = (int)min((long long)CHUNK, t.row_bytes - off);
    char* at = t.base + chunk / per_row * t.lead_stride + off;
    const unsigned long long align = (unsigned long long)t.base | t.lead_stride | t.row_stride | t.row_bytes;
    if (align % 16 == 0) move_columns<16>(at, t, bytes, n, row, parent, wanted, stage);
    else if (align % 4 == 0) move_columns<4>(at, t, bytes, n, row, parent, wanted, stage);
    else if (align % 2 == 0) move_columns<2>(at, t, bytes, n, row, parent, wanted, stage);
    else move_columns<1>(at, t, bytes, n, row, parent, wanted, stage);
}

}  // namespace

// tensors: `count` times (address, tables in it, bytes from table to table, rows of a table, bytes from row to row, bytes of a row), int64 on the host.
// rows, parents int32 [num_rows], group_start int32 [groups + 1]; most: rows of the largest group.  Returns the number of launches, or an error below 0
// (a CUDA error e as -1000 - e).
MI_EXPORT int mi_reorder_rows(const long long* tensors, int count, const int* rows, const int* parents, const int* group_start, int groups, int num_rows, int most,
                              cudaStream_t stream) {
    if (count < 0 || groups < 0 || groups > 65535 || num_rows < 0 || most < 0 || most > MOST_ROWS) return -2;
    if (!count || !groups || !num_rows || !most) return 0;
    const size_t smem = (size_t)most * CHUNK;
    if (smem > 40 * 1024) {                          // (with the lists; up to 48 KB need no leave)
        const cudaError_t fit = cudaFuncSetAttribute(reorder_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_ROWS * CHUNK);
        if (fit != cudaSuccess) return -1000 - (int)fit;
    }
    int launches = 0;
    for (int first = 0; first < count;) {
        RowTensors all = {};
        long long chunks = 0;
        for (; first < count && all.n < MOST_TENSORS; ++first) {
            const long long* d = tensors + 6 * first;
            const long long more = d[1] * ((d[5] + CHUNK - 1) / CHUNK);
            if (d[1] < 0 || d[3] < 0 || d[5] < 0 || more > 0x7fffffff) return -2;
            if (more == 0) continue;
            if (chunks + more > 0x7fffffff) break;
            all.t[all.n++] = RowTensor{(char*)d[0], d[2], d[4], d[5], d[3], chunks};
            chunks += more;
        }
        if (!all.n) continue;
        const cudaError_t e = launch_pdl(reorder_kernel, dim3((unsigned)chunks, groups), dim3(THREADS), smem, stream, all, rows, parents, group_start, num_rows, most);
        if (e != cudaSuccess) return -1000 - (int)e;
        ++launches;
    }
    return launches;
}

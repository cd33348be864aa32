// Block tables, slot maps, positions and tree masks of one step, built on the GPU from the requests' lengths.
//
// A request b has cached[b] tokens in a paged cache and takes new[b] more this step. Its row of the block table lists
// held[b] blocks of block_size tokens; token j of the request lives in slot table[b][j / bs] * bs + j % bs. The step
// needs need[b] = max(0, ceil((cached + new) / bs) - held) more blocks, taken from the top of a stack of free block
// ids: with P the inclusive prefix sum of need over the requests, request b is served while P[b] <= free_count, and
// the k-th block given out is free[free_count - 1 - k]. Every quantity is a prefix sum or a search in one, so nothing
// is sequential in the requests and the result does not depend on timing. The entries that a request which is not
// served wanted become -1, no block. new[b] < 0 ends a request: its blocks go back onto the stack, after this step's
// were taken.
//
// Drafted tokens may form a tree: parents[t] is the index (within its request) of token t's parent, -1 for one that
// follows the context. depth = number of ancestors; position = cached + depth; the mask word has a bit for the token
// itself and each ancestor, so a walk up the parents (at most 64 steps) gives both.
//
// Bound by latency: a few KB to a MB moved. One block does the prefix sums and the stack (its barriers replace a
// grid-wide one) and, with few token rows, fills those too; more rows are shared out over the blocks of one cluster,
// which wait for the first at the cluster's barrier, so the step stays one launch, and above ROWS_CLUSTER_MAX rows over a
// grid of their own (a second launch that overlaps the first's tail by programmatic dependent launch). 8300 rows of 256
// trees: a call from the host takes 20.5 us with the cluster and 23.4 us with the grid, which is why the cluster does
// them; in a captured step, where only the device counts, it takes 8.2 us and the grid would take 7.0 us. 67000 rows of
// 64 prompts: 11.9 us on the device with the cluster, 5.1 us with the grid.
#include <limits.h>

#include "common.cuh"
#include "host_util.h"

namespace vt {

constexpr int ST_SHORT = 1, ST_NARROW = 2, ST_TOKENS = 4, ST_TREE = 8, ST_FREE_FULL = 16;
constexpr int ROWS_ONE_BLOCK = 1024, ROWS_CLUSTER = 8;   // rows up to which one block is enough; blocks above
constexpr int ROWS_CLUSTER_MAX = 16384;
constexpr int STEP_MAX_REQUESTS = 4096;

struct StepArgs {
    int *table;
    long long table_stride;
    int width, B, T, bs, free_cap;
    int *held, *free_blocks, *free_count;
    const int *cached, *newl, *parents;
    int *cu, *seq_lens, *status;
    long long *positions, *slots, *mask;
};

// The smallest b in [0, n) with incl[b] > x (incl non-decreasing), n - 1 if there is none.
__device__ __forceinline__ int first_above(const int *incl, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (incl[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// a + b for a, b >= 0, at most INT_MAX: the sums are over what the caller's lengths say, and one that wrapped would be
// searched, and give places in the table, as if it were small. Saturating sums stay sorted in any order of adding.
__device__ __forceinline__ int sat_add(int a, int b) {
    return (int)min((unsigned)a + (unsigned)b, (unsigned)INT_MAX);
}

__device__ __forceinline__ int clamp_held(const StepArgs &A, int b) { return min(max(A.held[b], 0), A.width); }

// One token row: its position, slot and mask word. cu_end[b] = first token after request b; parents of token t at
// parents[t - p0] (its own and the at most 63 before it).
__device__ __forceinline__ void token_row(const StepArgs &A, const int *cu_end, int total, const int *parents, int p0,
                                          int t) {
    long long pos = 0, slot = -1;
    unsigned long long mask = 0;
    if (t < total) {
        const int b = first_above(cu_end, A.B, t);
        const int start = b ? cu_end[b - 1] : 0, i = t - start;
        const int c = max(A.cached[b], 0);
        int depth = i;
        if (parents && i < 64) {
            int node = i;
            depth = -1;
            while (node >= 0) {   // strictly decreasing: at most 64 steps
                mask |= 1ull << node;
                ++depth;
                const int p = parents[start + node - p0];
                node = p < node ? p : -1;
            }
        }
        pos = (long long)c + depth;
        const unsigned j = (unsigned)c + (unsigned)i, page = j / (unsigned)A.bs;   // both below 2^31
        if (page < (unsigned)clamp_held(A, b)) {
            const int blk = A.table[b * A.table_stride + page];
            if (blk >= 0) slot = (long long)blk * A.bs + (j - page * (unsigned)A.bs);
        }
    }
    A.positions[t] = pos;
    A.slots[t] = slot;
    if (A.mask) A.mask[t] = (long long)mask;
}

// The requests' prefix sums and the stack; cu, need and rel are [B] ints of shared memory.
__device__ __forceinline__ void step_requests(const StepArgs &A, int *cu, int *need, int *rel) {
    __shared__ int wsum[3][32];
    __shared__ int carry[3], flags;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
    if (tid < 3) carry[tid] = 0;
    if (tid == 0) flags = 0;
    const int count = min(min(max(A.free_count[0], 0), A.free_cap), INT_MAX - 1);   // below a saturated sum
    __syncthreads();
    for (int b0 = 0; b0 < A.B; b0 += blockDim.x) {
        const int b = b0 + tid;
        int v[3] = {0, 0, 0};
        if (b < A.B) {
            const int n = A.newl[b], c = max(A.cached[b], 0), h = clamp_held(A, b);
            if (n < 0) {
                v[2] = h;
            } else {
                v[0] = n;
                const long long want = ((long long)c + n + A.bs - 1) / A.bs;
                if (want > A.width) atomicOr(&flags, ST_NARROW);
                else v[1] = max((int)want - h, 0);
                if (A.parents && n > 64) atomicOr(&flags, ST_TREE);
            }
            A.seq_lens[b] = n < 0 ? 0 : (int)min((long long)c + n, (long long)INT_MAX);
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, v[k], o);
                if (lane >= o) v[k] = sat_add(v[k], x);
            }
            if (lane == 31) wsum[k][warp] = v[k];
        }
        __syncthreads();
        if (warp < 3) {   // warp k scans the warps' sums of quantity k and adds what came before
            int x = lane < nw ? wsum[warp][lane] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x = sat_add(x, y);
            }
            const int before = carry[warp];
            __syncwarp();
            x = sat_add(before, x);
            wsum[warp][lane] = x;
            if (lane == 31) carry[warp] = x;
        }
        __syncthreads();
        if (b < A.B) {
            cu[b] = sat_add(v[0], warp ? wsum[0][warp - 1] : (b0 ? cu[b0 - 1] : 0));
            need[b] = sat_add(v[1], warp ? wsum[1][warp - 1] : (b0 ? need[b0 - 1] : 0));
            rel[b] = sat_add(v[2], warp ? wsum[2][warp - 1] : (b0 ? rel[b0 - 1] : 0));
        }
        __syncthreads();
    }
    // blocks given out: all requests up to the last one whose inclusive sum still fits
    int lo = 0, hi = A.B;   // requests [0, lo) are served
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (need[mid] <= count) lo = mid + 1;
        else hi = mid;
    }
    const int served = lo, given = served ? need[served - 1] : 0, total = cu[A.B - 1], freed = rel[A.B - 1];
    for (int k = tid; k < given; k += blockDim.x) {
        const int b = first_above(need, A.B, k);
        const int col = clamp_held(A, b) + k - (b ? need[b - 1] : 0);
        if (col < A.width) A.table[b * A.table_stride + col] = A.free_blocks[count - 1 - k];
    }
    // A request that got none keeps its tokens, and seq_lens counts them: its row must not lead to whatever block ids
    // lie past those it holds.
    if (served < A.B || (flags & ST_NARROW)) {
        for (int b = tid >> 5; b < A.B; b += blockDim.x >> 5) {
            const int n = A.newl[b], h = clamp_held(A, b);
            const long long want = ((long long)max(A.cached[b], 0) + n + A.bs - 1) / A.bs;
            if (n < 0 || (b < served && want <= A.width)) continue;
            const int end = (int)min(want, (long long)A.width);
            for (int col = h + lane; col < end; col += 32) A.table[b * A.table_stride + col] = -1;
        }
    }
    __syncthreads();   // the entries taken have been read: the stack may be written
    const int room = A.free_cap - (count - given);
    for (int k = tid; k < min(freed, room); k += blockDim.x) {
        const int b = first_above(rel, A.B, k);
        int *e = A.table + b * A.table_stride + (k - (b ? rel[b - 1] : 0));
        A.free_blocks[count - given + k] = *e;
        *e = -1;
    }
    __syncthreads();
    for (int b = tid; b < A.B; b += blockDim.x) {
        const int h = clamp_held(A, b), got = b < served ? need[b] - (b ? need[b - 1] : 0) : 0;
        A.held[b] = A.newl[b] < 0 ? 0 : h + got;
        A.cu[b + 1] = cu[b];
    }
    if (tid == 0) {
        A.cu[0] = 0;
        A.free_count[0] = count - given + min(freed, room);
        int f = flags;
        if (served < A.B) f |= ST_SHORT;
        if (total > A.T) f |= ST_TOKENS;
        if (freed > room) f |= ST_FREE_FULL;
        A.status[0] = f;
    }
}

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// One block, or a cluster of `blocks` (0: one block, for the requests alone). The searches and the walks up the parents
// are chains of dependent reads, so what they read is brought to shared memory first.
__global__ void __launch_bounds__(1024) step_tables_kernel(StepArgs A, int blocks) {
    extern __shared__ int sm[];   // [3][B] prefix sums, then the parents of 63 + blockDim.x rows
    int *cu = sm, *par = sm + 3 * A.B;
    const int tid = threadIdx.x, rank = blocks > 1 ? (int)cluster_rank() : 0;
    pdl_launch_dependents();
    pdl_wait();
    if (rank == 0) step_requests(A, cu, sm + A.B, sm + 2 * A.B);
    if (blocks == 0) return;   // the rows have a grid of their own
    if (blocks > 1) {
        cluster_barrier();   // the first block's tables can be read
        if (rank > 0)
            for (int b = tid; b < A.B; b += blockDim.x) cu[b] = A.cu[b + 1];
    }
    const int per = (A.T + blocks - 1) / blocks, t1 = min(A.T, (rank + 1) * per);
    __syncthreads();
    const int total = cu[A.B - 1];
    if (!A.parents) {
#pragma unroll 4
        for (int t = rank * per + tid; t < t1; t += blockDim.x) token_row(A, cu, total, nullptr, 0, t);
        return;
    }
    for (int t0 = rank * per; t0 < t1; t0 += blockDim.x) {
        const int p0 = max(t0 - 63, 0), t = t0 + tid;
        for (int i = p0 + tid; i < min(t0 + (int)blockDim.x, t1); i += blockDim.x) par[i - p0] = A.parents[i];
        __syncthreads();
        if (t < t1) token_row(A, cu, total, par, p0, t);
        __syncthreads();
    }
}

constexpr int ROWS_THREADS = 256;
__global__ void __launch_bounds__(ROWS_THREADS) step_rows_kernel(StepArgs A) {
    extern __shared__ int sm[];   // [B] ends of the requests, then the parents of 63 + ROWS_THREADS rows
    int *par = sm + A.B;
    pdl_launch_dependents();
    pdl_wait();
    const int t0 = blockIdx.x * ROWS_THREADS, p0 = max(t0 - 63, 0);
    for (int b = threadIdx.x; b < A.B; b += ROWS_THREADS) sm[b] = A.cu[b + 1];
    if (A.parents)
        for (int t = p0 + threadIdx.x; t < min(t0 + ROWS_THREADS, A.T); t += ROWS_THREADS) par[t - p0] = A.parents[t];
    __syncthreads();
    const int t = t0 + threadIdx.x;
    if (t < A.T) token_row(A, sm, sm[A.B - 1], A.parents ? par : nullptr, p0, t);
}

}  // namespace vt

using namespace vt;

extern "C" int vt_step_tables(void *table, long long table_stride, int width, void *held, void *free_blocks,
                              int free_cap, void *free_count, const void *cached, const void *new_lens,
                              const void *parents, int B, int T, int block_size, void *cu, void *seq_lens,
                              void *positions, void *slots, void *mask, void *status, void *stream) {
    // (an empty stack has no address)
    if (!table || !held || (free_cap > 0 && !free_blocks) || !free_count || !cached || !new_lens || !cu || !seq_lens ||
        !status || B < 1 || B > STEP_MAX_REQUESTS || T < 0 || width < 1 || table_stride < width || free_cap < 0 ||
        block_size < 1 || (T > 0 && (!positions || !slots)) || (parents && T > 0 && !mask))
        return VT_EARG;
    StepArgs A{};
    A.table = (int *)table;
    A.table_stride = table_stride;
    A.width = width;
    A.B = B;
    A.T = T;
    A.bs = block_size;
    A.free_cap = free_cap;
    A.held = (int *)held;
    A.free_blocks = (int *)free_blocks;
    A.free_count = (int *)free_count;
    A.cached = (const int *)cached;
    A.newl = (const int *)new_lens;
    A.parents = (const int *)parents;
    A.cu = (int *)cu;
    A.seq_lens = (int *)seq_lens;
    A.status = (int *)status;
    A.positions = (long long *)positions;
    A.slots = (long long *)slots;
    A.mask = parents ? (long long *)mask : nullptr;
    cudaStream_t s = (cudaStream_t)stream;
    const int blocks = T <= ROWS_ONE_BLOCK ? 1 : T <= ROWS_CLUSTER_MAX ? ROWS_CLUSTER : 0;
    const int threads = (B <= 256 && T <= 256) ? 256 : 1024;
    const size_t smem = (size_t)(3 * B + 63 + threads) * sizeof(int);
    if (smem > 40 * 1024) {   // past the default limit together with the static arrays
        const int dev = cur_device();
        static std::atomic<bool> attr[VT_MAX_DEV];
        if (dev < 0 || dev >= VT_MAX_DEV) return VT_EARG;
        if (!attr[dev]) {
            if (cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (3 * STEP_MAX_REQUESTS + 63 + 1024) * (int)sizeof(int)) != cudaSuccess)
                return (int)cudaGetLastError();
            attr[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks ? blocks : 1);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (blocks > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = blocks;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        ++n;
    }
    if (pdl_enabled()) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    if (const cudaError_t e = cudaLaunchKernelEx(&cfg, step_tables_kernel, A, blocks)) return (int)e;
    if (blocks) return (int)cudaGetLastError();
    return launch_k(step_rows_kernel, dim3((T + ROWS_THREADS - 1) / ROWS_THREADS), dim3(ROWS_THREADS),
                    (size_t)(B + 63 + ROWS_THREADS) * sizeof(int), s, true, A);
}

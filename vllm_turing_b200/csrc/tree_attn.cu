// Attention of a step's new tokens over a paged cache: single tokens, chains and trees of drafted tokens.
//
// Request b has L = seq_lens[b] keys in the cache, the last n = cu[b + 1] - cu[b] of them this step's own tokens. Query
// token i of the request sees every key before those (j < ctx = L - n), and of its own step the tokens whose bit is
// set in its mask word (bit jj = token jj), or tokens 0 .. i without masks. Out = softmax(scale q K^T) V over the keys
// it sees, 0 where it sees none. A key in a block whose table entry is out of range is not seen.
#include <math.h>

#include "common.cuh"
#include "host_util.h"

namespace vt {

constexpr int TA_MAX_NEW = 64;

struct TaArgs {
    const void *q, *k, *v;
    void *out;
    long long q_t, q_h, o_t, o_h, k_b, k_r, k_h, v_b, v_r, v_h;
    const int *table, *cu, *seq_lens;
    const long long *mask;
    long long table_stride;
    int width, B, T, max_new, Hq, Hkv, D, bs, num_blocks;
    float scale;
};

// One block per (query token, head): its warps take the keys in turn, each with a running maximum, sum and output.
template <typename T>
__global__ void __launch_bounds__(256) tree_attn_simple_kernel(TaArgs A) {
    __shared__ float sm_o[8][256], sm_m[8], sm_l[8];
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, h = blockIdx.y, hk = h / (A.Hq / A.Hkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (t >= A.cu[A.B]) return;
    int lo = 0, hi = A.B - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (A.cu[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    const int b = lo, i = t - A.cu[b], n = A.cu[b + 1] - A.cu[b], L = A.seq_lens[b], ctx = L - n;
    if (i >= A.max_new) return;
    const unsigned long long see = A.mask ? (unsigned long long)A.mask[t] : (2ull << i) - 1;
    const T *q = (const T *)A.q + t * A.q_t + h * A.q_h;
    float qr[8], o[8], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        qr[e] = lane + 32 * e < A.D ? t2f<T>(q[lane + 32 * e]) * A.scale : 0.0f;
        o[e] = 0.0f;
    }
    for (int j = warp; j < L; j += 8) {
        const int jj = j - ctx;
        if (jj >= 0 && (jj >= 64 || !((see >> jj) & 1))) continue;
        const int page = j / A.bs;
        if (page >= A.width) continue;
        const int blk = A.table[b * A.table_stride + page];
        if (blk < 0 || blk >= A.num_blocks) continue;
        const T *k = (const T *)A.k + blk * A.k_b + (j - page * A.bs) * A.k_r + hk * A.k_h;
        const T *v = (const T *)A.v + blk * A.v_b + (j - page * A.bs) * A.v_r + hk * A.v_h;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (lane + 32 * e < A.D) s += qr[e] * t2f<T>(k[lane + 32 * e]);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.0f : mn;
        const float c = expf(m - mu), p = expf(s - mu);
        l = l * c + p;
        m = mn;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (lane + 32 * e < A.D) o[e] = o[e] * c + p * t2f<T>(v[lane + 32 * e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sm_o[warp][lane + 32 * e] = o[e];
    if (lane == 0) {
        sm_m[warp] = m;
        sm_l[warp] = l;
    }
    __syncthreads();
    float mx = -INFINITY, sum = 0.0f, acc = 0.0f;
    for (int w = 0; w < 8; ++w) mx = fmaxf(mx, sm_m[w]);
    if (mx == -INFINITY) mx = 0.0f;
    for (int w = 0; w < 8; ++w) {
        const float c = expf(sm_m[w] - mx);
        sum += c * sm_l[w];
        acc += c * sm_o[w][threadIdx.x];
    }
    if (threadIdx.x < A.D)
        ((T *)A.out)[t * A.o_t + h * A.o_h + threadIdx.x] = f2t<T>(sum == 0.0f ? 0.0f : acc / sum);
}

}  // namespace vt

using namespace vt;

extern "C" {

size_t vt_tree_attention_ws_bytes(int max_new, int Hq, int Hkv, int D) {
    (void)max_new;
    (void)Hq;
    (void)Hkv;
    (void)D;
    return 256;
}

int vt_tree_attention(const void *q, const void *k_cache, const void *v_cache, void *out, const long long *strides,
                      const void *block_table, long long table_stride, int table_width, const void *cu,
                      const void *seq_lens, const void *mask, int B, int T, int max_new, int Hq, int Hkv, int D,
                      long long num_blocks, int block_size, float scale, int dtype, void *workspace, size_t ws_bytes,
                      void *stream) {
    if (!q || !k_cache || !v_cache || !out || !strides || !block_table || !cu || !seq_lens || B < 1 || T < 0 ||
        max_new < 1 || max_new > TA_MAX_NEW || Hkv < 1 || Hq < Hkv || Hq % Hkv || D < 8 || D > 256 || D % 8 ||
        block_size < 8 || block_size % 8 || table_width < 0 || num_blocks < 0 || (dtype != 0 && dtype != 1) ||
        !workspace || ws_bytes < vt_tree_attention_ws_bytes(max_new, Hq, Hkv, D))
        return VT_EARG;
    TaArgs A{};
    A.q = q;
    A.k = k_cache;
    A.v = v_cache;
    A.out = out;
    A.q_t = strides[0];
    A.q_h = strides[1];
    A.o_t = strides[2];
    A.o_h = strides[3];
    A.k_b = strides[4];
    A.k_r = strides[5];
    A.k_h = strides[6];
    A.v_b = strides[7];
    A.v_r = strides[8];
    A.v_h = strides[9];
    A.table = (const int *)block_table;
    A.table_stride = table_stride;
    A.width = table_width;
    A.cu = (const int *)cu;
    A.seq_lens = (const int *)seq_lens;
    A.mask = (const long long *)mask;
    A.B = B;
    A.T = T;
    A.max_new = max_new;
    A.Hq = Hq;
    A.Hkv = Hkv;
    A.D = D;
    A.bs = block_size;
    A.num_blocks = (int)num_blocks;
    A.scale = scale;
    if (T == 0) return 0;
    cudaStream_t s = (cudaStream_t)stream;
    const dim3 grid(T, Hq);
    if (dtype == 0) return launch_k(tree_attn_simple_kernel<__half>, grid, dim3(256), 0, s, true, A);
    return launch_k(tree_attn_simple_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, true, A);
}

}  // extern "C"

// Rotary positions of query and key heads, alone or fused with the write of keys and values into a paged cache.
//
// Of each head the first `rot` of D values are rotated in pairs by the token's position, the others pass through:
//   a = position * w_i,  (y1, y2) = factor * (x1 cos a - x2 sin a, x2 cos a + x1 sin a)
// with pairs (i, i + rot / 2) ("half") or (2 i, 2 i + 1) ("interleaved"). transpose negates the sine: the map's
// transpose, which is the gradient of the rotation. The frequencies come as turns w_i / 2 pi in 64 bits: position *
// turns is reduced to [-1/2, 1/2] turns in 64 bits before the 32-bit sine and cosine, so that a position of a million
// keeps the full 32-bit accuracy (the product rounded to 32 bits would be off by up to 0.06 rad there).
//
// HBM bound: each value is read once and written once, so the kernel has to spend few instructions on a value and keep
// many loads in flight. Heads of up to 256 values that 16-byte vectors fit go through shared memory, whole, as rows of a
// warp's 32 vectors (two or more heads side by side when they are short). A warp takes a token and a share of its heads
// (of q, k and v in one list), up to RO_ROWS rows of them, at a time, copies the next share's to its own part of shared
// memory asynchronously, makes the token's sines and cosines (a chain of loads and arithmetic of about 2 us) and writes
// the share that has arrived: first the vectors that pass through, then the rotated ones, a pair of vectors a lane over
// all heads of the share, so that no lane idles where only part of the head rotates. Warps do not wait for one another.
// Everything else, larger heads or sizes and addresses that vectors do not fit, takes the second kernel, a unit (vector
// or element, and its partner) a thread. 16384 tokens of 32 + 8 heads: 58 us for heads of 128 (floor 51), 44 us for heads
// of 80 all rotated (floor 32); with 40 of the 80 rotated in half pairs, which vectors of 8 do not fit, 187 us.
#include "common.cuh"
#include "host_util.h"

namespace vt {

constexpr int RO_THREADS = 256;
constexpr int RO_MAX_HALF = 512;   // pairs a head may have
constexpr int RO_BLOCKS = 3;         // resident blocks an SM
constexpr int RO_ROWS = 8;           // heads of a share, per lane

struct RotArgs {
    const void *q, *k, *v;
    void *qo, *ko, *kc, *vc;                          // ko: rotary alone; kc / vc: the caches (fused form)
    long long q_t, q_h, k_t, k_h, v_t, v_h;           // strides in elements: token, head
    long long qo_t, qo_h, ko_t, ko_h;
    long long kc_b, kc_r, kc_h, vc_b, vc_r, vc_h;     // cache strides: block, row, head
    const long long *positions, *slots;
    const double *turns;
    float factor;
    int transpose, T, Hq, Hkv, D, rot, bs;
    int shares;                                       // shares a token's heads are dealt in (warp kernel)
    int dt, ds;                                       // tokens and shares from a warp's item to its next
    long long num_slots;
    int q_rest, k_rest;                               // copy the values past rot (0: rotated in place)
};

template <int V> struct RoVec;
template <> struct RoVec<8> { using type = uint4; };
template <> struct RoVec<1> { using type = uint16_t; };

template <typename T, int V> struct RoReg {
    T e[V];
    __device__ __forceinline__ void load(const T *p) {
        *reinterpret_cast<typename RoVec<V>::type *>(e) = *reinterpret_cast<const typename RoVec<V>::type *>(p);
    }
    __device__ __forceinline__ void store(T *p) const {
        *reinterpret_cast<typename RoVec<V>::type *>(p) = *reinterpret_cast<const typename RoVec<V>::type *>(e);
    }
};

// Unit u of a head of x (source) to y: the first `rot_units` are rotated, the others copied.
template <typename T, int V, bool INTER>
__device__ __forceinline__ void rotate_unit(const T *x, T *y, int u, int rot_units, int rot, const float2 *cs,
                                            bool rest) {
    constexpr int P = INTER ? 2 : 1;   // elements per pair that lie side by side
    if (u < rot_units) {
        if constexpr (INTER && V == 8) {
            __align__(16) RoReg<T, 8> r;
            r.load(x + u * 8);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 c = cs[u * 4 + j];
                const float a = t2f<T>(r.e[2 * j]), b = t2f<T>(r.e[2 * j + 1]);
                r.e[2 * j] = f2t<T>(a * c.x - b * c.y);
                r.e[2 * j + 1] = f2t<T>(b * c.x + a * c.y);
            }
            r.store(y + u * 8);
        } else {
            const int i1 = u * V * P, i2 = INTER ? i1 + 1 : i1 + rot / 2;
            __align__(16) RoReg<T, V> r1;
            __align__(16) RoReg<T, V> r2;
            r1.load(x + i1);
            r2.load(x + i2);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float2 c = cs[u * V + j];
                const float a = t2f<T>(r1.e[j]), b = t2f<T>(r2.e[j]);
                r1.e[j] = f2t<T>(a * c.x - b * c.y);
                r2.e[j] = f2t<T>(b * c.x + a * c.y);
            }
            r1.store(y + i1);
            r2.store(y + i2);
        }
    } else if (rest) {
        const int i = rot + (u - rot_units) * V;
        __align__(16) RoReg<T, V> r;
        r.load(x + i);
        r.store(y + i);
    }
}

template <typename T, int V, bool INTER, bool CACHE>
__global__ void __launch_bounds__(RO_THREADS) rotary_any_kernel(const __grid_constant__ RotArgs A) {
    __shared__ float2 cs[RO_MAX_HALF];
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x;
    const double pos = (double)A.positions[t];
    for (int i = threadIdx.x; i < A.rot / 2; i += RO_THREADS) {
        double r = pos * A.turns[i];
        r -= rint(r);
        float s, c;
        sincospif(2.0f * (float)r, &s, &c);
        cs[i] = make_float2(c * A.factor, A.transpose ? -s * A.factor : s * A.factor);
    }
    long long blk = -1;
    int row = 0;
    if (CACHE) {
        const long long slot = A.slots[t];
        if (slot >= 0 && slot < A.num_slots) {
            blk = slot / A.bs;
            row = (int)(slot - blk * A.bs);
        }
    }
    __syncthreads();
    const int rot_units = (INTER && V == 8) ? A.rot / 8 : A.rot / (2 * V);
    const int units = rot_units + (A.D - A.rot) / V, vunits = A.D / V;
    const int nq = A.Hq * units, nk = A.Hkv * units, all = nq + nk + (CACHE ? A.Hkv * vunits : 0);
    for (int w = blockIdx.y * RO_THREADS + threadIdx.x; w < all; w += gridDim.y * RO_THREADS) {
        if (w < nq) {
            const int h = w / units, u = w - h * units;
            rotate_unit<T, V, INTER>((const T *)A.q + t * A.q_t + h * A.q_h, (T *)A.qo + t * A.qo_t + h * A.qo_h, u,
                                     rot_units, A.rot, cs, A.q_rest);
        } else if (w < nq + nk) {
            const int h = (w - nq) / units, u = (w - nq) - h * units;
            const T *x = (const T *)A.k + t * A.k_t + h * A.k_h;
            if (!CACHE)
                rotate_unit<T, V, INTER>(x, (T *)A.ko + t * A.ko_t + h * A.ko_h, u, rot_units, A.rot, cs, A.k_rest);
            else if (blk >= 0)
                rotate_unit<T, V, INTER>(x, (T *)A.kc + blk * A.kc_b + row * A.kc_r + h * A.kc_h, u, rot_units, A.rot,
                                         cs, true);
        } else if (CACHE && blk >= 0) {
            const int h = (w - nq - nk) / vunits, u = (w - nq - nk) - h * vunits;
            __align__(16) RoReg<T, V> r;
            r.load((const T *)A.v + t * A.v_t + h * A.v_h + u * V);
            r.store((T *)A.vc + blk * A.vc_b + row * A.vc_r + h * A.vc_h + u * V);
        }
    }
}

__device__ __forceinline__ void ro_copy16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}


// Shared memory of a block: two shares a warp, [warp][2][RO_ROWS][32 lanes] vectors, then the cosines [warp][128].
constexpr int RO_SMEM = RO_THREADS / 32 * (2 * RO_ROWS * 32 * 16 + 128 * 8);

template <typename T, bool INTER, bool CACHE>
__global__ void __launch_bounds__(RO_THREADS, RO_BLOCKS) rotary_warp_kernel(const __grid_constant__ RotArgs A) {
    constexpr int WARPS = RO_THREADS / 32, NC = INTER ? 4 : 8;
    extern __shared__ __align__(16) unsigned char ro_sm[];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = A.rot / 2;
    uint4(*buf)[RO_ROWS][32] = reinterpret_cast<uint4(*)[RO_ROWS][32]>(ro_sm) + 2 * warp;
    float2 *cs = reinterpret_cast<float2 *>(ro_sm + WARPS * 2 * RO_ROWS * 32 * 16) + warp * 128;
    // a row: hpw heads of vph vectors; this lane's head and vector
    const int vph = A.D / 8, hpw = 32 / vph, sub = lane / vph, v = lane - sub * vph;
    const bool there = sub < hpw, rest = there && v * 8 >= A.rot;
    // rotating: hpr heads at a time, upr units (pairs of vectors; vectors of pairs when interleaved) of each
    const int hv = half / 8, upr = max(INTER ? A.rot / 8 : hv, 1), hpr = 32 / upr, rh = lane / upr, u = lane - rh * upr;
    const unsigned by_hpw = 65536u / (unsigned)hpw + 1u;   // n / hpw = n by_hpw >> 16 for n < 256
    const int HK = A.Hq + A.Hkv, E = HK + (CACHE ? A.Hkv : 0), step = A.shares * hpw;   // heads: q, k, then v
    int it = blockIdx.x * WARPS + warp, t = it / A.shares, share = it - t * A.shares;   // item: token and share
    pdl_wait();
    auto next = [&](int &tk, int &sh) {
        tk += A.dt;
        sh += A.ds;
        if (sh >= A.shares) sh -= A.shares, ++tk;
    };
    auto fetch = [&](int tk, int sh, int b) {
        if (tk < A.T && there) {
            const T *q = (const T *)A.q + tk * A.q_t + v * 8, *k = (const T *)A.k + tk * A.k_t + v * 8;
            const T *vv = CACHE ? (const T *)A.v + tk * A.v_t + v * 8 : nullptr;
#pragma unroll
            for (int i = 0; i < RO_ROWS; ++i) {
                const int e = sh * hpw + sub + i * step;
                if (e >= E) break;
                ro_copy16(&buf[b][i][lane], e < A.Hq ? q + e * A.q_h
                                            : e < HK ? k + (e - A.Hq) * A.k_h : vv + (e - HK) * A.v_h);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(t, share, 0);
    for (int b = 0; t < A.T; b ^= 1) {
        int tn = t, sn = share;
        next(tn, sn);
        const double pos = (double)A.positions[t];
        const long long slot = CACHE ? A.slots[t] : 0;
        fetch(tn, sn, b ^ 1);
        for (int i = lane; i < half; i += 32) {
            double r = pos * A.turns[i];
            r -= rint(r);
            float s, c;
            sincospif(2.0f * (float)r, &s, &c);
            cs[i] = make_float2(c * A.factor, A.transpose ? -s * A.factor : s * A.factor);
        }
        T *qo = (T *)A.qo + t * A.qo_t, *ko, *vo = nullptr;
        if (CACHE) {
            const bool ok = slot >= 0 && slot < A.num_slots;
            const long long blk = ok ? slot / A.bs : 0, row = ok ? slot - blk * A.bs : 0;
            ko = ok ? (T *)A.kc + blk * A.kc_b + row * A.kc_r : nullptr;   // NULL: no place in the cache
            vo = (T *)A.vc + blk * A.vc_b + row * A.vc_r;
        } else {
            ko = (T *)A.ko + t * A.ko_t;
        }
        const long long ko_h = CACHE ? A.kc_h : A.ko_h;
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        const int e0 = share * hpw;
        if (CACHE || A.rot < A.D) {   // what passes through
#pragma unroll 4
            for (int i = 0; i < RO_ROWS; ++i) {
                const int e = e0 + sub + i * step;
                if (e >= E) break;
                T *y = nullptr;
                if (e < A.Hq) {
                    if (rest && A.q_rest) y = qo + e * A.qo_h;
                } else if (e < HK) {
                    if (rest && ko && (CACHE || A.k_rest)) y = ko + (e - A.Hq) * ko_h;
                } else if (there && ko) {
                    y = vo + (e - HK) * A.vc_h;
                }
                if (y) *reinterpret_cast<uint4 *>(y + v * 8) = buf[b][i][lane];
            }
        }
        if (half > 0 && rh < hpr) {   // what rotates
            float c[NC], s[NC];
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const float2 x = cs[u * NC + j];
                c[j] = x.x;
                s[j] = x.y;
            }
#pragma unroll 2
            for (int n = rh; n < RO_ROWS * hpw; n += hpr) {
                const int i = (int)((unsigned)n * by_hpw >> 16), sb = n - i * hpw, e = e0 + sb + i * step;
                if (e >= HK) break;
                T *y = qo + e * A.qo_h;
                if (e >= A.Hq) {
                    if (!ko) break;
                    y = ko + (e - A.Hq) * ko_h;
                }
                const uint4 *x = &buf[b][i][sb * vph + u];
                const uint4 r = x[0];
                uint32_t w[4] = {r.x, r.y, r.z, r.w};
                if constexpr (INTER) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 a = unpack2<T>(w[j]);
                        w[j] = pack2<T>(a.x * c[j] - a.y * s[j], a.y * c[j] + a.x * s[j]);
                    }
                } else {
                    const uint4 p = x[hv];
                    uint32_t o[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 a = unpack2<T>(w[j]), d = unpack2<T>(o[j]);
                        w[j] = pack2<T>(a.x * c[2 * j] - d.x * s[2 * j], a.y * c[2 * j + 1] - d.y * s[2 * j + 1]);
                        o[j] = pack2<T>(d.x * c[2 * j] + a.x * s[2 * j], d.y * c[2 * j + 1] + a.y * s[2 * j + 1]);
                    }
                    *reinterpret_cast<uint4 *>(y + half + u * 8) = make_uint4(o[0], o[1], o[2], o[3]);
                }
                *reinterpret_cast<uint4 *>(y + u * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        __syncwarp();   // read: the share after the next may be copied over it, and the next token's cosines written
        t = tn;
        share = sn;
    }
}

template <typename T, bool CACHE> static int launch_rotary(RotArgs A, bool inter, bool vec, cudaStream_t s) {
    const int sms = num_sms(cur_device());
    const dim3 block(RO_THREADS);
    if (vec && A.D <= 256) {
        const int dev = cur_device();
        static std::atomic<bool> attr[VT_MAX_DEV];
        auto kernel = inter ? rotary_warp_kernel<T, true, CACHE> : rotary_warp_kernel<T, false, CACHE>;
        if (dev < 0 || dev >= VT_MAX_DEV) return VT_EARG;
        if (!attr[dev]) {
            if (cudaFuncSetAttribute(rotary_warp_kernel<T, true, CACHE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     RO_SMEM) != cudaSuccess ||
                cudaFuncSetAttribute(rotary_warp_kernel<T, false, CACHE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     RO_SMEM) != cudaSuccess)
                return (int)cudaGetLastError();
            attr[dev] = true;
        }
        const int hpw = 32 / (A.D / 8), heads = A.Hq + A.Hkv * (CACHE ? 2 : 1), warps = RO_THREADS / 32;
        // the shares of a token: more of them where there are too few tokens to give every SM some warps
        const int least = (heads + RO_ROWS * hpw - 1) / (RO_ROWS * hpw), most = (heads + hpw - 1) / hpw;
        const int want = (2 * warps * sms + A.T - 1) / A.T;
        A.shares = want < least ? least : want < most ? want : most;
        const long long items = (long long)A.T * A.shares, blocks = (items + warps - 1) / warps;
        if (items > 0x3fffffff) return VT_EARG;
        const dim3 grid((unsigned)(blocks < RO_BLOCKS * sms ? blocks : RO_BLOCKS * sms));
        A.dt = (int)grid.x * warps / A.shares;
        A.ds = (int)grid.x * warps % A.shares;
        return launch_k(kernel, grid, block, RO_SMEM, s, true, A);
    }
    const long long units = (long long)(A.Hq + A.Hkv) * (A.rot / 2 + A.D - A.rot) / (vec ? 8 : 1);
    int split = (int)((units + RO_THREADS - 1) / RO_THREADS);
    const int want = (2 * sms + A.T - 1) / A.T;
    if (split > want) split = want;
    if (split < 1) split = 1;
    const dim3 grid(A.T, split);
    if (vec)
        return inter ? launch_k(rotary_any_kernel<T, 8, true, CACHE>, grid, block, 0, s, true, A)
                     : launch_k(rotary_any_kernel<T, 8, false, CACHE>, grid, block, 0, s, true, A);
    return inter ? launch_k(rotary_any_kernel<T, 1, true, CACHE>, grid, block, 0, s, true, A)
                 : launch_k(rotary_any_kernel<T, 1, false, CACHE>, grid, block, 0, s, true, A);
}

static bool vec_ok(const void *p, long long a, long long b, long long c) {
    return ((uintptr_t)p & 15) == 0 && ((a | b | c) & 7) == 0;
}

static bool rot_args_ok(const RotArgs &A) {
    return A.T >= 0 && A.Hq >= 0 && A.Hkv >= 0 && A.Hq + A.Hkv >= 1 && A.D >= 1 && A.rot >= 0 && (A.rot & 1) == 0 &&
           A.rot <= A.D && A.rot / 2 <= RO_MAX_HALF && A.positions && (A.turns || A.rot == 0);
}

}  // namespace vt

using namespace vt;

extern "C" {

int vt_rotary(const void *q, void *q_out, const void *k, void *k_out, const long long *strides,
              const void *positions, const void *turns, float factor, int interleaved, int transpose, int T, int Hq,
              int Hkv, int D, int rot, int dtype, void *stream) {
    RotArgs A{};
    if (!strides) return VT_EARG;
    A.q = q;
    A.qo = q_out;
    A.k = k;
    A.ko = k_out;
    A.q_t = strides[0];
    A.q_h = strides[1];
    A.qo_t = strides[2];
    A.qo_h = strides[3];
    A.k_t = strides[4];
    A.k_h = strides[5];
    A.ko_t = strides[6];
    A.ko_h = strides[7];
    A.positions = (const long long *)positions;
    A.turns = (const double *)turns;
    A.factor = factor;
    A.transpose = transpose;
    A.T = T;
    A.Hq = Hq;
    A.Hkv = Hkv;
    A.D = D;
    A.rot = rot;
    A.q_rest = q != q_out;
    A.k_rest = k != k_out;
    if (!rot_args_ok(A) || (Hq && (!q || !q_out)) || (Hkv && (!k || !k_out)) || (dtype != 0 && dtype != 1))
        return VT_EARG;
    if (T == 0) return 0;
    const bool vec = D % 8 == 0 && rot % (interleaved ? 8 : 16) == 0 &&
                     (!Hq || (vec_ok(q, A.q_t, A.q_h, 0) && vec_ok(q_out, A.qo_t, A.qo_h, 0))) &&
                     (!Hkv || (vec_ok(k, A.k_t, A.k_h, 0) && vec_ok(k_out, A.ko_t, A.ko_h, 0)));
    if (dtype == 0) return launch_rotary<__half, false>(A, interleaved != 0, vec, (cudaStream_t)stream);
    return launch_rotary<__nv_bfloat16, false>(A, interleaved != 0, vec, (cudaStream_t)stream);
}

int vt_rotary_cache(const void *q, void *q_out, const void *k, const void *v, void *k_cache, void *v_cache,
                    const long long *strides, const void *positions, const void *slots, const void *turns,
                    float factor, int interleaved, int T, int Hq, int Hkv, int D, int rot, long long num_blocks,
                    int block_size, int dtype, void *stream) {
    RotArgs A{};
    if (!strides) return VT_EARG;
    A.q = q;
    A.qo = q_out;
    A.k = k;
    A.v = v;
    A.kc = k_cache;
    A.vc = v_cache;
    A.q_t = strides[0];
    A.q_h = strides[1];
    A.qo_t = strides[2];
    A.qo_h = strides[3];
    A.k_t = strides[4];
    A.k_h = strides[5];
    A.v_t = strides[6];
    A.v_h = strides[7];
    A.kc_b = strides[8];
    A.kc_r = strides[9];
    A.kc_h = strides[10];
    A.vc_b = strides[11];
    A.vc_r = strides[12];
    A.vc_h = strides[13];
    A.positions = (const long long *)positions;
    A.slots = (const long long *)slots;
    A.turns = (const double *)turns;
    A.factor = factor;
    A.T = T;
    A.Hq = Hq;
    A.Hkv = Hkv;
    A.D = D;
    A.rot = rot;
    A.bs = block_size;
    A.q_rest = q != q_out;
    // (a cache without blocks has no address)
    if (!rot_args_ok(A) || Hkv < 1 || (Hq && (!q || !q_out)) || !k || !v ||
        (num_blocks > 0 && (!k_cache || !v_cache)) || !slots || num_blocks < 0 || block_size < 1 ||
        (dtype != 0 && dtype != 1))
        return VT_EARG;
    A.num_slots = num_blocks * block_size;
    if (T == 0) return 0;
    const bool vec = D % 8 == 0 && rot % (interleaved ? 8 : 16) == 0 &&
                     (!Hq || (vec_ok(q, A.q_t, A.q_h, 0) && vec_ok(q_out, A.qo_t, A.qo_h, 0))) &&
                     vec_ok(k, A.k_t, A.k_h, 0) && vec_ok(v, A.v_t, A.v_h, 0) &&
                     vec_ok(k_cache, A.kc_b, A.kc_r, A.kc_h) && vec_ok(v_cache, A.vc_b, A.vc_r, A.vc_h);
    if (dtype == 0) return launch_rotary<__half, true>(A, interleaved != 0, vec, (cudaStream_t)stream);
    return launch_rotary<__nv_bfloat16, true>(A, interleaved != 0, vec, (cudaStream_t)stream);
}

}  // extern "C"

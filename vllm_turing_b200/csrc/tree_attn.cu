// Attention of a step's new tokens over a paged cache: single tokens, chains and trees of drafted tokens.
//
// Request b has L = seq_lens[b] keys in the cache, the last n = cu[b + 1] - cu[b] of them this step's own tokens. Query
// token i of the request sees every key before those (j < ctx = L - n), and of its own step the tokens whose bit is
// set in its mask word (bit jj = token jj), or tokens 0 .. i without masks. Out = softmax(scale q K^T) V over the keys
// it sees, 0 where it sees none. A key in a block whose table entry is out of range is not seen.
//
// Rows: the n tokens x G = Hq / Hkv query heads of one cached head share its keys, so they are the rows of one product,
// whole tokens of up to 128 rows to a tile (tcgen05 M = 128; unused rows cost nothing that counts, since rows are
// independent and the stream of keys bounds the kernel below about 250 rows). Per tile of TK keys:
//   S [128, TK] = Q K^T       tcgen05 kind::f16, both K-major, 128-byte swizzle
//   P = 2^(S scale log2 e - m) in 16 bits, written over S in tensor memory; m, l: running maximum and sum (32 bits)
//   O [128, D] += P V         tcgen05 kind::f16, P from tensor memory, V from shared memory as it lies in the cache
//                             (keys x D: the "MN-major" operand)
// O stays in tensor memory for all tiles; a row's m is raised, and O and l rescaled, only when a tile's maximum passes
// m by more than 8 (a factor 2^8): the quotient O / l is the same, P stays below 2^8 (fp16 P is held 2^7 times larger,
// so that small weights keep their bits), and rescaling, which reads and writes all of O, is rare. (O is a sum before the
// division: with bf16 values past 2^120 / L in magnitude it can pass 32 bits where the quotient would not.)
// P has 16 bits because one MMA takes both operands in one type, V's: each weight is rounded once, by at most 2^-8 (bf16)
// or 2^-11 (fp16) of itself; maxima, l, O and the parts have 32 bits. On random inputs the output's error against 64
// bits, relative to its norm, is 0.0018 .. 0.0023 in bf16 where the output's own rounding alone gives 0.0017, and 0.00026
// for 0.00021 in fp16. Weights of 32 bits would take a second product with the remainders.
//
// The softmax of a tile must not take longer than its bytes take to arrive (about 2800 cycles for 64 KB of K and V), nor
// than its products where those bound. A thread holds a row, so with few rows one warp would do all the work; hence
//   REP = 4 or 2 (at most 32 or 64 rows): the rows are repeated in every 128 / REP lanes, and replica p takes only the
//     keys [p, p + 1) TK / REP of each tile (its P is zero elsewhere). Each replica has its own m, l and O; they are
//     joined when the item ends.
//   REP = 1 (more rows): two groups of four warps, GR = 2, take half the keys of each tile for the same rows; the two
//     threads of a row agree on its m through shared memory.
// Q is the A operand: in tensor memory where that leaves room beside O, S and (over S) P, which also leaves more shared
// memory to the rings; for REP = 1 and D <= 128, where the products bound, P has columns of its own instead, so that the
// score MMA need not wait for the P V MMA two tiles before it, and Q is in shared memory.
//
// Work: the key tiles of all (request, cached head, row tile) items form one line of units; each CTA (one per SM) takes
// an equal contiguous range (computed from the lengths on the device, so a captured graph follows them), whatever
// the lengths. A range that covers part of an item leaves (O, m, l) in the workspace, and a second kernel joins
// the parts in CTA order. Everything is in a fixed order: same inputs, same bits.
//
// CTA: the first warps hold rows; one warp each loads K and V tiles by TMA through the block table (a box holds a power
// of two of rows that divides block_size, so no box crosses a page), a lane per box, into two rings; one issues the
// MMAs; one fetches the next item's Q. The K warp walks the CTA's range and leaves each segment (an item's tiles in the
// range) in shared memory for the others. The score MMA of tile t + 1 runs while the softmax of tile t does. Every wait
// is bounded.
//
// What nothing sees must not matter, whatever the memory holds: scores are selected, not added to; in the tiles that
// reach past ctx the rows of V past L are set to zero in shared memory, and infinities and NaN in the step's own rows
// are taken out there (0 x inf is NaN) and added to the rows that see them at the end. Those of the context stay: every
// row sees them. But a weight may be 0 in the products where it is not by definition (a replica's for the keys of the
// others, one that underflows), so where a sum came out as NaN the context is looked through, and the value becomes the
// sum of the infinities and NaN found there (ta_fix_wild; the joining kernel does the same with its parts). Where sums
// are finite that costs adding them up: 64 ragged trees 208.6 -> 211.8 us, 256 single tokens 344 -> 347 us, one token
// 12.8 -> 13.0 us on the device. (Looking at each value for itself before it is written: 13.8 us for one token.)
#include <math.h>

#include "tc_core.cuh"

namespace vt {

constexpr int TA_MAX_NEW = 64;
constexpr int TA_ROWS = 128;
constexpr int TA_ITEM_COST = 2;      // what an item costs besides its tiles, in tiles, when the ranges are cut
constexpr float TA_RAISE = 8.0f;     // log2 of the factor by which weights may pass the running maximum

constexpr int MAX_SLOTS = 12;        // of the K and V rings together

template <int NCH, int REP> struct TaLayout {        // NCH: 64-value chunks of the head
    static constexpr int TK = NCH <= 2 ? 128 : 64;   // keys a tile: 16 .. 32 KB of K
    static constexpr int DP = NCH * 64;
    static constexpr int GR = REP == 1 ? 2 : 1;                    // groups of row warps
    static constexpr bool QT = !(REP == 1 && NCH <= 2);            // Q in tensor memory, P over S
    static constexpr int THREADS = 128 * GR + 128;                 // rows, then the K, MMA, V and Q warps
    static constexpr int RR = TA_ROWS / REP;                       // rows of an item
    // QT: the next item's Q waits in shared memory, QC chunks of its rows at a time in QB buffers, for the row warps to
    // copy; with replicas the buffer also stages their sums when an item ends. Otherwise Q is the MMA's operand there.
    static constexpr int QC = QT ? (REP < NCH ? REP : NCH) : NCH, QB = QT && REP == 1 ? 2 : 1;
    static constexpr int Q_ROUND = RR * QC * 128;                  // 16 KB (QT)
    static constexpr int STAGE_LD = 36;                            // floats a row of the staging area
    static constexpr int STAGE = REP > 1 ? TA_ROWS * STAGE_LD * 4 : 0;
    static constexpr int Q_BYTES = (QB * Q_ROUND > STAGE ? QB * Q_ROUND : STAGE + 1023) / 1024 * 1024;
    static constexpr int SLOT = NCH * TK * 128;
    // entries of the rings of segments and of "pages that are not there" words: more than the K ring's slots (half of
    // the 7 that fit, or of 12) + 2, which is how far the K warp can be ahead of the rows
    static constexpr int RING = SLOT >= 32768 ? 8 : 16;
    // barriers and small shared state, bytes (checked in the kernel)
    static constexpr int BARS =
        ((2 * MAX_SLOTS + 12 + RING) * 8 + RING * 56 + 40 + GR * 1024 + (7 + RING) * 4 + 127) / 128 * 128;
    // tensor memory: O | S0 S1 | P0 P1 or Q
    static constexpr int S_COL = DP, Q_COL = S_COL + 2 * TK, P_COL = QT ? S_COL : Q_COL, P_LD = QT ? TK : TK / 2;
    static_assert(Q_COL + (QT ? DP / 2 : TK) <= 512, "tensor memory");
};

struct TaArgs {
    const void *q, *v;
    void *out;
    long long q_t, q_h, o_t, o_h, v_b, v_r, v_h;   // strides in elements
    const int *table, *cu, *seq_lens;
    const long long *mask;
    long long table_stride;
    int width, B, T, max_new, Hkv, G, D, bs, num_blocks;
    int tile_tokens;         // tokens of an item: whole tokens, at most TA_ROWS rows of them
    int box_rows;            // rows a TMA box holds
    int fold, head_step;     // boxes hold all chunks of their rows; chunks from one head to the next (ta_map)
    int cs, gs;              // bytes in a tile from one 64-value chunk to the next, from 8 rows to the next 8
    int k_slots, v_slots;    // slots of the two rings
    int rows;                // rows of an item at most
    int q_map;               // TMA can read q (16-byte aligned)
    int o_vec;               // 16-byte accesses fit out (2: 32-byte ones)
    uint32_t negate;         // the MMA takes Q negated (a negative scale)
    float sl2;               // |scale| log2 e
    struct TaDesc *desc;     // [grid]
    float2 *stats;           // [2 grid][TA_ROWS] {m, l}
    float *parts;            // [2 grid][DP / 4][TA_ROWS][4]
    unsigned *status;
    uint64_t timeout_ns;
};

// What the joining kernel needs to know of the item that CTA c's range starts inside of.
struct TaDesc {
    int split;               // 1: c's range starts inside an item and c is the first to do so
    int first, parts;        // slot of the item's first part; CTAs that hold parts (then c, c + 1, ..: 2 c, 2 c + 2, ..)
    int tokens, tok0, h;     // the item's tokens, the first one's row, cached head
};

// ---- the units and a CTA's range of them ---------------------------------------------------------------------------
struct TaReq {
    int L, n, cu0, nt, rtn;
    long long units;
};
__device__ __forceinline__ TaReq ta_request(const TaArgs &A, int b, int tk) {
    TaReq r;
    r.cu0 = A.cu[b];
    r.n = max(A.cu[b + 1] - r.cu0, 0);
    r.L = min(max(A.seq_lens[b], 0), 0x7fff0000);   // the last tile's keys stay within an int
    // tiles past the table's columns hold nothing to see
    r.nt = max(1, (int)((min((long long)r.L, (long long)A.width * A.bs) + tk - 1) / tk));
    r.rtn = (min(r.n, A.max_new) + A.tile_tokens - 1) / A.tile_tokens;
    r.units = (long long)A.Hkv * r.rtn * (r.nt + TA_ITEM_COST);
    return r;
}

struct TaPlan {   // in shared memory
    long long lo, hi, total, base0;
    int b0, ge;
};

// x / y for x, y >= 0: a 64-bit division takes a few hundred cycles, and these stand in the way of the first load
__device__ __forceinline__ long long ta_div(long long x, int y) {
    return x >> 31 ? x / y : (long long)((unsigned)x / (unsigned)y);
}
// floor(total c / ge)
__device__ __forceinline__ long long ta_range_lo(long long total, int ge, int c) {
    const long long q = ta_div(total, ge);
    return q * c + (unsigned)((int)(total - q * ge) * c) / (unsigned)ge;
}

struct TaSeg {       // in shared memory
    long long t0;    // the item's first tile, as a unit
    int tiles;       // 0: the range has ended
    int b, h, rt, kt0, nt, L, n, cu0;
    int head;        // first segment of the CTA
    int whole;       // all of the item
};

struct TaIter {
    long long u, hi, base;
    int b;
    bool begun;
    TaReq r;
    __device__ __forceinline__ TaIter(const TaArgs &A, const TaPlan &p, int tk)
        : u(p.lo), hi(p.hi), base(p.base0), b(p.b0), begun(false) {
        if (u < hi) r = ta_request(A, b, tk);
    }
    // An item's units are TA_ITEM_COST without a tile, then its tiles.
    __device__ __forceinline__ void next(const TaArgs &A, int tk, TaSeg &s) {
        s.tiles = 0;
        while (u < hi) {
            while (u >= base + r.units) {
                base += r.units;
                r = ta_request(A, ++b, tk);
            }
            const int per = r.nt + TA_ITEM_COST;
            const long long x = u - base, item = ta_div(x, per);
            const int y = (int)(x - item * per), take = (int)min((long long)per - y, hi - u);
            const int kt0 = max(y - TA_ITEM_COST, 0), kt1 = max(y + take - TA_ITEM_COST, 0);
            s.t0 = u - y + TA_ITEM_COST;
            u += take;
            if (kt1 == kt0) continue;
            s.b = b;
            s.kt0 = kt0;
            s.tiles = kt1 - kt0;
            s.h = (int)ta_div(item, r.rtn);
            s.rt = (int)(item - (long long)s.h * r.rtn);
            s.nt = r.nt;
            s.L = r.L;
            s.n = r.n;
            s.cu0 = r.cu0;
            s.head = !begun;
            begun = true;
            s.whole = s.tiles == r.nt;
            return;
        }
    }
};

// Every thread calls it: total units by a block reduction, then the request that holds the range's first unit.
template <int THREADS>
__device__ __forceinline__ void ta_plan(const TaArgs &A, int tk, TaPlan *plan, long long *wsum) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (A.B + THREADS - 1) / THREADS, b0 = tid * per, b1 = min(A.B, b0 + per);
    long long sum = 0;
    for (int b = b0; b < b1; ++b) sum += ta_request(A, b, tk).units;
    long long x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += wsum[w];
        total += wsum[w];
    }
    const int ge = (int)max(1ll, min((long long)gridDim.x, total));
    const int c = blockIdx.x;
    const long long lo = c < ge ? ta_range_lo(total, ge, c) : total, hi = c < ge ? ta_range_lo(total, ge, c + 1) : total;
    if (tid == 0) {
        plan->lo = lo;
        plan->hi = hi;
        plan->total = total;
        plan->ge = ge;
    }
    long long start = before + x - sum;
    if (lo < hi && lo >= start && lo < start + sum) {   // exactly one thread
        int b = b0;
        for (;; ++b) {
            const long long u = ta_request(A, b, tk).units;
            if (lo < start + u) break;
            start += u;
        }
        plan->b0 = b;
        plan->base0 = start;
    }
    __syncthreads();
}

// ---- small pieces ----------------------------------------------------------------------------------------------------
__device__ __forceinline__ float ta_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <typename T> __device__ __forceinline__ bool ta_wild(uint32_t half) {
    constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
    return (half & E) == E;
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// n limits, at most 2^62 ns (added to the timer it must not wrap)
__device__ __forceinline__ uint64_t ta_times(uint64_t limit, uint64_t n) {
    constexpr uint64_t MOST = 1ull << 62;
    return __umul64hi(limit, n) != 0 || limit * n > MOST ? MOST : limit * n;
}
// Waits for the phase of `parity` to complete; false when that takes longer than timeout_ns. The bound is each wait's
// own (a call over a very long context may run longer than it); the timer is read every 1024 polls.
__device__ __forceinline__ bool ta_wait(uint64_t *bar, uint32_t parity, uint64_t timeout_ns) {
    uint32_t polls = 0;
    uint64_t deadline = 0;
    while (!mbar_try_wait(bar, parity)) {
        if ((++polls & 1023u) != 0) continue;
        const uint64_t now = globaltimer();
        if (deadline == 0) deadline = now + timeout_ns;
        else if (now > deadline) return false;
    }
    return true;
}
__device__ __forceinline__ bool ta_warp_wait(uint64_t *bar, uint32_t parity, uint64_t timeout_ns) {
    return __all_sync(0xffffffffu, ta_wait(bar, parity, timeout_ns)) != 0;
}
// K as it lies in the cache, [keys][64 values] rows of 128 bytes: groups of 8 keys `gs` bytes apart (stride offset).
__device__ __forceinline__ uint64_t ta_k_desc(uint32_t saddr, int gs) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)1u << 16;
    d |= (uint64_t)(((uint32_t)gs >> 4) & 0x3FFFu) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}
// V the same way, but the MMA's N (values) is contiguous: 64-value chunks `cs` bytes apart (leading offset).
__device__ __forceinline__ uint64_t ta_v_desc(uint32_t saddr, int cs, int gs) {
    return (ta_k_desc(saddr, gs) & ~((uint64_t)0x3FFFu << 16)) | (uint64_t)(((uint32_t)cs >> 4) & 0x3FFFu) << 16;
}
// Called by a whole warp on uniform values; one elected lane issues. D (TMEM, fp32) (+)= A . B^T, kind::f16, A from
// shared memory or (ts) tensor memory; and the commit of what that lane has issued.
__device__ __forceinline__ void umma_f16_e(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts_e(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_commit_e(uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int x, int y, int z, int w,
                                            uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tma_load_5d(void *dst, const CUtensorMap *map, int x, int y, int z, int w, int u,
                                            uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
        "[%7];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(u), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
            "r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
// 32 bytes to global memory, 32-byte aligned
__device__ __forceinline__ void st_global32(void *p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
// N (16 or 32) consecutive tensor-memory columns of the warp's lanes from / to registers.
template <int N> __device__ __forceinline__ void ta_ld(uint32_t taddr, uint32_t *r) {
    static_assert(N == 16 || N == 32, "columns");
    if constexpr (N == 32) tmem_ld32(taddr, *reinterpret_cast<uint32_t(*)[32]>(r));
    else tmem_ld16(taddr, *reinterpret_cast<uint32_t(*)[32]>(r));
}
template <int N> __device__ __forceinline__ void ta_st(uint32_t taddr, const uint32_t *r) {
    static_assert(N == 16 || N == 32, "columns");
    if constexpr (N == 32) tmem_st32(taddr, *reinterpret_cast<const uint32_t(*)[32]>(r));
    else
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
            "%14, %15, %16};" ::"r"(taddr),
            "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
            "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
            : "memory");
}

// Bits kk = 0 .. 31: key c0-relative index kk0 + kk is seen, where keys below c0 all are and key c0 + jj has bit jj of
// `see`.
__device__ __forceinline__ uint32_t ta_seen(unsigned long long see, int kk0, int c0) {
    const int jj = kk0 - c0;
    if (jj <= -32) return 0xffffffffu;
    if (jj < 0) return (uint32_t)(see << -jj) | ((1u << -jj) - 1u);
    return jj < 64 ? (uint32_t)(see >> jj) : 0u;
}

// After an item's values are written, by whole warps some of whose rows got a NaN that is not their scores': where the
// context that the segment covers (keys j0 .. j1 - 1 of request b, cached head h) holds infinities or NaN, every row's
// value is their sum and that of the wild values of the step's own tokens it sees (wn). The lanes share out the keys, for
// 8 columns at a time: those of the warp, `share` from part * share on of every `width`. parts: the segment is a part of
// the item, and this row's values are TA_ROWS apart there, by fours; else they are at dst.
template <typename T>
__device__ __noinline__ void ta_fix_wild(const TaArgs &A, int b, int h, int j0, int j1, int width, int share, int part,
                                         int ctx, int seg_k0, int seg_k1, unsigned long long wn, bool ok, T *dst,
                                         float *parts) {
    constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;   // exponent; the mantissa is below it
    const int *trow = A.table + (long long)b * A.table_stride;
    auto values = [&](int j) -> const T * {   // of key j; null if its page is not there
        const int page = j / A.bs, blk = page < A.width ? trow[page] : -1;
        if (blk < 0 || blk >= A.num_blocks) return nullptr;
        return reinterpret_cast<const T *>(A.v) + blk * A.v_b + (j - page * A.bs) * A.v_r + h * A.v_h;
    };
#pragma unroll 1
    for (int c = 0; c < A.D; c += 8) {
        if (c % width / share != part) continue;
        uint32_t pos = 0, neg = 0;   // bit e: column c + e holds +inf, -inf; NaN counts as both
        for (int k = j0; k < j1 && (pos & neg) != 0xffu; k += 4 * 32) {   // nothing is added to 8 columns of NaN
            uint4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = k + 32 * i + (int)(threadIdx.x & 31);
                const T *v = j < j1 ? values(j) : nullptr;
                x[i] = v ? *reinterpret_cast<const uint4 *>(v + c) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t u = (w[e >> 1] >> (16 * (e & 1))) & 0xffffu;
                    if ((u & E) != E) continue;
                    const bool nan = (u & (E ^ 0x7fffu)) != 0;
                    if (nan || !(u & 0x8000u)) pos |= 1u << e;
                    if (nan || (u & 0x8000u)) neg |= 1u << e;
                }
            }
            pos = __reduce_or_sync(0xffffffffu, pos);
            neg = __reduce_or_sync(0xffffffffu, neg);
        }
        for (uint32_t left = ok ? pos | neg : 0u; left; left &= left - 1) {
            const int e = __ffs((int)left) - 1;
            float sum = !((neg >> e) & 1u) ? INFINITY : !((pos >> e) & 1u) ? -INFINITY : NAN;
            for (unsigned long long own = wn; own; own &= own - 1) {
                const int j = ctx + __ffsll((long long)own) - 1;
                const T *v = j >= seg_k0 && j < seg_k1 ? values(j) : nullptr;
                const float f = v ? t2f<T>(v[c + e]) : 0.0f;
                if (!isfinite(f)) sum += f;
            }
            if (parts) parts[(c + e) / 4 * (TA_ROWS * 4) + (c + e) % 4] = sum;
            else dst[c + e] = f2t<T>(sum);
        }
        __syncwarp();
    }
}

// ---- the kernel ------------------------------------------------------------------------------------------------------
template <typename T, int NCH, int REP>
__global__ void __launch_bounds__(TaLayout<NCH, REP>::THREADS, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                     const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ TaArgs A) {
    using Lay = TaLayout<NCH, REP>;
    constexpr int TK = Lay::TK, DP = Lay::DP, GR = Lay::GR;
    constexpr int ROW_WARPS = 4 * GR, K_WARP = ROW_WARPS, MMA_WARP = ROW_WARPS + 1, V_WARP = ROW_WARPS + 2,
                  Q_WARP = ROW_WARPS + 3;
    constexpr bool QT = Lay::QT;
    constexpr int TA_RING = Lay::RING;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *qs = smem_raw;   // 1024-byte aligned (checked below): the block has no static shared memory
    const int SK = A.k_slots, SV = A.v_slots;
    unsigned char *kring = qs + Lay::Q_BYTES, *vring = kring + (size_t)SK * Lay::SLOT;
    float *stage = reinterpret_cast<float *>(qs);   // [128][STAGE_LD] (REP > 1)
    uint64_t *kfull = reinterpret_cast<uint64_t *>(vring + (size_t)SV * Lay::SLOT);
    uint64_t *kempty = kfull + SK;
    uint64_t *vfull = kempty + SK;
    uint64_t *vempty = vfull + SV;
    uint64_t *sfull = vempty + SV;      // [2] scores in S buffer
    uint64_t *pfull = sfull + 2;        // [2] weights from them (and V ready for use), the row warps arrive
    uint64_t *pvdone = pfull + 2;       // [2] the MMAs that read them (and added to O) have completed
    uint64_t *qfull = pvdone + 2;       // [1] Q in place for the MMA (QT: the row warps arrive, else the Q warp)
    uint64_t *qbfull = qfull + 1;       // [2] QT: Q buffer loaded
    uint64_t *qbempty = qbfull + 2;     // [2] Q buffer free (QT: the row warps arrive, else the item's last scores)
    uint64_t *drain = qbempty + 2;
    uint64_t *segfull = drain + 1;      // [TA_RING]
    TaSeg *segs = reinterpret_cast<TaSeg *>(segfull + TA_RING);   // [TA_RING]
    TaPlan *plan = reinterpret_cast<TaPlan *>(segs + TA_RING);
    float2 *ml = reinterpret_cast<float2 *>(plan + 1);            // REP > 1: [128] m and l of the replicas
    float(*hm)[2][TA_ROWS] = reinterpret_cast<float(*)[2][TA_ROWS]>(ml);   // GR == 2: [tile & 1][group] maxima, sums
    long long *wsum = reinterpret_cast<long long *>(ml);          // [warps], before
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(hm + (GR == 2 ? 2 : 1));
    uint32_t *wild = tmem_slot + 1;                               // [2 segments][2 words]
    volatile uint32_t *more = wild + 4;                           // [segment & 1] the rows have another segment
    volatile uint32_t *bad = wild + 6;                            // [TA_RING] 8-row groups not there
    // what stands between kfull and here, at the most slots, fits the bytes that the host adds to Q and the rings
    static_assert(sizeof(TaSeg) == 56 && sizeof(TaPlan) == 40 &&
                      8 * (2 * MAX_SLOTS + 2 + 2 + 2 + 1 + 2 + 2 + 1 + TA_RING) + TA_RING * (int)sizeof(TaSeg) +
                              (int)sizeof(TaPlan) + GR * 2 * TA_ROWS * 4 + 4 * (1 + 4 + 2 + TA_RING) <=
                          Lay::BARS,
                  "shared state");
    static_assert(Lay::THREADS / 32 * 8 <= GR * 2 * TA_ROWS * 4, "sums of the plan");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    if (smem_u32(smem_raw) & 1023u) {   // the tiles' swizzle needs it
        pdl_wait();
        if (threadIdx.x == 0) {
            A.desc[blockIdx.x].split = 0;
            report(A.status, ST_PIPE_TIMEOUT | 0x2f0u);
        }
        return;
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < SK; ++s) {
            mbar_init(&kfull[s], 1);
            mbar_init(&kempty[s], 1);
        }
        for (int s = 0; s < SV; ++s) {
            mbar_init(&vfull[s], 1);
            mbar_init(&vempty[s], 1);
        }
        for (int s = 0; s < TA_RING; ++s) mbar_init(&segfull[s], 1);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&sfull[b], 1);
            mbar_init(&pfull[b], ROW_WARPS);
            mbar_init(&pvdone[b], 1);
            mbar_init(&qbfull[b], 1);
            mbar_init(&qbempty[b], QT ? ROW_WARPS : 1);
        }
        mbar_init(qfull, QT ? ROW_WARPS : 1);
        mbar_init(drain, 1);
        for (int i = 0; i < 4; ++i) wild[i] = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
        if (A.q_map) tma_prefetch_desc(&tmap_q);
    }
    if (warp == MMA_WARP) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    pdl_wait();
    tc_fence_before();
    ta_plan<Lay::THREADS>(A, TK, plan, wsum);   // synchronises the block
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t *>(tmem_slot);
    const uint64_t limit = A.timeout_ns;   // of every wait

    if (warp == K_WARP || warp == V_WARP) {
        // ---------------- K and V tiles ----------------
        // A tile is at most 32 boxes, one a lane: all chunks (fold), or 64-value chunk lane % NCH, of box_rows rows.
        // The table entries of the next tile are loaded while this one's copies are issued.
        const bool is_k = warp == K_WARP;
        const CUtensorMap *map = is_k ? &tmap_k : &tmap_v;
        uint64_t *full = is_k ? kfull : vfull, *empty = is_k ? kempty : vempty;
        unsigned char *ring = is_k ? kring : vring;
        const int S = is_k ? SK : SV;
        const int box = A.box_rows, per = A.fold ? 1 : NCH, p = lane / per, c = lane - p * per;
        const int box_bytes = box * 128 * (A.fold ? NCH : 1);
        const uint32_t dst0 = (uint32_t)((box >> 3) * p * A.gs + c * A.cs);
        bool dead = false;
        int g = 0, s = 0, seg = 0;   // tiles, ring slot, segments
        uint32_t phase = 1;          // of the slot's release: the first round finds all slots free
        TaIter it(A, *plan, TK);
        while (!dead) {
            TaSeg *sp = segs + seg % TA_RING;
            if (is_k) {
                TaSeg x;
                it.next(A, TK, x);
                if (lane == 0) {
                    *sp = x;
                    mbar_arrive(&segfull[seg % TA_RING]);
                }
                __syncwarp();
            } else if (!ta_warp_wait(&segfull[seg % TA_RING], (uint32_t)(seg / TA_RING) & 1u, limit)) {
                if (lane == 0) report(A.status, ST_PIPE_TIMEOUT | 0x218u);
                break;
            }
            const int tiles = sp->tiles, kt0 = sp->kt0, L = sp->L, h = sp->h;
            if (tiles == 0) break;
            const int *trow = A.table + (long long)sp->b * A.table_stride;
            auto entry_of = [&](int kt, int &r0) {   // this lane's table entry; -1: none needed or none there
                const int row = kt * TK + p * box, page = row / A.bs;
                r0 = row - page * A.bs;
                return row < L && page < A.width && p * box < TK ? trow[page] : -1;
            };
            int r0, ent = entry_of(kt0, r0);
            for (int kt = kt0; kt < kt0 + tiles; ++kt, ++g) {
                const int boxes = (min(max(L - kt * TK, 0), TK) + box - 1) / box * per;
                const int blk = (ent < 0 || ent >= A.num_blocks) ? A.num_blocks : ent;   // num_blocks reads as zeros
                const int y0 = r0;
                if (kt + 1 < kt0 + tiles) ent = entry_of(kt + 1, r0);
                int ok = 1;
                if (lane == 0) {
                    ok = ta_wait(&empty[s], phase, limit);
                    if (!ok) report(A.status, ST_PIPE_TIMEOUT | 0x210u);
                }
                if (!__shfl_sync(0xffffffffu, ok, 0)) {
                    dead = true;
                    break;
                }
                if (is_k) {   // groups of 8 rows whose page is not there
                    const bool none = lane < boxes && blk == A.num_blocks;
                    const uint32_t gone = __reduce_or_sync(
                        0xffffffffu, none ? ((1u << (box >> 3)) - 1u) << (p * (box >> 3)) : 0u);
                    if (lane == 0) bad[g % TA_RING] = gone;
                }
                if (lane == 0) mbar_arrive_expect_tx(&full[s], (uint32_t)(boxes * box_bytes));
                __syncwarp();
                if (lane < boxes) {
                    unsigned char *dst = ring + (size_t)s * Lay::SLOT + dst0;
                    if (A.fold) tma_load_5d(dst, map, 0, 0, h * A.head_step, y0 >> 3, blk, &full[s]);
                    else tma_load_4d(dst, map, c * 64, y0, h, blk, &full[s]);
                }
                if (++s == S) s = 0, phase ^= 1u;
            }
            ++seg;
        }
        if (lane == 0) {
            if (is_k && dead) {   // no further segment: whoever waits for one need not wait out its limit
                segs[(seg + 1) % TA_RING].tiles = 0;
                mbar_arrive(&segfull[(seg + 1) % TA_RING]);
            }
            // the copies issued land before the shared memory is released (those that were consumed have)
            for (int j = (g > S ? g - S : 0); j < g; ++j) ta_wait(&full[j % S], (uint32_t)(j / S) & 1u, limit);
        }
        __syncwarp();
    } else if (warp == MMA_WARP) {
        // ---------------- MMA issuer ----------------
        // The whole warp runs the loop on warp-uniform values and one elected lane issues: operands stay in uniform
        // registers. (A loop inside `if (lane == 0)` took about 120 cycles an MMA to issue, more than the MMAs.)
        const uint32_t id_s = idesc_f16<T>(TA_ROWS, TK) | (A.negate << 13);
        constexpr uint32_t id_o = idesc_f16<T>(TA_ROWS, DP) | (1u << 16);   // B (V) is MN-major
        const uint32_t tb = __shfl_sync(0xffffffffu, tmem_base, 0), kring0 = smem_u32(kring), vring0 = smem_u32(vring);
        const uint64_t qd = sw128_desc(smem_u32(qs));
        int g = 0, seg = 0, ks = 0, vs = 0;   // tiles, segments, ring slots
        uint32_t kphase = 0, vphase = 0;
        auto wait = [&](uint64_t *bar, uint32_t parity, unsigned code) {
            if (ta_warp_wait(bar, parity, limit)) {
                tc_fence_after();
                return true;
            }
            if (lane == 0) report(A.status, ST_PIPE_TIMEOUT | code);
            return false;
        };
        auto scores = [&](int gt) {   // S[gt] = Q K^T of the next K tile
            if (!wait(&kfull[ks], kphase, 0x220u)) return false;
            if (QT && gt > 1 && !wait(&pvdone[gt & 1], ((uint32_t)(gt >> 1) & 1u) ^ 1u, 0x228u)) return false;   // P over S
            const uint64_t kd = ta_k_desc(kring0 + (uint32_t)(ks * Lay::SLOT), A.gs);
            const uint32_t d = tb + Lay::S_COL + (uint32_t)((gt & 1) * TK);
#pragma unroll
            for (int i = 0; i < NCH * 4; ++i) {   // 16 values a step; past D both operands hold zeros
                const uint64_t kdi = kd + (uint64_t)((i >> 2) * (A.cs >> 4) + 2 * (i & 3));
                if constexpr (QT) umma_f16_ts_e(d, tb + Lay::Q_COL + 8 * i, kdi, id_s, i > 0);
                else umma_f16_e(d, qd + (i >> 2) * (TA_ROWS * 128 / 16) + 2 * (i & 3), kdi, id_s, i > 0);
            }
            umma_commit_e(&sfull[gt & 1]);
            umma_commit_e(&kempty[ks]);
            if (++ks == SK) ks = 0, kphase ^= 1u;
            return true;
        };
        bool ok = true;
        while (ok && (ok = wait(&segfull[seg % TA_RING], (uint32_t)(seg / TA_RING) & 1u, 0x238u))) {
            const int N = __shfl_sync(0xffffffffu, segs[seg % TA_RING].tiles, 0);
            if (N == 0) break;
            ok = wait(qfull, (uint32_t)seg & 1u, 0x230u) && scores(g);
            for (int t = 0; ok && t < N; ++t, ++g) {
                if (t + 1 < N) ok = scores(g + 1);
                else if (!QT) umma_commit_e(&qbempty[0]);
                ok = ok && wait(&pfull[g & 1], (uint32_t)(g >> 1) & 1u, 0x240u);
                ok = ok && wait(&vfull[vs], vphase, 0x250u);
                if (!ok) break;
                const uint32_t p = tb + Lay::P_COL + (uint32_t)((g & 1) * Lay::P_LD);
                const uint64_t v = ta_v_desc(vring0 + (uint32_t)(vs * Lay::SLOT), A.cs, A.gs);
#pragma unroll
                for (int i = 0; i < TK / 16; ++i)   // 16 keys a step: 8 columns of P, two groups of rows of V
                    umma_f16_ts_e(tb, p + 8 * i, v + (uint64_t)(i * (A.gs >> 3)), id_o, (t > 0 || i > 0) ? 1u : 0u);
                umma_commit_e(&pvdone[g & 1]);
                umma_commit_e(&vempty[vs]);
                if (++vs == SV) vs = 0, vphase ^= 1u;
            }
            ++seg;
        }
        umma_commit_e(drain);   // every MMA issued has completed once it flips
        ta_warp_wait(drain, 0u, limit);
    } else if (warp == Q_WARP) {
        // ---------------- Q of the items ----------------
        // [chunk][row] of 128 bytes (64 values), swizzled: one TMA box a chunk (its tokens past the request's end give
        // rows that nothing uses), or, for a q that TMA cannot read, element by element.
        constexpr int QC = Lay::QC, QB = Lay::QB;
        int round = 0;
        bool ok = true;
        uint64_t tiles = 0;   // of the segment before: the K warp hands out the next one after as many waits of its own
        for (int seg = 0; ok; ++seg) {
            ok = ta_warp_wait(&segfull[seg % TA_RING], (uint32_t)(seg / TA_RING) & 1u, ta_times(limit, tiles + 1));
            const TaSeg &sg = segs[seg % TA_RING];
            if (!ok || sg.tiles == 0) break;
            tiles = (uint64_t)sg.tiles;
            const int tok0 = sg.cu0 + sg.rt * A.tile_tokens, h0 = sg.h * A.G;
            const int rows = min(A.tile_tokens, A.max_new) * A.G;
            for (int c0 = 0; ok && c0 < NCH; c0 += QC, ++round) {
                const int b = round % QB, nc = min(QC, NCH - c0);
                uint64_t *bar = QT ? &qbfull[b] : qfull;
                ok = ta_warp_wait(&qbempty[b], ((uint32_t)(round / QB) & 1u) ^ 1u, limit);
                if (!ok) break;
                unsigned char *buf = qs + b * Lay::Q_ROUND;
                if (A.q_map) {
                    if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(nc * rows * 128));
                    __syncwarp();
                    if (lane < nc) tma_load_3d(buf + lane * (Lay::RR * 128), &tmap_q, (c0 + lane) * 64, h0, tok0, bar);
                    continue;
                }
                for (int i = lane; i < nc * rows * 64; i += 32) {
                    const int c = i / (rows * 64), r = i / 64 % rows, d = i % 64, t = r / A.G, tok = tok0 + t;
                    T x = f2t<T>(0.0f);
                    if ((c0 + c) * 64 + d < A.D && tok >= 0 && tok < A.T)
                        x = reinterpret_cast<const T *>(A.q)[(long long)tok * A.q_t +
                                                             (long long)(h0 + r - t * A.G) * A.q_h + (c0 + c) * 64 + d];
                    reinterpret_cast<T *>(buf + c * (Lay::RR * 128) + r * 128 + (((d >> 3) ^ (r & 7)) << 4))[d & 7] = x;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            }
        }
        if (lane == 0) {
            if (!ok) report(A.status, ST_PIPE_TIMEOUT | 0x2b0u);
            for (int j = (round > QB ? round - QB : 0); j < round; ++j)   // as the K and V warps do
                ta_wait(QT ? &qbfull[j % QB] : qfull, (uint32_t)(j / QB) & 1u, limit);
        }
        __syncwarp();
    } else if (warp < ROW_WARPS) {
        // ---------------- rows: softmax and output ----------------
        const int q4 = warp & 3, grp = warp >> 2;
        const int tid = q4 * 32 + lane;             // lane of tensor memory this thread holds
        constexpr int RR = TA_ROWS / REP, CPT = TK / REP / GR;   // rows; keys of a tile a thread takes
        const int row = tid % RR, part = GR == 2 ? grp : tid / RR;
        const uint32_t lane_base = tmem_base + ((uint32_t)(q4 * 32) << 16);
        bool dead = false;
        auto wait = [&](uint64_t *bar, uint32_t parity, unsigned code) {
            if (dead) return;   // the loops go on without data, so that the barriers among these warps stay matched
            if (!ta_warp_wait(bar, parity, limit)) {
                if (lane == 0) report(A.status, ST_PIPE_TIMEOUT | code);
                dead = true;
            }
            tc_fence_after();
        };
        int g = 0, seg = 0, qround = 0;
        // the next segment, if there is one, and its Q into tensor memory
        auto open = [&]() {
            wait(&segfull[seg % TA_RING], (uint32_t)(seg / TA_RING) & 1u, 0x258u);
            // One thread decides, since the warps' barriers must match. Two words in turn: a word is written again only
            // after the next segment's barrier, which a warp reaches after it has read this one's.
            if (threadIdx.x == 0) more[seg & 1] = !dead && segs[seg % TA_RING].tiles != 0;
            named_sync(TC_EPI_BAR, 128 * GR);
            if (!more[seg & 1]) return false;
            if constexpr (QT) {
                constexpr int QC = Lay::QC, QB = Lay::QB;
#pragma unroll
                for (int c0 = 0; c0 < NCH; c0 += QC, ++qround) {
                    const int b = qround % QB;
                    wait(&qbfull[b], (uint32_t)(qround / QB) & 1u, 0x2b8u);
                    const unsigned char *buf = qs + b * Lay::Q_ROUND + row * 128;
#pragma unroll
                    for (int c = 0; c < QC && c0 + c < NCH; ++c) {   // rows past the item's hold anything
                        if (GR == 2 && ((c0 + c) & 1) != grp) continue;
                        uint32_t w[32];
#pragma unroll
                        for (int v = 0; v < 8; ++v) {
                            const uint4 x = *reinterpret_cast<const uint4 *>(buf + c * (Lay::RR * 128) +
                                                                             ((v ^ (row & 7)) << 4));
                            w[4 * v] = x.x, w[4 * v + 1] = x.y, w[4 * v + 2] = x.z, w[4 * v + 3] = x.w;
                        }
                        tmem_st32(lane_base + Lay::Q_COL + 32 * (c0 + c), w);
                    }
                    // with replicas the buffer is the staging area too: free once the item before is written
                    __syncwarp();
                    if (lane == 0 && (REP == 1 || seg == 0 || c0 + QC < NCH)) mbar_arrive(&qbempty[b]);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(qfull);
            }
            return true;
        };
        bool has = open();
        if (threadIdx.x == 0) {
            A.desc[blockIdx.x].split = 0;
            if (has && segs[0].kt0 > 0) {
                const TaSeg &x = segs[0];
                const int c = blockIdx.x, ge = plan->ge;
                const long long total = plan->total, before = ta_range_lo(total, ge, c - 1), last = x.t0 + x.nt - 1;
                int c1 = (int)(last * ge / total);   // the CTA holding the item's last tile
                while (c1 + 1 < ge && ta_range_lo(total, ge, c1 + 1) <= last) ++c1;
                TaDesc d;
                d.split = x.t0 >= before;
                d.first = 2 * (c - 1) + (before >= x.t0 - TA_ITEM_COST ? 0 : 1);   // its first or last segment
                d.parts = c1 - c + 2;
                d.tokens = min(min(x.n, A.max_new) - x.rt * A.tile_tokens, A.tile_tokens);
                d.tok0 = x.cu0 + x.rt * A.tile_tokens;
                d.h = x.h;
                A.desc[c] = d;
            }
        }
        while (has) {
            const TaSeg &sg = segs[seg % TA_RING];
            // (of a request with more tokens than keys, by more than the mask's 64 bits, no token has a key it sees)
            const int N = sg.tiles, L = sg.L, ctx = max(L - sg.n, -64), kt0 = sg.kt0;
            const int live = min(min(sg.n, A.max_new) - sg.rt * A.tile_tokens, A.tile_tokens) * A.G;
            const int row_i = row / A.G, tok_i = sg.rt * A.tile_tokens + row_i, tok = sg.cu0 + tok_i;
            const bool mine = row < live && tok >= 0 && tok < A.T;
            const bool warp_live = (REP > 1 ? 0 : q4 * 32) < live;
            unsigned long long see = 0;
            if (mine) {
                see = A.mask ? (unsigned long long)A.mask[tok] : (2ull << tok_i) - 1ull;
                if (sg.n < 64) see &= (1ull << sg.n) - 1ull;
            }
            float m = -INFINITY, l = 0.0f;
            for (int t = 0; t < N; ++t, ++g) {
                const int buf = g & 1;
                const int k0 = (kt0 + t) * TK;
                const uint32_t use = (uint32_t)(g >> 1);
                const bool past = k0 + TK > ctx;
                const uint32_t s_col = lane_base + Lay::S_COL + (uint32_t)(buf * TK);
                const uint32_t p_col = lane_base + Lay::P_COL + (uint32_t)(buf * Lay::P_LD);
                wait(&sfull[buf], use & 1u, 0x260u);
                const uint32_t gone = bad[g % TA_RING];
                if (warp_live) {
                    constexpr int LD = CPT < 32 ? CPT : 32;
                    float x[CPT < 32 ? 32 : CPT];
#pragma unroll
                    for (int c = 0; c < CPT; c += LD)
                        ta_ld<LD>(s_col + (uint32_t)(part * CPT + c), reinterpret_cast<uint32_t *>(&x[c]));
                    tmem_ld_wait();
                    if (past || gone != 0) {
#pragma unroll
                        for (int c = 0; c < CPT; c += LD) {
                            const int kk = part * CPT + c;
                            uint32_t vis = ta_seen(see, k0 + kk, ctx);
                            const uint32_t g4 = (gone >> (kk / 8)) & 15u;
                            vis &= ~(((g4 * 0x00204081u) & 0x01010101u) * 255u);
#pragma unroll
                            for (int j = 0; j < LD; ++j) x[c + j] = (vis >> j) & 1u ? x[c + j] : -INFINITY;
                        }
                    }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int j = 0; j < CPT; ++j) mx[j & 3] = fmaxf(mx[j & 3], x[j]);
                    float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    if (GR == 2) {   // the two warps that hold these rows (and have read their scores: P may go there)
                        hm[buf][grp][row] = top;
                        named_sync(TC_EPI_BAR + 1 + q4, 64);
                        top = fmaxf(top, hm[buf][grp ^ 1][row]);
                    }
                    const float tm = top * A.sl2;   // sl2 > 0
                    // (a row that is none holds anything: it must not make its warp rescale)
                    const bool raise = row < live && (tm > m + TA_RAISE || (m == -INFINITY && tm > m));
                    if (__any_sync(0xffffffffu, raise)) {
                        const float f = raise ? ta_exp2(m - tm) : 1.0f;
                        if (raise) m = tm;
                        l *= f;
                        if (t > 0) {   // O of the tiles before this one; a group's share of its columns
                            wait(&pvdone[(g - 1) & 1], (uint32_t)((g - 1) >> 1) & 1u, 0x270u);
#pragma unroll 1
                            for (int c = grp * (DP / GR); c < (grp + 1) * (DP / GR); c += 32) {
                                uint32_t o[32];
                                tmem_ld32(lane_base + (uint32_t)c, o);
                                tmem_ld_wait();
#pragma unroll
                                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                                tmem_st32(lane_base + (uint32_t)c, o);
                            }
                        }
                    }
                    constexpr float BIAS = std::is_same<T, __half>::value ? 7.0f : 0.0f;
                    const float off = (m == -INFINITY ? 0.0f : -m) + BIAS;
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    uint32_t w[CPT / 2];
#pragma unroll
                    for (int j = 0; j < CPT; j += 2) {   // a hidden key: 2^-inf = 0
                        const float a = ta_exp2(__fmaf_rn(x[j], A.sl2, off));
                        const float b = ta_exp2(__fmaf_rn(x[j + 1], A.sl2, off));
                        sum[j & 2] += a;
                        sum[(j & 2) + 1] += b;
                        w[j >> 1] = pack2<T>(a, b);
                    }
                    // P's columns are free: sfull was committed after the MMAs that read them two tiles ago
                    if constexpr (REP == 1) ta_st<CPT / 2>(p_col + (uint32_t)(part * (CPT / 2)), w);
                    if constexpr (REP > 1) {
                        // the replica's CPT / 2 columns of P, zeros in the others'
#pragma unroll
                        for (int c = 0; c < TK / 2; c += 32) {
                            uint32_t z[32];
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                z[j] = (c + j) / (CPT / 2) == part ? w[j % (CPT / 2)] : 0u;
                            ta_st<32>(p_col + (uint32_t)c, z);
                        }
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tmem_st_wait();
                }
                if (past) {
                    // rows of V that not every row sees: zeros past the length, no infinities or NaN before it
                    const int r0 = max(ctx - k0, 0);
                    wait(&vfull[g % SV], (uint32_t)(g / SV) & 1u, 0x290u);
                    unsigned char *vs = vring + (size_t)(g % SV) * Lay::SLOT;
                    for (int idx = threadIdx.x; idx < (TK - r0) * NCH * 8 && !dead; idx += 128 * GR) {
                        const int r = r0 + idx / (NCH * 8), v = idx % (NCH * 8), j = k0 + r;
                        uint4 *p = reinterpret_cast<uint4 *>(vs + (r >> 3) * A.gs + (v >> 3) * A.cs + (r & 7) * 128 +
                                                             (((v & 7) ^ (r & 7)) << 4));
                        if (j >= L) {
                            *p = make_uint4(0, 0, 0, 0);
                            continue;
                        }
                        uint4 y = *p;
                        uint32_t *w = reinterpret_cast<uint32_t *>(&y);
                        bool any = false;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (ta_wild<T>(w[e])) w[e] &= 0xffff0000u, any = true;
                            if (ta_wild<T>(w[e] >> 16)) w[e] &= 0x0000ffffu, any = true;
                        }
                        if (any) {
                            *p = y;
                            const int jj = j - ctx;   // < n; a wild one past the mask's 64 bits is seen by no row
                            if (jj < 64) atomicOr(&wild[(seg & 1) * 2 + (jj >> 5)], 1u << (jj & 31));
                        }
                    }
                    fence_proxy_async();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[buf]);
            }
            // the next item's Q may go in: this one's last scores are done
            ++seg;
            has = open();
            wait(&pvdone[(g - 1) & 1], (uint32_t)((g - 1) >> 1) & 1u, 0x2a0u);
            if (threadIdx.x == 0) {   // the words of the segment after this one
                wild[(seg & 1) * 2] = 0;
                wild[(seg & 1) * 2 + 1] = 0;
            }
            // the sums of the replicas or of the two groups: a factor for the replica's, and the common m and l
            float f0 = 1.0f;
            if constexpr (GR == 2) {
                float *mine2 = hm[(g - 1) & 1][grp];   // the last tile's maxima have been read
                mine2[row] = l;
                named_sync(TC_EPI_BAR, 256);
                l = hm[(g - 1) & 1][0][row] + hm[(g - 1) & 1][1][row];
            } else if constexpr (REP > 1) {
                ml[tid] = make_float2(m, l);
                named_sync(TC_EPI_BAR, 128);
                const float m0 = m;
                l = 0.0f;
#pragma unroll
                for (int r = 0; r < REP; ++r) m = fmaxf(m, ml[r * RR + row].x);
                const float mz = m == -INFINITY ? 0.0f : m;
#pragma unroll
                for (int r = 0; r < REP; ++r) {
                    const float2 o = ml[r * RR + row];
                    l += ta_exp2(o.x - mz) * o.y;
                }
                f0 = ta_exp2(m0 - mz);
            }
            const volatile uint32_t *wv = wild + ((seg & 1) ^ 1) * 2;
            const unsigned long long wn = see & (wv[0] | (unsigned long long)wv[1] << 32);
            const bool whole = sg.whole;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const size_t slot = (size_t)(2 * blockIdx.x + (sg.head ? 0 : 1));
            T *dst = reinterpret_cast<T *>(A.out) + (long long)tok * A.o_t +
                     (long long)(sg.h * A.G + row - row_i * A.G) * A.o_h;
            // NV values of the row from column c: the parts go to the workspace in 32 bits, a whole item's to the output.
            float odd = 0.0f;   // the sum of what was written: NaN if any of it is (or infinities of both signs are)
            auto put = [&](auto &o, int c) {
                constexpr int NV = sizeof(o) / sizeof(float);
                float x[4] = {o[0], o[1], o[2], o[3]};
#pragma unroll
                for (int e = 4; e < NV; ++e) x[e & 3] += o[e];
                odd += (x[0] + x[1]) + (x[2] + x[3]);
                if (wn) {   // the values taken out above, for the rows that see them
                    for (unsigned long long left = wn; left; left &= left - 1) {
                        const int j = ctx + __ffsll((long long)left) - 1, page = j / A.bs;
                        if (j < kt0 * TK || j >= (kt0 + N) * TK || page >= A.width) continue;
                        const int blk = A.table[(long long)sg.b * A.table_stride + page];
                        if (blk < 0 || blk >= A.num_blocks) continue;
                        const T *v = reinterpret_cast<const T *>(A.v) + blk * A.v_b + (j - page * A.bs) * A.v_r +
                                     sg.h * A.v_h;
#pragma unroll
                        for (int e = 0; e < NV; ++e) {
                            if (c + e >= A.D) break;
                            const float f = t2f<T>(v[c + e]);
                            if (!isfinite(f)) o[e] += f;
                        }
                    }
                }
                if (!whole) {   // a warp's rows side by side
                    float4 *w = reinterpret_cast<float4 *>(A.parts) + (slot * (DP / 4) + c / 4) * TA_ROWS + row;
#pragma unroll
                    for (int e = 0; e < NV / 4; ++e)
                        w[e * TA_ROWS] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    return;
                }
                uint32_t w[NV / 2 < 12 ? 12 : NV / 2];
#pragma unroll
                for (int e = 0; e < NV / 2; ++e) w[e] = pack2<T>(o[2 * e] * inv, o[2 * e + 1] * inv);
#pragma unroll
                for (int e = 0; e < NV; e += 8) {
                    if (c + e >= A.D) break;
                    if constexpr (NV >= 16) {   // 32 bytes at a time where they fit
                        if (A.o_vec == 2 && (e & 8 || c + e + 8 < A.D)) {
                            if (e & 8) continue;
                            st_global32(dst + c + e, *reinterpret_cast<const uint32_t(*)[8]>(&w[e / 2]));
                            continue;
                        }
                    }
                    if (A.o_vec) {
                        *reinterpret_cast<uint4 *>(dst + c + e) =
                            make_uint4(w[e / 2], w[e / 2 + 1], w[e / 2 + 2], w[e / 2 + 3]);
                    } else {
                        uint16_t *d16 = reinterpret_cast<uint16_t *>(dst + c + e);
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            d16[2 * h] = (uint16_t)w[e / 2 + h];
                            d16[2 * h + 1] = (uint16_t)(w[e / 2 + h] >> 16);
                        }
                    }
                }
            };
            if constexpr (REP > 1) {
                // The replicas' sums through shared memory, `width` columns at a time; a thread then adds up the REP
                // replicas of width / REP of its row's. 32 columns fit the staging area; when the CTA has no further
                // item, the K and V rings are idle and hold them all. (One loop for both: this runs once per item, from
                // a cold instruction cache.)
                const int width = has ? 32 : DP, ld = width + 4;
                float *area = has ? stage : reinterpret_cast<float *>(kring);
#pragma unroll 1
                for (int c0 = 0; c0 < DP; c0 += width) {
#pragma unroll 1
                    for (int c = 0; c < width; c += 64) {
                        float o[64];
                        const bool two = c + 32 < width;
                        const uint32_t col = lane_base + (uint32_t)(c0 + c);
                        tmem_ld32(col, *reinterpret_cast<uint32_t(*)[32]>(o));
                        if (two) tmem_ld32(col + 32, *reinterpret_cast<uint32_t(*)[32]>(o + 32));
                        tmem_ld_wait();
                        float4 *y = reinterpret_cast<float4 *>(area + tid * ld + c);
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            if ((e == 8 && !two) || row >= live) break;   // only the item's rows
                            y[e] = f0 == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                              : make_float4(o[4 * e] * f0, o[4 * e + 1] * f0, o[4 * e + 2] * f0,
                                                            o[4 * e + 3] * f0);
                        }
                    }
                    named_sync(TC_EPI_BAR, 128);
                    if (mine && !dead) {
#pragma unroll 2
                        for (int c = part * (width / REP); c < (part + 1) * (width / REP); c += 8) {
                            float r[8] = {};
#pragma unroll
                            for (int k = 0; k < REP; ++k) {
                                const float4 *y = reinterpret_cast<const float4 *>(area + (k * RR + row) * ld + c);
                                const float4 a = y[0], b = y[1];
                                r[0] += a.x, r[1] += a.y, r[2] += a.z, r[3] += a.w;
                                r[4] += b.x, r[5] += b.y, r[6] += b.z, r[7] += b.w;
                            }
                            put(r, c0 + c);
                        }
                    }
                    if (has) named_sync(TC_EPI_BAR, 128);
                }
                if (!whole && mine && part == 0) A.stats[slot * TA_ROWS + row] = make_float2(m, l);
            } else if (warp_live) {
                constexpr int SHARE = DP / GR;   // a group's share of the columns
#pragma unroll 1
                for (int c = grp * SHARE; c < (grp + 1) * SHARE; c += 32) {
                    float o[32];
                    tmem_ld32(lane_base + (uint32_t)c, *reinterpret_cast<uint32_t(*)[32]>(o));
                    tmem_ld_wait();
                    if (mine && !dead) put(o, c);
                }
                if (!whole && mine && grp == 0) A.stats[slot * TA_ROWS + row] = make_float2(m, l);
            }
            if (__any_sync(0xffffffffu, odd != odd && l == l)) {   // (scores that are NaN make l, and the row, NaN)
                const int width = REP > 1 && has ? 32 : DP, k0 = kt0 * TK, k1 = (kt0 + N) * TK;
                float *at = A.parts + (slot * (DP / 4) * TA_ROWS + row) * 4;
                ta_fix_wild<T>(A, sg.b, sg.h, k0, min(ctx, k1), width, width / (REP * GR), part, ctx, k0, k1, wn,
                               mine && !dead && l == l, dst, whole ? nullptr : at);
            }
            if constexpr (REP > 1) {   // the staging area is the Q buffer again, which the next copy writes
                fence_proxy_async();
                __syncwarp();
                if (has && lane == 0) mbar_arrive(&qbempty[0]);
            }
            tc_fence_before();
        }
    }
    // all roles done: free TMEM after every TMEM access and MMA of the CTA has completed
    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// Joins the parts of the items that a range boundary cuts. Each block reads which CTAs start inside an item, as the
// first to do so (desc.split), and lists them; the blocks then share out the (item, 32 rows, 8 columns) tasks, a lane a
// row. A task is a warp's, or that of 2, 4 or 8 warps of a block, which share its contributors, where there are few
// tasks (one token over a long context is cut into many parts). A row's contributors are the CTAs c - 1 .. c1 in order;
// the warps' sums add up in warp order.
constexpr int TJ_THREADS = 256, TJ_WARPS = TJ_THREADS / 32, TJ_COLS = 8;

// Column col of row r of the item that CTA c's range starts inside of, when some of the row's are NaN: a value that is
// infinite or NaN in parts is the sum of those parts, whatever their weights (one that is 0 is so by underflow).
template <int DP> __device__ __noinline__ float tj_fix_wild(const TaArgs &A, int c, int r, int col, float joined) {
    const TaDesc d = A.desc[c];
    float sum = 0.0f;
    for (int j = 0; j < d.parts; ++j) {
        const size_t s = j == 0 ? d.first : 2 * (c - 1 + j);
        const float x = A.parts[((s * (DP / 4) + col / 4) * TA_ROWS + r) * 4 + col % 4];
        if (!isfinite(x)) sum += x;
    }
    return isfinite(sum) ? joined : sum;
}

template <typename T, int NCH>
__global__ void __launch_bounds__(TJ_THREADS) tree_join_kernel(const __grid_constant__ TaArgs A, int ctas) {
    constexpr int DP = NCH * 64, CBS = DP / TJ_COLS;
    __shared__ float acc_sm[TJ_WARPS][TJ_COLS][32];
    __shared__ float2 ml_sm[TJ_WARPS][32];
    __shared__ short list[TJ_THREADS];
    __shared__ int found[TJ_WARPS];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // up to TJ_THREADS cut items at a time (one pass, unless the GPU has more SMs than that)
    for (int base = 0; base < ctas; base += TJ_THREADS) {
        const bool cut = base + tid < ctas && A.desc[base + tid].split != 0;
        const unsigned bal = __ballot_sync(0xffffffffu, cut);
        if (lane == 0) found[warp] = __popc(bal);
        __syncthreads();
        int at = __popc(bal & ((1u << lane) - 1u)), items = 0;
        for (int w = 0; w < TJ_WARPS; ++w) {
            if (w < warp) at += found[w];
            items += found[w];
        }
        if (cut) list[at] = (short)tid;
        __syncthreads();
        const int rbs = (A.rows + 31) / 32, per = rbs * CBS, tasks = items * per;
        int wpr = TJ_WARPS;
        while (wpr > 1 && (long long)tasks * wpr > (long long)gridDim.x * TJ_WARPS) wpr >>= 1;
        const int groups = TJ_WARPS / wpr, grp = warp / wpr, wr = warp - grp * wpr;
        for (int w0 = blockIdx.x * groups; w0 < tasks; w0 += gridDim.x * groups) {
            const int task = w0 + grp, item = task / per, q = task - item * per, cb = q % CBS;
            const int r = q / CBS * 32 + lane;
            float acc[TJ_COLS], l = 0.0f, m = -INFINITY;
#pragma unroll
            for (int e = 0; e < TJ_COLS; ++e) acc[e] = 0.0f;
            T *dst = nullptr;
            if (task < tasks) {
                const int c = base + list[item];
                const TaDesc d = A.desc[c];
                const int i = r / A.G, tok = d.tok0 + i;
                if (i < d.tokens && tok >= 0 && tok < A.T)
                    dst = reinterpret_cast<T *>(A.out) + (long long)tok * A.o_t +
                          (long long)(d.h * A.G + r - i * A.G) * A.o_h + cb * TJ_COLS;
                if (dst) {
#pragma unroll 4
                    for (int j = wr; j < d.parts; j += wpr) {
                        const size_t s = j == 0 ? d.first : 2 * (c - 1 + j);
                        const float2 st = A.stats[s * TA_ROWS + r];
                        const float4 *p =
                            reinterpret_cast<const float4 *>(A.parts) + (s * (DP / 4) + cb * 2) * TA_ROWS + r;
                        const float4 a = p[0], b = p[TA_ROWS];
                        const float v[TJ_COLS] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                        const float mn = fmaxf(m, st.x), mz = mn == -INFINITY ? 0.0f : mn;
                        const float f = ta_exp2(m - mz), w = ta_exp2(st.x - mz);
                        m = mn;
                        l = l * f + w * st.y;
#pragma unroll
                        for (int e = 0; e < TJ_COLS; ++e)   // (a part that is all hidden from the row holds zeros)
                            acc[e] = __fmaf_rn(w, v[e], acc[e] * f);
                    }
                }
            }
            if (wpr > 1) {
                ml_sm[warp][lane] = make_float2(m, l);
#pragma unroll
                for (int e = 0; e < TJ_COLS; ++e) acc_sm[warp][e][lane] = acc[e];
                __syncthreads();
                if (wr == 0) {
                    for (int w = warp + 1; w < warp + wpr; ++w) {
                        const float2 st = ml_sm[w][lane];
                        const float mn = fmaxf(m, st.x), mz = mn == -INFINITY ? 0.0f : mn;
                        const float f = ta_exp2(m - mz), g = ta_exp2(st.x - mz);
                        m = mn;
                        l = l * f + g * st.y;
#pragma unroll
                        for (int e = 0; e < TJ_COLS; ++e) acc[e] = acc[e] * f + g * acc_sm[w][e][lane];
                    }
                }
                __syncthreads();
            }
            if (!dst || wr > 0) continue;
            const float odd = ((acc[0] + acc[1]) + (acc[2] + acc[3])) + ((acc[4] + acc[5]) + (acc[6] + acc[7]));
            if (odd != odd && l == l) {
#pragma unroll
                for (int e = 0; e < TJ_COLS; ++e)
                    acc[e] = tj_fix_wild<DP>(A, base + list[item], r, cb * TJ_COLS + e, acc[e]);
            }
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            uint32_t w[TJ_COLS / 2];
#pragma unroll
            for (int e = 0; e < TJ_COLS / 2; ++e) w[e] = pack2<T>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
            if (cb * TJ_COLS >= A.D) continue;
            if (A.o_vec) {
                *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
                uint16_t *d16 = reinterpret_cast<uint16_t *>(dst);
#pragma unroll
                for (int e = 0; e < TJ_COLS / 2; ++e) {
                    d16[2 * e] = (uint16_t)w[e];
                    d16[2 * e + 1] = (uint16_t)(w[e] >> 16);
                }
            }
        }
        __syncthreads();
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
// The cache as TMA sees it, any strides (elements, multiples of 8); what lies outside reads as 0.
// Plain: [num_blocks][heads][rows][D], a box is 64 values of box_rows rows, so a tile of D values takes D / 64 boxes a
// page. Folded (D % 64 == 0, head stride % 64 == 0): [num_blocks][rows / 8][head and chunk][8 rows][64 values]; a box is
// all chunks of box_rows rows, in the order [rows / 8][chunk][8][64] that the MMA's strides describe as well. A box
// takes about 60 cycles to issue, so for 16-row pages the plain form bounds the stream (D = 256: 16 boxes of 2 KB for
// 32 KB, 3.8 TB/s against 5.3 TB/s with one box).
static bool ta_map(CUtensorMap *m, const void *base, int D, int bs, int Hkv, int nb, long long sr, long long sh,
                   long long sb, int box_rows, bool fold) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint32_t nch = (cuuint32_t)(D / 64), br = (cuuint32_t)box_rows;
    cuuint64_t dims[5] = {(cuuint64_t)D, (cuuint64_t)bs, (cuuint64_t)Hkv, (cuuint64_t)nb, 0};
    cuuint64_t strides[4] = {(cuuint64_t)sr * 2, (cuuint64_t)sh * 2, (cuuint64_t)sb * 2, 0};
    cuuint32_t box[5] = {64, br, 1, 1, 1}, estr[5] = {1, 1, 1, 1, 1};
    if (fold) {
        const cuuint64_t d5[5] = {64, 8, (cuuint64_t)(Hkv - 1) * (cuuint64_t)(sh / 64) + nch, (cuuint64_t)bs / 8,
                                  (cuuint64_t)nb};
        const cuuint64_t s5[4] = {(cuuint64_t)sr * 2, 128, (cuuint64_t)sr * 16, (cuuint64_t)sb * 2};
        const cuuint32_t b5[5] = {64, 8, nch, br / 8, 1};
        for (int i = 0; i < 5; ++i) dims[i] = d5[i], box[i] = b5[i];
        for (int i = 0; i < 4; ++i) strides[i] = s5[i];
    }
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, fold ? 5 : 4, const_cast<void *>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// q [T][Hq][D]; a box is 64 values of the G heads of one cached head, for an item's tokens.
static bool ta_q_map(CUtensorMap *m, const void *base, int D, int Hq, int T, long long sh, long long st, int G,
                     int tokens) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)Hq, (cuuint64_t)T};
    cuuint64_t strides[2] = {(cuuint64_t)sh * 2, (cuuint64_t)st * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)tokens}, estr[3] = {1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int ta_tile_tokens(int G) { return TA_ROWS / G; }
static int ta_rows(int max_new, int G) { return (max_new < ta_tile_tokens(G) ? max_new : ta_tile_tokens(G)) * G; }
static size_t ta_desc_bytes(int grid) { return ((size_t)grid * sizeof(TaDesc) + 255) & ~(size_t)255; }
static size_t ta_stats_bytes(int grid) { return (size_t)2 * grid * TA_ROWS * sizeof(float2); }

template <typename T, int NCH, int REP>
static int launch_ta(const CUtensorMap &mk, const CUtensorMap &mv, const CUtensorMap &mq, TaArgs A, cudaStream_t s) {
    using Lay = TaLayout<NCH, REP>;
    const int dev = cur_device();
    if (dev < 0 || dev >= VT_MAX_DEV) return VT_EARG;
    const int fixed = Lay::BARS + Lay::Q_BYTES;
    int slots = (max_smem_optin(dev) - fixed) / Lay::SLOT;
    if (slots > MAX_SLOTS) slots = MAX_SLOTS;
    if (slots < 4 || (REP > 1 && slots * Lay::SLOT < TA_ROWS * (Lay::DP + 4) * 4)) return VT_EARG;
    A.k_slots = (slots + 1) / 2;
    A.v_slots = slots / 2;
    A.cs = A.fold ? 1024 : Lay::TK * 128;
    A.gs = A.fold ? NCH * 1024 : 1024;
    const int smem = fixed + slots * Lay::SLOT;
    static std::atomic<bool> attr[VT_MAX_DEV];
    if (!attr[dev]) {
        if (cudaFuncSetAttribute(tree_attn_kernel<T, NCH, REP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
            cudaSuccess)
            return (int)cudaGetLastError();
        attr[dev] = true;
    }
    const int grid = num_sms(dev);
    if (int rc = launch_k(tree_attn_kernel<T, NCH, REP>, dim3(grid), dim3(Lay::THREADS), smem, s, true, mk, mv, mq, A))
        return rc;
    if (grid < 2) return 0;
    return launch_k(tree_join_kernel<T, NCH>, dim3(4 * grid), dim3(TJ_THREADS), 0, s, true, A, grid);
}

template <typename T, int NCH>
static int dispatch_rep(const CUtensorMap &mk, const CUtensorMap &mv, const CUtensorMap &mq, const TaArgs &A,
                        cudaStream_t s) {
    const int rows = A.max_new * A.G;
    if (rows <= 32) return launch_ta<T, NCH, 4>(mk, mv, mq, A, s);
    if (rows <= 64) return launch_ta<T, NCH, 2>(mk, mv, mq, A, s);
    return launch_ta<T, NCH, 1>(mk, mv, mq, A, s);
}

template <typename T>
static int dispatch_ta(const CUtensorMap &mk, const CUtensorMap &mv, const CUtensorMap &mq, const TaArgs &A,
                       cudaStream_t s) {
    if (A.D <= 64) return dispatch_rep<T, 1>(mk, mv, mq, A, s);
    if (A.D <= 128) return dispatch_rep<T, 2>(mk, mv, mq, A, s);
    if (A.D <= 192) return dispatch_rep<T, 3>(mk, mv, mq, A, s);
    return dispatch_rep<T, 4>(mk, mv, mq, A, s);
}

}  // namespace vt

using namespace vt;

extern "C" {

size_t vt_tree_attention_ws_bytes(int max_new, int Hq, int Hkv, int D) {
    if (max_new < 1 || max_new > TA_MAX_NEW || Hkv < 1 || Hq < Hkv || Hq / Hkv > TA_ROWS || D < 1 || D > 256) return 0;
    const int grid = num_sms(cur_device()), dp = (D + 63) / 64 * 64;
    return ta_desc_bytes(grid) + ta_stats_bytes(grid) + (size_t)2 * grid * TA_ROWS * dp * sizeof(float);
}

int vt_tree_attention(const void *q, const void *k_cache, const void *v_cache, void *out, const long long *strides,
                      const void *block_table, long long table_stride, int table_width, const void *cu,
                      const void *seq_lens, const void *mask, int B, int T, int max_new, int Hq, int Hkv, int D,
                      long long num_blocks, int block_size, float scale, int dtype, void *workspace, size_t ws_bytes,
                      void *stream) {
    if (!q || !k_cache || !v_cache || !out || !strides || !block_table || !cu || !seq_lens || B < 1 || T < 0 ||
        max_new < 1 || max_new > TA_MAX_NEW || Hkv < 1 || Hq < Hkv || Hq % Hkv || Hq / Hkv > TA_ROWS || D < 8 ||
        D > 256 || D % 8 || block_size < 8 || block_size % 8 || table_width < 1 || num_blocks < 1 || num_blocks > 0x7ffffffe ||
        (dtype != 0 && dtype != 1) || !workspace || ((uintptr_t)workspace & 255) ||
        ws_bytes < vt_tree_attention_ws_bytes(max_new, Hq, Hkv, D) || ((uintptr_t)k_cache & 15) ||
        ((uintptr_t)v_cache & 15) || !(scale == scale))
        return VT_EARG;
    for (int i = 4; i < 10; ++i)
        if (strides[i] < 0 || strides[i] % 8) return VT_EARG;
    if (T == 0) return 0;
    cudaStream_t s = (cudaStream_t)stream;
    void *scratch;
    TaArgs A{};
    if (int rc = ws_acquire(0, s, &scratch, &A.status)) return rc;
    int box = 8;   // the largest power of two of rows that divides the block, at most a tile
    const int tk = D <= 128 ? 128 : 64;
    while (box * 2 <= tk && block_size % (box * 2) == 0) box *= 2;
    CUtensorMap mk, mv, mq;
    const bool fold = D % 64 == 0 && strides[6] % 64 == 0 && strides[9] == strides[6];
    if (!ta_map(&mk, k_cache, D, block_size, Hkv, (int)num_blocks, strides[5], strides[6], strides[4], box, fold) ||
        !ta_map(&mv, v_cache, D, block_size, Hkv, (int)num_blocks, strides[8], strides[9], strides[7], box, fold))
        return VT_EARG;
    A.fold = fold;
    A.head_step = (int)(strides[6] / 64);
    A.q = q;
    A.v = v_cache;
    A.out = out;
    A.q_t = strides[0];
    A.q_h = strides[1];
    A.o_t = strides[2];
    A.o_h = strides[3];
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
    A.Hkv = Hkv;
    A.G = Hq / Hkv;
    A.tile_tokens = ta_tile_tokens(A.G);
    A.D = D;
    A.bs = block_size;
    A.num_blocks = (int)num_blocks;
    A.box_rows = box;
    A.q_map = ((uintptr_t)q & 15) == 0 && ((A.q_t | A.q_h) & 7) == 0 && A.q_t >= 0 && A.q_h >= 0 &&
              ta_q_map(&mq, q, D, Hq, T, A.q_h, A.q_t, A.G, max_new < A.tile_tokens ? max_new : A.tile_tokens);
    A.o_vec = ((uintptr_t)out & 15) == 0 && ((A.o_t | A.o_h) & 7) == 0;
    if (A.o_vec && ((uintptr_t)out & 31) == 0 && ((A.o_t | A.o_h) & 15) == 0) A.o_vec = 2;
    A.negate = scale < 0.0f;
    A.sl2 = fmaxf(fabsf(scale) * 1.4426950408889634f, 1.2e-38f);   // above 0: a hidden key's -inf stays -inf
    A.rows = ta_rows(max_new, A.G);
    A.timeout_ns = pipe_timeout_ns();
    const int grid = num_sms(cur_device());
    char *ws = (char *)workspace;
    A.desc = (TaDesc *)ws;
    A.stats = (float2 *)(ws + ta_desc_bytes(grid));
    A.parts = (float *)(ws + ta_desc_bytes(grid) + ta_stats_bytes(grid));
    if (dtype == 0) return dispatch_ta<__half>(mk, mv, mq, A, s);
    return dispatch_ta<__nv_bfloat16>(mk, mv, mq, A, s);
}

}  // extern "C"

// s2d_cache_tc.cu -- attention of many query rows over paged keys and values
// on tcgen05 (sm_100a): the pooled rows of a batch against the shared prefix,
// and the rows of prompts against prefix and own pages.
//
// A CTA takes items of 256 query rows of one KV head as two tiles of 128 (the
// M of every MMA) and walks the positions of an item in tiles of 128:
//   S = Q K^T        both operands in shared memory, S in TMEM
//   P = 2^(s - m)    one thread per row, S read from TMEM, P written over it
//   O += P V         P from TMEM, V from shared memory (MN-major), O in TMEM
// The two row tiles alternate: while one is in its softmax, the tensor core
// runs the products of the other.  An item of one row tile is walked by both
// warpgroups in the same way, tile by tile in turn; or by one of them, the next
// such item by the other, where it is short or the ring holds no more than
// three tiles (f32 heads of 128).  One CTA per SM draws items from a counter,
// the longest first; one item's first loads run under the last one's epilogue.
//
// What bounds it: bf16 prompts of 500 to 2,048 tokens behind 2,000 positions (32
// and 8 heads of 128) take 255 us, 860 TFLOP/s; the products alone take 200,
// the softmax alone 219 (without its exponentials 177: TMEM reads, the
// hand-overs, the items' starts and ends), so the two row tiles overlap most
// of the smaller one.  S in halves of 64 positions, one under the other's
// softmax, is slower (259): the products alone then take 227.  f32 prompts of
// 33 to 400 tokens behind 727: 167 us, 290 TFLOP/s of the formula's and 580 of
// f16 products.  Short items pay 7 us to start and end.
//
// 16-bit queries: Q as it is, P rounded once to the cache's type (its relative
// error, half a step of that type, is that of the output's own rounding).
//
// f32 queries: Q and P enter as f16 pairs hi + lo (two MMAs into one
// accumulator, about 22 bits).
//
// Every MMA step of 16 positions truncates its sum to f32, always toward zero:
// up to 1.0e-7 of the result a step (equal weights, values of one sign).  So O
// is moved and added up with rounding every kFlush tiles: of f32 rows every two
// tiles, into registers (1.5e-6 at any length); of 16-bit rows, which have no
// registers left, every kTcHold = 64 into device memory that the CTA keeps to
// itself (p.held, which stays in L2): 5e-5 at any length, a ninth of half an f16
// step, where 131,072 positions without it came out 8.4e-4 too small and 2^20
// 6.7e-3.
//
// m is not the running maximum itself but a reference that follows it: it is
// set kBelow below the first tile's maximum and moves (and what is summed so far
// is rescaled) only when a tile's maximum is more than kAbove above it.  For f16
// these are 9 and 15: P stays below 2^15, and half of f16's smallest step is
// 2^-34 of the largest weight, so that what is rounded away stays below 2e-5
// over 2^18 positions (set 6 below, 2^-31: as many positions 31 binades below one
// of them were lost, 1.1e-4 of the result).  bf16 has f32's exponents, and 6 and
// 14 move the reference less often.
//
// Warps: 0-3 and 4-7 softmax and epilogue of row tiles 0 and 1 (warp w owns
// TMEM lanes 32 (w % 4) ..), 8 loads K and V pages by TMA (one page of 64
// positions x 64 columns a box, 128-byte swizzle) into a ring of tiles,
// 9 issues the MMAs (10 and 11 only give up registers).  Every wait is bounded;
// one that gives up sets the status word's S2D_CACHE_ABORTED, and the CTA
// leaves with its TMEM freed.
#include <cuda.h>

#include "s2d_cache_attn.cuh"
#include "s2d_tc_common.cuh"

#include <algorithm>
#include <type_traits>

namespace s2d {

namespace {

constexpr int kTcThreads = 384;
// Tiles of positions up to which one warpgroup takes an item of one row tile
// alone.  128 sequences of 16 bf16 tokens, 32 and 8 heads: over 16 positions 67
// us, shared by both 82; over 350 97 and 101; over 850 140 (8) and 137.
constexpr int kTcAlone = 5;
constexpr int kTcSorted = 64;  // sequences whose row tiles are ordered
constexpr int kTcRows = 128;
constexpr int kTcItemRows = 2 * kTcRows;
constexpr int kTcColumns = 512;

// Byte offset of 16-byte chunk c of row r in a 128-byte-swizzled region.
__device__ __forceinline__ uint32_t swizzle(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

__device__ __forceinline__ void tma_page(void *dst, const CUtensorMap *map, int x, int g, int page, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            su32(dst)),
        "l"(map), "r"(x), "r"(0), "r"(g), "r"(page), "r"(su32(bar))
        : "memory");
}
// D (+)= A B, A and B in shared memory, by the thread whose `one` is set.  The
// whole warp runs the instruction under a predicate, not under a branch: its
// operands live in uniform registers, which a branch on the elected thread
// makes the compiler rebuild for every MMA (80 cycles each to issue).
__device__ __forceinline__ void umma_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one));
}
// the same with A in TMEM (lane = row, two 16-bit elements per column)
__device__ __forceinline__ void umma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one));
}
__device__ __forceinline__ void commit_one(uint32_t one, uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(su32(bar)),
        "r"(one)
        : "memory");
}
#define S2D_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define S2D_I8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void lds16(uint32_t addr, float (&x)[4]) {
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void sts16(uint32_t addr, const uint32_t (&x)[4]) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
}
// One thread of the warp, the same one each time.
__device__ __forceinline__ uint32_t elect() {
    uint32_t yes;
    asm volatile("{ .reg .pred q; elect.sync _|q, 0xffffffff; selp.u32 %0, 1, 0, q; }" : "=r"(yes));
    return yes;
}
// A bounded wait of a whole warp; gives up early once *abort is set.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t par, const volatile int *abort) {
    for (uint32_t i = 0; !__all_sync(0xffffffffu, mb_try(bar, par)); ++i)
        if (i >= kTcSpin || ((i & 255u) == 255u && *abort)) return false;
    return true;
}
// 32 columns of this thread's lane; the values are there after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : S2D_R8(r, 0), S2D_R8(r, 8), S2D_R8(r, 16), S2D_R8(r, 24)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : S2D_R8(r, 0), S2D_R8(r, 8)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::S2D_I8(r, 0),
        S2D_I8(r, 8), S2D_I8(r, 16), S2D_I8(r, 24), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::S2D_I8(r, 0), "r"(addr) : "memory");
}
// 2^x on the special-function unit; results below 2^-126 are 0.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two f32 sums or products in one instruction.
__device__ __forceinline__ uint64_t two(float x, float y) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ float2 untwo(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// The maximum of N scores (NaN left out) in four chains.
template <int N>
__device__ __forceinline__ float max_of(const uint32_t (&s)[N]) {
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < N; i += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k) m[k] = max3(m[k], __uint_as_float(s[i + 2 * k]), __uint_as_float(s[i + 2 * k + 1]));
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
// Scores of columns [0, N) that the row does not see: -inf.
template <int N>
__device__ __forceinline__ void mask(uint32_t (&s)[N], int vis) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = i < vis ? s[i] : 0xff800000u;
}

template <typename Q, int HD>
struct TcShape {
    static constexpr bool kF32 = sizeof(Q) == 4;
    static constexpr int BN = kTcTilePositions;            // positions per tile
    static constexpr int kPages = BN / kCachePage;         // pages per tile
    static constexpr int kHalves = HD / 64;                // 128-byte column blocks of a row
    static constexpr int kSplit = kF32 ? 2 : 1;            // hi and lo
    static constexpr int kQHalf = kTcRows * 128;           // one column block of one row tile
    static constexpr int kQTile = kHalves * kSplit * kQHalf;
    static constexpr int kKvHalf = BN * 128;               // one column block of a K or V tile
    static constexpr int kSlot = kHalves * kKvHalf;        // a K or a V tile
    static constexpr int kFit = (224 * 1024 - 2 * kQTile) / kSlot;
    static constexpr int kSlots = kFit < 8 ? kFit : 8;     // K and V tiles in flight
    static constexpr int kSmem = 2 * kQTile + kSlots * kSlot + 1024;
    static constexpr int kFlush = kF32 ? 2 : kTcHold;      // tiles that O takes before it moves, f32: to registers, else to p.held
    static constexpr uint32_t kO = 2 * BN;                 // TMEM: S0, S1 (BN columns each), O0, O1 (HD each)
    static_assert(kO + 2 * HD <= kTcColumns, "TMEM columns");
    static_assert(kSlots >= 3, "K and V of a tile and the next K");
};

// What is put aside of O of a 16-bit row (see the top): by the row's thread, 16
// columns at a time, in functions of their own between two tiles, where no score
// is held in registers: inline, or in the midst of a tile, long prompts take 1 %
// more.
//
// held = by * held + O, or O alone
template <int HD>
__device__ __noinline__ void hold(uint32_t ot, float4 *held, bool more, float by) {
#pragma unroll 1
    for (int i = 0; i < HD; i += 16) {
        uint32_t o[16];
        tmem_ld16(ot + i, o);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const float4 x = more ? held[(i + e) / 4 * kTcRows] : make_float4(0.f, 0.f, 0.f, 0.f);
            held[(i + e) / 4 * kTcRows] = make_float4(fmaf(x.x, by, __uint_as_float(o[e])), fmaf(x.y, by, __uint_as_float(o[e + 1])),
                                                      fmaf(x.z, by, __uint_as_float(o[e + 2])), fmaf(x.w, by, __uint_as_float(o[e + 3])));
        }
    }
}
// O += by * held
template <int HD>
__device__ __noinline__ void hold_back(uint32_t ot, const float4 *held, float by) {
#pragma unroll 1
    for (int i = 0; i < HD; i += 16) {
        uint32_t o[16];
        tmem_ld16(ot + i, o);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
            const float4 x = held[(i + e) / 4 * kTcRows], y = held[((i + e) / 4 + 1) * kTcRows];
            const float add[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = __float_as_uint(fmaf(add[k], by, __uint_as_float(o[e + k])));
            tmem_st8(ot + i + e, w);
        }
    }
    tmem_wait_st();
}

// Where an item lies.
struct TcPlace {
    int some;       // 0: no further item
    int pooled, g, split, tile, b;  // own items: row tile `tile` of sequence b
    int half;                       // 0 or 1: that half of the row tile's rows; -1: all
};

struct TcShared {
    uint64_t full[8], empty[8], s_full[2], p_half[2][2], pv_done[2], q_full[2], item_full[2], item_empty[2], pair_full, pair_free;
    TcPlace item[2];
    float2 ml[kTcRows];  // the second warpgroup's (m, l), where both take one row tile
    uint32_t tmem;
    int abort;
};

// The k-th own row tile when all sequences' tiles are ordered by the own slots
// they see, in steps of 128, the most first: CTAs that draw in this order end
// nearly together.
// A tile's slots follow from its sequence's length, so the step of the k-th is
// found by bisection over the count of tiles that see as much.  By one warp.
// Without an order the k-th is the k-th by sequence, looked for from b0 on,
// before which there are `past` of them; a later call has a larger k.
// k < 0: the number of own row tiles.
struct TcCursor {
    int b0, past;
};
__device__ __noinline__ int find_own_tile(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p, int k, int &b, TcCursor &from) {
    const int lane = threadIdx.x & 31;
    // tiles of sequence i that see at least x steps; they are its last ones
    auto count = [&](int i, int x, int &tiles) {
        int first;
        const int nt = cache_tokens(a.q_start, a.tokens, i, first, c.status);
        tiles = (nt * p.rep + kTcItemRows - 1) / kTcItemRows;
        const int64_t need = (int64_t)(x - 1) * 128 - (cache_length(c, i) - nt);  // first token that sees so much
        return x <= 0 || need <= 0 ? tiles : need >= nt ? 0 : tiles - (int)(need * p.rep / kTcItemRows);
    };
    auto total = [&](int x) {
        int sum = 0, tiles;
        for (int i = lane; i < c.n_seq; i += 32) sum += count(i, x, tiles);
        return __reduce_add_sync(0xffffffffu, sum);
    };
    if (k < 0) return total(0);
    // Items of split positions are short: any order will do, and the bisection
    // costs more than it saves (8 sequences, 122.4 us with it, 120.5 without).
    // So it does with many sequences, which need no order for an even end: 32 of
    // 400 tokens 171 us with it, 178 without; 128 of 16 142 and 121; 1,024 of 2
    // 2,860 and 648.
    const bool sorted = p.own_splits == 1 && c.n_seq <= kTcSorted;
    int lo = 0, hi = sorted ? c.max_pages * kCachePage / 128 + 1 : 0;  // total(lo) > k (it is for 0); total(hi + 1) = 0
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (total(mid) > k) lo = mid;
        else hi = mid - 1;
    }
    const int above = sorted ? lo + 1 : INT32_MAX;  // among those that see exactly lo steps (unsorted: all), by sequence
    if (sorted) k -= total(above), from = {};
    else k -= from.past;
    for (int b0 = from.b0; b0 < c.n_seq; b0 += 32) {
        int tiles = 0, more = 0, n = 0;
        if (b0 + lane < c.n_seq) more = count(b0 + lane, above, tiles), n = count(b0 + lane, lo, tiles) - more;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, sum > k);
        if (past) {
            const int l = __ffs(past) - 1;
            b = b0 + l;
            from.b0 = b0;
            return __shfl_sync(0xffffffffu, tiles - more - 1, l) - (k - __shfl_sync(0xffffffffu, sum - n, l));
        }
        const int tiles32 = __shfl_sync(0xffffffffu, sum, 31);
        k -= tiles32, from.past += tiles32;
    }
    return 0;
}

// What an item is: its rows, its positions, where its results go.
template <int BN, bool DUAL>
struct TcItem {
    int g, split, b, first, rows, r0, back;  // back: own slots before the sequence's first token
    int pre0, pre1, own0, own1;              // prefix positions and own slots of the item
    int jp, tiles, J[2];                     // prefix tiles; all tiles; those of each warpgroup
    // one row tile only: both warpgroups take it, with the even and the odd
    // tiles, or one alone (`by`), in turn, under the end of the other's item
    bool pooled, dual, solo;
    int by;

    // own slots that rows [0, n) of the item see together
    __device__ __forceinline__ int seen(int n, int rep) const { return pooled ? 0 : max(0, back + (r0 + n - 1) / rep + 1); }
    // positions of tile j that exist
    __device__ __forceinline__ int valid(int j) const { return j < jp ? pre1 - pre0 - j * BN : own1 - own0 - (j - jp) * BN; }

    // The fields of the MMA warp's loops, known to be alike in all lanes.
    __device__ __forceinline__ void uniform() {
        auto u = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
        pre0 = u(pre0), pre1 = u(pre1), own0 = u(own0), own1 = u(own1), jp = u(jp), tiles = u(tiles), dual = DUAL && u(dual), solo = u(solo), by = u(by), J[0] = u(J[0]), J[1] = u(J[1]);
    }

    // The CTA's n-th item.  false: nothing to do.
    __device__ bool get(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p, const TcPlace &at, int n) {
        pooled = at.pooled, g = at.g, split = at.split, b = at.b;
        const int tile = at.tile, splits = pooled ? p.prefix_splits : p.own_splits;
        first = back = pre0 = pre1 = own0 = own1 = 0;
        if (pooled) {
            rows = real_tokens(a, c.n_seq) * p.rep - tile * kTcItemRows;
            const int tiles = (a.prefix_len + BN - 1) / BN, per = (tiles + splits - 1) / splits;
            pre0 = min(a.prefix_len, split * per * BN), pre1 = min(a.prefix_len, pre0 + per * BN);
        } else {
            const int nt = cache_tokens(a.q_start, a.tokens, b, first, c.status);
            back = cache_length(c, b) - nt;
            rows = nt * p.rep - tile * kTcItemRows;
            if (p.fused) pre1 = a.prefix_len;
        }
        r0 = tile * kTcItemRows + max(0, at.half) * kTcRows, rows -= max(0, at.half) * kTcRows;
        if (rows <= 0) return false;
        rows = min(rows, at.half >= 0 ? kTcRows : kTcItemRows);
        if (!pooled) {
            const int span = seen(rows, p.rep), tiles = (span + BN - 1) / BN, per = (tiles + splits - 1) / splits;
            own0 = min(span, split * per * BN), own1 = min(span, own0 + per * BN);
        }
        jp = (pre1 - pre0 + BN - 1) / BN;
        tiles = jp + (own1 - own0 + BN - 1) / BN;
        const bool one = rows <= kTcRows;
        dual = DUAL && one && tiles > kTcAlone, solo = one && !dual, by = n & 1;
        J[0] = dual ? (tiles + 1) / 2 : solo ? (by == 0 ? tiles : 0) : jp + max(0, (min(seen(kTcRows, p.rep), own1) - own0 + BN - 1) / BN);
        J[1] = dual ? tiles / 2 : solo ? (by == 1 ? tiles : 0) : tiles;
        return true;
    }
};

template <typename Q, typename E, int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
    rows_tc_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const S2dCacheView c,
                   const S2dCacheAttention a, const AttnPlan p) {
    using Sh = TcShape<Q, HD>;
    constexpr int BN = Sh::BN;
    extern __shared__ uint8_t raw[];
    __shared__ TcShared sh;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sbase = su32(smem);
    // through a shuffle, so that the compiler knows it alike in all lanes: what
    // the MMA warp computes from such values stays in uniform registers, where
    // the MMAs take their operands (80 cycles an MMA to issue otherwise)
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    volatile int *abort_v = &sh.abort;

    grid_dep_launch();  // every CTA is resident: what follows may use what they leave of the GPU
    if (threadIdx.x == 0) {
        for (int i = 0; i < Sh::kSlots; ++i) mb_init(&sh.full[i], 1), mb_init(&sh.empty[i], 1);
        for (int i = 0; i < 2; ++i) mb_init(&sh.s_full[i], 1), mb_init(&sh.p_half[i][0], 4), mb_init(&sh.p_half[i][1], 4), mb_init(&sh.pv_done[i], 1), mb_init(&sh.q_full[i], 4),
            mb_init(&sh.item_full[i], 1), mb_init(&sh.item_empty[i], 9);
        mb_init(&sh.pair_full, 4), mb_init(&sh.pair_free, 4);
        sh.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&sh.tmem)),
                     "r"(kTcColumns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // all 512 columns are this CTA's: its TMEM starts at 0, which the MMAs'
    // addresses then need not be told at run time
    constexpr uint32_t tmem = 0;
    if (sh.tmem != 0) {
        if (threadIdx.x == 0) cache_flag(c.status, S2D_CACHE_ABORTED);
        if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem), "r"(kTcColumns));
        return;
    }
    TcItem<BN, (Sh::kSlots >= 5)> it;

    // The CTA's n-th item, which the loader draws and places, through a ring of
    // two; false at the end.  For the MMA and softmax warps.
    auto take = [&](int n, TcPlace &at, bool &ok) {
        const int s = n & 1;
        if (!(ok = warp_wait(&sh.item_full[s], (n >> 1) & 1, abort_v))) return false;
        at = sh.item[s];
        __syncwarp();
        if (lane == 0) mb_arrive(&sh.item_empty[s]);
        return at.some != 0;
    };
    // Registers: 168 a thread at launch (three warps on a scheduler); warps
    // 8-11 give theirs to the softmax warps: 2 x 216 + 72 = 3 x 168.
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 8) {
            // ---- loader: K then V of every tile of every item ----
            int issued = 0;
            bool ok = true;
            const int G = c.kv_heads, prefix_items = p.prefix_tiles * p.prefix_splits * G;
            TcPlace next = {};
            TcCursor cursor = {};
            // Own items of whole row tiles, and behind them the last few, where
            // they are at most half a round of the CTAs, as halves: 616 items on
            // 148 SMs would else end with 24 SMs at work on a fifth.  Not more
            // of them: a half reads as many keys and values.
            const int tiles = p.own_tiles ? find_own_tile(c, a, p, -1, next.b, cursor) * p.own_splits * G : 0;
            const int odd = tiles % (int)gridDim.x, whole = Sh::kSlots >= 5 && odd <= (int)gridDim.x / 2 ? tiles - odd : tiles;
            const int items = prefix_items + whole + 2 * (tiles - whole);
            // places item `item` in `next` and hands it to the others as the n-th
            auto put = [&](int n, int item) {
                next.some = item < items;
                if (next.some) {
                    next.pooled = item < prefix_items;
                    if (!next.pooled) item -= prefix_items;
                    next.half = next.pooled || item < whole ? -1 : (item - whole) & 1;
                    if (next.half >= 0) item = whole + (item - whole) / 2;
                    next.g = item % G, item /= G;
                    const int splits = next.pooled ? p.prefix_splits : p.own_splits;
                    next.split = item % splits, next.tile = item / splits;
                    if (!next.pooled) next.tile = find_own_tile(c, a, p, next.tile, next.b, cursor);
                }
                const int s = n & 1, use = n >> 1;
                if (use > 0 && !warp_wait(&sh.item_empty[s], (use - 1) & 1, abort_v)) return false;
                if (lane == 0) {
                    sh.item[s] = next;
                    mb_arrive(&sh.item_full[s]);
                }
                __syncwarp();
                return true;
            };
            ok = put(0, (int)blockIdx.x);
            for (int n = 0; ok && next.some; ++n) {
                const TcPlace at = next;
                // the next item is drawn here, and placed once this one's loads are issued
                int item = items;
                if (p.next_item && lane == 0) item = (int)gridDim.x + atomicAdd(p.next_item, 1);
                const bool real = it.get(c, a, p, at, n);
                const int32_t *own_table = c.page_table + (int64_t)it.b * c.table_stride;  // pooled: unused
                int ids = 0, have = -1;  // page ids 32 * have + lane of the current segment
                for (int j = 0; real && j < it.tiles && ok; ++j) {
                    const bool own = j >= it.jp;
                    if (j == it.jp) have = -1;
                    const int32_t *table = own ? own_table : a.prefix_pages;
                    const int page0 = own ? it.own0 / kCachePage + (j - it.jp) * Sh::kPages : it.pre0 / kCachePage + j * Sh::kPages;
                    const int n_pages = min(Sh::kPages, (it.valid(j) + kCachePage - 1) / kCachePage);
                    const int last = ((own ? it.own1 : it.pre1) - 1) / kCachePage;  // last page of the segment
                    int page[Sh::kPages];
    #pragma unroll
                    for (int i = 0; i < Sh::kPages; ++i) {
                        const int at = min(page0 + i, last);
                        if (at / 32 != have) {
                            have = at / 32;
                            ids = __ldg(table + min(have * 32 + lane, last));
                            if ((uint32_t)ids >= (uint32_t)c.n_pages) {
                                cache_flag(c.status, S2D_CACHE_BAD_PAGE);
                                ids = 0;
                            }
                        }
                        page[i] = __shfl_sync(0xffffffffu, ids, at & 31);
                    }
    #pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        const int s = issued % Sh::kSlots, use = issued / Sh::kSlots;
                        if (use > 0 && !warp_wait(&sh.empty[s], (use & 1) ^ 1, abort_v)) {
                            ok = false;
                            break;
                        }
                        if (lane == 0) {
                            uint8_t *slot = smem + 2 * Sh::kQTile + s * Sh::kSlot;
                            mb_expect_tx(&sh.full[s], (uint32_t)(n_pages * Sh::kHalves * kCachePage * 128));
    #pragma unroll
                            for (int i = 0; i < Sh::kPages; ++i)
                                if (i < n_pages)
    #pragma unroll
                                    for (int h = 0; h < Sh::kHalves; ++h)
                                        tma_page(slot + h * Sh::kKvHalf + i * kCachePage * 128, kv ? &mv : &mk, 64 * h, it.g, page[i], &sh.full[s]);
                        }
                        __syncwarp();
                        ++issued;
                    }
                }
                if (ok) ok = put(n + 1, __shfl_sync(0xffffffffu, item, 0));
            }
            if (!ok) *abort_v = 1;
            // neither a copy nor the arrival that frees its slot may still be landing when the CTA leaves
            for (int i = max(0, issued - Sh::kSlots); i < issued; ++i) {
                (void)mb_wait(&sh.full[i % Sh::kSlots], (i / Sh::kSlots) & 1, abort_v, false);
                (void)mb_wait(&sh.empty[i % Sh::kSlots], (i / Sh::kSlots) & 1, abort_v);
            }
        } else if (warp == 9) {
            // ---- MMA issuer ----
            constexpr uint32_t type = std::is_same<E, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
            constexpr uint32_t id_s = idesc_f16_f32(kTcRows, BN) | type, id_o = idesc_f16_f32_bmn(kTcRows, HD) | type;
            auto wait = [&](uint64_t *bar, uint32_t par) { return warp_wait(bar, par, abort_v); };
            auto slot_wait = [&](int i) { return wait(&sh.full[i % Sh::kSlots], (uint32_t)(i / Sh::kSlots) & 1); };
            auto slot_base = [&](int i) { return sbase + 2 * Sh::kQTile + (uint32_t)(i % Sh::kSlots) * Sh::kSlot; };
            int kv = 0;                // tiles of earlier items: tile j's K is load 2 (kv + j), its V the next
            uint32_t np[2] = {0, 0};   // P tiles taken so far
            uint32_t nitem[2] = {0, 0};
            bool ok = true;
            const uint32_t one = elect();
            auto issue_s = [&](int q, int j) {
                const int load = 2 * (kv + j);
                const uint32_t k = slot_base(load), qt = sbase + (uint32_t)q * Sh::kQTile, d = tmem + (uint32_t)(q * BN);
#pragma unroll
                for (int part = Sh::kSplit - 1; part >= 0; --part)  // the remainders first: their sums are small
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        const uint32_t half = (uint32_t)(kk >> 2), off = (uint32_t)((kk & 3) * 32);
                        umma_ss(one, d, desc_k_sw128(qt + (uint32_t)(part * Sh::kHalves * Sh::kQHalf) + half * Sh::kQHalf + off),
                                 desc_k_sw128(k + half * Sh::kKvHalf + off), id_s, (uint32_t)(part != Sh::kSplit - 1 || kk > 0));
                    }
                commit_one(one, &sh.s_full[q]);
                if (q == 1 || it.dual || it.solo) commit_one(one, &sh.empty[load % Sh::kSlots]);
            };
            auto issue_pv = [&](int q, int j, int half) {  // half: of the tile's positions
                const int load = 2 * (kv + j) + 1;
                const uint32_t v = slot_base(load) + (uint32_t)(half * (BN / 32) * 2048), d = tmem + Sh::kO + (uint32_t)(q * HD);
                const uint32_t pt = tmem + (uint32_t)(q * BN + half * (Sh::kF32 ? BN / 2 : BN / 4));
                const int jj = it.dual ? j >> 1 : j;  // the warpgroup's own count
                const bool fresh = jj % Sh::kFlush == 0;
#pragma unroll
                for (int part = 0; part < Sh::kSplit; ++part)
#pragma unroll
                    for (int kk = 0; kk < BN / 32; ++kk)
                        // 16-bit: 8 columns a step; f32: 8 of hi and 8 of lo over the 16 that S leaves
                        umma_ts(one, d, pt + (uint32_t)(Sh::kF32 ? kk * 16 + part * 8 : kk * 8), desc_mn_sw128(v + (uint32_t)kk * 2048u, Sh::kKvHalf), id_o,
                                (uint32_t)(!fresh || part || kk || half));
                if (half == 0) return;
                commit_one(one, &sh.pv_done[q]);
                if (q == 1 || it.dual || it.solo) commit_one(one, &sh.empty[load % Sh::kSlots]);
            };
            TcPlace at;
            for (int n = 0; ok && take(n, at, ok); ++n) {
                if (!it.get(c, a, p, at, n)) continue;
                it.uniform();
                const int J = it.tiles, step = it.dual ? 2 : 1;  // step: to the warpgroup's next tile
                for (int q = 0; q < 2 && ok; ++q) {
                    if (it.J[q] == 0) continue;  // solo: the other warpgroup; or a range of positions that the rows do not reach
                    ok = wait(&sh.q_full[q], nitem[q]++ & 1);
                    tc_fence_after();
                    const int j = it.dual ? q : 0;
                    if (ok && (ok = slot_wait(2 * (kv + j)))) issue_s(q, j);
                }
                for (int j = 0; j < J && ok; ++j) {
                    const int load = 2 * (kv + j) + 1;
                    bool v_ready = false;
                    for (int q = 0; q < 2 && ok; ++q) {
                        if (it.dual ? (j & 1) != q : j >= it.J[q]) continue;
                        if (!(ok = wait(&sh.p_half[q][0], np[q] & 1))) break;
                        tc_fence_after();
                        const bool more = it.dual ? j + 2 < J : j + 1 < it.J[q];
                        if (!v_ready) {
                            if (!(ok = slot_wait(load))) break;
                            v_ready = true;
                            const int n0 = it.valid(j);
                            if (n0 < BN) {
                                // rows of V past the last position hold anything: their weights are 0, and 0 times a NaN is not
                                const uint32_t v = slot_base(load);
                                for (int i = lane; i < (BN - n0) * 8 * Sh::kHalves; i += 32) {
                                    const int h = i / ((BN - n0) * 8), at = i % ((BN - n0) * 8);
                                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v + (uint32_t)(h * Sh::kKvHalf + n0 * 128 + at * 16)), "r"(0) : "memory");
                                }
                                fence_proxy_async_smem();
                                __syncwarp();
                            }
                        }
                        issue_pv(q, j, 0);
                        if (!(ok = wait(&sh.p_half[q][1], np[q]++ & 1))) break;
                        tc_fence_after();
                        issue_pv(q, j, 1);
                        if (more) {
                            if (!(ok = slot_wait(2 * (kv + j + step)))) break;
                            issue_s(q, j + step);
                        }
                    }
                }
                kv += J;
            }
            if (!ok) *abort_v = 1;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ---- softmax and epilogue of row tile q: one thread per row ----
        const int q = warp >> 2, r = 32 * (warp & 3) + lane;
        const uint32_t lane_t = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t st = lane_t + (uint32_t)(q * BN), ot = lane_t + Sh::kO + (uint32_t)(q * HD);
        const uint32_t qdst = sbase + (uint32_t)q * Sh::kQTile;
        constexpr float kBelow = std::is_same<E, __half>::value ? 9.f : 6.f, kAbove = std::is_same<E, __half>::value ? 15.f : 14.f;
        uint32_t ns = 0, nd = 0;  // S tiles taken so far (P V tiles done are as many); items shared by both warpgroups
        bool ok = true;
        TcPlace at;
            for (int n = 0; ok && take(n, at, ok); ++n) {
            if (!it.get(c, a, p, at, n) || (it.solo && q != it.by)) continue;
            const int tile0 = it.dual || it.solo ? 0 : q * kTcRows, row = tile0 + r, J = it.J[q];  // tile0: the warpgroup's first row
            const bool real = row < it.rows;
            const int rr = it.r0 + (real ? row : 0), rt = row_token(p, rr), tok = it.first + rt, head = it.g * p.rep + rr - rt * p.rep;
            // The warp's 32 query rows, 16 bytes a lane with a row's lanes side by
            // side, all in flight at once.  Compact loops, here and below: code
            // that runs once an item comes from L2, at about six cycles an
            // instruction.
            constexpr int kLanes = HD * (int)sizeof(Q) / 16, kTogether = 32 / kLanes;  // lanes of a row, rows of a load
            auto q_slot = [&](int w, int slot) { return qdst + (uint32_t)((slot >> 3) * Sh::kQHalf) + swizzle(32 * (warp & 3) + w, slot & 7); };
            // Scores are taken with |scale|: the rows' sign takes the scale's, so
            // that their maximum is that of q . k.
            float qmul = fabsf(a.scale) * kLog2e;
            // Without tiles there is nothing to load or to hand over, and the issuer
            // does not wait: the warpgroup could be two items ahead of it.
            if (J > 0) {
                const int c16 = lane % kLanes;  // 16-byte chunk of the row
                // 16-bit: chunk c to its place.  f32: chunks 2k and 2k + 1 to where their elements' hi and lo will be.
                const int to_slot = Sh::kF32 ? (c16 & 1) * (kLanes / 2) + (c16 >> 1) : c16;
#pragma unroll 4
                for (int i = 0; i < kLanes; ++i) {
                    const int w = i * kTogether + lane / kLanes, wr = it.r0 + tile0 + 32 * (warp & 3) + w, wt = row_token(p, wr);
                    const bool is = tile0 + 32 * (warp & 3) + w < it.rows;
                    const Q *src = static_cast<const Q *>(a.q);
                    if (is) src += (int64_t)(it.first + wt) * a.q_stride + (int64_t)(it.g * p.rep + wr - wt * p.rep) * HD + c16 * (16 / (int)sizeof(Q));
                    cp_async16(q_slot(w, to_slot), src, is);
                }
                cp_commit();
                cp_wait<0>();
                __syncwarp();
                if constexpr (Sh::kF32) {
                    // a thread splits its row into hi + lo, scaled by the power of two that puts its largest element near 2^14: the
                    // remainders stay normal f16 (at most by 2^114, which keeps rows of subnormal numbers finite)
                    float amax = 0.f;
#pragma unroll 4
                    for (int k = 0; k < kLanes; ++k) {
                        float x[4];
                        lds16(q_slot(lane, k), x);
                        amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x[0]), fabsf(x[1]))), fmaxf(fabsf(x[2]), fabsf(x[3])));
                    }
                    const int ex = max((int)(__float_as_uint(amax) >> 23) - 126, -100);
                    const float up = copysignf(__uint_as_float((uint32_t)(127 + 14 - ex) << 23), a.scale);
                    qmul *= __uint_as_float((uint32_t)(127 + ex - 14) << 23);
#pragma unroll 2
                    for (int k = 0; k < kLanes / 2; ++k) {
                        float x[4], y[4];
                        uint32_t hi[4], lo[4];
                        lds16(q_slot(lane, k), x);
                        lds16(q_slot(lane, kLanes / 2 + k), y);
                        split2<E>(x[0] * up, x[1] * up, hi[0], lo[0]);
                        split2<E>(x[2] * up, x[3] * up, hi[1], lo[1]);
                        split2<E>(y[0] * up, y[1] * up, hi[2], lo[2]);
                        split2<E>(y[2] * up, y[3] * up, hi[3], lo[3]);
                        sts16(q_slot(lane, k), hi);
                        sts16(q_slot(lane, kLanes / 2 + k), lo);
                    }
                } else if (a.scale < 0.f) {
#pragma unroll 1
                    for (int k = 0; k < kLanes; ++k) {
                        float x[4];
                        lds16(q_slot(lane, k), x);
                        const uint32_t y[4] = {__float_as_uint(x[0]) ^ 0x80008000u, __float_as_uint(x[1]) ^ 0x80008000u, __float_as_uint(x[2]) ^ 0x80008000u,
                                               __float_as_uint(x[3]) ^ 0x80008000u};
                        sts16(q_slot(lane, k), y);
                    }
                }
                qmul = fmaxf(qmul, 1e-38f);  // a masked score stays -inf when the scale is 0
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mb_arrive(&sh.q_full[q]);
            }

            const int own_limit = min(it.pooled ? 0 : max(0, it.back + rt + 1), it.own1) - it.own0;  // own slots of the item that this row sees
            float mref = -INFINITY, l = 0.f, fade = 1.f;  // fade: what `held` is to be rescaled by
            float acc[Sh::kF32 ? HD : 1];
#pragma unroll
            for (int i = 0; i < (Sh::kF32 ? HD : 1); ++i) acc[i] = 0.f;
            // 16-bit: where O goes after kFlush tiles, elements 4 i .. 4 i + 3 of the row at [128 i]
            float4 *const held = reinterpret_cast<float4 *>(p.held) + ((int64_t)blockIdx.x * 2 + q) * (HD / 4) * kTcRows + r;
            // acc += O (f32), once P V of the last tile is done
            auto flush = [&](bool clear) {
                if constexpr (Sh::kF32) {
#pragma unroll
                    for (int i = 0; i < HD; i += 32) {
                        uint32_t o[32];
                        tmem_ld(ot + i, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) acc[i + e] += __uint_as_float(o[e]);
                        if (clear) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = 0;
                            tmem_st32(ot + i, o);
                        }
                    }
                }
            };
            for (int jj = 0; jj < J; ++jj, ++ns) {
                const int j = it.dual ? 2 * jj + q : jj;
                if (!Sh::kF32 && jj > 0 && jj % Sh::kFlush == 0) {
                    // the next P V starts O anew
                    if (!(ok = warp_wait(&sh.pv_done[q], (ns - 1) & 1, abort_v))) break;
                    tc_fence_after();
                    hold<HD>(ot, held, jj > Sh::kFlush, fade);
                    fade = 1.f;
                }
                if (!(ok = warp_wait(&sh.s_full[q], ns & 1, abort_v))) break;
                tc_fence_after();
                const int vis = !real ? BN : j < it.jp ? it.pre1 - it.pre0 - j * BN : own_limit - (j - it.jp) * BN;
                const bool whole = __all_sync(0xffffffffu, vis >= BN);
                uint32_t s[Sh::kF32 ? 32 : BN];
                float mx;
                if constexpr (Sh::kF32) {
                    mx = -INFINITY;
#pragma unroll 1
                    for (int h = 0; h < BN / 32; ++h) {
                        tmem_ld(st + 32 * h, s);
                        tmem_wait_ld();
                        if (!whole) mask(s, vis - 32 * h);
                        mx = fmaxf(mx, max_of(s));
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < BN / 32; ++h) tmem_ld(st + 32 * h, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * h]));
                    tmem_wait_ld();
                    if (!whole) mask(s, vis);
                    mx = max_of(s);
                }
                mx *= qmul;
                const bool up = mx > mref + kAbove;
                const float mnew = up ? mx - kBelow : mref;
                const float corr = up && mref > -INFINITY ? ex2(mref - mnew) : 1.f;
                const bool rescale = jj > 0 && __any_sync(0xffffffffu, corr != 1.f);
                const bool flushes = Sh::kF32 && jj > 0 && (rescale || jj % Sh::kFlush == 0);
                if (rescale || flushes) {
                    // O holds the tiles before this once P V of the last one is done
                    if (!(ok = warp_wait(&sh.pv_done[q], (ns - 1) & 1, abort_v))) break;
                    tc_fence_after();
                }
                if constexpr (Sh::kF32) {
                    if (flushes) flush(jj % Sh::kFlush != 0);
                    if (rescale) {
#pragma unroll
                        for (int i = 0; i < HD; ++i) acc[i] *= corr;
                    }
                } else if (rescale) {
#pragma unroll 1
                    for (int i = 0; i < HD; i += 32) {
                        uint32_t o[32];
                        tmem_ld(ot + i, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                        tmem_st32(ot + i, o);
                    }
                }
                l *= corr, fade *= corr;
                mref = mnew;
                const float base = mref == -INFINITY ? 0.f : mref;  // nothing seen yet: every score is -inf
                const uint64_t qm2 = two(qmul, qmul), nb2 = two(-base, -base);
                uint64_t sum[2] = {0, 0};
                // half of P is written: P V of its positions may run under the other half's softmax
                auto hand_over = [&](int half) {
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mb_arrive(&sh.p_half[q][half]);
                };
                if constexpr (Sh::kF32) {
#pragma unroll 2
                    for (int h = 0; h < BN / 16; ++h) {
                        uint32_t x[16], hi[8], lo[8];
                        tmem_ld16(st + 16 * h, x);
                        tmem_wait_ld();
                        if (!whole) mask(x, vis - 16 * h);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float2 y = untwo(fma2(two(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), qm2, nb2));
                            const float w0 = ex2(y.x), w1 = ex2(y.y);
                            sum[i & 1] = add2(sum[i & 1], two(w0, w1));
                            split2<E>(w0, w1, hi[i], lo[i]);
                        }
                        tmem_st8(st + 16 * h, hi);
                        tmem_st8(st + 16 * h + 8, lo);
                        if (h % (BN / 32) == BN / 32 - 1) hand_over(h / (BN / 32));
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < BN / 64; ++h) {  // P of columns 64 h .. into TMEM columns 32 h ..: all of S has been read
                        uint32_t w[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float2 y = untwo(fma2(two(__uint_as_float(s[64 * h + 2 * i]), __uint_as_float(s[64 * h + 2 * i + 1])), qm2, nb2));
                            const float w0 = ex2(y.x), w1 = ex2(y.y);
                            sum[i & 1] = add2(sum[i & 1], two(w0, w1));
                            w[i] = pack2<E>(w0, w1);
                        }
                        tmem_st32(st + 32 * h, w);
                        hand_over(h);
                    }
                }
                const float2 total = untwo(add2(sum[0], sum[1]));
                l += total.x + total.y;
            }
            if (ok && J > 0) ok = warp_wait(&sh.pv_done[q], (ns - 1) & 1, abort_v);
            if (!ok) break;
            tc_fence_after();
            if (J > 0) flush(false);
            if (!Sh::kF32 && J > Sh::kFlush) hold_back<HD>(ot, held, fade);
            float mine = 1.f, other = 0.f;  // what this warpgroup's and the other's O count
            if (it.dual) {
                // the second warpgroup's part goes to the first, which shares its TMEM lanes: O is there (f32: put there), (m, l)
                // through shared memory
                if (q == 1) {
                    if constexpr (Sh::kF32) {
#pragma unroll
                        for (int i = 0; i < HD; i += 32) {
                            uint32_t o[32];
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(acc[i + e]);
                            tmem_st32(ot + i, o);
                        }
                        tmem_wait_st();
                    }
                    sh.ml[r] = make_float2(mref, l);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mb_arrive(&sh.pair_full);
                    // until the first has read it
                    if (!(ok = warp_wait(&sh.pair_free, nd++ & 1, abort_v))) break;
                    continue;
                }
                if (!(ok = warp_wait(&sh.pair_full, nd++ & 1, abort_v))) break;
                tc_fence_after();
                const float2 b = sh.ml[r];
                const float m = fmaxf(mref, b.x);
                mine = part_factor(mref, l, m), other = part_factor(b.x, b.y, m);
                l = l * mine + b.y * other, mref = m;
            }
            const int64_t id = (int64_t)tok * a.heads + head;
            const bool parts = p.parts > 0;
            const int part = it.pooled ? it.split : p.prefix_splits + it.split;
            const float inv = parts ? 1.f : l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: zeros
            if (real) {
                if (parts) {
                    p.ml[id * p.parts + part] = make_float2(mref, l);
                } else {
                    const float lse2 = l == 0.f ? -INFINITY : mref + log2f(l);
                    if (a.lse) a.lse[id] = lse2 * kLn2;
                    if (p.lse2) p.lse2[id] = lse2;
                }
            }
            // O, scaled, through the warp's own rows of the Q tile (free by now), so
            // that a global store writes whole rows: kBlocks blocks of 128 bytes a
            // row, swizzled like Q, as often as an output row of OB bytes takes
            constexpr int kBlocks = Sh::kHalves * Sh::kSplit;
            auto store = [&](auto *to_rows, auto row_offset) {
                using O = std::remove_reference_t<decltype(*to_rows)>;
                constexpr int kEach = 16 / (int)sizeof(O), kCols = kBlocks * 8 * kEach < HD ? kBlocks * 8 * kEach : HD;  // elements of a chunk; columns of a pass
                constexpr int kChunks = kCols / kEach, kRows = 32 / (kChunks < 32 ? kChunks : 32);                       // chunks of a row; rows of a store
#pragma unroll(Sh::kF32 ? HD / kCols : 1)
                for (int c0 = 0; c0 < HD; c0 += kCols) {
#pragma unroll(Sh::kF32 ? kCols / 32 : 1)
                    for (int i = c0; i < c0 + kCols; i += 32) {
                        float o[32];
                        if constexpr (Sh::kF32) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = acc[i + e] * (mine * inv);
                        } else {
                            uint32_t raw_o[32];
#pragma unroll
                            for (int e = 0; e < 32; ++e) raw_o[e] = 0;
                            if (J > 0) {
                                tmem_ld(ot + i, raw_o);  // warp-collective
                                tmem_wait_ld();
                            }
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(raw_o[e]) * (mine * inv);
                        }
                        if (it.dual && it.J[1] > 0) {
                            uint32_t two_o[32];
                            tmem_ld(ot + HD + i, two_o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = fmaf(__uint_as_float(two_o[e]), other * inv, o[e]);
                        }
#pragma unroll
                        for (int e = 0; e < 32; e += kEach) {
                            const int ch = (i - c0 + e) / kEach;
                            uint32_t w[4];
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                if constexpr (sizeof(O) == 4) w[x] = __float_as_uint(o[e + x]);
                                else w[x] = pack2<O>(o[e + 2 * x], o[e + 2 * x + 1]);
                            }
                            sts16(q_slot(lane, ch), w);
                        }
                    }
                    __syncwarp();
#pragma unroll 4
                    for (int i = 0; i < 32; i += kRows) {
                        const int tr = 32 * (warp & 3) + i + lane / kChunks, w = tile0 + tr, ch = lane % kChunks;
                        float x[4];
                        lds16(q_slot(tr - 32 * (warp & 3), ch), x);
                        if (w < it.rows) *reinterpret_cast<uint4 *>(to_rows + row_offset(it.r0 + w) + c0 + ch * kEach) =
                            make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
                    }
                    __syncwarp();
                }
            };
            auto at_row = [&](int wr, int64_t stride, int step) {  // offset of a row's token and head
                const int wt = row_token(p, wr);
                return (int64_t)(it.first + wt) * stride + (int64_t)(it.g * p.rep + wr - wt * p.rep) * step;
            };
            if (parts) store(p.part + part * HD, [&](int wr) { return at_row(wr, (int64_t)a.heads * p.parts * HD, p.parts * HD); });
            else store(static_cast<Q *>(a.out), [&](int wr) { return at_row(wr, a.out_stride, HD); });
            if (it.dual) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mb_arrive(&sh.pair_free);
            }
        }
        if (!ok) *abort_v = 1;
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_v) cache_flag(c.status, S2D_CACHE_ABORTED);
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTcColumns));
    }
}

// ---------------------------------------------------------------------------
// weights of many rows
// ---------------------------------------------------------------------------

// mass[b][g][slot] += sum over the rows that see the slot of 2^(s - lse2), the
// scores computed again with the slots as rows: S^T = K Q^T, so that a slot is
// a TMEM lane and one thread adds its weights, in the order of the rows.
//
// A CTA takes up to kWeighTiles tiles of 128 slots of one (sequence, KV head)
// and its query rows 128 at a time: the rows are loaded once, the keys stream
// through a ring of two tiles, and two warpgroups take every other tile, each
// with a TMEM buffer of its own.  Warps 0-7 load the rows and add the weights,
// 8 loads keys, 9 issues the MMAs; with 16-bit queries two CTAs share an SM.
// Every wait is bounded, as above.
//
// Bound by latency: 8 sequences of 1,968 to 8,160 slots, 32 tokens each, 8 KV
// heads of 128 take 37 us, of which reading the keys is 13.  The whole call: 106
// us with 2 tiles a CTA, 99 to 104 with 4 to 16.
constexpr int kWeighTiles = 8, kWeighThreads = 320;

template <typename Q, int HD>
struct WeighShape {
    static constexpr bool kF32 = sizeof(Q) == 4;
    static constexpr int kHalves = HD / 64, kSplit = kF32 ? 2 : 1;
    static constexpr int kQHalf = kTcRows * 128, kQ = kHalves * kSplit * kQHalf;  // query rows: a column block; all
    static constexpr int kKHalf = kTcRows * 128, kK = kHalves * kKHalf;           // a tile of keys
    static constexpr int kSmem = kQ + 2 * kK + 1024;
};

template <typename Q, typename E, int HD>
__global__ void __launch_bounds__(kWeighThreads) weigh_tc_kernel(const __grid_constant__ CUtensorMap mk, const S2dCacheView c, const S2dCacheAttention a,
                                                                 const AttnPlan p) {
    using Sh = WeighShape<Q, HD>;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t k_full[2], k_empty[2], s_full[2], s_free[2], q_full, q_free;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ __align__(16) float2 s_row[kTcRows];  // a row's (multiplier of its scores, lse2); lse2 inf: no weight
    __shared__ int s_seen[kTcRows];                  // slots that a row sees
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sbase = su32(smem);
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31, b = blockIdx.y, g = blockIdx.z;
    const int p0 = (int)blockIdx.x * kWeighTiles * kTcRows;
    int first;
    const int n = cache_length(c, b), nt = cache_tokens(a.q_start, a.tokens, b, first, c.status);
    if (p0 >= n || nt == 0) {
        // the grid must not end before the one that it was launched behind
        if (blockIdx.x + blockIdx.y + blockIdx.z == 0) grid_dep_wait();
        return;
    }
    const int back = n - nt, rows = nt * p.rep;
    volatile int *abort_v = &s_abort;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) mb_init(&k_full[i], 1), mb_init(&k_empty[i], 1), mb_init(&s_full[i], 1), mb_init(&s_free[i], 4);
        mb_init(&q_full, 8), mb_init(&q_free, 8);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&s_tmem)), "r"(2 * kTcRows));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    // row tiles before this one see none of the CTA's slots
    const int r_first = (int)min((int64_t)rows, (int64_t)max(0, p0 - back) * p.rep) / kTcRows * kTcRows;
    // tiles of slots that the rows from r0 on see (the last of them the most)
    auto tiles_of = [&](int r0) {
        const int seen = min(n, back + row_token(p, min(rows, r0 + kTcRows) - 1) + 1);
        return __shfl_sync(0xffffffffu, min(kWeighTiles, (seen - p0 + kTcRows - 1) / kTcRows), 0);
    };
    bool ok = true;
    if (warp == 8) {
        const int32_t *table = c.page_table + (int64_t)b * c.table_stride + p0 / kCachePage;
        int loads = 0;
        for (int r0 = r_first; r0 < rows && ok; r0 += kTcRows) {
            const int tiles = tiles_of(r0);
            for (int t = 0; t < tiles && ok; ++t, ++loads) {
                const int s = loads & 1, use = loads >> 1;
                if (use > 0 && !(ok = warp_wait(&k_empty[s], (use & 1) ^ 1, abort_v))) break;
                const int n_pages = min(2, (n - p0 - t * kTcRows + kCachePage - 1) / kCachePage);
                if (lane == 0) {
                    mb_expect_tx(&k_full[s], (uint32_t)(n_pages * Sh::kHalves * kCachePage * 128));
                    for (int i = 0; i < n_pages; ++i) {
                        int page = __ldg(table + 2 * t + i);
                        if ((uint32_t)page >= (uint32_t)c.n_pages) {
                            cache_flag(c.status, S2D_CACHE_BAD_PAGE);
                            page = 0;
                        }
                        for (int h = 0; h < Sh::kHalves; ++h)
                            tma_page(smem + Sh::kQ + s * Sh::kK + h * Sh::kKHalf + i * kCachePage * 128, &mk, 64 * h, g, page, &k_full[s]);
                    }
                }
                __syncwarp();
            }
        }
        if (!ok) *abort_v = 1;
        // neither a copy nor the arrival that frees its slot may still be landing when the CTA leaves
        for (int i = max(0, loads - 2); i < loads; ++i) {
            (void)mb_wait(&k_full[i & 1], (i >> 1) & 1, abort_v, false);
            (void)mb_wait(&k_empty[i & 1], (i >> 1) & 1, abort_v);
        }
    } else if (warp == 9) {
        constexpr uint32_t id_s = idesc_f16_f32(kTcRows, kTcRows) | (std::is_same<E, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u);
        const uint32_t one = elect();
        int loads = 0;
        uint32_t turn = 0, used[2] = {0, 0};  // row tiles; tiles that a buffer has held
        for (int r0 = r_first; r0 < rows && ok; r0 += kTcRows, ++turn) {
            const int tiles = tiles_of(r0);
            if (!(ok = warp_wait(&q_full, turn & 1, abort_v))) break;
            for (int t = 0; t < tiles && ok; ++t, ++loads) {
                const int s = loads & 1, w = t & 1;
                if (!(ok = warp_wait(&k_full[s], (loads >> 1) & 1, abort_v))) break;
                if (used[w] > 0 && !(ok = warp_wait(&s_free[w], (used[w] - 1) & 1, abort_v))) break;
                ++used[w];
                tc_fence_after();
                const uint32_t k = sbase + Sh::kQ + (uint32_t)s * Sh::kK;
#pragma unroll
                for (int part = Sh::kSplit - 1; part >= 0; --part)  // the remainders first: their sums are small
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        const uint32_t half = (uint32_t)(kk >> 2), off = (uint32_t)((kk & 3) * 32);
                        umma_ss(one, tmem + (uint32_t)(w * kTcRows), desc_k_sw128(k + half * Sh::kKHalf + off),
                                desc_k_sw128(sbase + (uint32_t)(part * Sh::kHalves * Sh::kQHalf) + half * Sh::kQHalf + off), id_s,
                                (uint32_t)(part != Sh::kSplit - 1 || kk > 0));
                    }
                commit_one(one, &s_full[w]);
                commit_one(one, &k_empty[s]);
            }
        }
        if (!ok) *abort_v = 1;
    } else {
        const int wg = warp >> 2;
        const uint32_t st = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)(wg * kTcRows);
        float sum[kWeighTiles / 2] = {};
        bool waited = false;
        uint32_t turn = 0, taken = 0;  // row tiles; tiles of this warpgroup
        for (int r0 = r_first; r0 < rows && ok; r0 += kTcRows, ++turn) {
            // 128 query rows: 16 a warp, 16 bytes a lane
            constexpr int kLanes = HD * (int)sizeof(Q) / 16, kTogether = 32 / kLanes, kLoads = 16 / kTogether;
            const int c16 = lane % kLanes, tiles = tiles_of(r0);
            uint4 qv[kLoads];
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int w = r0 + 16 * warp + i * kTogether + lane / kLanes, wt = row_token(p, w);
                const Q *src = static_cast<const Q *>(a.q) + (int64_t)(first + wt) * a.q_stride + (int64_t)(g * p.rep + w - wt * p.rep) * HD;
                qv[i] = w < rows ? reinterpret_cast<const uint4 *>(src)[c16] : make_uint4(0, 0, 0, 0);
            }
            if (!waited) grid_dep_wait(), waited = true;  // the rows' sums are there
            // the last rows are used up: their MMAs are done and their weights added
            if (turn > 0 && !(ok = warp_wait(&q_free, (turn - 1) & 1, abort_v))) break;
            if (threadIdx.x < kTcRows) {
                const int w = r0 + (int)threadIdx.x, wt = row_token(p, w);
                float l = INFINITY;
                if (w < rows) l = __ldcg(&p.lse2[(int64_t)(first + wt) * a.heads + g * p.rep + w - wt * p.rep]);
                s_row[threadIdx.x].y = l == -INFINITY ? INFINITY : l;
                if (!Sh::kF32) s_row[threadIdx.x].x = a.scale * kLog2e;
                s_seen[threadIdx.x] = w < rows ? back + wt + 1 : 0;
            }
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int w = 16 * warp + i * kTogether + lane / kLanes;
                if constexpr (Sh::kF32) {
                    const float x[4] = {__uint_as_float(qv[i].x), __uint_as_float(qv[i].y), __uint_as_float(qv[i].z), __uint_as_float(qv[i].w)};
                    float amax = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
                    for (int o = kLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                    const int ex = max((int)(__float_as_uint(amax) >> 23) - 126, -100);  // as in the kernel above
                    const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
                    if (c16 == 0) s_row[w].x = a.scale * kLog2e * __uint_as_float((uint32_t)(127 + ex - 14) << 23);
                    uint32_t hi[2], lo[2];
                    split2<E>(x[0] * up, x[1] * up, hi[0], lo[0]);
                    split2<E>(x[2] * up, x[3] * up, hi[1], lo[1]);
                    const uint32_t at = sbase + (uint32_t)((c16 >> 4) * Sh::kQHalf) + swizzle(w, (c16 >> 1) & 7) + (c16 & 1) * 8;
                    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(hi[0]), "r"(hi[1]) : "memory");
                    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + (uint32_t)(Sh::kHalves * Sh::kQHalf)), "r"(lo[0]), "r"(lo[1]) : "memory");
                } else {
                    const uint32_t x[4] = {qv[i].x, qv[i].y, qv[i].z, qv[i].w};
                    sts16(sbase + (uint32_t)((c16 >> 3) * Sh::kQHalf) + swizzle(w, c16 & 7), x);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mb_arrive(&q_full);
            if (!(ok = warp_wait(&q_full, turn & 1, abort_v))) break;  // the other warps' entries of s_row
#pragma unroll
            for (int i = 0; i < kWeighTiles / 2; ++i) {
                const int t = 2 * i + wg;
                if (t >= tiles || !ok) continue;
                if (!(ok = warp_wait(&s_full[wg], taken++ & 1, abort_v))) continue;
                tc_fence_after();
                const int slot = p0 + t * kTcRows + 32 * (warp & 3) + lane;  // this thread's slot
                // 128 rows that all see the tile's slots, or not
                const bool whole = r0 + kTcRows <= rows && s_seen[0] >= min(n, p0 + (t + 1) * kTcRows);
#pragma unroll 1
                for (int h = 0; h < kTcRows / 32; ++h) {
                    uint32_t x[32];
                    tmem_ld(st + 32 * h, x);
                    tmem_wait_ld();
                    float part[2] = {0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float4 r = *reinterpret_cast<const float4 *>(&s_row[32 * h + e]);
                        const float w0 = ex2(fmaf(__uint_as_float(x[e]), r.x, -r.y)), w1 = ex2(fmaf(__uint_as_float(x[e + 1]), r.z, -r.w));
                        part[0] += whole || slot < s_seen[32 * h + e] ? w0 : 0.f;
                        part[1] += whole || slot < s_seen[32 * h + e + 1] ? w1 : 0.f;
                    }
                    sum[i] += part[0] + part[1];
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mb_arrive(&s_free[wg]);
            }
            __syncwarp();
            if (lane == 0) mb_arrive(&q_free);
        }
        if (!waited) grid_dep_wait();
        if (!ok) *abort_v = 1;
        float *mass = c.mass + ((int64_t)b * c.kv_heads + g) * c.max_pages * kCachePage;
#pragma unroll
        for (int i = 0; i < kWeighTiles / 2; ++i) {
            const int slot = p0 + (2 * i + wg) * kTcRows + 32 * (warp & 3) + lane;
            if (ok && slot < n) mass[slot] += sum[i];
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_v) cache_flag(c.status, S2D_CACHE_ABORTED);
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kTcRows));
    }
}

// The pool as [page][head][position][element], boxes of one page's 64
// positions x 64 elements with 128-byte swizzle.
bool page_map(CUtensorMap *m, const S2dCacheView &c, void *base) {
    EncodeTiled enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, kCachePage, (cuuint64_t)c.kv_heads, (cuuint64_t)c.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.head_dim * 2, (cuuint64_t)c.head_stride * 2, (cuuint64_t)c.page_stride * 2};
    const cuuint32_t box[4] = {64, kCachePage, 1, 1}, one[4] = {1, 1, 1, 1};
    return enc(m, c.type == S2D_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, strides, box, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename Q, typename E, int HD>
cudaError_t launch(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p, cudaStream_t s) {
    CUtensorMap mk, mv;
    if (!page_map(&mk, c, c.k) || !page_map(&mv, c, c.v)) return cudaErrorInvalidValue;
    constexpr int smem = TcShape<Q, HD>::kSmem;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = smem_limit(done, rows_tc_kernel<Q, E, HD>, c.device, smem);
    if (e) return e;
    // at most: own_tiles is a bound, and any of them may be two halves
    const int64_t items = ((int64_t)p.prefix_tiles * p.prefix_splits + 2 * (int64_t)p.own_tiles * p.own_splits) * c.kv_heads;
    if (items > 0x7fffffff - 1024) return cudaErrorInvalidValue;
    int sms = 0;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, c.device))) return e;
    AttnPlan q = p;
    sms = std::min(sms, kCacheSms);  // p.held has room for as many CTAs
    if (items <= sms) q.next_item = nullptr;  // one item each
    if (q.next_item && (e = cudaMemsetAsync(q.next_item, 0, sizeof(int), s))) return e;
    rows_tc_kernel<Q, E, HD><<<(unsigned)std::min<int64_t>(items, sms), kTcThreads, smem, s>>>(mk, mv, c, a, q);
    return cudaGetLastError();
}

template <typename Q, typename E, int HD>
cudaError_t weigh(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p, cudaStream_t s) {
    CUtensorMap mk;
    if (!page_map(&mk, c, c.k)) return cudaErrorInvalidValue;
    constexpr int smem = WeighShape<Q, HD>::kSmem;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = smem_limit(done, weigh_tc_kernel<Q, E, HD>, c.device, smem);
    if (e) return e;
    const int slots = kWeighTiles * kTcRows;
    const dim3 grid((unsigned)((c.max_pages * kCachePage + slots - 1) / slots), (unsigned)c.n_seq, (unsigned)c.kv_heads);
    // its first keys and queries are loaded while the rows' sums are still computed
    return s2d_launch(weigh_tc_kernel<Q, E, HD>, grid, dim3(kWeighThreads), smem, s, true, mk, c, a, p);
}

}  // namespace

cudaError_t launch_weigh_tc(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p, cudaStream_t s) {
    const bool wide = c.head_dim == 128;
    if (a.type == S2D_TYPE_F32) return wide ? weigh<float, __half, 128>(c, a, p, s) : weigh<float, __half, 64>(c, a, p, s);
    if (a.type == S2D_TYPE_F16) return wide ? weigh<__half, __half, 128>(c, a, p, s) : weigh<__half, __half, 64>(c, a, p, s);
    return wide ? weigh<__nv_bfloat16, __nv_bfloat16, 128>(c, a, p, s) : weigh<__nv_bfloat16, __nv_bfloat16, 64>(c, a, p, s);
}

cudaError_t launch_rows_tc(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p, cudaStream_t s) {
    const bool wide = c.head_dim == 128;
    if (a.type == S2D_TYPE_F32) return wide ? launch<float, __half, 128>(c, a, p, s) : launch<float, __half, 64>(c, a, p, s);
    if (a.type == S2D_TYPE_F16) return wide ? launch<__half, __half, 128>(c, a, p, s) : launch<__half, __half, 64>(c, a, p, s);
    return wide ? launch<__nv_bfloat16, __nv_bfloat16, 128>(c, a, p, s) : launch<__nv_bfloat16, __nv_bfloat16, 64>(c, a, p, s);
}

}  // namespace s2d

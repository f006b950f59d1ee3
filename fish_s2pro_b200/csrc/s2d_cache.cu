// s2d_cache.cu -- paged-cache operators of include/s2d_cache.h: appending new
// tokens and evicting slots, and the checks of the C entry points.  The
// attention kernels are in s2d_cache_attn.cu.
#include "s2d_cache.cuh"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace s2d {

const char *cache_view_fault(const S2dCacheView *c) {
    if (!c) return "cache view is null";
    if (!c->k || !c->v || !c->page_table || !c->lengths) return "cache view has a null buffer";
    if (c->head_dim != 64 && c->head_dim != 128) return "head_dim must be 64 or 128";
    if (c->type != S2D_TYPE_F16 && c->type != S2D_TYPE_BF16) return "cache type must be F16 or BF16";
    if (c->n_seq <= 0 || c->kv_heads <= 0 || c->n_pages <= 0 || c->max_pages <= 0) return "cache sizes must be positive";
    if (c->n_seq > 65535 || c->kv_heads > 1024) return "at most 65535 sequences and 1024 KV heads";
    if (c->max_pages > (1 << 18)) return "at most 2^18 pages per sequence";  // slots and their products stay inside int
    if (c->table_stride < c->max_pages) return "page-table rows overlap";
    const int64_t page = (int64_t)kCachePage * c->head_dim;
    if (c->head_stride < page || c->head_stride % 8) return "head_stride must be a multiple of 8 of at least 64 * head_dim";
    if (c->page_stride < c->head_stride * (c->kv_heads - 1) + page || c->page_stride % 8)
        return "page_stride must be a multiple of 8 and hold every KV head's rows";
    if (!cache_aligned16(c->k) || !cache_aligned16(c->v)) return "misaligned buffer: k and v must be 16-byte aligned";
    return nullptr;
}

namespace {

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------

// frac(rope_base^(-2i / head_dim) / 2 pi) in 2^-64 turns, per pair: a
// position times an entry, modulo 2^64, is the pair's angle as an exact
// fraction of a turn, however far the position (a product of floats is 2e-3
// off at position 32,768).
struct RopeTurns {
    uint64_t turn[64];
};

// The table of a rope_base: computed once, as the base is a model's.
const RopeTurns &rope_turns(double base, int hd) {
    thread_local RopeTurns r;
    thread_local double have = 0.0;
    thread_local int have_hd = 0;
    if (base != have || hd != have_hd) {
        const long double two_pi = 6.283185307179586476925286766559005768L;
        for (int i = 0; i < hd / 2; ++i) {
            const long double f = powl((long double)base, -2.0L * i / hd) / two_pi;
            r.turn[i] = (uint64_t)((f - floorl(f)) * 0x1p64L);  // f - floor(f) < 1
        }
        have = base, have_hd = hd;
    }
    return r;
}

// 16 bytes of elements of type T as f32, and back.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4 &v, float (&x)[16 / sizeof(T)]) {
    if constexpr (sizeof(T) == 4) {
        x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(w[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
}
// N elements of type T from f32, in one store of 8 or 16 bytes.
template <typename T, int N>
__device__ __forceinline__ void store_pack(T *to, const float (&x)[N]) {
    if constexpr (sizeof(T) == 4) {
        static_assert(N == 4, "16 bytes");
        *reinterpret_cast<float4 *>(to) = make_float4(x[0], x[1], x[2], x[3]);
    } else if constexpr (N == 4) {
        *reinterpret_cast<uint2 *>(to) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
    } else {
        static_assert(N == 8, "16 bytes");
        *reinterpret_cast<uint4 *>(to) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
}

// A block takes `group` consecutive tokens (at most kGroup): one thread each
// finds a token's sequence, slot and page, the block computes the tokens' sines
// and cosines for all their heads, and then every group of L lanes takes head
// rows of the tokens in turn.  A head row of HD elements is read 16 bytes a
// lane, so its lanes are neighbours in one warp (8 to 32) and sum the squares
// with shuffles.
//
// HBM bound: every row is read and written once; 36,900 bf16 tokens of 32 and 8
// heads of 128 take 168 to 180 us, 5.1 to 5.4 TB/s.  What a token needs before its rows (four
// dependent loads) is paid once for the group (8 tokens a group: 177 us, 4:
// 196), and kAhead rows of a lane are under way at once (2, with more blocks:
// 184; 8, with fewer: 192).
constexpr int kGroup = 32, kAhead = 4;

template <typename Q, typename E, int HD>
__global__ void __launch_bounds__(256, 4) append_kernel(const S2dCacheView c, const S2dCacheAppend a, const __grid_constant__ RopeTurns turns, int tokens) {
    constexpr int W = 16 / (int)sizeof(Q), L = HD / W, kRows = 256 / L;
    __shared__ __align__(16) float2 s_turn[kGroup][HD / 2];  // (cos, sin) of the tokens' pairs
    __shared__ __align__(16) float s_gain[2][HD];            // of queries and keys
    __shared__ int64_t s_at[kGroup], s_side[kGroup];         // a token's cache rows and its positions / mass, of head 0; -1: none
    __shared__ int s_pos[kGroup];
    const int G = c.kv_heads, cap = c.max_pages * kCachePage, tid = threadIdx.x;
    // the rows of sequences: [first_row, last), none of them negative, so that their differences are ints; those before and behind stay as they are
    const int first_row = a.q_start ? max(0, __ldg(a.q_start)) : 0, last = a.q_start ? max(0, min(a.tokens, __ldg(a.q_start + c.n_seq))) : min(a.tokens, c.n_seq);
    const int t0 = max((int)blockIdx.x * tokens, first_row), n = (int)min((int64_t)(blockIdx.x + 1) * tokens, (int64_t)last) - t0;
    // lengths of every sequence, tokens or none
    for (int b = (int)blockIdx.x * 256 + tid; b < c.n_seq; b += (int)gridDim.x * 256) {
        int first;
        const int m = cache_tokens(a.q_start, a.tokens, b, first, c.status), p = a.past[b];
        if (p < 0 || p > cap) cache_flag(c.status, S2D_CACHE_BAD_LENGTH);
        c.lengths[b] = min(cap, min(max(p, 0), cap) + m);
    }
    if (n <= 0) return;
    int before = t0;  // sequences that end at or before the group's first token
    if (a.q_start) {
        before = 0;
        for (int b0 = 0; b0 < c.n_seq; b0 += 256) before += __syncthreads_count(b0 + tid < c.n_seq && __ldg(a.q_start + min(b0 + tid, c.n_seq - 1) + 1) <= t0);
    }
    if (tid < n) {
        const int t = t0 + tid;
        int seq = t, i = 0;
        if (a.q_start) {
            seq = before;
            while (seq < c.n_seq && __ldg(a.q_start + seq + 1) <= t) ++seq;
            i = seq < c.n_seq ? t - __ldg(a.q_start + seq) : -1;  // an unordered q_start: lengths has set the status
        }
        const int past = i >= 0 ? __ldg(a.past + seq) : -1;
        const bool sane = past >= 0 && past <= cap, fits = sane && i < cap - past;
        if (!fits) cache_flag(c.status, sane ? S2D_CACHE_FULL : S2D_CACHE_BAD_LENGTH);
        s_at[tid] = fits ? cache_row(c, c.page_table + (int64_t)seq * c.table_stride, 0, past + i) : -1;
        s_side[tid] = fits ? (int64_t)seq * G * cap + past + i : -1;
        s_pos[tid] = __ldg(a.pos + t);
    }
    for (int e = tid; e < 2 * HD; e += 256) {
        const float *gain = e < HD ? a.q_norm : a.k_norm;
        s_gain[e / HD][e % HD] = gain ? __ldg(gain + e % HD) : 1.f;
    }
    __syncthreads();
    for (int i = tid; i < n * (HD / 2); i += 256) {
        const int64_t x = (int64_t)((uint64_t)(int64_t)s_pos[i / (HD / 2)] * turns.turn[i % (HD / 2)]);  // [-1/2, 1/2) turn
        float sn, cs;
        sincospif((float)x * 0x1p-63f, &sn, &cs);
        s_turn[i / (HD / 2)][i % (HD / 2)] = make_float2(cs, sn);
    }
    for (int i = tid; i < n * G; i += 256) {
        const int64_t at = s_side[i / G];
        if (at >= 0 && c.positions) c.positions[at + (int64_t)(i % G) * cap] = s_pos[i / G];
        if (at >= 0 && c.mass) c.mass[at + (int64_t)(i % G) * cap] = 0.f;
    }
    __syncthreads();

    const int d0 = tid % L * W;
    const uint32_t mates = (L == 32 ? 0xffffffffu : (1u << L) - 1u) << ((tid & 31) / L * L);  // the row's lanes
    // The head rows of one kind (0 queries, 1 keys, 2 values) of the group's
    // tokens: lane group tid / L takes rows tid / L, + kRows, ... of them.
    auto rows_of = [&](auto kind_of, const void *from, int64_t stride, int heads) {
        constexpr int kind = decltype(kind_of)::value;
        const bool normed = kind == 0 ? a.q_norm != nullptr : kind == 1 && a.k_norm != nullptr;
        const Q *src = static_cast<const Q *>(from) + (int64_t)t0 * stride + d0;
        const int next_tok = kRows / heads, next_head = kRows % heads;
        int tok = tid / L / heads, head = tid / L % heads;
        while (tok < n) {
            uint4 in[kAhead];
            int its_tok[kAhead], its_head[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                its_tok[k] = tok, its_head[k] = head;
                if (tok < n) in[k] = *reinterpret_cast<const uint4 *>(src + tok * stride + head * HD);
                tok += next_tok, head += next_head;
                if (head >= heads) head -= heads, ++tok;
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (its_tok[k] >= n) break;  // whole rows: the row's lanes together
                float x[W];
                unpack16<Q>(in[k], x);
                if (kind < 2) {
                    if (normed) {
                        float ss = 0.f;
#pragma unroll
                        for (int e = 0; e < W; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
                        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mates, ss, o);
                        const float norm = rsqrtf(ss * (1.f / HD) + a.eps);
#pragma unroll
                        for (int e = 0; e < W; e += 4) {
                            const float4 gain = *reinterpret_cast<const float4 *>(&s_gain[kind][d0 + e]);
                            x[e] *= norm * gain.x, x[e + 1] *= norm * gain.y, x[e + 2] *= norm * gain.z, x[e + 3] *= norm * gain.w;
                        }
                    }
#pragma unroll
                    for (int p = 0; p < W / 2; p += 2) {
                        const float4 r = *reinterpret_cast<const float4 *>(&s_turn[its_tok[k]][d0 / 2 + p]);
                        const float u0 = x[2 * p], w0 = x[2 * p + 1], u1 = x[2 * p + 2], w1 = x[2 * p + 3];
                        x[2 * p] = u0 * r.x - w0 * r.y, x[2 * p + 1] = fmaf(u0, r.y, w0 * r.x);
                        x[2 * p + 2] = u1 * r.z - w1 * r.w, x[2 * p + 3] = fmaf(u1, r.w, w1 * r.z);
                    }
                }
                if constexpr (kind == 0) {
                    store_pack(static_cast<Q *>(a.q_out) + (int64_t)(t0 + its_tok[k]) * a.q_out_stride + its_head[k] * HD + d0, x);
                } else {
                    const int64_t at = s_at[its_tok[k]];
                    if (at >= 0) store_pack(static_cast<E *>(kind == 1 ? c.k : c.v) + at + (int64_t)its_head[k] * c.head_stride + d0, x);
                }
            }
        }
    };
    rows_of(std::integral_constant<int, 0>{}, a.q, a.q_stride, a.heads);
    rows_of(std::integral_constant<int, 1>{}, a.k, a.k_stride, G);
    rows_of(std::integral_constant<int, 2>{}, a.v, a.v_stride, G);
}

template <typename Q, typename E>
cudaError_t append_launch(const S2dCacheView &c, const S2dCacheAppend &a, const RopeTurns &r, cudaStream_t s) {
    // as few waves of blocks as groups of kGroup tokens take, all of them full:
    // of 36,900 tokens, groups of 32 (1.95 waves) take 168 us, of 28 (2.2) 188
    constexpr int kRun = kCacheSms * 4;
    const int waves = std::max(1, (int)(((int64_t)a.tokens + kRun * kGroup - 1) / (kRun * kGroup)));
    const int tokens = std::max(1, (int)(((int64_t)a.tokens + kRun * waves - 1) / (kRun * waves)));
    const unsigned blocks = (unsigned)std::max<int64_t>(1, ((int64_t)a.tokens + tokens - 1) / tokens);
    if (c.head_dim == 64) append_kernel<Q, E, 64><<<blocks, 256, 0, s>>>(c, a, r, tokens);
    else append_kernel<Q, E, 128><<<blocks, 256, 0, s>>>(c, a, r, tokens);
    return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// evict
// ---------------------------------------------------------------------------

// f32 -> u32 with the same order; NaN as -inf, -0 as 0.  Never all ones.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// A reduction over the block, in every thread.
template <int WARPS, typename F>
__device__ __forceinline__ int block_reduce(int v, int *sh, F warp_op, int none) {
    v = warp_op(v);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = warp_op((threadIdx.x & 31) < WARPS ? sh[threadIdx.x & 31] : none);
    __syncthreads();
    return v;
}
// Exclusive prefix sum over the block's threads; total receives the sum.
template <int WARPS>
__device__ __forceinline__ int block_scan(int v, int *sh, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int in = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += x;
    }
    if (lane == 31) sh[warp] = in;
    __syncthreads();
    int w = lane < WARPS ? sh[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += x;
    }
    const int before = warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
    total = __shfl_sync(0xffffffffu, w, 31);
    __syncthreads();
    return before + in - v;
}

// counts[0 .. n), n <= N, replaced by their exclusive prefix sums; total receives the sum.
template <int THREADS, int N>
__device__ __forceinline__ void scan_counts(int *counts, int n, int *sh, int &total) {
    constexpr int PER = (N + THREADS - 1) / THREADS;
    int mine = 0, run[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = (int)threadIdx.x * PER + i;
        run[i] = mine;
        mine += at < n ? counts[at] : 0;
    }
    const int before = block_scan<THREADS / 32>(mine, sh, total);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = (int)threadIdx.x * PER + i;
        if (at < n) counts[at] = before + run[i];
    }
    __syncthreads();
}

// One (sequence, KV head) per block, or per cluster of blocks that all choose
// and then share the moves.  A slot's key is its mass in an order that unsigned
// comparison follows, or all ones where it is recent.
//
//  choose  the smallest key that stays, by a radix select in digits of 11 bits
//          (histogram in shared memory, scan from the top), and how many of
//          the slots that equal it stay, the lowest first;
//  list    the freed slots below the budget and the kept rows above it, both
//          ascending: a ballot per warp and KPT slots a thread, then one scan
//          over the warps' counts;
//  move    row i of the second list into slot i of the first.  A row is read
//          from a slot >= budget and written to one < budget, so no move reads
//          what another writes.
//
// Up to THREADS * KPT slots the keys stay in registers (read once); longer
// caches read them again in each of the passes.  The moves are HBM bound, so
// kMoves 16-byte units of a thread are under way at once.  bf16, 16 sequences
// of 6,000 to 8,192 slots to 4,096, 8 heads of 128: 74 us; 64 sequences that
// give up one of 2,049 slots, which is the choice alone: 20 us, a chain of
// block-wide steps.
constexpr int kDigit = 11, kMoves = 8;

template <int THREADS, int KPT>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) evict_kernel(const S2dCacheView c, const S2dCacheEvict a, int32_t *lists, int share) {
    constexpr int WARPS = THREADS / 32, ROUND = THREADS * KPT, BINS = 1 << kDigit, PER = BINS / THREADS;
    static_assert(KPT <= 32 && WARPS * KPT <= 1024 && PER >= 1, "counts of a round fit the scan");
    __shared__ int sh[32];
    __shared__ int hist[BINS];  // and the warps' counts of a round
    __shared__ longlong2 s_move[THREADS];  // (to, from) elements of rows to move
    __shared__ uint32_t s_digit;
    __shared__ int s_need, s_in;
    const int G = c.kv_heads, pair = (int)blockIdx.x / share, part = (int)blockIdx.x % share, b = pair / G, g = pair % G, tid = threadIdx.x;
    const int cap = c.max_pages * kCachePage, lane = tid & 31, warp = tid >> 5;
    const int n = cache_length(c, b), budget = a.budget;
    if (g == 0 && part == 0 && tid == 0 && a.past) a.past[b] = min(n, budget);
    if (n <= budget) return;  // the whole cluster
    int32_t *pos = c.positions + ((int64_t)b * G + g) * cap;
    float *mass = c.mass + ((int64_t)b * G + g) * cap;
    const int32_t *table = c.page_table + (int64_t)b * c.table_stride;
    const int rounds = (n + ROUND - 1) / ROUND;
    // slot of a thread's i-th key in a round
    auto slot = [&](int r, int i) { return r * ROUND + i * THREADS + tid; };

    // keys of a thread that a round uses
    auto used = [&](int r) { return min(KPT, (n - r * ROUND + THREADS - 1) / THREADS); };

    uint32_t key[KPT];
    float weight[KPT];
    int newest = INT32_MIN;
    for (int r = 0; r < rounds; ++r) {
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            if (i >= used(r)) break;
            const int j = slot(r, i);
            key[i] = (uint32_t)(j < n ? pos[j] : INT32_MIN);  // the position, for now
            weight[i] = rounds == 1 && j < n ? mass[j] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            if (i >= used(r)) break;
            newest = max(newest, (int)key[i]);
        }
    }
    newest = block_reduce<WARPS>(newest, sh, [](int v) { return __reduce_max_sync(0xffffffffu, v); }, INT32_MIN);
    const int64_t edge = (int64_t)newest - a.recent;
    int recents = 0;
    for (int r = 0; r < rounds; ++r)
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            if (i >= used(r)) break;
            const int j = slot(r, i);
            if (j < n && (int64_t)(rounds > 1 ? pos[j] : (int)key[i]) > edge) ++recents;
        }
    recents = block_reduce<WARPS>(recents, sh, [](int v) { return __reduce_add_sync(0xffffffffu, v); }, 0);
    // More recent slots than the budget (positions that repeat): only they can
    // stay, by their mass.  Otherwise all of them stay.
    const bool crowded = recents > budget;
    auto key_of = [&](int position, float w) {
        const bool late = (int64_t)position > edge;
        return late == crowded ? ordered(w) : late ? 0xffffffffu : 0u;
    };
    if (rounds == 1) {
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            if (i >= used(0)) break;
            key[i] = slot(0, i) < n ? key_of((int)key[i], weight[i]) : 0u;
        }
    }
    auto load = [&](int r) {
        if (rounds == 1) return;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            if (i >= used(r)) break;
            const int j = slot(r, i);
            key[i] = j < n ? key_of(pos[j], mass[j]) : 0u;
        }
    };

    // the digits of the smallest key that stays, from the top; need: how many
    // of the keys that share its digits so far stay
    uint32_t least = crowded ? 0u : 0xffffffffu;
    int need = crowded ? budget : budget - recents;
    if (need > 0) {
        // the bits that all of them share are settled; weights are close to
        // one another, and keys that all fall into a few bins wait in line
        uint32_t any = 0, all = 0xffffffffu;
        for (int r = 0; r < rounds; ++r) {
            load(r);
#pragma unroll
            for (int i = 0; i < KPT; ++i) {
                if (i >= used(r)) break;
                if (slot(r, i) < n && key[i] != 0xffffffffu) any |= key[i], all &= key[i];
            }
        }
        any = block_reduce<WARPS>(any, sh, [](uint32_t v) { return __reduce_or_sync(0xffffffffu, v); }, 0u);
        all = block_reduce<WARPS>(all, sh, [](uint32_t v) { return __reduce_and_sync(0xffffffffu, v); }, 0xffffffffu);
        const int open = 32 - __clz(any ^ all);
        uint32_t prefix = open < 32 ? all >> open << open : 0u;
        least = prefix;
        for (int shift = open; shift > 0;) {
            const int from = shift, width = min(kDigit, shift);
            shift -= width;
            for (int i = tid; i < BINS; i += THREADS) hist[i] = 0;
            __syncthreads();
            for (int r = 0; r < rounds; ++r) {
                load(r);
#pragma unroll
                for (int i = 0; i < KPT; ++i) {
                    if (i >= used(r)) break;
                    const uint32_t k = key[i];
                    if (slot(r, i) < n && k != 0xffffffffu && (from == 32 || (k >> from) == (prefix >> from)))
                        atomicAdd(&hist[(k >> shift) & ((1u << width) - 1u)], 1);
                }
            }
            __syncthreads();
            int mine = 0, total;
#pragma unroll
            for (int i = 0; i < PER; ++i) mine += hist[BINS - 1 - tid * PER - i];  // bins from the top, PER a thread
            int above = block_scan<WARPS>(mine, sh, total);
            if (above < need && above + mine >= need) {
#pragma unroll 1
                for (int i = 0; i < PER; ++i) {
                    const int bin = BINS - 1 - tid * PER - i, in = hist[bin];
                    if (above + in >= need) {
                        s_digit = (uint32_t)bin, s_need = need - above, s_in = in;
                        break;
                    }
                    above += in;
                }
            }
            __syncthreads();
            prefix |= s_digit << shift;
            need = s_need;
            least = prefix;
            if (s_in == need) {  // all of them stay: every key from here on
                least = prefix - 1, need = 0;
                break;
            }
            __syncthreads();
        }
    }

    // lists, round by round
    const int most = min(budget, cap - budget);
    int32_t *holes = lists + (int64_t)blockIdx.x * 2 * most, *rows = holes + most;
    int equals = 0, n_holes = 0, n_rows = 0;
    for (int r = 0; r < rounds; ++r) {
        load(r);
        uint32_t keep = 0;  // bit i: the thread's i-th slot of the round stays
        if (need > 0) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < KPT; ++i) {
                if (i >= used(r)) break;
                const uint32_t same = __ballot_sync(0xffffffffu, slot(r, i) < n && key[i] == least);
                if (lane == 0) hist[i * WARPS + warp] = __popc(same);
            }
            __syncthreads();
            int total = 0;
            scan_counts<THREADS, WARPS * KPT>(hist, used(r) * WARPS, sh, total);
#pragma unroll
            for (int i = 0; i < KPT; ++i) {
                if (i >= used(r)) break;
                const bool is = slot(r, i) < n && key[i] == least;
                const uint32_t same = __ballot_sync(0xffffffffu, is);
                const int rank = equals + hist[i * WARPS + warp] + __popc(same & ((1u << lane) - 1u));
                if (is && rank < need) keep |= 1u << i;
            }
            equals += total;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            if (i >= used(r)) break;
            const int j = slot(r, i);
            if (j < n && (key[i] > least || key[i] == 0xffffffffu)) keep |= 1u << i;
            const uint32_t hole = __ballot_sync(0xffffffffu, j < budget && !((keep >> i) & 1u)), row = __ballot_sync(0xffffffffu, j >= budget && ((keep >> i) & 1u));
            if (lane == 0) hist[i * WARPS + warp] = __popc(hole) | __popc(row) << 16;
        }
        __syncthreads();
        int total = 0;
        scan_counts<THREADS, WARPS * KPT>(hist, used(r) * WARPS, sh, total);
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            if (i >= used(r)) break;
            const int j = slot(r, i);
            const bool hole = j < budget && !((keep >> i) & 1u), row = j >= budget && ((keep >> i) & 1u);
            const uint32_t h = __ballot_sync(0xffffffffu, hole), w = __ballot_sync(0xffffffffu, row), below = (1u << lane) - 1u;
            const int at = hist[i * WARPS + warp];
            if (hole) holes[n_holes + (at & 0xffff) + __popc(h & below)] = j;
            if (row) rows[n_rows + (int)((uint32_t)at >> 16) + __popc(w & below)] = j;
        }
        n_holes += total & 0xffff, n_rows += (int)((uint32_t)total >> 16);
    }
    // every block of the cluster has read the positions and the mass that the
    // moves change (and this block has written its lists)
    if (share > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }

    // THREADS rows at a time: a thread works out where one goes, then all copy
    const int units = c.head_dim / 4, half = units / 2;  // 16-byte units of a slot's key and value rows (powers of two)
    const int shift = 31 - __clz(units);
    const int row0 = (int)((int64_t)n_rows * part / share), row1 = (int)((int64_t)n_rows * (part + 1) / share);
    for (int m0 = row0; m0 < row1; m0 += THREADS) {
        const int m = m0 + tid;
        if (m < row1) {
            const int to = holes[m], from = rows[m];
            const int64_t x = cache_row(c, table, g, to), y = cache_row(c, table, g, from);
            s_move[tid] = x < 0 || y < 0 ? make_longlong2(-1, -1) : make_longlong2(x, y);
            pos[to] = pos[from];
            mass[to] = mass[from];
        }
        __syncthreads();
        const int count = min(THREADS, row1 - m0) * units;
        for (int i0 = tid; i0 < count; i0 += kMoves * THREADS) {
            uint4 v[kMoves];
            int64_t to[kMoves];
#pragma unroll
            for (int k = 0; k < kMoves; ++k) {
                const int i = i0 + k * THREADS, u = i & (units - 1);  // the same for all k: THREADS is a multiple of units
                to[k] = -1;
                if (i >= count) continue;
                const longlong2 at = s_move[i >> shift];
                to[k] = at.x;
                if (at.x >= 0) v[k] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(u < half ? c.k : c.v) + at.y + (u & (half - 1)) * 8);
            }
            const int u = i0 & (units - 1);
            uint16_t *base = static_cast<uint16_t *>(u < half ? c.k : c.v) + (u & (half - 1)) * 8;
#pragma unroll
            for (int k = 0; k < kMoves; ++k)
                if (to[k] >= 0) *reinterpret_cast<uint4 *>(base + to[k]) = v[k];
        }
        __syncthreads();
    }
}

// List entries of one (sequence, KV head): at most the slots below the budget
// are freed, at most the slots above it are moved.
size_t evict_list(const S2dCacheView &c, const S2dCacheEvict &a) {
    const int64_t cap = (int64_t)c.max_pages * kCachePage;
    return (size_t)std::max<int64_t>(0, std::min<int64_t>(a.budget, cap - a.budget));
}

// Threads of a block: 16 of a sequence's slots each, in registers, or 32 with
// the most threads; several smaller blocks run on an SM together.
int evict_threads(const S2dCacheView &c) {
    const int64_t cap = (int64_t)c.max_pages * kCachePage;
    return cap <= 256 * 16 ? 256 : cap <= 512 * 16 ? 512 : 1024;
}
// Blocks that share the moves of one (sequence, KV head): as many (up to 8) as
// run at once, as each chooses for itself.
int evict_share(const S2dCacheView &c) {
    const int64_t pairs = (int64_t)c.n_seq * c.kv_heads, most = kCacheSms * (1024 / evict_threads(c));
    int share = 1;
    while (share < 8 && pairs * share * 2 <= most) share *= 2;
    return share;
}

const char *evict_fault(const S2dCacheView *c, const S2dCacheEvict *a) {
    if (const char *f = cache_view_fault(c)) return f;
    if (!a) return "evict arguments are null";
    if (!c->positions || !c->mass) return "eviction needs the cache's positions and mass";
    if (a->budget < 1) return "budget must be at least 1";
    if (a->recent < 0 || a->recent > a->budget) return "recent must be in [0, budget]";
    if (cache_overlap(a->past, sizeof(int32_t) * c->n_seq, c->lengths, sizeof(int32_t) * c->n_seq))
        return "past and lengths must not overlap";
    return nullptr;
}

const char *append_fault(const S2dCacheView *c, const S2dCacheAppend *a) {
    if (const char *f = cache_view_fault(c)) return f;
    if (!a) return "append arguments are null";
    if (a->tokens < 0) return "tokens must not be negative";
    if (!a->past || (a->tokens && (!a->q || !a->k || !a->v || !a->q_out || !a->pos))) return "append has a null buffer";
    if (a->heads <= 0 || a->heads % c->kv_heads) return "heads must be a positive multiple of kv_heads";
    if (a->heads / c->kv_heads > kCacheMaxRep) return "at most 16 query heads per KV head";
    if (!a->q_start && a->tokens > c->n_seq) return "without q_start there is one token per sequence";
    if (a->type != c->type && !(a->type == S2D_TYPE_F32 && c->type == S2D_TYPE_F16))
        return "q, k and v must have the cache's type, or F32 with an F16 cache";
    const int w = a->type == S2D_TYPE_F32 ? 4 : 8;
    const int64_t qrow = (int64_t)a->heads * c->head_dim;
    if (a->q_stride % w || a->k_stride % w || a->v_stride % w || a->q_out_stride % w || !cache_aligned16(a->q) ||
        !cache_aligned16(a->k) || !cache_aligned16(a->v) || !cache_aligned16(a->q_out))
        return "misaligned buffer: rows of q, k, v and q_out must be 16-byte aligned";
    if (a->q_stride < 0 || a->k_stride < 0 || a->v_stride < 0 || (a->tokens > 1 && a->q_out_stride < qrow))
        return "token strides must not be negative, and rows of q_out must not overlap";
    if (a->tokens > 0) {
        // blocks write q_out while others still read q, k and v
        const int64_t es = a->type == S2D_TYPE_F32 ? 4 : 2, kvrow = (int64_t)c->kv_heads * c->head_dim;
        const CacheRows out{a->q_out, a->q_out_stride * es, qrow * es};
        auto shares = [&](const void *p, int64_t stride, int64_t row) { return cache_rows_overlap(out, {p, stride * es, row * es}, a->tokens); };
        if (!(a->q == a->q_out && a->q_stride == a->q_out_stride) && shares(a->q, a->q_stride, qrow)) return "q_out must be q itself or not overlap it";
        if (shares(a->k, a->k_stride, kvrow) || shares(a->v, a->v_stride, kvrow)) return "q_out must not overlap k or v";
    }
    if (!(a->rope_base > 0.0) || !std::isfinite(a->rope_base)) return "rope_base must be positive and finite";
    if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return "eps must be finite and not negative";
    // a block writes lengths while others still read these
    const size_t lengths = sizeof(int32_t) * c->n_seq;
    if (cache_overlap(a->past, lengths, c->lengths, lengths) || cache_overlap(a->q_start, lengths + sizeof(int32_t), c->lengths, lengths) ||
        (a->tokens && cache_overlap(a->pos, sizeof(int32_t) * (size_t)a->tokens, c->lengths, lengths)))
        return "lengths must not overlap past, pos or q_start";
    return nullptr;
}

}  // namespace
}  // namespace s2d

using namespace s2d;

extern "C" int32_t s2d_cache_append(const S2dCacheView *view, const S2dCacheAppend *args, void *stream, char *err,
                                    size_t err_cap) {
    if (const char *f = append_fault(view, args)) return cache_fail(err, err_cap, S2D_EINVAL, f);
    const RopeTurns &r = rope_turns(args->rope_base, view->head_dim);
    DeviceGuard guard(view->device);
    if (guard.error) return cache_cuda(err, err_cap, "cache append: device", guard.error);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = args->type == S2D_TYPE_F32    ? append_launch<float, __half>(*view, *args, r, s)
                          : args->type == S2D_TYPE_F16 ? append_launch<__half, __half>(*view, *args, r, s)
                                                       : append_launch<__nv_bfloat16, __nv_bfloat16>(*view, *args, r, s);
    return cache_cuda(err, err_cap, "cache append", e);
}

extern "C" int32_t s2d_cache_evict_workspace(const S2dCacheView *view, const S2dCacheEvict *args, size_t *bytes, char *err,
                                             size_t err_cap) {
    if (const char *f = evict_fault(view, args)) return cache_fail(err, err_cap, S2D_EINVAL, f);
    if (!bytes) return cache_fail(err, err_cap, S2D_EINVAL, "bytes is null");
    *bytes = sizeof(int32_t) * 2 * evict_list(*view, *args) * (size_t)view->n_seq * view->kv_heads * evict_share(*view);
    return S2D_OK;
}

extern "C" int32_t s2d_cache_evict(const S2dCacheView *view, const S2dCacheEvict *args, void *stream, char *err,
                                   size_t err_cap) {
    size_t need = 0;
    if (const int32_t rc = s2d_cache_evict_workspace(view, args, &need, err, err_cap)) return rc;
    if (need && (!args->workspace || args->workspace_bytes < need || ((uintptr_t)args->workspace & 255u)))
        return cache_fail(err, err_cap, S2D_EINVAL, "workspace is null, too small or not 256-byte aligned");
    DeviceGuard guard(view->device);
    if (guard.error) return cache_cuda(err, err_cap, "cache evict: device", guard.error);
    const int threads = evict_threads(*view), share = evict_share(*view);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)view->n_seq * (unsigned)view->kv_heads * (unsigned)share), cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)share, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr, cfg.numAttrs = 1;
    int32_t *lists = static_cast<int32_t *>(args->workspace);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, threads == 256 ? evict_kernel<256, 16> : threads == 512 ? evict_kernel<512, 16> : evict_kernel<1024, 32>, *view, *args, lists, share);
    return cache_cuda(err, err_cap, "cache evict", e);
}

extern "C" int32_t s2d_cache_status(const S2dCacheView *view, int32_t *bits, void *stream, char *err, size_t err_cap) {
    if (const char *f = cache_view_fault(view)) return cache_fail(err, err_cap, S2D_EINVAL, f);
    if (!bits || !view->status) return cache_fail(err, err_cap, S2D_EINVAL, "no status word to read");
    DeviceGuard guard(view->device);
    cudaError_t e = guard.error;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (!e) e = cudaStreamIsCapturing(s, &capture);
    if (!e && capture != cudaStreamCaptureStatusNone) return cache_fail(err, err_cap, S2D_EINVAL, "the status cannot be read while the stream is captured");
    if (!e) e = cudaMemcpyAsync(bits, view->status, sizeof(int32_t), cudaMemcpyDeviceToHost, s);
    if (!e) e = cudaMemsetAsync(view->status, 0, sizeof(int32_t), s);
    if (!e) e = cudaStreamSynchronize(s);
    return cache_cuda(err, err_cap, "cache status", e);
}

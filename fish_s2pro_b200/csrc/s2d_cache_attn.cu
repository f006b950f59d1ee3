// s2d_cache_attn.cu -- attention over a shared prefix and paged caches
// (s2d_cache_attention, include/s2d_cache.h).
//
// The softmax of a query row over [prefix ; own slots] is put together from
// parts: over any set of positions, m = max s, l = sum 2^(s - m) and
// O = sum 2^(s - m) v (s = scale * log2(e) * q . k) are enough, and parts
// join by rescaling with 2^(m_i - m).  The prefix is the same for every
// sequence, so the query rows of all sequences that share a KV head
// (tokens * heads / kv_heads of them) are its rows together.
#include "s2d_cache.cuh"

#include <math.h>

#include <algorithm>

namespace s2d {

namespace {

__device__ __forceinline__ void cp_async16(void *dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)),
                 "l"(src), "r"(valid ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p)));
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p)));
}
// c += A (16 x 16) . B (16 x 8) in the element type of the cache, f32 sums
template <typename E>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename E>
__device__ __forceinline__ uint32_t pack2(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename E>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&v));
}
// (x, y) = hi + lo, both of the cache's type
template <typename E>
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    hi = pack2<E>(x, y);
    const float2 h = unpack2<E>(hi);
    lo = pack2<E>(x - h.x, y - h.y);
}

__device__ __forceinline__ void store_out(float *p, float x) { *p = x; }
__device__ __forceinline__ void store_out(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void store_out(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

constexpr float kLog2e = 1.4426950408889634f;

// What a part (pm, pl) counts in a softmax whose maximum is m: nothing if it
// saw no position (or only scores of -inf), all of it if its scores are NaN
// (which fmaxf leaves out of pm), so that a NaN reaches its row.
__device__ __forceinline__ float part_factor(float pm, float pl, float m) {
    return pm == -INFINITY ? (pl == 0.f ? 0.f : 1.f) : exp2f(pm - m);
}

// How the call is cut up (from sizes that the host knows).
struct AttnPlan {
    int rep;                        // query heads per KV head
    int prefix_tiles, prefix_splits;  // row tiles over the pooled rows; position splits
    int own_tiles, own_splits;      // at most this many row tiles over all sequences
    int parts;                      // prefix_splits (0 without a prefix) + own_splits
    float *part;                    // [tokens][heads][parts][2 + head_dim]
    float *lse2;                    // [tokens][heads], base 2 (weigh)
};
constexpr int kTileRows = 8;

// Rows that belong to some sequence: tokens [0, this).
__device__ __forceinline__ int real_tokens(const S2dCacheAttention &a, int n_seq) {
    const int n = a.q_start ? __ldg(a.q_start + n_seq) : n_seq;
    return max(0, min(n, a.tokens));
}

// The sequence and its row tile behind own tile `tile` (tiles of `rows` rows,
// the sequences' tiles one after the other); b = -1 when there is none.
// Called by a whole warp.
__device__ __forceinline__ void find_tile(const S2dCacheView &c, const S2dCacheAttention &a, int rep, int rows, int &tile,
                                          int &b) {
    if (!a.q_start) {
        const int per = (rep + rows - 1) / rows;
        b = tile / per, tile %= per;
        if (b >= min(c.n_seq, a.tokens)) b = -1;
        return;
    }
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < c.n_seq; b0 += 32) {
        int first, n = 0;
        if (b0 + lane < c.n_seq) n = (int)(((int64_t)cache_tokens(a.q_start, a.tokens, b0 + lane, first, c.status) * rep + rows - 1) / rows);
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, sum > tile);
        if (past) {
            const int l = __ffs(past) - 1;
            tile -= __shfl_sync(0xffffffffu, sum - n, l);
            b = b0 + l;
            return;
        }
        tile -= __shfl_sync(0xffffffffu, sum, 31);
    }
    b = -1;
}

// The query row of a lane's MMA row (g = lane / 4), as A fragments: rows g
// hold q (its rounding to the cache's type if q is f32), rows g + 8 the f32
// remainder.  f32 rows are scaled by the power of two that puts their largest
// element near 2^14, so that the remainder stays a normal f16; qmul takes it
// out of the scores again, along with scale * log2(e).
template <typename Q, typename E, int HD>
__device__ __forceinline__ void load_q(const Q *row, float scale, int t, uint32_t (&qa)[HD / 16][4], float &qmul) {
    if constexpr (sizeof(Q) == 4) {
        float qv[HD / 16][4], amax = 0.f;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            float2 v0 = make_float2(0.f, 0.f), v1 = v0;
            if (row) {
                v0 = *reinterpret_cast<const float2 *>(row + 16 * k + 2 * t);
                v1 = *reinterpret_cast<const float2 *>(row + 16 * k + 2 * t + 8);
            }
            qv[k][0] = v0.x, qv[k][1] = v0.y, qv[k][2] = v1.x, qv[k][3] = v1.y;
#pragma unroll
            for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(qv[k][e]));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        int ex = 0;
        frexpf(amax, &ex);
        ex = max(ex, -100);  // 2^(14 - ex) stays finite for the smallest rows
        const float up = ldexpf(1.f, 14 - ex);
        qmul = scale * kLog2e * ldexpf(1.f, ex - 14);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            split2<E>(qv[k][0] * up, qv[k][1] * up, qa[k][0], qa[k][1]);
            split2<E>(qv[k][2] * up, qv[k][3] * up, qa[k][2], qa[k][3]);
        }
    } else {
        qmul = scale * kLog2e;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            qa[k][0] = row ? *reinterpret_cast<const uint32_t *>(row + 16 * k + 2 * t) : 0u;
            qa[k][2] = row ? *reinterpret_cast<const uint32_t *>(row + 16 * k + 2 * t + 8) : 0u;
            qa[k][1] = qa[k][3] = 0u;
        }
    }
}

// One block: 8 query rows (MMA rows 0-7 their values, 8-15 the remainders of
// what the cache's type rounds: f32 queries, and the weights of every type)
// against one split of the positions, four warps taking its 16-position
// chunks in turn.
template <typename Q, typename E, int HD>
__global__ void __launch_bounds__(128) part_kernel(const S2dCacheView c, const S2dCacheAttention a, const AttnPlan p) {
    constexpr int KC = 16, NO = HD / 8, UNITS = HD / 8, PITCH = HD * 2 + 16, STAGE = 2 * KC * PITCH, NW = 4;
    extern __shared__ __align__(16) uint8_t sm[];
    const int G = c.kv_heads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, t = lane & 3;
    const int prefix_items = p.prefix_tiles * p.prefix_splits * G;
    int item = (int)blockIdx.x;
    const bool own = item >= prefix_items;
    if (own) item -= prefix_items;
    const int g = item % G;
    item /= G;
    const int splits = own ? p.own_splits : p.prefix_splits, split = item % splits;
    int tile = item / splits, b = 0, first = 0, n_rows, span, limit;
    const int32_t *table = a.prefix_pages;
    if (own) {
        find_tile(c, a, p.rep, kTileRows, tile, b);
        if (b < 0) return;
        const int nt = cache_tokens(a.q_start, a.tokens, b, first, c.status), n = cache_length(c, b);
        table = c.page_table + (int64_t)b * c.table_stride;
        n_rows = nt * p.rep - tile * kTileRows;
        const int tok = tile * kTileRows + min(gl, n_rows - 1), last = tile * kTileRows + min(kTileRows, n_rows) - 1;
        limit = max(0, n - nt + tok / p.rep + 1);
        span = max(0, n - nt + last / p.rep + 1);
    } else {
        n_rows = real_tokens(a, c.n_seq) * p.rep - tile * kTileRows;
        if (n_rows <= 0) return;
        limit = span = a.prefix_len;
    }
    n_rows = min(n_rows, kTileRows);
    const int r = tile * kTileRows + gl, tok = first + r / p.rep, head = g * p.rep + r % p.rep;
    const bool real = gl < n_rows;
    const int nch = (span + KC - 1) / KC, per = (nch + splits - 1) / splits;
    const int ch0 = min(nch, split * per), ch1 = min(nch, ch0 + per);

    uint8_t *ring = sm + (size_t)warp * 2 * STAGE;
    auto issue = [&](int ch, int stage) {
        uint8_t *kt = ring + (size_t)stage * STAGE, *vt = kt + KC * PITCH;
        const int64_t at = cache_row(c, table, g, ch * KC);  // a chunk never spans two pages
        const int n = at < 0 ? 0 : min(KC, span - ch * KC);
        const char *ks = static_cast<const char *>(c.k) + 2 * max(at, (int64_t)0), *vs = static_cast<const char *>(c.v) + 2 * max(at, (int64_t)0);
#pragma unroll
        for (int i = 0; i < KC * UNITS / 32; ++i) {
            const int u = lane + 32 * i, row = u / UNITS, cc = u % UNITS;
            const int64_t src = (int64_t)(row < n ? row : 0) * (HD * 2) + cc * 16;
            cp_async16(kt + row * PITCH + cc * 16, ks + src, row < n);
            cp_async16(vt + row * PITCH + cc * 16, vs + src, row < n);
        }
        cp_commit();
        return n;
    };
    uint32_t qa[HD / 16][4];
    float qmul;
    load_q<Q, E, HD>(real ? static_cast<const Q *>(a.q) + (int64_t)tok * a.q_stride + (int64_t)head * HD : nullptr, a.scale, t, qa, qmul);

    float o[NO][4];
#pragma unroll
    for (int j = 0; j < NO; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float mrun = -INFINITY, lrun = 0.f;
    int ch = ch0 + warp, have = 0, next = 0;
    if (ch < ch1) have = issue(ch, 0);
    for (int stage = 0; ch < ch1; ch += NW, stage ^= 1, have = next) {
        if (ch + NW < ch1) next = issue(ch + NW, stage ^ 1);
        else cp_commit();
        cp_wait<1>();
        __syncwarp();
        const uint8_t *kt = ring + (size_t)stage * STAGE, *vt = kt + KC * PITCH;
        float s[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < HD / 32; ++kk)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t kf[4];
                ldsm4(kf, kt + (q * 8 + (lane & 7)) * PITCH + (kk * 32 + (lane >> 3) * 8) * 2);
                mma<E>(s[q], qa[2 * kk], kf[0], kf[1]);
                mma<E>(s[q], qa[2 * kk + 1], kf[2], kf[3]);
            }
        float x[2][2], mx = -INFINITY;
        const int vis = min(have, limit - ch * KC);
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                x[q][e] = q * 8 + 2 * t + e < vis ? (s[q][e] + s[q][2 + e]) * qmul : -INFINITY;
                mx = fmaxf(mx, x[q][e]);
            }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mnew = fmaxf(mrun, mx), base = mnew == -INFINITY ? 0.f : mnew;  // nothing seen yet: all weights 0
        const float corr = exp2f(mrun - base);
        mrun = mnew;
        uint32_t pa[4];
        float sum = 0.f;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const float p0 = exp2f(x[q][0] - base), p1 = exp2f(x[q][1] - base);
            sum += p0 + p1;
            split2<E>(p0, p1, pa[2 * q], pa[2 * q + 1]);
        }
        lrun = fmaf(lrun, corr, sum);
#pragma unroll
        for (int j = 0; j < NO; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] *= corr;
#pragma unroll
        for (int nd = 0; nd < HD / 16; ++nd) {
            uint32_t vf[4];
            ldsm4_trans(vf, vt + ((lane & 7) + ((lane >> 3) & 1) * 8) * PITCH + (nd * 16 + (lane >> 4) * 8) * 2);
            mma<E>(o[2 * nd], pa, vf[0], vf[1]);
            mma<E>(o[2 * nd + 1], pa, vf[2], vf[3]);
        }
        __syncwarp();  // the stage is read before it is filled again
    }
    cp_wait<0>();
    __syncthreads();

    // join the warps: [warp][row][2 + HD] over the drained rings
    float *ms = reinterpret_cast<float *>(sm);
    lrun += __shfl_xor_sync(0xffffffffu, lrun, 1);
    lrun += __shfl_xor_sync(0xffffffffu, lrun, 2);
    float *w = ms + (warp * kTileRows + gl) * (HD + 2);
    if (t == 0) w[0] = mrun, w[1] = lrun;
#pragma unroll
    for (int j = 0; j < NO; ++j) {
        w[2 + j * 8 + 2 * t] = o[j][0] + o[j][2];
        w[2 + j * 8 + 2 * t + 1] = o[j][1] + o[j][3];
    }
    __syncthreads();
    const int part = own ? (p.parts - p.own_splits) + split : split;
    for (int i = threadIdx.x; i < n_rows * HD; i += 128) {
        const int row = i / HD, d = i % HD, rr = tile * kTileRows + row;
        float m = -INFINITY, l = 0.f, sum = 0.f;
#pragma unroll
        for (int k = 0; k < NW; ++k) m = fmaxf(m, ms[(k * kTileRows + row) * (HD + 2)]);
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            const float *ws = ms + (k * kTileRows + row) * (HD + 2);
            const float f = part_factor(ws[0], ws[1], m);
            l = fmaf(ws[1], f, l), sum = fmaf(ws[2 + d], f, sum);
        }
        float *to = p.part + (((int64_t)(first + rr / p.rep) * a.heads + g * p.rep + rr % p.rep) * p.parts + part) * (HD + 2);
        if (d == 0) to[0] = m, to[1] = l;
        to[2 + d] = sum;
    }
}

// One warp per (token, head): joins its parts in their order.
template <typename Q, int HD>
__global__ void __launch_bounds__(128) join_kernel(const S2dCacheView c, const S2dCacheAttention a, const AttnPlan p) {
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (id >= (int64_t)real_tokens(a, c.n_seq) * a.heads) return;
    const int64_t tok = id / a.heads;
    const int head = (int)(id % a.heads);
    const float *part = p.part + id * p.parts * (HD + 2);
    float m = -INFINITY, l = 0.f, o[HD / 32] = {};
    for (int k = 0; k < p.parts; ++k) m = fmaxf(m, part[k * (HD + 2)]);
    for (int k = 0; k < p.parts; ++k) {
        const float *w = part + k * (HD + 2);
        const float f = part_factor(w[0], w[1], m);
        l = fmaf(w[1], f, l);
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) o[i] = fmaf(w[2 + lane + 32 * i], f, o[i]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: zeros
    Q *out = static_cast<Q *>(a.out) + tok * a.out_stride + (int64_t)head * HD;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) store_out(out + lane + 32 * i, o[i] * inv);
    if (lane == 0) {
        const float lse2 = l == 0.f ? -INFINITY : m + log2f(l);
        if (a.lse) a.lse[id] = lse2 * 0.6931471805599453f;
        if (p.lse2) p.lse2[id] = lse2;
    }
}

// mass[b][g][slot] += sum over the rows that see the slot of 2^(s - lse2): the
// scores again, as S^T = K Q^T, so that a slot's weights lie in one quad's
// registers and are added in the order of the rows.  A block takes 64 slots,
// a warp 16 of them.
template <typename Q, typename E, int HD>
__global__ void __launch_bounds__(128) weigh_kernel(const S2dCacheView c, const S2dCacheAttention a, const AttnPlan p) {
    const int G = c.kv_heads, b = blockIdx.y, g = blockIdx.z, lane = threadIdx.x & 31, gl = lane >> 2, t = lane & 3;
    int first;
    const int n = cache_length(c, b), nt = cache_tokens(a.q_start, a.tokens, b, first, c.status);
    const int j0 = (int)blockIdx.x * kCachePage + (threadIdx.x >> 5) * 16;
    if (j0 >= n || nt == 0) return;
    const int64_t at = cache_row(c, c.page_table + (int64_t)b * c.table_stride, g, j0);
    if (at < 0) return;
    const uint16_t *k = static_cast<const uint16_t *>(c.k) + at;
    uint32_t ka[HD / 16][4];  // slots j0 + gl and j0 + gl + 8
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = gl + 8 * (i & 1);
            ka[kk][i] = j0 + row < n ? *reinterpret_cast<const uint32_t *>(k + (int64_t)row * HD + 16 * kk + 8 * (i >> 1) + 2 * t) : 0u;
        }
    float sum[2] = {};
    const int rows = nt * p.rep;
    // rows before this one see none of the block's slots
    const int skip = max(0, j0 - (n - nt)) * p.rep / 8 * 8;
    for (int r0 = skip; r0 < rows; r0 += 8) {
        const int r = r0 + gl;  // the lane loads query row r as column gl of B
        uint32_t qa[HD / 16][4];
        float qmul;
        load_q<Q, E, HD>(r < rows ? static_cast<const Q *>(a.q) + (int64_t)(first + r / p.rep) * a.q_stride + (int64_t)(g * p.rep + r % p.rep) * HD : nullptr,
                         a.scale, t, qa, qmul);
        const float mine = r < rows ? p.lse2[(int64_t)(first + r / p.rep) * a.heads + g * p.rep + r % p.rep] : -INFINITY;
        float s[4] = {};
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
            mma<E>(s, ka[kk], qa[kk][0], qa[kk][2]);
            if constexpr (sizeof(Q) == 4) mma<E>(s, ka[kk], qa[kk][1], qa[kk][3]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int col = 2 * t + e;
            const float lse2 = __shfl_sync(0xffffffffu, mine, col * 4), qm = __shfl_sync(0xffffffffu, qmul, col * 4);
            const int seen = n - nt + (r0 + col) / p.rep + 1;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (lse2 != -INFINITY && j0 + gl + 8 * i < seen) sum[i] += exp2f(fmaf(s[2 * i + e], qm, -lse2));
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
        const int j = j0 + gl + 8 * i;
        if (t == 0 && j < n) c.mass[((int64_t)b * G + g) * c.max_pages * kCachePage + j] += sum[i];
    }
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

const char *attention_fault(const S2dCacheView *c, const S2dCacheAttention *a) {
    if (const char *f = cache_view_fault(c)) return f;
    if (!a) return "attention arguments are null";
    if (a->tokens < 0) return "tokens must not be negative";
    if (a->tokens && (!a->q || !a->out)) return "attention has a null buffer";
    if (a->heads <= 0 || a->heads % c->kv_heads) return "heads must be a positive multiple of kv_heads";
    if (a->heads / c->kv_heads > kCacheMaxRep) return "at most 16 query heads per KV head";
    if (!a->q_start && a->tokens > c->n_seq) return "without q_start there is one token per sequence";
    if (a->type != c->type && !(a->type == S2D_TYPE_F32 && c->type == S2D_TYPE_F16))
        return "q must have the cache's type, or F32 with an F16 cache";
    if (a->prefix_len < 0 || a->prefix_len > (1 << 24)) return "prefix_len must be in [0, 2^24]";
    if (a->prefix_len && !a->prefix_pages) return "a prefix needs its pages";
    if (a->weigh && !c->mass) return "weighing needs the cache's mass";
    if (!std::isfinite(a->scale)) return "scale must be finite";
    if ((int64_t)a->tokens * a->heads > (1 << 26)) return "at most 2^26 query rows";
    const int w = a->type == S2D_TYPE_F32 ? 4 : 8;
    const int64_t row = (int64_t)a->heads * c->head_dim;
    if (a->q_stride % w || a->out_stride % w || !cache_aligned16(a->q) || !cache_aligned16(a->out))
        return "misaligned buffer: rows of q and out must be 16-byte aligned";
    if (a->q_stride < 0 || (a->tokens > 1 && a->out_stride < row)) return "q_stride must not be negative, and rows of out must not overlap";
    return nullptr;
}

void make_plan(const S2dCacheView &c, const S2dCacheAttention &a, AttnPlan &p, size_t &bytes) {
    p = {};
    p.rep = a.heads / c.kv_heads;
    const int64_t rows = (int64_t)a.tokens * p.rep;
    const int target = 2 * 148;
    auto cut = [&](int64_t blocks, int64_t positions) {  // splits that fill the GPU, of at least 64 positions
        const int64_t want = (target + blocks - 1) / std::max<int64_t>(blocks, 1);
        return (int)std::max<int64_t>(1, std::min<int64_t>({want, (positions + 63) / 64, 64}));
    };
    if (a.prefix_len) {
        p.prefix_tiles = (int)((rows + kTileRows - 1) / kTileRows);
        p.prefix_splits = cut((int64_t)p.prefix_tiles * c.kv_heads, a.prefix_len);
    }
    p.own_tiles = (int)(a.q_start ? rows / kTileRows + c.n_seq : (int64_t)a.tokens * ((p.rep + kTileRows - 1) / kTileRows));
    p.own_splits = cut((int64_t)p.own_tiles * c.kv_heads, (int64_t)c.max_pages * kCachePage);
    p.parts = p.prefix_splits + p.own_splits;
    const size_t part = align256(sizeof(float) * (size_t)a.tokens * a.heads * p.parts * (c.head_dim + 2));
    bytes = part + (a.weigh ? align256(sizeof(float) * (size_t)a.tokens * a.heads) : 0);
    char *w = static_cast<char *>(a.workspace);
    p.part = reinterpret_cast<float *>(w);
    p.lse2 = a.weigh && w ? reinterpret_cast<float *>(w + part) : nullptr;
}

template <typename Q, typename E, int HD>
cudaError_t attention_launch(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p, cudaStream_t s) {
    const size_t smem = (size_t)4 * 2 * 2 * 16 * (HD * 2 + 16);  // also holds the join: 4 warps x 8 rows x (HD + 2) floats
    cudaError_t e = cudaFuncSetAttribute(part_kernel<Q, E, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e) return e;
    const int64_t items = ((int64_t)p.prefix_tiles * p.prefix_splits + (int64_t)p.own_tiles * p.own_splits) * c.kv_heads;
    if (items > 0x7fffffff) return cudaErrorInvalidValue;
    part_kernel<Q, E, HD><<<(unsigned)items, 128, smem, s>>>(c, a, p);
    if ((e = cudaGetLastError())) return e;
    join_kernel<Q, HD><<<(unsigned)(((int64_t)a.tokens * a.heads + 3) / 4), 128, 0, s>>>(c, a, p);
    if ((e = cudaGetLastError()) || !a.weigh) return e;
    weigh_kernel<Q, E, HD><<<dim3((unsigned)c.max_pages, (unsigned)c.n_seq, (unsigned)c.kv_heads), 128, 0, s>>>(c, a, p);
    return cudaGetLastError();
}

template <typename Q, typename E>
cudaError_t attention_launch(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p, cudaStream_t s) {
    return c.head_dim == 64 ? attention_launch<Q, E, 64>(c, a, p, s) : attention_launch<Q, E, 128>(c, a, p, s);
}

}  // namespace
}  // namespace s2d

using namespace s2d;

extern "C" int32_t s2d_cache_attention_workspace(const S2dCacheView *view, const S2dCacheAttention *args, size_t *bytes,
                                                 char *err, size_t err_cap) {
    if (const char *f = attention_fault(view, args)) return cache_fail(err, err_cap, S2D_EINVAL, f);
    if (!bytes) return cache_fail(err, err_cap, S2D_EINVAL, "bytes is null");
    AttnPlan p;
    make_plan(*view, *args, p, *bytes);
    return S2D_OK;
}

extern "C" int32_t s2d_cache_attention(const S2dCacheView *view, const S2dCacheAttention *args, void *stream, char *err,
                                       size_t err_cap) {
    if (const char *f = attention_fault(view, args)) return cache_fail(err, err_cap, S2D_EINVAL, f);
    if (args->tokens == 0) return S2D_OK;
    AttnPlan p;
    size_t need = 0;
    make_plan(*view, *args, p, need);
    if (need && (!args->workspace || args->workspace_bytes < need || ((uintptr_t)args->workspace & 255u)))
        return cache_fail(err, err_cap, S2D_EINVAL, "workspace is null, too small or not 256-byte aligned");
    DeviceGuard guard(view->device);
    if (guard.error) return cache_cuda(err, err_cap, "cache attention: device", guard.error);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = args->type == S2D_TYPE_F32    ? attention_launch<float, __half>(*view, *args, p, s)
                          : args->type == S2D_TYPE_F16 ? attention_launch<__half, __half>(*view, *args, p, s)
                                                       : attention_launch<__nv_bfloat16, __nv_bfloat16>(*view, *args, p, s);
    return cache_cuda(err, err_cap, "cache attention", e);
}

// s2d_cache_attn.cu -- attention over a shared prefix and paged caches
// (s2d_cache_attention, include/s2d_cache.h).
//
// The softmax of a query row over [prefix ; own slots] is put together from
// parts: over any set of positions, m = max s, l = sum 2^(s - m) and
// O = sum 2^(s - m) v (s = scale * log2(e) * q . k) are enough, and parts
// join by rescaling with 2^(m_i - m).  The prefix is the same for every
// sequence, so the query rows of all sequences that share a KV head
// (tokens * heads / kv_heads of them) are its rows together.
#include "s2d_cache_attn.cuh"

#include <math.h>
#include <string.h>

#include <type_traits>

#include <algorithm>

namespace s2d {

namespace {

__device__ __forceinline__ void cp_async16(void *dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)),
                 "l"(src), "r"(valid ? 16 : 0)
                 : "memory");
}

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

__device__ __forceinline__ void store_out4(float *p, const float (&x)[4]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
template <typename E>
__device__ __forceinline__ void store_out4(E *p, const float (&x)[4]) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<E>(x[0], x[1]), pack2<E>(x[2], x[3]));
}

// All threads of the cluster's CTAs (of the CTA where it is alone).
__device__ __forceinline__ void cluster_sync(int size) {
    if (size == 1) {
        __syncthreads();
        return;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// *p in the shared memory of CTA `rank` of the cluster
template <typename T>
__device__ __forceinline__ T cluster_get(const T *p, int rank, int size) {
    static_assert(sizeof(T) == 4 || sizeof(T) == 8 || sizeof(T) == 16, "one, two or four words");
    if (size == 1) return *p;
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    T v;
    if constexpr (sizeof(T) == 4) {
        uint32_t x;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
        memcpy(&v, &x, 4);
    } else if constexpr (sizeof(T) == 16) {
        uint4 x;
        asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
        memcpy(&v, &x, 16);
    } else {
        uint2 x;
        asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(x.x), "=r"(x.y) : "r"(at) : "memory");
        memcpy(&v, &x, 8);
    }
    return v;
}

// The query row of a lane's MMA row (g = lane / 4, t = lane % 4), as A
// fragments: rows g hold q (its rounding to the cache's type if q is f32), rows
// g + 8 the f32 remainder.  f32 rows are scaled by the power of two that puts
// their largest element near 2^14, so that the remainder stays a normal f16
// (at most by 2^114, which keeps rows of subnormal numbers finite); qmul takes
// it out of the scores again, along with scale * log2(e).
template <typename Q, typename E, int HD>
struct QueryRow {
    uint2 raw[HD / 16][2];  // elements 16 k + 2 t and 16 k + 2 t + 8 with the next, under way (f32: two words; else one)

    __device__ __forceinline__ void load(const Q *row, int t) {
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const Q *at = row + 16 * k + 8 * i + 2 * t;
                raw[k][i] = make_uint2(0u, 0u);
                if (!row) continue;
                if constexpr (sizeof(Q) == 4) raw[k][i] = *reinterpret_cast<const uint2 *>(at);
                else raw[k][i].x = *reinterpret_cast<const uint32_t *>(at);
            }
    }
    __device__ __forceinline__ void fragments(float scale, uint32_t (&qa)[HD / 16][4], float &qmul) const {
        qmul = scale * kLog2e;
        if constexpr (sizeof(Q) == 4) {
            float amax = 0.f;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(raw[k][i].x)), fabsf(__uint_as_float(raw[k][i].y))));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int ex = max((int)(__float_as_uint(amax) >> 23) - 126, -100);
            const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
            qmul *= __uint_as_float((uint32_t)(127 + ex - 14) << 23);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    split2<E>(__uint_as_float(raw[k][i].x) * up, __uint_as_float(raw[k][i].y) * up, qa[k][2 * i], qa[k][2 * i + 1]);
        } else {
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) qa[k][2 * i] = raw[k][i].x, qa[k][2 * i + 1] = 0u;
        }
    }
};

constexpr int kMaxParts = 64;  // position splits of the prefix, or of own slots: parts of a row are at most as many and two

// Single tokens: the rep <= 8 query heads of one (sequence, KV head) against
// the sequence's own slots, shared by the CTAs of a cluster (chunks of 16
// slots, contiguous ranges) and in each by four warps in turn, every warp with
// its own two-stage copy ring.  MMA rows 0-7 hold the heads' values, rows 8-15
// the remainders of what the cache's type rounds (f32 queries, and the weights
// of every type), so the sums have f32's precision at no extra MMA.  f16 has no
// exponents below 2^-24: weights are taken from a reference 2^14 below the
// maximum, which leaves every one of them right to 2^-39 of the largest (from
// the maximum itself it was 2^-25: 32,768 slots 25 binades below one of them
// lost a quarter of what they add, 2.4e-4).  An MMA truncates what it adds to, so
// each chunk starts from 0 and is added to O with rounding, in the instruction
// that rescales O anyway (summed in the MMAs, equal weights over 32,768 slots
// came out 5.1e-5 too small, over 131,072 2.1e-4).
//
// The CTAs' parts meet through distributed shared memory; without a prefix the
// call needs no kernel to join them.  KEEP (weighing): the scores stay in
// shared memory until the row's sum over prefix and own slots is known, and
// each CTA adds its slots' weights to the mass: the keys are read once and no
// score leaves the SM.  What a CTA reads at its end (the mass, the prefix's
// parts) is under way before the parts meet: 1 us a read, 140 us a call
// instead of 146.
//
// HBM bound: f16, 64 sequences of 1,025 to 4,096 slots, 32 and 8 heads of 128,
// weighing: 140 us, 4.9 TB/s with the prefix's launch.  Two CTAs share an SM;
// the rest is their beginnings and ends, which more and smaller CTAs do not
// hide (2 warps: 139 us, 1: 147).
template <typename Q, typename E, int HD, bool KEEP>
__global__ void __launch_bounds__(128) token_kernel(const S2dCacheView c, const S2dCacheAttention a, const AttnPlan p, int score_pitch) {
    constexpr int KC = 16, NO = HD / 8, UNITS = HD / 8, PITCH = HD * 2 + 16, STAGE = 2 * KC * PITCH, NW = 4, R = 8;
    constexpr float kBelow = std::is_same<E, __half>::value ? 14.f : 0.f;  // the reference of the weights below their maximum
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ float2 s_ml[R];        // this CTA's (m, l) of each row
    __shared__ float s_lse[R];        // lse2 of each row
    __shared__ float s_rank[R][16];   // what each CTA's part counts, over the row's sum
    float *s_o = reinterpret_cast<float *>(sm + NW * 2 * STAGE);  // [R][HD]: this CTA's O
    float *s_pre = s_o + R * HD;                                  // [R][parts]: what each prefix part counts
    float *s_score = s_pre + R * p.parts;                         // [rep][score_pitch]
    const int G = c.kv_heads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, t = lane & 3;
    const int S = p.own_splits, rank = (int)blockIdx.x % S;
    int item = (int)blockIdx.x / S;
    const int groups = (p.rep + R - 1) / R, grp = item % groups;  // more than 8 heads: groups of 8
    item /= groups;
    const int g = item % G, b = item / G;
    const int head0 = g * p.rep + grp * R, n_rows = min(R, p.rep - grp * R);
    const int32_t *table = c.page_table + (int64_t)b * c.table_stride;
    // what the first copies and scores wait for, all under way together: the
    // length, 32 page ids (id `lane` of a window, read again as the window
    // moves on), the query rows
    int ids = __ldg(table + min(lane, c.max_pages - 1)), window = 0;
    QueryRow<Q, E, HD> query;
    query.load(gl < n_rows ? static_cast<const Q *>(a.q) + (int64_t)b * a.q_stride + (int64_t)(head0 + gl) * HD : nullptr, t);
    const int n = cache_length(c, b), nch = (n + KC - 1) / KC, per = (nch + S - 1) / S;
    const int ch0 = min(nch, rank * per), ch1 = min(nch, ch0 + per);

    uint8_t *ring = sm + (size_t)warp * 2 * STAGE;
    auto issue = [&](int ch, int stage) {
        uint8_t *kt = ring + (size_t)stage * STAGE, *vt = kt + KC * PITCH;
        const int at_page = ch * KC / kCachePage;  // a chunk never spans two pages
        if (at_page / 32 != window) {
            window = at_page / 32;
            ids = __ldg(table + min(window * 32 + lane, c.max_pages - 1));
        }
        const int page = __shfl_sync(0xffffffffu, ids, at_page & 31);
        const bool good = (uint32_t)page < (uint32_t)c.n_pages;
        if (!good) cache_flag(c.status, S2D_CACHE_BAD_PAGE);
        const int have = good ? min(KC, n - ch * KC) : 0;
        const int64_t at = (int64_t)(good ? page : 0) * c.page_stride + (int64_t)g * c.head_stride + (int64_t)(ch * KC % kCachePage) * HD;
        const char *ks = static_cast<const char *>(c.k) + 2 * at, *vs = static_cast<const char *>(c.v) + 2 * at;
#pragma unroll
        for (int i = 0; i < KC * UNITS / 32; ++i) {
            const int u = lane + 32 * i, row = u / UNITS, cc = u % UNITS;
            const int src = (row < have ? row : 0) * (HD * 2) + cc * 16;
            cp_async16(kt + row * PITCH + cc * 16, ks + src, row < have);
            cp_async16(vt + row * PITCH + cc * 16, vs + src, row < have);
        }
        cp_commit();
        return have;
    };
    int ch = ch0 + warp, have = 0, next = 0;
    if (ch < ch1) have = issue(ch, 0);
    uint32_t qa[HD / 16][4];
    float qmul;
    query.fragments(a.scale, qa, qmul);

    float o[NO][4];
#pragma unroll
    for (int j = 0; j < NO; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float mrun = -INFINITY, lrun = 0.f;
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
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                x[q][e] = q * 8 + 2 * t + e < have ? (s[q][e] + s[q][2 + e]) * qmul : -INFINITY;
                mx = fmaxf(mx, x[q][e]);
            }
            if (KEEP && gl < n_rows)
                *reinterpret_cast<float2 *>(s_score + gl * score_pitch + (ch - ch0) * KC + q * 8 + 2 * t) = make_float2(x[q][0], x[q][1]);
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mnew = fmaxf(mrun, mx - kBelow), base = mnew == -INFINITY ? 0.f : mnew;  // nothing seen yet: all weights 0
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
        for (int nd = 0; nd < HD / 16; ++nd) {
            uint32_t vf[4];
            ldsm4_trans(vf, vt + ((lane & 7) + ((lane >> 3) & 1) * 8) * PITCH + (nd * 16 + (lane >> 4) * 8) * 2);
            float d[2][4] = {};
            mma<E>(d[0], pa, vf[0], vf[1]);
            mma<E>(d[1], pa, vf[2], vf[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[2 * nd][e] = fmaf(o[2 * nd][e], corr, d[0][e]), o[2 * nd + 1][e] = fmaf(o[2 * nd + 1][e], corr, d[1][e]);
        }
        __syncwarp();  // the stage is read before it is filled again
    }
    cp_wait<0>();
    __syncthreads();

    // join the warps, over the drained rings: [warp][row][HD + 2]
    float *ms = reinterpret_cast<float *>(sm);
    lrun += __shfl_xor_sync(0xffffffffu, lrun, 1);
    lrun += __shfl_xor_sync(0xffffffffu, lrun, 2);
    float *w = ms + (warp * R + gl) * (HD + 2);
    if (t == 0) w[0] = mrun, w[1] = lrun;
#pragma unroll
    for (int j = 0; j < NO; ++j) {
        w[2 + j * 8 + 2 * t] = o[j][0] + o[j][2];
        w[2 + j * 8 + 2 * t + 1] = o[j][1] + o[j][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n_rows * HD; i += 128) {
        const int row = i / HD, d = i % HD;
        float m = -INFINITY, l = 0.f, sum = 0.f;
#pragma unroll
        for (int k = 0; k < NW; ++k) m = fmaxf(m, ms[(k * R + row) * (HD + 2)]);
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            const float *ws = ms + (k * R + row) * (HD + 2);
            const float f = part_factor(ws[0], ws[1], m);
            l = fmaf(ws[1], f, l), sum = fmaf(ws[2 + d], f, sum);
        }
        if (d == 0) s_ml[row] = make_float2(m, l);
        s_o[row * HD + d] = sum;
    }
    // With a prefix and kept scores the row's sum is needed here: wait for the
    // prefix's parts.  With a prefix alone the own part goes to the workspace
    // like the others, for the join kernel: no block holds its SM until the
    // prefix is done, but the last one, so that the grid ends after it.
    const bool late = !KEEP && p.parts;
    const int parts = KEEP ? p.parts : 0;  // prefix parts that are joined here
    if (p.parts && (KEEP || blockIdx.x == gridDim.x - 1)) grid_dep_wait();
    // the mass so far of kMass slots a thread, under way while the parts meet
    constexpr int kMass = 16;
    const int slot0 = ch0 * KC + (int)threadIdx.x, slot1 = min(n, ch1 * KC);
    float *mass = c.mass + ((int64_t)b * G + g) * c.max_pages * kCachePage, before[kMass];
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < kMass; ++i) before[i] = slot0 + 128 * i < slot1 ? mass[slot0 + 128 * i] : 0.f;
    }
    // and the first prefix parts of its outputs
    constexpr int kPre = 8;
    const int out0 = rank * 128 + (int)threadIdx.x;
    float4 pv[kPre];
    if (parts && out0 < n_rows * (HD / 4)) {
        const float4 *part = reinterpret_cast<const float4 *>(p.part + ((int64_t)b * a.heads + head0 + out0 / (HD / 4)) * p.parts * HD + out0 % (HD / 4) * 4);
#pragma unroll
        for (int k = 0; k < kPre; ++k)
            if (k < parts) pv[k] = __ldcg(part + k * (HD / 4));
    }
    cluster_sync(S);

    // what every part counts in the row's softmax: ranks, then prefix parts
    for (int row = warp; row < n_rows; row += NW) {
        const int64_t id = (int64_t)b * a.heads + head0 + row;
        const float2 none = make_float2(-INFINITY, 0.f);
        float2 mine = none, pre[kMaxParts / 32];
#pragma unroll
        for (int i = 0; i < kMaxParts / 32; ++i) pre[i] = lane + 32 * i < parts ? __ldcg(&p.ml[id * p.parts + lane + 32 * i]) : none;
        if (lane < S) mine = cluster_get(&s_ml[row], lane, S);
        float m = mine.x;
#pragma unroll
        for (int i = 0; i < kMaxParts / 32; ++i) m = fmaxf(m, pre[i].x);
        m = warp_max(m);
        const float f = lane < S ? part_factor(mine.x, mine.y, m) : 0.f;
        float l = lane < S ? f * mine.y : 0.f, fp[kMaxParts / 32];
#pragma unroll
        for (int i = 0; i < kMaxParts / 32; ++i) fp[i] = part_factor(pre[i].x, pre[i].y, m), l = fmaf(pre[i].y, fp[i], l);
        l = warp_sum(l);
        const float inv = late ? 1.f : l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: zeros
        if (lane < S) s_rank[row][lane] = f * inv;
#pragma unroll
        for (int i = 0; i < kMaxParts / 32; ++i)
            if (lane + 32 * i < parts) s_pre[row * p.parts + lane + 32 * i] = fp[i] * inv;
        if (lane == 0) {
            const float lse2 = l == 0.f ? -INFINITY : m + log2f(l);
            s_lse[row] = l == 0.f ? 0.f : lse2;
            if (late && rank == 0) p.ml[id * p.parts + p.parts - 1] = make_float2(m, l);
            if (!late && rank == 0) {
                if (a.lse) a.lse[id] = lse2 * kLn2;
                if (p.lse2) p.lse2[id] = lse2;
            }
        }
    }
    __syncthreads();
    // the outputs, four elements a thread, shared by the ranks
    for (int i = out0; i < n_rows * (HD / 4); i += S * 128) {
        const int row = i / (HD / 4), d = i % (HD / 4) * 4;
        const int64_t id = (int64_t)b * a.heads + head0 + row;
        float sum[4] = {};
        auto add = [&](float4 v, float f) {
            sum[0] = fmaf(v.x, f, sum[0]), sum[1] = fmaf(v.y, f, sum[1]), sum[2] = fmaf(v.z, f, sum[2]), sum[3] = fmaf(v.w, f, sum[3]);
        };
        for (int k = 0; k < S; ++k) add(cluster_get(reinterpret_cast<const float4 *>(&s_o[row * HD + d]), k, S), s_rank[row][k]);
        const float4 *part = reinterpret_cast<const float4 *>(p.part + id * p.parts * HD + d);
        for (int k0 = 0; k0 < parts; k0 += kPre) {
            if (k0 || i != out0) {
#pragma unroll
                for (int k = 0; k < kPre; ++k)
                    if (k0 + k < parts) pv[k] = __ldcg(part + (k0 + k) * (HD / 4));
            }
#pragma unroll
            for (int k = 0; k < kPre; ++k)
                if (k0 + k < parts) add(pv[k], s_pre[row * p.parts + k0 + k]);
        }
        if (late) store_out4(p.part + (id * p.parts + p.parts - 1) * HD + d, sum);
        else store_out4(static_cast<Q *>(a.out) + (int64_t)b * a.out_stride + (int64_t)(head0 + row) * HD + d, sum);
    }
    if constexpr (KEEP) {
        for (int j0 = slot0; j0 < slot1; j0 += 128 * kMass) {
            if (j0 != slot0) {
#pragma unroll
                for (int i = 0; i < kMass; ++i) before[i] = j0 + 128 * i < slot1 ? mass[j0 + 128 * i] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < kMass; ++i) {
                const int j = j0 + 128 * i;
                if (j >= slot1) break;
                float sum = 0.f;
                for (int row = 0; row < n_rows; ++row) sum += exp2f(s_score[row * score_pitch + j - ch0 * KC] - s_lse[row]);
                mass[j] = before[i] + sum;
            }
        }
    }
    cluster_sync(S);  // no CTA leaves while another may read its part
}

// One warp per (token, head): joins its parts, eight in flight, in their order.
// A call of a few us (128 tokens of 32 heads with 10 parts: 8), bound by its
// launch and two dependent reads.
template <typename Q, int HD>
__global__ void __launch_bounds__(128) join_kernel(const S2dCacheView c, const S2dCacheAttention a, const AttnPlan p) {
    constexpr int V = HD / 32;  // elements of a lane
    using Vec = std::conditional_t<V == 4, float4, float2>;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    grid_dep_wait();
    grid_dep_launch();
    const int64_t from = first_token(a), to = real_tokens(a, c.n_seq);  // both loads under way together
    if (id < from * a.heads || id >= to * a.heads) return;
    const int64_t tok = id / a.heads;
    const int head = (int)(id % a.heads);
    const Vec *part = reinterpret_cast<const Vec *>(p.part + id * p.parts * HD) + lane;
    float m = -INFINITY;
    for (int k = lane; k < p.parts; k += 32) m = fmaxf(m, p.ml[id * p.parts + k].x);
    m = warp_max(m);
    float l = 0.f, o[V] = {};
    for (int k0 = 0; k0 < p.parts; k0 += 32) {
        // lane k holds part k0 + k's share
        const float2 e = k0 + lane < p.parts ? p.ml[id * p.parts + k0 + lane] : make_float2(-INFINITY, 0.f);
        const float f = part_factor(e.x, e.y, m);
        l += warp_sum(e.y * f);
        for (int k1 = 0; k1 < min(32, p.parts - k0); k1 += 8) {
            Vec v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k0 + k1 + k < p.parts) v[k] = part[(int64_t)(k0 + k1 + k) * 32];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float fk = __shfl_sync(0xffffffffu, f, k1 + k);
                if (k0 + k1 + k < p.parts) {
                    const float *x = reinterpret_cast<const float *>(&v[k]);
#pragma unroll
                    for (int i = 0; i < V; ++i) o[i] = fmaf(x[i], fk, o[i]);
                }
            }
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: zeros
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] *= inv;
    Q *out = static_cast<Q *>(a.out) + tok * a.out_stride + (int64_t)head * HD + V * lane;
    if constexpr (V == 4) {
        store_out4(out, o);
    } else {
        if constexpr (sizeof(Q) == 4) *reinterpret_cast<float2 *>(out) = make_float2(o[0], o[1]);
        else *reinterpret_cast<uint32_t *>(out) = pack2<Q>(o[0], o[1]);
    }
    if (lane == 0) {
        const float lse2 = l == 0.f ? -INFINITY : m + log2f(l);
        if (a.lse) a.lse[id] = lse2 * kLn2;
        if (p.lse2) p.lse2[id] = lse2;
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
    const int64_t es = a->type == S2D_TYPE_F32 ? 4 : 2;
    if (a->tokens && cache_rows_overlap({a->q, a->q_stride * es, row * es}, {a->out, a->out_stride * es, row * es}, a->tokens))
        return "out must not overlap q";
    return nullptr;
}

constexpr int kTcTile = 256;      // query rows of a tcgen05 item
constexpr int kMaxCluster = 8;    // CTAs that share one (sequence, KV head) of single tokens
constexpr int kSms = kCacheSms;
constexpr int kTokenSmemMost = 224 * 1024;
constexpr int kTokenSmemTwo = 111 * 1024;  // of each of two CTAs on an SM

// Shared memory of the token kernel: rings (16 slots x 2 stages x 4 warps of
// K and V), the CTA's part, the factors of the prefix parts, the scores.
size_t token_smem(const S2dCacheView &c, const AttnPlan &p, int pitch) {
    return (size_t)4 * 2 * 2 * 16 * (c.head_dim * 2 + 16) + sizeof(float) * 8 * ((size_t)c.head_dim + p.parts) +
           sizeof(float) * (size_t)std::min(p.rep, 8) * pitch;
}
// Floats between the rows of kept scores, 0 if none are kept; + 8 spreads the
// rows over the banks.  Kept where they fit the splits that make_plan has
// chosen: 64 sequences of up to 4,096 slots 128 us, computed again from the keys
// 212; of up to 12,288, which leaves one CTA an SM, 431 and 579.  No splits are
// added for longer tables (beyond 19,400 slots of 64 sequences, 9,600 of 128, at
// 8 KV heads of 128), where the keys are read twice: 64 sequences that fill
// tables of 32,768 take 1,932 us, 1,013 without weights.
int score_pitch(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p) {
    if (!a.weigh || p.rep > 8) return 0;
    const int chunks = c.max_pages * (kCachePage / 16), pitch = (chunks + p.own_splits - 1) / p.own_splits * 16 + 8;
    return token_smem(c, p, pitch) <= (size_t)kTokenSmemMost ? pitch : 0;
}

void make_plan(const S2dCacheView &c, const S2dCacheAttention &a, AttnPlan &p, size_t &bytes) {
    p = {};
    p.rep = a.heads / c.kv_heads;
    p.rep_inv = p.rep > 1 ? (uint32_t)(((1ull << 32) + p.rep - 1) / p.rep) : 0;
    const int64_t rows = (int64_t)a.tokens * p.rep;
    // splits that give `fill` items to fill, of at least `least` positions
    auto cut = [&](int64_t items, int64_t positions, int64_t least, int64_t fill) {
        const int64_t want = fill / std::max<int64_t>(items, 1);
        return (int)std::max<int64_t>(1, std::min<int64_t>({want, (positions + least - 1) / least, kMaxParts}));
    };
    const int64_t pooled = (rows + kTcTile - 1) / kTcTile;
    if (!a.q_start) {
        if (a.prefix_len) {
            p.prefix_tiles = (int)pooled;
            // The token kernel runs on the SMs that the prefix's items leave.
            // With 3.5 tiles of 128 positions a SM (64 sequences behind 8,192
            // positions) 33 us on 88 SMs and 41 on all, with 27 tiles (128
            // behind 32,000) 123 and 90.
            const int64_t tiles = pooled * c.kv_heads * ((a.prefix_len + 127) / 128);
            p.prefix_splits = cut(pooled * c.kv_heads, a.prefix_len, 128, tiles < 8 * kSms ? 88 : kSms);
        }
        const int64_t items = (int64_t)a.tokens * c.kv_heads;
        // A cluster per item until four CTAs an SM run, of at least 8 pages
        // each: 512 items of 1,025 to 4,096 slots take 191 us on one CTA each,
        // 148 on two, 163 on four.
        p.own_splits = 1;
        while (p.own_splits < kMaxCluster && items * p.own_splits < 4 * kSms && c.max_pages > 8 * p.own_splits) p.own_splits *= 2;
        p.parts = p.prefix_splits;
        // Kept scores: twice the CTAs where two of them then fit an SM and one
        // does not leave room (64 sequences in tables of 8,192 slots, filled to
        // 2,048 and more 300 us and 235, to 100 and more 56 and 59).  Once only:
        // 128 sequences in such tables, which four splits would need, stay at
        // one CTA an SM (801 us, 527 without weights).
        auto two_fit = [&](int splits) {
            AttnPlan t = p;
            t.own_splits = splits;
            const int pitch = score_pitch(c, a, t);
            return pitch && token_smem(c, t, pitch) <= (size_t)kTokenSmemTwo;
        };
        if (p.own_splits < kMaxCluster && !two_fit(p.own_splits) && two_fit(2 * p.own_splits)) p.own_splits *= 2;
        if (p.parts && !score_pitch(c, a, p)) ++p.parts;  // the own part goes with them
    } else {
        const int64_t own = rows / kTcTile + std::min<int64_t>(c.n_seq, rows);  // sum of ceil(rows of b / 256) is no more
        // Row tiles that fill the SMs take all their positions; fewer are
        // split by positions and joined: 8 sequences of 32 tokens and 1,968 to
        // 8,160 slots take 111 us with 2 items an SM, 102 with 3, 109 with 4,
        // 127 with 8.
        const bool fill = own * c.kv_heads >= kSms;
        p.own_tiles = (int)own;
        p.own_splits = fill ? 1 : cut(own * c.kv_heads, (int64_t)c.max_pages * kCachePage, 512, 3 * kSms);
        // They take the prefix as well (`fused`) unless its tiles in the rows
        // that each sequence leaves empty, about n_seq / 2 row tiles, cost more
        // than items and parts of their own.  64 sequences of 48 tokens of 32
        // bf16 heads, fused and not: behind 727 positions (8 of these units)
        // 102 and 161 us, 2,000 (23) 170 and 202, 8,000 (78) 564 and 471; f32,
        // with twice the products: 193 and 239, 343 and 325, 861 and 746.
        const int64_t waste = (int64_t)c.n_seq * ((a.prefix_len + 127) / 128);
        p.fused = a.prefix_len && fill && waste <= pooled * (a.type == S2D_TYPE_F32 ? 12 : 32);
        if (a.prefix_len && !p.fused) {
            p.prefix_tiles = (int)pooled;
            p.prefix_splits = cut(pooled * c.kv_heads, a.prefix_len, 128, kSms);
        }
        p.parts = p.prefix_splits + p.own_splits;
        if (p.parts == 1) p.parts = 0;  // an item sees all that its rows see
    }
    size_t at = 0;
    char *w = static_cast<char *>(a.workspace);
    auto take = [&](size_t n) {
        char *to = w && n ? w + at : nullptr;
        at += align256(n);
        return to;
    };
    const size_t ids = (size_t)a.tokens * a.heads;
    p.part = reinterpret_cast<float *>(take(sizeof(float) * ids * p.parts * c.head_dim));
    p.ml = reinterpret_cast<float2 *>(take(sizeof(float2) * ids * p.parts));
    p.next_item = reinterpret_cast<int *>(take(p.prefix_tiles || p.own_tiles ? sizeof(int) : 0));
    const bool again = a.weigh && (a.q_start || !score_pitch(c, a, p));  // weights by computing the scores again
    p.lse2 = reinterpret_cast<float *>(take(again ? sizeof(float) * ids : 0));
    // the most tiles that an item may take
    auto tiles_of = [](int64_t positions, int splits) { return ((positions + kTcTilePositions - 1) / kTcTilePositions + splits - 1) / splits; };
    const int64_t pooled_tiles = p.prefix_tiles ? tiles_of(a.prefix_len, p.prefix_splits) : 0;
    const int64_t own_tiles = p.own_tiles ? (p.fused ? tiles_of(a.prefix_len, 1) : 0) + tiles_of((int64_t)c.max_pages * kCachePage, p.own_splits) : 0;
    const bool hold = a.type != S2D_TYPE_F32 && std::max(pooled_tiles, own_tiles) > kTcHold;
    p.held = reinterpret_cast<float *>(take(hold ? sizeof(float) * kSms * kTcTile * c.head_dim : 0));
    bytes = at;
}

template <typename Q, typename E, int HD, bool KEEP>
cudaError_t token_launch(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p, int pitch, cudaStream_t s) {
    const size_t smem = token_smem(c, p, pitch);
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = smem_limit(done, token_kernel<Q, E, HD, KEEP>, c.device, kTokenSmemMost);
    if (e) return e;
    const int64_t blocks = (int64_t)a.tokens * c.kv_heads * ((p.rep + 7) / 8) * p.own_splits;
    if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks), cfg.blockDim = dim3(128), cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.own_splits, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    // behind the prefix's items: may start while they end, and waits for them before it reads their parts
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = p.parts ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, token_kernel<Q, E, HD, KEEP>, c, a, p, pitch);
}

template <typename Q, typename E, int HD>
cudaError_t attention_launch(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p, cudaStream_t s) {
    cudaError_t e = cudaSuccess;
    if (p.prefix_tiles || p.own_tiles) e = launch_rows_tc(c, a, p, s);
    const int pitch = a.q_start ? 0 : score_pitch(c, a, p);
    if (!e && !a.q_start) e = pitch ? token_launch<Q, E, HD, true>(c, a, p, pitch, s) : token_launch<Q, E, HD, false>(c, a, p, 0, s);
    if (!e && p.parts && !pitch)
        e = s2d_launch(join_kernel<Q, HD>, dim3((unsigned)(((int64_t)a.tokens * a.heads + 3) / 4)), dim3(128), 0, s, true, c, a, p);
    if (e || !p.lse2) return e;
    return launch_weigh_tc(c, a, p, s);
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

// s2d_cache.cu -- paged-cache operators of include/s2d_cache.h: appending new
// tokens and evicting slots, and the checks of the C entry points.  The
// attention kernels are in s2d_cache_attn.cu.
#include "s2d_cache.cuh"

#include <math.h>

#include <algorithm>

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

// [a, a + na) and [b, b + nb) share a byte
bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && x < y + nb && y < x + na;
}

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

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(float x) { return x; }
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

// One block per token.  A head row of HD elements is read 16 bytes a thread,
// so the row's threads are neighbouring lanes of one warp (8 to 32), which
// sum the squares with shuffles.  A thread keeps its place in the row over
// all the rows it takes, so its pairs' sines and cosines are computed once
// per token and serve all H + Hkv heads.
template <typename Q, typename E, int HD>
__global__ void __launch_bounds__(256) append_kernel(const S2dCacheView c, const S2dCacheAppend a, const RopeTurns turns) {
    constexpr int W = 16 / (int)sizeof(Q), L = HD / W, ROWS = 256 / L;
    const int t = blockIdx.x, G = c.kv_heads, cap = c.max_pages * kCachePage;
    // lengths of every sequence, tokens or none
    for (int b = t * 256 + (int)threadIdx.x; b < c.n_seq; b += (int)gridDim.x * 256) {
        int first;
        const int n = cache_tokens(a.q_start, a.tokens, b, first, c.status), p = a.past[b];
        if (p < 0 || p > cap) cache_flag(c.status, S2D_CACHE_BAD_LENGTH);
        c.lengths[b] = min(cap, min(max(p, 0), cap) + n);
    }
    if (t >= a.tokens) return;
    // the token's sequence: how many end at or before it
    int seq = t, i = 0;
    if (a.q_start) {
        seq = 0;
        for (int b0 = 0; b0 < c.n_seq; b0 += 256) {
            const int b = b0 + (int)threadIdx.x;
            seq += __syncthreads_count(b < c.n_seq && __ldg(a.q_start + b + 1) <= t);
        }
        if (seq >= c.n_seq) return;  // padding
        i = t - __ldg(a.q_start + seq);
    }
    if (seq >= c.n_seq) return;
    const int slot = __ldg(a.past + seq) + i;
    const bool fits = i >= 0 && slot >= i && slot < cap;  // slot >= i: past >= 0 and no overflow
    if (!fits && threadIdx.x == 0) cache_flag(c.status, i < 0 || slot < i ? S2D_CACHE_BAD_LENGTH : S2D_CACHE_FULL);
    const int pos = __ldg(a.pos + t);

    const int group = threadIdx.x / L, lane = threadIdx.x % L, d0 = lane * W;
    float cs[W / 2], sn[W / 2];
#pragma unroll
    for (int p = 0; p < W / 2; ++p) {
        const int64_t turn = (int64_t)((uint64_t)(int64_t)pos * turns.turn[d0 / 2 + p]);  // [-1/2, 1/2) turn
        sincospif((float)turn * 0x1p-63f, &sn[p], &cs[p]);
    }
    const uint32_t mates = (L == 32 ? 0xffffffffu : (1u << L) - 1u) << ((threadIdx.x & 31) / L * L);  // the row's lanes
    const int rows = a.heads + 2 * G;
    for (int r = group; r < rows; r += ROWS) {
        const bool is_q = r < a.heads, is_k = !is_q && r < a.heads + G;
        const int h = is_q ? r : is_k ? r - a.heads : r - a.heads - G;
        const Q *src = static_cast<const Q *>(is_q ? a.q : is_k ? a.k : a.v) +
                       (int64_t)t * (is_q ? a.q_stride : is_k ? a.k_stride : a.v_stride) + (int64_t)h * HD + d0;
        const Pack<Q, W> in = *reinterpret_cast<const Pack<Q, W> *>(src);
        float x[W];
#pragma unroll
        for (int e = 0; e < W; ++e) x[e] = to_float(in.v[e]);
        const float *gain = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
        if (gain) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < W; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mates, ss, o);
            const float s = rsqrtf(ss * (1.f / HD) + a.eps);
#pragma unroll
            for (int e = 0; e < W; ++e) x[e] = x[e] * s * __ldg(gain + d0 + e);
        }
        if (is_q || is_k) {
#pragma unroll
            for (int p = 0; p < W / 2; ++p) {
                const float u = x[2 * p], w = x[2 * p + 1];
                x[2 * p] = u * cs[p] - w * sn[p];
                x[2 * p + 1] = fmaf(u, sn[p], w * cs[p]);
            }
        }
        if (is_q) {
            Pack<Q, W> o;
#pragma unroll
            for (int e = 0; e < W; ++e) o.v[e] = from_float<Q>(x[e]);
            *reinterpret_cast<Pack<Q, W> *>(static_cast<Q *>(a.q_out) + (int64_t)t * a.q_out_stride + (int64_t)h * HD + d0) = o;
        } else if (fits) {
            const int64_t at = cache_row(c, c.page_table + (int64_t)seq * c.table_stride, h, slot);
            if (at < 0) continue;
            Pack<E, W> o;
#pragma unroll
            for (int e = 0; e < W; ++e) o.v[e] = from_float<E>(x[e]);
            *reinterpret_cast<Pack<E, W> *>(static_cast<E *>(is_k ? c.k : c.v) + at + d0) = o;
        }
    }
    if (fits)
        for (int g = threadIdx.x; g < G; g += 256) {
            const int64_t at = ((int64_t)seq * G + g) * cap + slot;
            if (c.positions) c.positions[at] = pos;
            if (c.mass) c.mass[at] = 0.f;
        }
}

template <typename Q, typename E>
cudaError_t append_launch(const S2dCacheView &c, const S2dCacheAppend &a, const RopeTurns &r, cudaStream_t s) {
    const unsigned blocks = (unsigned)std::max(1, a.tokens);
    if (c.head_dim == 64) append_kernel<Q, E, 64><<<blocks, 256, 0, s>>>(c, a, r);
    else append_kernel<Q, E, 128><<<blocks, 256, 0, s>>>(c, a, r);
    return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// evict
// ---------------------------------------------------------------------------

constexpr int kEvictThreads = 1024;

// f32 -> u32 with the same order; NaN as -inf, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ int block_max(int v, int *sh) {
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = __reduce_max_sync(0xffffffffu, sh[threadIdx.x & 31]);
    __syncthreads();
    return v;
}
// Exclusive prefix sum over the block's threads; total receives the sum.
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
    int w = sh[lane];
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

// One block per (sequence, KV head): the budget-th largest key by a radix
// select of four 8-bit digits, then the freed slots and the rows to move
// listed in ascending order (block scans over the slots in order), then the
// moves.  A row is read from a slot >= budget and written to a slot < budget,
// so no move reads what another writes.
__global__ void __launch_bounds__(kEvictThreads) evict_kernel(const S2dCacheView c, const S2dCacheEvict a, int32_t *lists) {
    __shared__ int sh[32];
    __shared__ int hist[256];
    __shared__ uint32_t s_digit;
    __shared__ int s_need;
    const int G = c.kv_heads, b = blockIdx.x / G, g = blockIdx.x % G, cap = c.max_pages * kCachePage;
    const int n = cache_length(c, b), budget = a.budget;
    if (g == 0 && threadIdx.x == 0 && a.past) a.past[b] = min(n, budget);
    if (n <= budget) return;
    int32_t *pos = c.positions + ((int64_t)b * G + g) * cap;
    float *mass = c.mass + ((int64_t)b * G + g) * cap;
    const int32_t *table = c.page_table + (int64_t)b * c.table_stride;

    int newest = INT32_MIN;
    for (int j = threadIdx.x; j < n; j += kEvictThreads) newest = max(newest, pos[j]);
    newest = block_max(newest, sh);
    const int64_t edge = (int64_t)newest - a.recent;
    // More recent slots than the budget (positions that repeat): only they
    // can stay, by their mass.  Otherwise all of them stay.
    int recents = 0;
    for (int j = threadIdx.x; j < n; j += kEvictThreads) recents += (int64_t)pos[j] > edge;
    int all_recents;
    block_scan(recents, sh, all_recents);
    const bool crowded = all_recents > budget;
    auto key = [&](int j) {
        const bool late = (int64_t)pos[j] > edge;
        return late == crowded ? ordered(mass[j]) : late ? 0xffffffffu : 0u;
    };

    // digits of the budget-th largest key, from the top; need: how many of
    // the keys that share the digits so far are kept
    uint32_t prefix = 0;
    int need = budget;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) hist[threadIdx.x] = 0;
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += kEvictThreads) {
            const uint32_t k = key(j);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255u], 1);
        }
        __syncthreads();
        int total;
        const int digit = 255 - (int)threadIdx.x;  // descending over the threads
        const int mine = threadIdx.x < 256 ? hist[digit] : 0;
        const int above = block_scan(mine, sh, total);
        if (threadIdx.x < 256 && above < need && above + mine >= need) s_digit = (uint32_t)digit, s_need = need - above;
        __syncthreads();
        prefix |= s_digit << shift;
        need = s_need;
        __syncthreads();
    }

    // slots in order: equals are kept while they are among the first `need`
    const int most = min(budget, cap - budget);
    int32_t *holes = lists + (int64_t)blockIdx.x * 2 * most, *rows = holes + most;
    int equals = 0, n_holes = 0, n_rows = 0;
    for (int j0 = 0; j0 < n; j0 += kEvictThreads) {
        const int j = j0 + (int)threadIdx.x;
        const uint32_t k = j < n ? key(j) : 0u;
        const bool same = j < n && k == prefix;
        int total;
        const int eq = equals + block_scan(same, sh, total);
        equals += total;
        const bool keep = j < n && (k > prefix || (same && eq < need));
        const bool hole = j < budget && !keep, row = j >= budget && keep;
        const int at = block_scan(hole | (row << 16), sh, total);
        if (hole) holes[n_holes + (at & 0xffff)] = j;
        if (row) rows[n_rows + (at >> 16)] = j;
        n_holes += total & 0xffff, n_rows += total >> 16;
    }
    __syncthreads();

    const int units = c.head_dim / 8;  // 16-byte units of a row
    for (int i = threadIdx.x; i < n_rows * 2 * units; i += kEvictThreads) {
        const int m = i / (2 * units), u = i % (2 * units);
        const int64_t to = cache_row(c, table, g, holes[m]), from = cache_row(c, table, g, rows[m]);
        if (to < 0 || from < 0) continue;
        uint16_t *base = static_cast<uint16_t *>(u < units ? c.k : c.v) + (u % units) * 8;
        *reinterpret_cast<uint4 *>(base + to) = *reinterpret_cast<const uint4 *>(base + from);
    }
    for (int m = threadIdx.x; m < n_rows; m += kEvictThreads) {
        pos[holes[m]] = pos[rows[m]];
        mass[holes[m]] = mass[rows[m]];
    }
}

// List entries of one (sequence, KV head): at most the slots below the budget
// are freed, at most the slots above it are moved.
size_t evict_list(const S2dCacheView &c, const S2dCacheEvict &a) {
    const int64_t cap = (int64_t)c.max_pages * kCachePage;
    return (size_t)std::max<int64_t>(0, std::min<int64_t>(a.budget, cap - a.budget));
}

const char *evict_fault(const S2dCacheView *c, const S2dCacheEvict *a) {
    if (const char *f = cache_view_fault(c)) return f;
    if (!a) return "evict arguments are null";
    if (!c->positions || !c->mass) return "eviction needs the cache's positions and mass";
    if (a->budget < 1) return "budget must be at least 1";
    if (a->recent < 0 || a->recent > a->budget) return "recent must be in [0, budget]";
    if (overlap(a->past, sizeof(int32_t) * c->n_seq, c->lengths, sizeof(int32_t) * c->n_seq))
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
    if (!(a->rope_base > 0.0) || !std::isfinite(a->rope_base)) return "rope_base must be positive and finite";
    if (!(a->eps >= 0.f)) return "eps must not be negative";
    if (overlap(a->past, sizeof(int32_t) * c->n_seq, c->lengths, sizeof(int32_t) * c->n_seq))
        return "past and lengths must not overlap";
    return nullptr;
}

}  // namespace
}  // namespace s2d

using namespace s2d;

extern "C" int32_t s2d_cache_append(const S2dCacheView *view, const S2dCacheAppend *args, void *stream, char *err,
                                    size_t err_cap) {
    if (const char *f = append_fault(view, args)) return cache_fail(err, err_cap, S2D_EINVAL, f);
    RopeTurns r;
    const int hd = view->head_dim;
    const long double two_pi = 6.283185307179586476925286766559005768L;
    for (int i = 0; i < hd / 2; ++i) {
        const long double f = powl((long double)args->rope_base, -2.0L * i / hd) / two_pi;
        r.turn[i] = (uint64_t)((f - floorl(f)) * 0x1p64L);  // f - floor(f) < 1
    }
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
    *bytes = sizeof(int32_t) * 2 * evict_list(*view, *args) * (size_t)view->n_seq * view->kv_heads;
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
    evict_kernel<<<(unsigned)view->n_seq * (unsigned)view->kv_heads, kEvictThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        *view, *args, static_cast<int32_t *>(args->workspace));
    return cache_cuda(err, err_cap, "cache evict", cudaGetLastError());
}

extern "C" int32_t s2d_cache_status(const S2dCacheView *view, int32_t *bits, void *stream, char *err, size_t err_cap) {
    if (const char *f = cache_view_fault(view)) return cache_fail(err, err_cap, S2D_EINVAL, f);
    if (!bits || !view->status) return cache_fail(err, err_cap, S2D_EINVAL, "no status word to read");
    DeviceGuard guard(view->device);
    cudaError_t e = guard.error;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!e) e = cudaMemcpyAsync(bits, view->status, sizeof(int32_t), cudaMemcpyDeviceToHost, s);
    if (!e) e = cudaMemsetAsync(view->status, 0, sizeof(int32_t), s);
    if (!e) e = cudaStreamSynchronize(s);
    return cache_cuda(err, err_cap, "cache status", e);
}

// s2d_cache.cuh -- shared parts of the paged-cache operators (s2d_cache.cu,
// s2d_cache_attn.cu; the interface is include/s2d_cache.h).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>

#include "../../include/s2d_cache.h"
#include "s2d_common.cuh"

namespace s2d {

constexpr int kCachePage = S2D_CACHE_PAGE;
constexpr int kCacheMaxRep = 16;
constexpr int kCacheSms = 148;  // SMs of a B200, which grids and plans are made for

// Two f32 as a pair of 16-bit elements, and back.
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
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void cache_flag(int32_t *status, int bits) {
    if (status) atomicOr(status, bits);
}

// Element offset of slot t's row of KV head g, page table row `table`; -1
// (and the status bit) when the page id is outside the pool.
__device__ __forceinline__ int64_t cache_row(const S2dCacheView &c, const int32_t *table, int g, int t) {
    const int page = __ldg(table + t / kCachePage);
    if ((uint32_t)page >= (uint32_t)c.n_pages) {
        cache_flag(c.status, S2D_CACHE_BAD_PAGE);
        return -1;
    }
    return (int64_t)page * c.page_stride + (int64_t)g * c.head_stride + (int64_t)(t % kCachePage) * c.head_dim;
}

// A sequence's length, held inside its page table.
__device__ __forceinline__ int cache_length(const S2dCacheView &c, int b) {
    const int n = __ldg(c.lengths + b), cap = c.max_pages * kCachePage;
    if (n < 0 || n > cap) {
        cache_flag(c.status, S2D_CACHE_BAD_LENGTH);
        return n < 0 ? 0 : cap;
    }
    return n;
}

// Rows [first, first + count) of a packed batch that belong to sequence b,
// held inside [0, tokens].  Rows before the first sequence's belong to none, and
// are reported as an entry out of range.
__device__ __forceinline__ int cache_tokens(const int32_t *q_start, int tokens, int b, int &first, int32_t *status) {
    if (!q_start) {
        first = b;
        return b < tokens ? 1 : 0;
    }
    const int t0 = __ldg(q_start + b), t1 = __ldg(q_start + b + 1);
    if (t0 < 0 || t1 < t0 || t1 > tokens) {
        cache_flag(status, S2D_CACHE_BAD_LENGTH);
        first = 0;
        return 0;
    }
    if (b == 0 && t0 > 0) cache_flag(status, S2D_CACHE_BAD_LENGTH);
    first = t0;
    return t1 - t0;
}

// Runs the enclosed host code with `device` current.
struct DeviceGuard {
    int before = -1;
    cudaError_t error;
    explicit DeviceGuard(int device) {
        error = cudaGetDevice(&before);
        if (!error && before != device) error = cudaSetDevice(device);
        else if (!error) before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
};

inline int32_t cache_fail(char *err, size_t cap, int32_t code, const char *msg) {
    if (err && cap) snprintf(err, cap, "%s", msg);
    return code;
}
inline int32_t cache_cuda(char *err, size_t cap, const char *what, cudaError_t e) {
    if (!e) return S2D_OK;
    if (err && cap) snprintf(err, cap, "%s: %s", what, cudaGetErrorString(e));
    return S2D_ECUDA;
}

// Raises a kernel's dynamic shared memory limit to `bytes`, once per device.
// `done` is the kernel's own; every caller asks for the same size.
template <typename K>
inline cudaError_t smem_limit(std::atomic<uint64_t> &done, K kernel, int device, int bytes) {
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (!e) done.fetch_or(bit, std::memory_order_release);
    return e;
}

// nullptr if the view can be used, else what is wrong with it.
const char *cache_view_fault(const S2dCacheView *c);
// [a, a + na) and [b, b + nb) share a byte
inline bool cache_overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && x < y + nb && y < x + na;
}
// n rows of `row` bytes from p, `stride` >= 0 bytes apart
struct CacheRows {
    const void *p;
    int64_t stride, row;
};
// Some row of a shares a byte with some row of b, both of n > 0 rows.  Slices of
// one packed buffer lie between each other's rows and share none.  Row i of a
// can only meet the last row of b that starts before its end, as that one ends
// last too.
inline bool cache_rows_overlap(const CacheRows &a, const CacheRows &b, int64_t n) {
    if (!cache_overlap(a.p, (size_t)(a.stride * (n - 1) + a.row), b.p, (size_t)(b.stride * (n - 1) + b.row))) return false;
    const int64_t off = (int64_t)((uintptr_t)b.p - (uintptr_t)a.p);  // row j of b starts here + j * b.stride from a's first
    auto meets = [&](int64_t i) {
        const int64_t at = i * a.stride, reach = at + a.row - 1 - off;
        if (reach < 0) return false;
        const int64_t j = b.stride && reach / b.stride < n ? reach / b.stride : n - 1;
        return off + j * b.stride + b.row > at;
    };
    if (a.stride == b.stride && a.stride) {
        // j - i is the same for all i that meet a row at all, up to b's last row:
        // the first of them, and the first that only b's last row can meet
        int64_t d = (a.row - 1 - off) / a.stride;
        if (d * a.stride > a.row - 1 - off) --d;
        const int64_t first = d < 0 ? -d : 0, last = n - d > 0 ? n - d : 0;
        return (first < n && meets(first)) || (last < n && meets(last));
    }
    for (int64_t i = 0; i < n; ++i)
        if (meets(i)) return true;
    return false;
}
inline bool cache_aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace s2d

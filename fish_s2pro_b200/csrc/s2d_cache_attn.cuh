// s2d_cache_attn.cuh -- what the paged attention kernels share
// (s2d_cache_attn.cu: single tokens, joining, weighing; s2d_cache_tc.cu: many
// rows on tcgen05).
#pragma once

#include "s2d_cache.cuh"

namespace s2d {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// (x, y) = hi + lo, both of the cache's type
template <typename E>
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    hi = pack2<E>(x, y);
    const float2 h = unpack2<E>(hi);
    lo = pack2<E>(x - h.x, y - h.y);
}

// What a part (pm, pl) counts in a softmax whose reference is m: nothing if it
// saw no position (or only scores of -inf), all of it if its scores are NaN
// (which fmaxf leaves out of pm), so that a NaN reaches its row.
__device__ __forceinline__ float part_factor(float pm, float pl, float m) {
    return pm == -INFINITY ? (pl == 0.f ? 0.f : 1.f) : exp2f(pm - m);
}

// How a call is cut up, from sizes that the host knows.  A query row is a
// (token, query head); a row's results over a set of positions are its part:
// (m, l) and O with l = sum 2^(s - m), O = sum 2^(s - m) v in base 2.
struct AttnPlan {
    int rep;                          // query heads per KV head
    uint32_t rep_inv;                 // ceil(2^32 / rep), 0 for 1: see row_token
    int prefix_tiles, prefix_splits;  // items over the pooled rows and the prefix
    int own_tiles, own_splits;        // at most this many row tiles over all sequences, and position splits
    int fused;                        // own items walk the prefix too
    int parts;                        // parts per row in the workspace; 0: items write the results
    float *part;                      // [tokens][heads][parts][head_dim]
    float2 *ml;                       // [tokens][heads][parts]
    int *next_item;                   // what the tcgen05 CTAs draw further items from
    float *lse2;                      // [tokens][heads] in base 2, for the weigh kernel, or NULL
    float *held;                      // [CTAs][2][head_dim / 4][128][4]: O of earlier tiles, where an item of 16-bit rows may take over kTcHold; or NULL
};

// Tiles of positions, and the tiles that O of 16-bit rows takes in the tensor
// core's accumulator before it is added up in f32 with rounding.
constexpr int kTcTilePositions = 128, kTcHold = 64;

// row / rep without a division, for rows below 2^28 (rep <= 16).
__device__ __forceinline__ int row_token(const AttnPlan &p, int row) { return p.rep_inv ? (int)__umulhi((uint32_t)row, p.rep_inv) : row; }

// No token at or past this belongs to a sequence, nor one before first_token.
__device__ __forceinline__ int real_tokens(const S2dCacheAttention &a, int n_seq) {
    const int n = a.q_start ? __ldg(a.q_start + n_seq) : n_seq;
    return max(0, min(n, a.tokens));
}

__device__ __forceinline__ int first_token(const S2dCacheAttention &a) { return a.q_start ? max(0, __ldg(a.q_start)) : 0; }

// s2d_cache_tc.cu: the items of `p` on tcgen05, and the weights of its rows by
// computing their scores again (from p.lse2).
cudaError_t launch_rows_tc(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p, cudaStream_t s);

cudaError_t launch_weigh_tc(const S2dCacheView &c, const S2dCacheAttention &a, const AttnPlan &p, cudaStream_t s);

}  // namespace s2d

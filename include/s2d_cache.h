/* s2d_cache.h -- C ABI of the operators on a paged KV cache.
 *
 * One layer's cache of n_seq sequences: pages of S2D_CACHE_PAGE positions
 * drawn from a pool, a page-table row per sequence, the page layout of the
 * batched token loop.  A sequence's cached rows sit in slots 0 .. length - 1
 * of its page-table row; after an eviction a slot no longer says which
 * position it holds, so each (sequence, KV head) keeps its slots' positions
 * and, for the choice of what to evict, the attention weight that each slot
 * has received (its "mass").
 *
 *   s2d_cache_append     QK-norm and rotary position of new tokens, their key
 *                        and value rows written into the pages
 *   s2d_cache_attention  the new tokens over a prefix that every sequence
 *                        shares (computed once for all of them) and over
 *                        their own sequences; optionally adds the softmax
 *                        weights of the own slots to the mass
 *   s2d_cache_evict      brings every sequence down to a budget of slots
 *
 * The reference keeps one growing cache per request (slow_ar.rs:372-528,
 * attention.rs:14-170) and has no counterpart of the last two; the first is
 * rms_norm_heads + apply_rope_normal + write_token (attention.rs:56-76,
 * 172-206) over a batch.
 *
 * Every buffer is device memory of the view's device, except the structs
 * themselves, which are read before the call returns.  Calls are enqueued on
 * `stream` (a cudaStream_t; NULL: the legacy default stream) and return
 * without waiting, so they can be captured into a CUDA graph; they keep no
 * state of their own.  A workspace belongs to one call at a time: calls that
 * may overlap on the GPU, graphs among them, need one each.  All sizes that
 * change from step to step (lengths, past, q_start) are read on the device.
 *
 * Errors in the arguments return S2D_EINVAL before any device work, with the
 * message in err.  What only the device can see (a page id outside the pool,
 * a length outside the page table, a sequence that is full) sets bits in the
 * view's status word; what the sequences concerned get is then unspecified,
 * but nothing outside the buffers is touched.  s2d_cache_status reads the
 * word.
 *
 * Limits (S2D_EINVAL beyond): head_dim 64 or 128, heads / kv_heads <= 16,
 * kv_heads <= 1024, n_seq <= 65,535, max_pages <= 2^18; of attention, prefix_len
 * <= 2^24 and tokens * heads <= 2^26.
 *
 * Precision: norms, rotations, softmax statistics, lse and mass are f32, and
 * results are rounded to their type once.  Attention with f32 queries takes
 * queries and softmax weights as f16 pairs of about 22 bits: its results are
 * within 2e-5 of the largest value over up to 2^18 positions, for scores of up
 * to some tens (a score is right to some 2^-22 of itself).  With f16 or bf16 queries the weights of
 * packed tokens (q_start), and those of a prefix's positions, are rounded to that
 * type before they meet the values, by up to half a step each, which adds on
 * average as much again as the result's own rounding; the own slots of single
 * tokens are weighed without it.  f32 queries avoid it at twice the products.
 *
 * Pages may be shared by sequences that only read them.  Append and evict
 * write their sequence's pages, so a page that they reach belongs to one
 * sequence.  Key rows and value rows that no token may see yet enter with
 * weight 0, so an infinity or a NaN in the value row of a slot can reach the
 * sequence's earlier tokens of the same call (0 times it is a NaN, as in a
 * product over all slots); slots at and past the length
 * never count, whatever they hold.
 */
#ifndef S2D_CACHE_H
#define S2D_CACHE_H

#include "s2d.h"

#ifdef __cplusplus
extern "C" {
#endif

#define S2D_CACHE_PAGE 64 /* positions per page */

/* Element types, by ggml's numbers. */
#define S2D_TYPE_F32 0
#define S2D_TYPE_F16 1
#define S2D_TYPE_BF16 30

/* Bits of the status word. */
#define S2D_CACHE_BAD_PAGE 1   /* a page id outside [0, n_pages)             */
#define S2D_CACHE_BAD_LENGTH 2 /* a length, past or q_start entry out of range */
#define S2D_CACHE_FULL 4       /* a token past the last slot of its sequence   */
#define S2D_CACHE_ABORTED 8    /* a kernel gave up waiting: results incomplete  */

typedef struct S2dCacheView {
    /* The row of (page p, KV head g, place r) starts at element
     * p * page_stride + g * head_stride + r * head_dim of k and of v.  Both
     * 16-byte aligned, strides multiples of 8 elements. */
    void *k, *v;
    int64_t page_stride, head_stride;
    const int32_t *page_table; /* [n_seq][max_pages], rows table_stride apart   */
    int64_t table_stride;
    int32_t *lengths;          /* [n_seq]: cached slots of each sequence         */
    int32_t *positions;        /* [n_seq][kv_heads][max_pages * 64], or NULL     */
    float *mass;               /* the same shape, or NULL                        */
    int32_t *status;           /* one word, or NULL                              */
    int32_t n_seq, kv_heads, head_dim; /* head_dim 64 or 128                      */
    int32_t n_pages;           /* pages in the pool                              */
    int32_t max_pages;         /* page-table entries of a sequence               */
    int32_t type;              /* S2D_TYPE_F16 or S2D_TYPE_BF16                  */
    int32_t device;            /* CUDA device ordinal of every buffer            */
} S2dCacheView;

/* New tokens, packed: token t of sequence b is row q_start[b] + t, for
 * q_start[b + 1] - q_start[b] tokens; rows at and past q_start[n_seq] are
 * padding and left as they are.  q_start[0] is 0: if it is more, the rows before
 * it are left as they are too, and S2D_CACHE_BAD_LENGTH is set.  q_start NULL:
 * one token per sequence.
 * With heads rows per token of head_dim elements each: consecutive heads are
 * head_dim apart, tokens *_stride elements apart; all rows 16-byte aligned. */
typedef struct S2dCacheAppend {
    const void *q, *k, *v;     /* [tokens][heads | kv_heads | kv_heads][head_dim] */
    int64_t q_stride, k_stride, v_stride;
    void *q_out;               /* [tokens][heads][head_dim]; may be q itself, else its
                                  rows share no byte with those of q, k and v      */
    int64_t q_out_stride;
    const float *q_norm, *k_norm; /* [head_dim] gains, or NULL: no norm             */
    const int32_t *pos;        /* [tokens]: rotary position of each token           */
    const int32_t *past;       /* [n_seq]: slots filled before this call            */
    const int32_t *q_start;    /* [n_seq + 1] or NULL                               */
    int32_t tokens, heads, type; /* type of q, k, v and q_out: F32 with an F16 cache,
                                  or the cache's own type                          */
    float eps;
    double rope_base;
} S2dCacheAppend;

/* For every token: x / sqrt(mean(x^2) + eps) * gain of each query and key
 * head (no norm where the gain is NULL), adjacent pairs (2i, 2i + 1) rotated
 * by pos / rope_base^(2i / head_dim), the queries written to q_out, the key
 * and the value (as they are) to slot past[b] + t of their sequence;
 * positions[slot] = pos, mass[slot] = 0 where the view has them.  Then
 * lengths[b] = past[b] + tokens of b, for every sequence: lengths must not
 * overlap past, pos or q_start (S2D_EINVAL), and the layers of a model may
 * share them.
 * A token beyond the last slot is left out (S2D_CACHE_FULL). */
int32_t s2d_cache_append(const S2dCacheView *view, const S2dCacheAppend *args, void *stream, char *err,
                         size_t err_cap);

typedef struct S2dCacheAttention {
    const void *q;             /* [tokens][heads][head_dim]                        */
    int64_t q_stride;
    void *out;                 /* [tokens][heads][head_dim]; rows share no byte with q's */
    int64_t out_stride;
    float *lse;                /* [tokens][heads] natural log of the softmax's sum, or NULL */
    const int32_t *q_start;    /* [n_seq + 1] or NULL                               */
    const int32_t *prefix_pages; /* [ceil(prefix_len / 64)] page ids in the same pool */
    int32_t prefix_len;        /* positions of the shared prefix, 0: none           */
    int32_t tokens, heads, type; /* F32 with an F16 cache, or the cache's own type   */
    int32_t weigh;             /* nonzero: add the weights to the view's mass        */
    float scale;
    void *workspace;           /* s2d_cache_attention_workspace bytes, 256-byte aligned */
    size_t workspace_bytes;
} S2dCacheAttention;

/* Bytes of workspace that this call needs (may be 0); reads no buffer. */
int32_t s2d_cache_attention_workspace(const S2dCacheView *view, const S2dCacheAttention *args, size_t *bytes, char *err,
                                      size_t err_cap);
/* softmax(scale * q . k) v with heads / kv_heads query heads per KV head (at
 * most 16).  A sequence's tokens are its newest slots: token t of T sees the
 * whole prefix and the own slots below length - T + t + 1 (so call it after
 * the append and before the next eviction).  A row that sees nothing gives
 * zeros and lse -inf.  weigh: mass[b][g][slot] += the softmax weights that
 * the tokens of b give the slot, summed over g's query heads, in a fixed
 * order. */
int32_t s2d_cache_attention(const S2dCacheView *view, const S2dCacheAttention *args, void *stream, char *err,
                            size_t err_cap);

typedef struct S2dCacheEvict {
    int32_t budget;            /* slots to keep, >= 1                              */
    int32_t recent;            /* 0 .. budget                                      */
    int32_t *past;             /* [n_seq], receives min(length, budget), or NULL    */
    void *workspace;           /* s2d_cache_evict_workspace bytes, 256-byte aligned  */
    size_t workspace_bytes;
} S2dCacheEvict;

int32_t s2d_cache_evict_workspace(const S2dCacheView *view, const S2dCacheEvict *args, size_t *bytes, char *err,
                                  size_t err_cap);
/* Every (sequence, KV head) with more than budget slots keeps budget of them:
 * first those with positions above newest - recent (newest: the largest
 * position that it holds), then by mass, heaviest first, equals by slot (a
 * NaN mass counts as -inf).  Kept rows at slots >= budget move into the slots
 * below budget that were freed, both in ascending order, with their
 * positions and mass.  Sequences within the budget are not touched.  lengths
 * stays as it is (past must not overlap it): the next append takes past.
 * Needs the view's positions and mass. */
int32_t s2d_cache_evict(const S2dCacheView *view, const S2dCacheEvict *args, void *stream, char *err, size_t err_cap);

/* Waits for `stream`, returns the status word in *bits and clears it: not
 * while `stream` is captured (S2D_EINVAL), and a bit that a call on another
 * stream sets meanwhile may be cleared unread. */
int32_t s2d_cache_status(const S2dCacheView *view, int32_t *bits, void *stream, char *err, size_t err_cap);

#ifdef __cplusplus
}
#endif
#endif /* S2D_CACHE_H */

/*
 * fmx_cache.h -- C-ABI of the KV cache's long-context operators (libfmx.so):
 * rotary positions of any layout, attention of a batch behind one shared
 * prefix, attention that adds up the weight each cached key gets, and the
 * eviction of keys by those weights. They stand beside fmx_rope_table,
 * fmx_attention_decode and the prefix cache of fmx_model.h; the reference has
 * mx::fast::rope (model.cpp:875-876) and mx::fast::
 * scaled_dot_product_attention (:879-882) at their place, and no counterpart
 * of the shared prefix, the weights and the eviction.
 *
 * Conventions as in fmx.h: device pointers, asynchronous on `stream`, status
 * codes, fmx_last_error(). Workspace: as there (NULL: allocated
 * stream-ordered by the call); it carries nothing from one call to the next,
 * so calls ordered on one stream, captured ones among them, may share one.
 */
#ifndef FMX_CACHE_H
#define FMX_CACHE_H

#include "fmx.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A strided view of rows of heads: element (b, l, h, d) is at
 * data + b * batch_stride + l * token_stride + h * head_stride + d, strides in
 * elements, not negative. For a cache, b is the slot and l the position. An
 * output's rows must not overlap one another (strides of 0 are refused). Nor,
 * except where a call says so, may they lie between an input's first and last
 * element (or an input's between theirs), or between those of another output:
 * such calls are refused. Keys and values alone may lie among each other. */
typedef struct fmx_heads {
  void* data;
  int64_t batch_stride;
  int64_t token_stride;
  int64_t head_stride;
} fmx_heads;

/* Limits of the operators below: batch * seq_len and the positions of a
 * cache or prefix at most 2^24. */
#define FMX_CACHE_MAX_ROWS (1 << 24)

/* ------------------------------------------------------------------------
 * Rotary positions
 * --------------------------------------------------------------------- */

/* How the angle per position f_i of pair i < dims / 2 follows from
 * g_i = base^(-2 i / dims), with s = factor:
 *   NONE    f = g
 *   LINEAR  f = g / s
 *   NTK     f = (base * s^(dims / (dims - 2)))^(-2 i / dims)  (dims >= 4)
 *   PARTS   f = t g + (1 - t) g / s, t from 0 to 1 as the turns over the
 *           trained length, original_max g / (2 pi), go from `low` to `high`
 *   YARN    the same with t from 1 to 0 as i goes from a to b: a the pair
 *           (rounded down, at least 0) that turns `high` times over
 *           original_max, b the pair (rounded up, at most dims - 1) that
 *           turns `low` times; results times 0.1 ln(s) + 1
 * attention_factor: results times this; 0: the scaling's own (1, or YARN's). */
typedef enum fmx_rope_scaling {
  FMX_ROPE_NONE = 0,
  FMX_ROPE_LINEAR = 1,
  FMX_ROPE_NTK = 2,
  FMX_ROPE_PARTS = 3,
  FMX_ROPE_YARN = 4
} fmx_rope_scaling;

typedef struct fmx_rope_config {
  int64_t dims;          /* rotated elements of a head: even, 2 .. 1024     */
  double base;           /* > 1                                             */
  int32_t scaling;       /* fmx_rope_scaling                                */
  double factor;         /* s >= 1 (ignored for NONE)                       */
  int64_t original_max;  /* PARTS, YARN: the trained length, >= 1           */
  double low, high;      /* PARTS, YARN: turns, 0 < low < high              */
  double attention_factor;
} fmx_rope_config;

/* freqs [dims / 2] (host) and the factor on the results. Host-side. */
int fmx_rope_frequencies(const fmx_rope_config* cfg, double* freqs, double* attention_factor);

/* What a rotation needs: the angles per position on the device, the factor
 * on the results and which elements pair up: (i, i + dims / 2) as
 * mx::fast::rope with traditional = false, or, interleaved, (2 i, 2 i + 1). */
typedef struct fmx_rope_angles {
  const double* freqs; /* [dims / 2] */
  int64_t dims;
  double factor;
  int32_t interleaved;
} fmx_rope_angles;

/* out[b, l, h] = x[b, l, h] with its first dims elements rotated to position
 * p = positions[b * seq_len + l] (device int32 [batch, seq_len], any value):
 * (a, b) -> factor * (a cos - b sin, a sin + b cos) of p f_i. The angle is
 * formed and reduced in fp64, its cosine and sine in fp32, the result is
 * rounded once. inverse: by -p f_i, which is the gradient of the forward
 * call. Elements from dims on are copied. x and out: FMX_BF16, FMX_F16 or
 * FMX_F32; out may be x itself, with the same strides. head_dim at most 1024
 * and at least dims. */
int fmx_rope(const fmx_rope_angles* angles, int dtype, int64_t batch, int64_t seq_len,
             int64_t n_heads, int64_t head_dim, const fmx_heads* x, const int32_t* positions,
             int inverse, const fmx_heads* out, fmx_stream stream);

/* The rotation of a step's new tokens together with the caches' append:
 * q_out = rotated q; token l of sequence b: its rotated keys and its values
 * go to position offsets[b] + l (device int32 [batch]) of cache slot
 * slots[b] (device int32 [batch], distinct; NULL: slot b). A row whose slot
 * is outside [0, n_slots) or whose position is outside [0, max_seq) is not
 * written. positions as in fmx_rope: a key's cache position and its rotary
 * position need not agree. q_out may be q itself, with the same strides, if no
 * new key or value is among its rows. (FMX_F32 caches: the attentions and the
 * eviction below take 16-bit ones.) */
int fmx_rope_append(const fmx_rope_angles* angles, int dtype, int64_t batch, int64_t seq_len,
                    int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, const fmx_heads* q,
                    const fmx_heads* k, const fmx_heads* v, const int32_t* positions,
                    const int32_t* offsets, const int32_t* slots, int64_t n_slots,
                    int64_t max_seq, const fmx_heads* q_out, const fmx_heads* k_cache,
                    const fmx_heads* v_cache, fmx_stream stream);

/* ------------------------------------------------------------------------
 * Attention over the cache
 * --------------------------------------------------------------------- */

/* n_heads a multiple of n_kv_heads (query head h reads kv head
 * h / (n_heads / n_kv_heads)); head_dim a multiple of 8, at most 256; scale
 * finite and positive. q, out, keys and values are FMX_BF16 or FMX_F16;
 * their data 16-byte aligned, strides multiples of 8, and the token strides
 * of keys and values at most 2^24. Calls whose work takes a launch of 2^32
 * threads or more are refused (FMX_ERR_UNSUPPORTED): those of 2^26 query rows
 * (batch * seq_len * n_heads) and of about 2^24 pairs of sequence and kv head.
 * Scores, weights and sums are fp32; in the products with the values a weight
 * has 16 bits (bf16) or 22 (float16), whatever the number of rows. */
typedef struct fmx_attention_shape {
  int32_t dtype;
  int64_t batch;
  int64_t seq_len; /* queries per sequence */
  int64_t n_heads;
  int64_t n_kv_heads;
  int64_t head_dim;
  float scale;
} fmx_attention_shape;

/* Attention of a batch whose sequences share their first prefix_len
 * positions: every query sees the whole prefix, and of its sequence's own
 * cache slot the positions 0 .. offsets[b] + l (queries are the newest
 * seq_len tokens, whose keys are in the cache already; offsets device int32
 * [batch], as in fmx_model_forward; a query whose offsets[b] + l is negative
 * sees none of its own, positions end at max_seq):
 *   out[b, l, h] = softmax(scale q . [prefix keys, own keys]) [values]
 *   lse[b, l, h] = ln sum exp(scale q . keys), fp32, contiguous; may be NULL
 * A query that sees no key gets 0 and lse -inf. k_prefix, v_prefix: token
 * stride per position (batch_stride unused; may be NULL when prefix_len is
 * 0). k_cache, v_cache: slots[b] as in fmx_rope_append (need not be
 * distinct); a slot outside [0, n_slots) has no keys. max_seq 0: no own keys
 * (the caches may then be NULL). Keys and values that a query may not see
 * do not reach its results, whatever they hold; an infinite value that it
 * sees leaves it infinity or NaN. */
size_t fmx_attention_shared_prefix_workspace_size(const fmx_attention_shape* shape,
                                                  int64_t prefix_len, int64_t max_seq);
int fmx_attention_shared_prefix(const fmx_attention_shape* shape, const fmx_heads* q,
                                const fmx_heads* k_prefix, const fmx_heads* v_prefix,
                                int64_t prefix_len, const fmx_heads* k_cache,
                                const fmx_heads* v_cache, int64_t n_slots, int64_t max_seq,
                                const int32_t* offsets, const int32_t* slots,
                                const fmx_heads* out, float* lse, void* workspace,
                                size_t workspace_bytes, fmx_stream stream);

/* Attention over the own caches alone that also adds up what weight every
 * key gets: for kv head g and position j of sequence b's slot
 *   weights_out[slot, g, j] = weights_in[slot, g, j]
 *                           + sum over l < seq_len and the query heads h of g
 *                             of softmax(..)[b, l, h, j]
 * (the weights that fmx_cache_evict goes by). weights fp32
 * [n_slots, n_kv_heads, max_seq], contiguous; weights_in NULL: 0;
 * weights_out may be weights_in. Positions that no query sees keep
 * weights_in's value (all do with seq_len 0); slots of no sequence are not
 * written. slots distinct. A slot's row starts from 0 when another sequence
 * takes it: the caller clears it.
 * The sums are in a fixed order: equal calls give equal bits. */
size_t fmx_attention_scored_workspace_size(const fmx_attention_shape* shape, int64_t max_seq);
int fmx_attention_scored(const fmx_attention_shape* shape, const fmx_heads* q,
                         const fmx_heads* k_cache, const fmx_heads* v_cache, int64_t n_slots,
                         int64_t max_seq, const int32_t* offsets, const int32_t* slots,
                         const float* weights_in, float* weights_out, const fmx_heads* out,
                         void* workspace, size_t workspace_bytes, fmx_stream stream);

/* ------------------------------------------------------------------------
 * Eviction
 * --------------------------------------------------------------------- */

/* Cuts each sequence of more than `budget` positions down to budget, for
 * every kv head on its own: kept are its first `sinks` and last `recent`
 * positions (sinks + recent <= budget) and of the others those with the
 * largest weights, of equal ones the lower positions (-0 equals 0, a NaN is
 * above all numbers). The kept keys, values and weights move to positions
 * 0 .. in their order; the rest of a weights row becomes 0, cache positions
 * behind the kept ones are left as they are. Shorter sequences keep
 * everything.
 *   lengths   [batch] device int32, positions in use (clamped to
 *             [0, max_seq]); lengths_out [batch] receives
 *             min(length, budget) and may be lengths
 *   kept      [batch, n_kv_heads, budget] device int32 or NULL: the kept
 *             positions, -1 behind the last
 *   slots     as in fmx_rope_append (distinct; one outside [0, n_slots) is
 *             skipped: length 0, kept -1)
 * k_out, v_out, weights_out: caches of out_max_seq >= min(budget, max_seq)
 * positions, weights [n_slots, n_kv_heads, out_max_seq], that overlap none
 * of the inputs; or all three NULL (out_max_seq ignored): in place. dtype:
 * FMX_BF16 or FMX_F16. head_dim at most 1024. batch * n_kv_heads below 2^22,
 * and no launch of 2^32 threads or more (FMX_ERR_UNSUPPORTED). */
size_t fmx_cache_evict_workspace_size(int64_t batch, int64_t n_kv_heads, int64_t budget);
int fmx_cache_evict(int dtype, int64_t batch, int64_t n_kv_heads, int64_t head_dim,
                    const fmx_heads* k_cache, const fmx_heads* v_cache, float* weights,
                    int64_t n_slots, int64_t max_seq, const int32_t* lengths,
                    const int32_t* slots, int64_t budget, int64_t sinks, int64_t recent,
                    const fmx_heads* k_out, const fmx_heads* v_out, float* weights_out,
                    int64_t out_max_seq, int32_t* lengths_out, int32_t* kept, void* workspace,
                    size_t workspace_bytes, fmx_stream stream);

#ifdef __cplusplus
}
#endif
#endif /* FMX_CACHE_H */

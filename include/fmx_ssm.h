/*
 * fmx_ssm.h -- C-ABI of the selective state space layer's operators
 * (libfmx.so): the short causal convolution, the selective scan, the norm of
 * groups with its gate, and one decoded token through all three. They stand
 * beside the Nemotron-H MoE block of fmx_nemotron.h; the reference has its
 * Mamba-2 mixer and ssm_kernel (nemotron_h.cpp:608-653) at their place.
 *
 * Conventions as in fmx_cache.h: device pointers, strided views (fmx_heads),
 * asynchronous on `stream`, status codes, fmx_last_error(). Workspace: as
 * there (NULL: allocated stream-ordered by the call); it carries nothing from
 * one call to the next, so calls ordered on one stream, captured ones among
 * them, may share one.
 *
 * Of all of them: sequence b's state is slot slots[b] (device int32 [batch],
 * distinct; NULL: slot b) of a pool of n_slots. A slot outside [0, n_slots)
 * is no slot: its sequence starts from 0 and leaves no state. lengths (device
 * int32 [batch], clamped to [0, seq_len]; NULL: seq_len): the tokens of each
 * sequence, the first ones of its rows; what the rows behind them hold does
 * not reach any result, and the output's are left as they are. batch * seq_len at
 * most 2^24; work that takes launches of 2^32 threads or more (rows of 16-byte
 * vectors go furthest) is FMX_ERR_UNSUPPORTED. An output must not lie between
 * the first and last element of an input or of another output, except where a
 * call says so.
 */
#ifndef FMX_SSM_H
#define FMX_SSM_H

#include "fmx_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------
 * Short causal convolution
 * --------------------------------------------------------------------- */

typedef enum fmx_activation {
  FMX_ACT_NONE = 0,
  FMX_ACT_SILU = 1
} fmx_activation;

#define FMX_SSM_MAX_TAPS 8

/* out[b, t, c] = act(bias[c] + sum over k < taps of weight[c, k] x[b, t - taps + 1 + k, c])
 * with the rows before the first from the slot's state, which holds the
 * taps - 1 rows before it, oldest first:
 *   state   [n_slots, taps - 1, channels], contiguous, of x's type
 *   state_in   NULL: 0. state_out: receives the last taps - 1 rows of each
 *              sequence (its state's among them where it is shorter); may be
 *              state_in; NULL: not kept. (Both are ignored for one tap.)
 * x, out: [batch, seq_len, channels], head_stride unused. weight
 * [channels, taps] and bias [channels] (NULL: 0) contiguous. All of dtype:
 * FMX_BF16, FMX_F16 or FMX_F32; sums in fp32, rounded once. SiLU, v / (1 +
 * e^-v), is off by 4 2^-23 of itself, and |v| 2^-23 more for negative v, and 0
 * for v below about -87 (here and as a gate below). taps 1 ..
 * FMX_SSM_MAX_TAPS, channels at most 2^20. */
int fmx_causal_conv(int dtype, int64_t batch, int64_t seq_len, int64_t channels, int64_t taps,
                    int activation, const fmx_heads* x, const void* weight, const void* bias,
                    const void* state_in, void* state_out, int64_t n_slots,
                    const int32_t* lengths, const int32_t* slots, const fmx_heads* out,
                    fmx_stream stream);

/* ------------------------------------------------------------------------
 * Selective scan
 * --------------------------------------------------------------------- */

/* n_heads a multiple of n_groups (head h reads group h / (n_heads /
 * n_groups)); head_dim and state_dim multiples of 8, at most 256. dtype
 * FMX_BF16 or FMX_F16. The time step of a token and head is v = dt + dt_bias
 * (dt alone), then ln(1 + e^v) if dt_softplus, then clamped to [dt_min,
 * dt_max] (dt_max may be infinite). */
typedef struct fmx_ssm_shape {
  int32_t dtype;
  int64_t batch;
  int64_t seq_len;
  int64_t n_heads;
  int64_t head_dim;
  int64_t n_groups;
  int64_t state_dim;
  int32_t dt_softplus;
  float dt_min;
  float dt_max;
} fmx_ssm_shape;

/* For every sequence and head, token by token, with its time step dt:
 *   S[p, n] = exp(dt a) S[p, n] + dt x[p] b[n]
 *   out[p]  = sum over n of c[n] S[p, n] + d x[p]
 * x, out [batch, seq_len, n_heads, head_dim]; b, c [batch, seq_len, n_groups,
 * state_dim]; dt [batch, seq_len, n_heads] (its element (b, l, h) at data +
 * b batch_stride + l token_stride + h head_stride); all of dtype. Data of x,
 * b, c and out 16-byte aligned, strides multiples of 8. a [n_heads] fp32 (a
 * negative number, -exp(A_log)); d, dt_bias [n_heads] fp32 or NULL (0).
 * state [n_slots, n_heads, head_dim, state_dim] fp32, contiguous, 16-byte
 * aligned: state_in NULL: 0; state_out receives S behind the last token, may
 * be state_in; NULL: not kept.
 * S, sums and decays are fp32 or more, out is rounded once. (float16 with more
 * than 8 tokens: S, where c takes it into out, is off by 2^-23 of itself and
 * 2^-37 of its row's largest; dt x with its decay, where b takes it into S, by
 * 2^-23 of itself and 2^-37 of the row's largest, be it S's or what up to 64
 * tokens bring.) What is infinite or NaN in a token's
 * rows reaches that token and later ones of its sequence, as either, and none
 * before it; of a state's row, that row. */
size_t fmx_ssm_scan_workspace_size(const fmx_ssm_shape* shape);
int fmx_ssm_scan(const fmx_ssm_shape* shape, const fmx_heads* x, const fmx_heads* dt,
                 const float* a, const fmx_heads* b, const fmx_heads* c, const float* d,
                 const float* dt_bias, const float* state_in, float* state_out, int64_t n_slots,
                 const int32_t* lengths, const int32_t* slots, const fmx_heads* out,
                 void* workspace, size_t workspace_bytes, fmx_stream stream);

/* ------------------------------------------------------------------------
 * Norm of groups with its gate
 * --------------------------------------------------------------------- */

/* With rms(v) = sqrt(mean of v^2 over the group + eps), groups of channels /
 * n_groups neighbouring channels, gate = z sigmoid(z):
 *   gate_first: u = x gate;  out = u / rms(u) weight
 *   otherwise:               out = x / rms(x) weight gate
 * z NULL: no gate. x, z, out [batch, seq_len, channels], head_stride unused;
 * weight [channels] (NULL: 1); all of dtype: FMX_BF16, FMX_F16 or FMX_F32.
 * fp32 throughout, rounded once (a sum of squares beyond fp32 makes its rms
 * infinite). channels a multiple of n_groups, at most
 * 2^20; eps positive. out may be x or z, with the same strides. */
int fmx_gated_norm(int dtype, int64_t batch, int64_t seq_len, int64_t channels,
                   int64_t n_groups, float eps, int gate_first, const fmx_heads* x,
                   const fmx_heads* z, const void* weight, const int32_t* lengths,
                   const fmx_heads* out, fmx_stream stream);

/* ------------------------------------------------------------------------
 * One decoded token
 * --------------------------------------------------------------------- */

/* A layer between its projections. Channels of the convolution: x (n_heads *
 * head_dim), b, then c (n_groups * state_dim each). Arrays as in the calls
 * above; conv_bias, d, dt_bias and norm_weight may be NULL. dtype FMX_BF16 or
 * FMX_F16; taps 2 .. FMX_SSM_MAX_TAPS. */
typedef struct fmx_ssm_layer {
  int32_t dtype;
  int64_t n_heads;
  int64_t head_dim;
  int64_t n_groups;
  int64_t state_dim;
  int64_t taps;
  int32_t activation;    /* of the convolution */
  const void* conv_weight; /* [channels, taps] */
  const void* conv_bias;   /* [channels] */
  const float* a;          /* [n_heads] */
  const float* d;
  const float* dt_bias;
  int32_t dt_softplus;
  float dt_min;
  float dt_max;
  const void* norm_weight; /* [n_heads * head_dim] */
  int64_t norm_groups;
  float eps;
  int32_t gate_first;
} fmx_ssm_layer;

/* What a prompt's three calls through a layer would refuse, before the first
 * of them moves a state: fmx_causal_conv of xbc into conv_rows, fmx_ssm_scan of
 * conv_rows' parts into scan_rows, fmx_gated_norm of scan_rows into out, states
 * in place; and outputs of one over what another reads. Launches nothing; taps
 * may be 1, and conv_state's pool of conv_slots another size than state's of
 * n_slots. conv_rows [batch, seq_len, channels] and scan_rows [batch, seq_len,
 * n_heads * head_dim] contiguous, 16-byte aligned. */
int fmx_ssm_prompt_check(const fmx_ssm_layer* layer, int64_t batch, int64_t seq_len,
                         const fmx_heads* xbc, const fmx_heads* dt, const fmx_heads* z,
                         void* conv_rows, void* scan_rows, void* conv_state, int64_t conv_slots,
                         float* state, int64_t n_slots, const int32_t* lengths,
                         const int32_t* slots, const fmx_heads* out);

/* fmx_causal_conv, fmx_ssm_scan and fmx_gated_norm of one token of each
 * sequence, states updated in place, in fp32 from the rows to the output,
 * which alone is rounded. xbc [batch, channels], z and out [batch, n_heads *
 * head_dim] (z NULL: no gate), dt [batch, n_heads]; of the views batch_stride
 * alone is used, and head_stride of dt. xbc, z and out need their type's
 * alignment only, conv_state [n_slots, taps - 1, channels] and state
 * [n_slots, n_heads, head_dim, state_dim] fp32, 16-byte aligned. */
size_t fmx_ssm_step_workspace_size(const fmx_ssm_layer* layer, int64_t batch);
int fmx_ssm_step(const fmx_ssm_layer* layer, int64_t batch, const fmx_heads* xbc,
                 const fmx_heads* dt, const fmx_heads* z, void* conv_state, float* state,
                 int64_t n_slots, const int32_t* slots, const fmx_heads* out, void* workspace,
                 size_t workspace_bytes, fmx_stream stream);

#ifdef __cplusplus
}
#endif
#endif /* FMX_SSM_H */

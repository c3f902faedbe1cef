/*
 * deltacore_layers.h — C ABI of the operators around the token mixers of a block stack, exported by the
 * same library as deltacore.h and under the same rules: row-major device buffers the caller owns, nothing
 * allocated, a dc_status returned before anything is enqueued when a check fails, work enqueued on `stream`
 * of the device that is current, sm_100 devices only.
 *
 *   dc_rms_norm            the residual stream's addition, the RMS norm of the sum, and its output in
 *                          float32, bfloat16 or 8 bits (e4m3) with scales; dc_rms_norm_bwd its backward
 *   dc_causal_conv         the short causal depthwise convolution, over a prompt or one token;
 *                          dc_causal_conv_bwd its backward
 *   dc_selective_scan      the selective state space scan over a prompt; dc_selective_scan_step one token;
 *                          dc_selective_scan_bwd the scan's backward
 *
 * They have no counterpart in burn-deltanet: the residual add and the norm in front of a block are Burn
 * modules there, and the selective scan is the diagonal relative of the delta rule that stacks of
 * linear-time mixers interleave with it.
 *
 * All sums, norms, states and exponentials are held in float32; a value is rounded once, when it is
 * written.  Every result is deterministic (no floating-point atomics).  Strides are in elements.
 */
#ifndef DELTACORE_LAYERS_H
#define DELTACORE_LAYERS_H

#include "deltacore.h"

#ifdef __cplusplus
extern "C" {
#endif

/* dc_rms_norm_args.out_dtype beside DC_F32 and DC_BF16: 8-bit floats of 4 exponent and 3 mantissa bits. */
#define DC_E4M3 2

/* Limits of dc_rms_norm / dc_rms_norm_bwd (width), dc_causal_conv (taps) and dc_selective_scan (state). */
#define DC_RMS_MAX_WIDTH 16384
#define DC_CONV_MAX_TAPS 8
#define DC_SCAN_MAX_STATE 64

/*
 * Over each row of `width` values:
 *   s = x + residual_in (s = x when residual_in is NULL), in float32;
 *   residual_out = s rounded to residual_dtype (not written when NULL);
 *   y = s / sqrt(mean(s^2) + eps) * weight (of the unrounded s), in out_dtype.
 * With out_dtype DC_E4M3, y is divided by a scale per `group` consecutive columns (group 32, 64, 128 or 256
 * dividing width; 0: one scale per row) and rounded to the nearest e4m3 value (the quotient is taken in float32 to about
 * 2^-22, so that a value within that of a tie may go either way):
 *   scale = max|y| / 448 over the group (at least 2^-126; 1 where every y is 0 or NaN), float32,
 *   [rows, width / group] (or [rows, 1]).
 * A row that holds a NaN is NaN throughout.  Row i of a tensor starts at i * its stride, columns are
 * contiguous.  residual_out may be residual_in or x, and y may be x or residual_in (same dtype and stride): in place.
 * Otherwise no output's rows may overlap another buffer's (columns or rows of one buffer beside each other do not).
 * rows may be 0.  1 <= width <= DC_RMS_MAX_WIDTH.
 */
typedef struct dc_rms_norm_args {
    int64_t rows, width;
    int64_t x_stride, residual_in_stride, residual_out_stride, y_stride;
    int32_t x_dtype, residual_dtype, out_dtype;
    int32_t group;
    float eps;
    const void *x;
    const void *residual_in;
    const float *weight; /* [width] */
    void *residual_out;
    void *y;
    float *scale; /* DC_E4M3 only */
} dc_rms_norm_args;

DC_API int dc_rms_norm(const dc_rms_norm_args *args, dc_stream_t stream);

/*
 * The backward of dc_rms_norm (a float32 or bfloat16 y), given r = residual_out (x itself where there was no
 * residual), d_y and the gradient d_r of residual_out (NULL: zero).  With inv = 1 / sqrt(mean(r^2) + eps):
 *   d = inv * weight * d_y - r * inv^3 * mean(weight * d_y * r) + d_r
 *   d_x = d in x_dtype, d_residual = d in r_dtype (either may be NULL)
 *   d_weight = sum over rows of d_y * r * inv, float32 [width] (may be NULL)
 * d_residual may be d_r, and d_x may be d_y or d_r (same dtype and stride); otherwise neither may overlap another buffer.
 * d_weight needs a workspace of dc_rms_norm_bwd_workspace_size bytes (16-byte aligned).
 */
typedef struct dc_rms_norm_bwd_args {
    int64_t rows, width;
    int64_t d_y_stride, d_r_stride, r_stride, d_x_stride, d_residual_stride;
    int32_t y_dtype, r_dtype, x_dtype; /* of d_y; of r, d_r and d_residual; of d_x */
    float eps;
    const void *d_y;
    const void *d_r;
    const void *r;
    const float *weight;
    void *d_x;
    void *d_residual;
    float *d_weight;
    void *workspace;
    uint64_t workspace_bytes;
} dc_rms_norm_bwd_args;

DC_API uint64_t dc_rms_norm_bwd_workspace_size(const dc_rms_norm_bwd_args *args);
DC_API int dc_rms_norm_bwd(const dc_rms_norm_bwd_args *args, dc_stream_t stream);

/*
 * Causal depthwise convolution of x [batch, seq, channels] with `taps` weights per channel:
 *   pre[t, c] = bias[c] + sum_j weight[c, j] * x[t - taps + 1 + j, c],  y = pre * sigma(pre) with DC_CONV_SILU,
 *   else y = pre.
 * Tokens before the first come from window_in [batch, channels, taps] (column taps + t holds token t < 0;
 * column 0 is not read by the sum; NULL: zeros), as in dc_qkv_prologue.  lengths[b] (NULL: seq) cuts sequence
 * b short, clamped to [0, seq]: x is not read past it and y is zero there.  window_out (or NULL) receives the
 * last `taps` columns of [window_in | x up to the length].  window_out may be window_in when seq == 1; they
 * must not overlap otherwise.  A decode step is seq = 1.  Token t of sequence b starts at b * batch_stride +
 * t * token_stride of its tensor; channels are contiguous.  y's rows must overlap neither x's nor one another
 * (slices of one buffer that lie beside each other do not).  x may have a batch stride of 0.  1 <= taps <=
 * DC_CONV_MAX_TAPS; up to 65535 * 32 channels; batch, seq and channels may be 0 (seq = 0 copies the window).
 */
#define DC_CONV_SILU 0x1u

typedef struct dc_causal_conv_args {
    int64_t batch, seq, channels;
    int64_t x_batch_stride, x_token_stride, y_batch_stride, y_token_stride;
    int32_t taps;
    int32_t in_dtype, out_dtype;
    uint32_t flags;
    const void *x;
    const float *weight; /* [channels, taps] */
    const float *bias;   /* [channels] or NULL */
    const float *window_in;
    const int32_t *lengths; /* [batch] or NULL */
    void *y;
    float *window_out;
} dc_causal_conv_args;

DC_API int dc_causal_conv(const dc_causal_conv_args *args, dc_stream_t stream);

/*
 * The backward of dc_causal_conv, given d_y (out_dtype) and the gradient d_window_out of window_out (NULL:
 * zero): d_x in in_dtype (zero past a sequence's length), d_weight [channels, taps], d_bias [channels] (or NULL)
 * and d_window_in [batch, channels, taps] (or NULL) in float32.  d_x's rows must overlap neither x's nor d_y's nor one
 * another, d_window_in neither d_window_out nor window_in.  Workspace: dc_causal_conv_bwd_workspace_size bytes, 16-byte
 * aligned.
 */
typedef struct dc_causal_conv_bwd_args {
    int64_t batch, seq, channels;
    int64_t x_batch_stride, x_token_stride, d_y_batch_stride, d_y_token_stride, d_x_batch_stride, d_x_token_stride;
    int32_t taps;
    int32_t in_dtype, out_dtype;
    uint32_t flags;
    const void *d_y;
    const float *d_window_out;
    const void *x;
    const float *weight;
    const float *bias;
    const float *window_in;
    const int32_t *lengths;
    void *d_x;
    float *d_weight;
    float *d_bias;
    float *d_window_in;
    void *workspace;
    uint64_t workspace_bytes;
} dc_causal_conv_bwd_args;

DC_API uint64_t dc_causal_conv_bwd_workspace_size(const dc_causal_conv_bwd_args *args);
DC_API int dc_causal_conv_bwd(const dc_causal_conv_bwd_args *args, dc_stream_t stream);

/*
 * The selective state space scan.  For every sequence and channel d of group e = d / (channels / groups), with a
 * state h of `state` float32 values:
 *   step_t = softplus(dt[t, d] + dt_bias[d])                 (without DC_SCAN_SOFTPLUS: dt + dt_bias)
 *   h_n    = exp(step_t * a[d, n]) * h_n + step_t * u[t, d] * b[t, e, n]
 *   y[t,d] = (sum_n c[t, e, n] * h_n + d[d] * u[t, d]) * z[t, d] * sigma(z[t, d])
 * exp(step_t * a) is 1 for a step of 0 whatever a is, -inf included (a state switched off: 0 for every other step).
 * dt_bias, d, z and state_in may be NULL (0, 0, no gate, 0).  u, dt, z, b and c share in_dtype; token t of
 * sequence s starts at s * batch_stride + t * token_stride of each tensor, with contiguous channels (u, dt, z,
 * y) or contiguous [groups, state] (b, c), so all of them may be column slices of projections.  lengths as in
 * dc_causal_conv: nothing is read past a sequence's length, y is zero there, and state_out [batch, channels,
 * state] is the state after its last token.  state_out may be state_in or NULL, and must not overlap it otherwise.
 * y's rows must overlap neither an input's nor one another nor state_out (slices of one buffer beside each other do not).
 * checkpoints (or NULL) receives the states that dc_selective_scan_bwd starts from:
 * dc_selective_scan_checkpoint_size bytes.  1 <= state <= DC_SCAN_MAX_STATE; batch, seq and channels may be 0.
 *
 * workspace: with a long sequence and few (sequence, channel) pairs, a workspace of
 * dc_selective_scan_workspace_size bytes (16-byte aligned; 0 where it would not help) lets the time axis be cut
 * into segments that run side by side.  NULL runs it in one piece.
 */
#define DC_SCAN_SOFTPLUS 0x1u

typedef struct dc_selective_scan_args {
    int64_t batch, seq, channels, state, groups;
    int64_t u_batch_stride, u_token_stride, dt_batch_stride, dt_token_stride, z_batch_stride, z_token_stride;
    int64_t b_batch_stride, b_token_stride, c_batch_stride, c_token_stride, y_batch_stride, y_token_stride;
    int32_t in_dtype, out_dtype;
    uint32_t flags;
    const void *u;
    const void *dt;
    const float *a; /* [channels, state] */
    const void *b;
    const void *c;
    const float *d;       /* [channels] or NULL */
    const void *z;
    const float *dt_bias; /* [channels] or NULL */
    const float *state_in;
    const int32_t *lengths;
    void *y;
    float *state_out;
    float *checkpoints;
    void *workspace;
    uint64_t workspace_bytes;
} dc_selective_scan_args;

DC_API uint64_t dc_selective_scan_checkpoint_size(const dc_selective_scan_args *args);
DC_API uint64_t dc_selective_scan_workspace_size(const dc_selective_scan_args *args);
DC_API int dc_selective_scan(const dc_selective_scan_args *args, dc_stream_t stream);

/* One token for every sequence: the same arguments with seq = 1 (token strides, lengths and checkpoints are not
 * read).  The state is read once and written once; state_out may be state_in. */
DC_API int dc_selective_scan_step(const dc_selective_scan_args *args, dc_stream_t stream);

/*
 * The backward of dc_selective_scan.  `fwd` is the forward's argument with the checkpoints it wrote (y,
 * state_out and workspace are not used; state_in is not read: it is the first checkpoint).  Given d_y
 * (fwd.out_dtype) and the gradient d_state_out of state_out (NULL: zero), writes every gradient that is not NULL:
 * d_u, d_dt, d_z [batch, seq, channels] and d_b, d_c [batch, seq, groups, state], contiguous, in fwd.in_dtype
 * (zero past a sequence's length); d_a [channels, state], d_d, d_dt_bias [channels] and d_state_in [batch,
 * channels, state] in float32.  d_u, d_dt, d_b, d_c and d_a are required, d_z when z is given.  No gradient may overlap
 * an input, nor d_state_in d_state_out.  Workspace:
 * dc_selective_scan_bwd_workspace_size bytes, 16-byte aligned.
 */
typedef struct dc_selective_scan_bwd_args {
    dc_selective_scan_args fwd;
    int64_t d_y_batch_stride, d_y_token_stride;
    const void *d_y;
    const float *d_state_out;
    void *d_u;
    void *d_dt;
    float *d_a;
    void *d_b;
    void *d_c;
    float *d_d;
    void *d_z;
    float *d_dt_bias;
    float *d_state_in;
    void *workspace;
    uint64_t workspace_bytes;
} dc_selective_scan_bwd_args;

DC_API uint64_t dc_selective_scan_bwd_workspace_size(const dc_selective_scan_bwd_args *args);
DC_API int dc_selective_scan_bwd(const dc_selective_scan_bwd_args *args, dc_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* DELTACORE_LAYERS_H */

/*
 * cc1d_mixer.h — C ABI of the operators that stand next to the causal convolution in a
 * linear-attention mixer: the gated delta rule (chunked forward and backward, recurrent step) and the
 * root-mean-square norm with the residual's addition (forward, backward, output in 8 bits).
 * No counterpart in Dao-AILab/causal-conv1d.
 *
 * Conventions are those of cc1d.h: raw device pointers, element strides as int64_t, sizes as int32_t,
 * an opaque stream handle, a cc1d_status from every function.  Nothing here allocates, frees,
 * synchronises the host or throws.
 */
#ifndef CC1D_MIXER_H_
#define CC1D_MIXER_H_

#include "cc1d.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------------------
 * The gated delta rule, per sequence and value head, state S (dim_k, dim_v) in fp32:
 *
 *   D   = exp(g[t]) S
 *   u   = beta[t] (v[t] - D^T k[t])
 *   S   = D + k[t] u^T
 *   out[t] = scale S^T q[t]
 *
 * Value head h reads q and k of head h / (v_heads / heads).  With qk_l2norm, q and k stand for
 * q rsqrt(sum q^2 + 1e-6) and k rsqrt(sum k^2 + 1e-6), each token and head for itself.
 * States, gradients and fp32 outputs are carried to fp32's precision whatever x_dtype is (products to 2^-25 of their factors'
 * values, sums in fp32; values below 2^-90 lose bits), and the gradients of q, k, v are rounded once as they are stored.  out of
 * 16 bits is rounded once too, in chunks from products whose factors (the state, and what a chunk's tokens add to it) carry 2^-17.
 *
 * Without cu_seqlens there are `batch` sequences of `seqlen` tokens.  With it (batch == 1) sequence n
 * is tokens cu_seqlens[n] .. cu_seqlens[n+1]-1, `sequences` of them (one at least where there are
 * tokens), ascending; empty ones are allowed, entries outside [0, seqlen] are clamped, and tokens of no sequence give zeros.
 * Short sequences go token by token, packed ones each by its own length; the others in chunks of 64 tokens, which are
 * worked out together: a NaN or infinity reaches its head's outputs from the start of its chunk on.
 * ---------------------------------------------------------------------------------- */
typedef struct cc1d_delta_params {
    int32_t batch, seqlen, heads, v_heads, dim_k, dim_v;
    int32_t sequences;               /* len(cu_seqlens) - 1; == batch without cu_seqlens */
    int32_t x_dtype;                 /* cc1d_dtype of q, k, v, out */
    int32_t g_dtype, beta_dtype;     /* any cc1d_dtype each */
    int32_t qk_l2norm;
    int32_t cu_seqlens_is_int64;
    float scale;
    int32_t reserved0;

    const void *q;                   /* (batch, seqlen, heads, dim_k), unit stride along dim_k */
    int64_t q_stride_b, q_stride_l, q_stride_h;
    const void *k;
    int64_t k_stride_b, k_stride_l, k_stride_h;
    const void *v;                   /* (batch, seqlen, v_heads, dim_v), unit stride along dim_v */
    int64_t v_stride_b, v_stride_l, v_stride_h;
    const void *g;                   /* (batch, seqlen, v_heads); the logarithm of the decay */
    int64_t g_stride_b, g_stride_l, g_stride_h;
    const void *beta;                /* (batch, seqlen, v_heads) */
    int64_t beta_stride_b, beta_stride_l, beta_stride_h;
    const void *cu_seqlens;          /* (sequences + 1,) contiguous, or NULL */
    const float *initial_states;     /* (sequences, v_heads, dim_k, dim_v), unit stride along dim_v, or NULL (zeros) */
    int64_t init_stride_n, init_stride_h, init_stride_k;
    void *out;                       /* (batch, seqlen, v_heads, dim_v), unit stride along dim_v */
    int64_t out_stride_b, out_stride_l, out_stride_h;
    float *final_states;             /* like initial_states (may be the same tensor), or NULL */
    int64_t final_stride_n, final_stride_h, final_stride_k;
    void *saved;                     /* NULL, or cc1d_delta_saved_bytes() of device memory, 256-byte aligned: what the
                                        backward needs of the forward (the state in front of every 64 tokens, and what
                                        they added to it), written by cc1d_delta_fwd, read by cc1d_delta_bwd */
} cc1d_delta_params;

int cc1d_validate_delta(const cc1d_delta_params *p);
/* Device memory the forward works in: 256-byte aligned, needs no initialisation, may be 0 bytes. */
int cc1d_delta_workspace_bytes(const cc1d_delta_params *p, size_t *bytes);
int cc1d_delta_saved_bytes(const cc1d_delta_params *p, size_t *bytes);
int cc1d_delta_fwd(const cc1d_delta_params *p, void *workspace, size_t workspace_bytes, cc1d_stream_t stream);

/* Backward.  `fwd` is the forward's block: `saved` is needed, `out` and `final_states` are ignored.  Tokens more than 2^25 bytes
 * apart (in v, out, dout or dv) are refused with CC1D_ERR_TOO_LARGE here and where `saved` is given to the forward. */
typedef struct cc1d_delta_bwd_params {
    cc1d_delta_params fwd;
    const void *dout;                /* (batch, seqlen, v_heads, dim_v) of x_dtype, unit stride along dim_v */
    int64_t dout_stride_b, dout_stride_l, dout_stride_h;
    const float *dfinal_states;      /* like initial_states, or NULL */
    int64_t dfinal_stride_n, dfinal_stride_h, dfinal_stride_k;
    void *dq;                        /* of x_dtype, unit stride along dim_k */
    int64_t dq_stride_b, dq_stride_l, dq_stride_h;
    void *dk;
    int64_t dk_stride_b, dk_stride_l, dk_stride_h;
    void *dv;                        /* of x_dtype, unit stride along dim_v */
    int64_t dv_stride_b, dv_stride_l, dv_stride_h;
    void *dg;                        /* (batch, seqlen, v_heads) contiguous, of g_dtype */
    void *dbeta;                     /* (batch, seqlen, v_heads) contiguous, of beta_dtype */
    float *dinitial_states;          /* or NULL */
    int64_t dinit_stride_n, dinit_stride_h, dinit_stride_k;
} cc1d_delta_bwd_params;

int cc1d_validate_delta_bwd(const cc1d_delta_bwd_params *p);
int cc1d_delta_bwd_workspace_bytes(const cc1d_delta_bwd_params *p, size_t *bytes);
int cc1d_delta_bwd(const cc1d_delta_bwd_params *p, void *workspace, size_t workspace_bytes, cc1d_stream_t stream);

/* The step of a decode loop: `seqlen` (one or a few) tokens of `batch` sequences, states advanced in
 * place.  state_indices[b] picks the state of entry b; a negative index, or one that is not below
 * state_slots, writes zeros to out[b] and leaves every state untouched.  Indices must not repeat. */
typedef struct cc1d_delta_step_params {
    int32_t batch, seqlen, heads, v_heads, dim_k, dim_v;
    int32_t state_slots;             /* state.size(0); == batch unless indices are given */
    int32_t x_dtype, g_dtype, beta_dtype;
    int32_t qk_l2norm;
    float scale;

    const void *q;
    int64_t q_stride_b, q_stride_l, q_stride_h;
    const void *k;
    int64_t k_stride_b, k_stride_l, k_stride_h;
    const void *v;
    int64_t v_stride_b, v_stride_l, v_stride_h;
    const void *g;
    int64_t g_stride_b, g_stride_l, g_stride_h;
    const void *beta;
    int64_t beta_stride_b, beta_stride_l, beta_stride_h;
    float *state;                    /* (state_slots, v_heads, dim_k, dim_v), unit stride along dim_v */
    int64_t state_stride_n, state_stride_h, state_stride_k;
    void *out;
    int64_t out_stride_b, out_stride_l, out_stride_h;
    const int32_t *state_indices;    /* (batch,) unit stride, or NULL */
} cc1d_delta_step_params;

int cc1d_validate_delta_step(const cc1d_delta_step_params *p);
int cc1d_delta_step(const cc1d_delta_step_params *p, cc1d_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Root-mean-square norm over rows of `dim` elements, with the residual's addition:
 *
 *   h = x + residual      (summed in fp32, rounded once to r_dtype; without residual h = x)
 *   y = h rsqrt(mean(h^2) + eps) weight
 *
 * y8 / scales instead of y: scales[row] = max|y| / 448 (to a unit in fp32's last place), y8 = the fp32 quotient
 * y / scales[row], to nearest, in e4m3, to nearest, ties to even both times; y is not rounded to x_dtype in between.  A
 * row of zeros has scale 0 and zeros.  A scale below 2^-126 is rounded to what fp32 has there after the quotients are formed.
 * ---------------------------------------------------------------------------------- */
typedef struct cc1d_norm_params {
    int64_t rows;
    int32_t dim;                     /* up to 2^31 - 8193; backward: 2^27 - 32 */
    int32_t x_dtype, r_dtype, w_dtype; /* of x and y; of residual and h; of weight */
    float eps;
    int32_t reserved0;
    const void *x;                   /* (rows, dim), unit stride along dim */
    int64_t x_stride;
    const void *residual;            /* (rows, dim), or NULL */
    int64_t residual_stride;
    const void *weight;              /* (dim,) contiguous */
    void *h;                         /* (rows, dim); needed with residual, else NULL.  May be residual itself */
    int64_t h_stride;
    void *y;                         /* (rows, dim) of x_dtype; NULL with y8 */
    int64_t y_stride;
    void *y8;                        /* (rows, dim) e4m3, or NULL */
    int64_t y8_stride;
    float *scales;                   /* (rows,) with y8 */
} cc1d_norm_params;

int cc1d_validate_norm(const cc1d_norm_params *p);
int cc1d_norm_fwd(const cc1d_norm_params *p, cc1d_stream_t stream);

/* Backward of y (and h): dx = dh + r (w dy) - h r^3 mean(h w dy), in x_dtype and / or r_dtype;
 * dweight = sum over rows of dy h r, rounded once to w_dtype.  Partial sums of dweight go to the
 * workspace and are added in a fixed order. */
typedef struct cc1d_norm_bwd_params {
    int64_t rows;
    int32_t dim;
    int32_t x_dtype, r_dtype, w_dtype;
    float eps;
    int32_t reserved0;
    const void *h;                   /* (rows, dim) of r_dtype */
    int64_t h_stride;
    const void *weight;
    const void *dy;                  /* (rows, dim) of x_dtype */
    int64_t dy_stride;
    const void *dh;                  /* (rows, dim) of r_dtype, or NULL */
    int64_t dh_stride;
    void *dx;                        /* (rows, dim) of x_dtype, or NULL */
    int64_t dx_stride;
    void *dresidual;                 /* (rows, dim) of r_dtype, or NULL */
    int64_t dresidual_stride;
    void *dweight;                   /* (dim,) of w_dtype */
} cc1d_norm_bwd_params;

int cc1d_validate_norm_bwd(const cc1d_norm_bwd_params *p);
int cc1d_norm_bwd_workspace_bytes(const cc1d_norm_bwd_params *p, size_t *bytes);
int cc1d_norm_bwd(const cc1d_norm_bwd_params *p, void *workspace, size_t workspace_bytes, cc1d_stream_t stream);

/* Rows of e4m3 values times their scales, as y_dtype. */
typedef struct cc1d_dequantize_params {
    int64_t rows;
    int32_t dim;
    int32_t y_dtype;
    const void *y8;                  /* (rows, dim) e4m3, unit stride along dim */
    int64_t y8_stride;
    const float *scales;             /* (rows,) contiguous */
    void *y;                         /* (rows, dim) */
    int64_t y_stride;
} cc1d_dequantize_params;

int cc1d_validate_dequantize(const cc1d_dequantize_params *p);
int cc1d_dequantize_rows(const cc1d_dequantize_params *p, cc1d_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* CC1D_MIXER_H_ */

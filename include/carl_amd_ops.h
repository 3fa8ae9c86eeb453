/*
 * carl_amd_ops.h - C-ABI of the learner's operators beside the step engine:
 * linear attention with a decay for each head (chunked and recurrent forms),
 * the gated feed-forward block, AdamW over many tensors, log-probabilities and
 * choices of actions, the root-mean-square norm, and products in 8 bits.
 *
 * Same conventions as carl_amd.h: plain pointers and sizes, CARL_OK or a
 * negative status, the message of the calling thread's last failure in
 * carl_last_error().  Every call checks its arguments on the host, queues its
 * kernels on `stream` (a hipStream_t; NULL is the default stream) of the
 * current device and returns; nothing is allocated, copied to the host or
 * kept between calls, so calls can be captured into a HIP graph (replays keep
 * the capture's numbers, AdamW's step and rate among them).  Device
 * pointers must be valid on that device; where a call needs scratch memory,
 * a *_workspace function says how many bytes, and the caller's buffer must be
 * 256-byte aligned and unused by other streams until the call's work is done.
 */
#ifndef CARL_AMD_OPS_H
#define CARL_AMD_OPS_H

#include <stdint.h>

#include "carl_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
enum { CARL_OP_F32 = 0, CARL_OP_BF16 = 1, CARL_OP_F16 = 2 };

/* ---- linear attention with a decay for each head ----------------------------
 * For each sequence and query head, with S a key_dim x value_dim memory:
 *   S_t = [start_t ? 0 : exp(log_decay) S_{t-1}] + k_t v_t^T
 *   o_t = scale S_t^T q_t
 * Query head h reads key and value head h / (heads / kv_heads).  A step whose
 * start is set sees nothing before it, whatever the memory holds (NaN and
 * infinities included); S before the first step is initial_state, or zero.
 * Steps of the chunked form run in chunks as products of matrices; long
 * sequences are split over workgroups and joined through the workspace.
 * q, k, v and out hold one element type, the memory is float32.  All sums are
 * float32.  With bfloat16 the weights of steps within a chunk are rounded to
 * that type before they meet v, and so is the memory where q reads it; what
 * enters the memory is kept to float32's precision where the memory is
 * returned, else to 16 bits.  float16's range would not hold the weights: its
 * intermediate values are float32.
 * Results do not depend on timing: there are no atomics. */
typedef struct carl_rows {
    void* data;                 /* a row: the head's contiguous elements */
    int64_t batch, step, head;  /* strides in elements */
} carl_rows;

typedef struct carl_attention {
    int64_t batch, steps;       /* may be 0; batch times heads at most 4,194,304 */
    int32_t heads, kv_heads;    /* heads is a multiple of kv_heads, at most 65535 */
    int32_t key_dim, value_dim; /* 1 to CARL_ATTENTION_MAX_DIM */
    int32_t type;               /* of q, k, v, out and their gradients */
    float scale;
    carl_rows q, k, v, out;
    const float* log_decay;     /* [heads], natural logarithm of the decay: at most 0 */
    const uint8_t* starts;      /* 0 or 1 for each sequence and step, or NULL */
    int64_t starts_batch, starts_step;
    const float* initial_state; /* [batch, heads, key_dim, value_dim], or NULL */
    float* final_state;         /* likewise, or NULL (backward: not used) */
    /* backward: d_out is read, d_q, d_k and d_v are written */
    carl_rows d_out, d_q, d_k, d_v;
    const float* d_final_state; /* or NULL */
    float* d_initial_state;     /* or NULL */
    void* workspace;            /* carl_linear_attention_workspace bytes, or NULL for 0 */
} carl_attention;

enum { CARL_ATTENTION_MAX_DIM = 128 };

int carl_linear_attention_workspace(const carl_attention* a, int backward, int64_t* bytes);
int carl_linear_attention(const carl_attention* a, void* stream);
int carl_linear_attention_backward(const carl_attention* a, void* stream);
/* One step of every sequence (steps is 1, the step strides are not used):
 * the memory `state` [batch, heads, key_dim, value_dim] is updated in place. */
int carl_linear_attention_step(const carl_attention* a, float* state, void* stream);

/* ---- gated feed-forward block -------------------------------------------------
 *   h = act(x w_gate^T) * (x w_up^T)        y = h w_down^T
 * and its gradients.  All matrices hold one element type; products are summed
 * in float32, and h (of more than 16 rows) and the gradients of both
 * projections are rounded to that type once, where the next product reads them
 * (float16's times a power of two that the largest possible one fits, so that
 * they do not leave its range; its h of up to 128 rows is not rounded).  The
 * backward pass needs only the inputs: it computes both projections again. */
enum { CARL_SILU = 0, CARL_GELU = 1 };  /* GELU in its tanh form */

typedef struct carl_ffn {
    int64_t rows;               /* at most 2^28; times the larger of width and inner, in tiles of
                                 * 128 x 128 (float32: 128 x 64), at most 2^36 elements */
    int32_t width, inner;       /* 1 to CARL_FFN_MAX_DIM */
    int32_t type, activation;
    const void* x;              /* [rows, width], rows x_row elements apart */
    int64_t x_row;
    const void *w_gate, *w_up;  /* [inner, width] */
    const void* w_down;         /* [width, inner] */
    void* y;                    /* [rows, width] */
    /* backward: dy is read; gradients that are NULL are left out */
    const void* dy;             /* [rows, width], rows dy_row elements apart */
    int64_t dy_row;
    void* dx;                   /* [rows, width] */
    void *dw_gate, *dw_up, *dw_down;
    void* workspace;            /* carl_gated_ffn_workspace bytes */
} carl_ffn;

enum { CARL_FFN_MAX_DIM = 65536 };

/* For the pointers and strides of the call to come (operands that are not
 * aligned to 16 bytes are laid out anew in the workspace). */
int carl_gated_ffn_workspace(const carl_ffn* f, int backward, int64_t* bytes);
int carl_gated_ffn(const carl_ffn* f, void* stream);
int carl_gated_ffn_backward(const carl_ffn* f, void* stream);

/* ---- AdamW ----------------------------------------------------------------
 * For each element, in float32 and in this order of roundings:
 *   m = m beta1 + g (1 - beta1)
 *   v = v beta2 + (g g) (1 - beta2)
 *   p = p (1 - lr weight_decay)
 *       - (m (lr / (1 - beta1^step))) / (sqrt(v) (1 / sqrt(1 - beta2^step)) + eps)
 * with g first multiplied by *grad_scale where that is given.  Parameters and
 * gradients may each be of any element type (a parameter is rounded once, to
 * nearest even, when it is written).
 *
 * Moments are float32, or 8-bit codes of blocks of CARL_ADAMW_BLOCK
 * consecutive elements of a tensor (its last block may be shorter) with one
 * float32 scale s per block, the block's largest magnitude:
 *   first moment   int8  c in [-127, 127]   value s (c/127) |c/127|
 *   second moment  uint8 c in [0, 255]      value s (c/255)^4
 * Codes are rounded to nearest even, and a second moment above zero never
 * gets code 0.  The square-law codes keep 1.6% (0.4% of its root for the
 * second moment) near a block's largest value and reach 4 (9) decades below
 * it.  A block that holds a NaN or an infinity gets the scale NaN and decodes
 * to NaN throughout. */
enum { CARL_ADAMW_BLOCK = 256 };

typedef struct carl_adamw_tensor {
    void* param;
    const void* grad;
    void* exp_avg;              /* float* or int8_t* */
    void* exp_avg_sq;           /* float* or uint8_t* */
    float* exp_avg_scale;       /* [ceil(n / 256)], or NULL with float moments */
    float* exp_avg_sq_scale;    /* likewise */
    int64_t n;                  /* elements, at most 2^33; a tensor of none is passed over */
    int32_t param_type, grad_type;
} carl_adamw_tensor;

typedef struct carl_adamw {
    double lr, beta1, beta2, eps, weight_decay;
    int64_t step;               /* of this update, the first is 1 */
    int32_t bits;               /* of the moments: 8 or 32 */
    const float* grad_scale;    /* device, or NULL */
} carl_adamw;

int carl_adamw_step(const carl_adamw_tensor* tensors, int count, const carl_adamw* hyper, void* stream);

/* The float32 values of n 8-bit moments' codes (one tensor's, or several whose
 * blocks follow one another). */
int carl_adamw_decode(const int8_t* exp_avg, const float* exp_avg_scale, const uint8_t* exp_avg_sq,
                      const float* exp_avg_sq_scale, int64_t n, float* exp_avg_out, float* exp_avg_sq_out,
                      void* stream);
/* The codes and scales of n float32 moments, as carl_adamw_step writes them. */
int carl_adamw_encode(const float* exp_avg, const float* exp_avg_sq, int64_t n, int8_t* exp_avg_out,
                      float* exp_avg_scale, uint8_t* exp_avg_sq_out, float* exp_avg_sq_scale, void* stream);

/* ---- actions ----------------------------------------------------------------
 * A row holds the logits of all action heads, one head after another.  A logit
 * is available where it is not masked and not -infinity; with x_j a head's
 * available logits
 *   log p_j = x_j - log(sum_i exp x_i)      H = -sum_j p_j log p_j
 * and a row's log-probability and entropy are its heads' sums, in order.  What
 * is not available weighs nothing whatever it holds, has the log-probability
 * -infinity and the gradient 0.  A head with nothing available has entropy 0.
 * An action below 0 is none: its head adds 0 to the log-probability (and takes
 * part in the entropy).  An action past its head's last makes the
 * log-probability NaN, and its head's gradients where there are some by the
 * log-probability.  A NaN or +infinity among the available logits makes its
 * head's results NaN.
 *
 * The best actions of a head are those with the largest keys, the available
 * logits plus noise (one float32 addition; without noise the logits), equal
 * ones by their index, a NaN before all others; with noise -log(-log u), u
 * uniform in (0, 1), the best one is a sample.  Where fewer than k are
 * available the rest have the action -1 and the log-probability -infinity. */
typedef struct carl_actions {
    int64_t rows;               /* at most 2^40 */
    int32_t type;               /* of logits and their gradients */
    int32_t heads;              /* 1 to CARL_ACTIONS_MAX_HEADS */
    const int32_t* sizes;       /* on the host, [heads]: at least 1, CARL_ACTIONS_MAX_LOGITS in all */
    const void* logits;         /* [rows, logits], rows logits_row elements apart */
    int64_t logits_row;
    const uint8_t* mask;        /* likewise: 1 where available, 0 where masked; or NULL */
    int64_t mask_row;
    /* log-probabilities */
    const void* actions;        /* [rows, heads], rows actions_row apart: int32_t, or int64_t */
    int64_t actions_row;
    int32_t actions_wide;       /* 1 for int64_t */
    float *log_prob, *entropy;  /* [rows], of the choice log_prob is [rows, heads, k] */
    /* backward: gradients of both outputs, row_step apart (0: one value for all rows), NULL for zero */
    const float *d_log_prob, *d_entropy;
    int64_t d_log_prob_step, d_entropy_step;
    void* d_logits;             /* [rows, logits] */
    /* the best actions */
    const float* noise;         /* [rows, logits], rows noise_row apart, or NULL */
    int64_t noise_row;
    int32_t k;                  /* 1 to CARL_ACTIONS_MAX_K */
    int32_t* best;              /* [rows, heads, k] */
} carl_actions;

enum { CARL_ACTIONS_MAX_HEADS = 64, CARL_ACTIONS_MAX_LOGITS = 16384, CARL_ACTIONS_MAX_K = 64 };

int carl_action_log_prob(const carl_actions* a, void* stream);
int carl_action_log_prob_backward(const carl_actions* a, void* stream);
int carl_top_actions(const carl_actions* a, void* stream);

/* ---- root-mean-square norm, rows in 8 bits -------------------------------------
 *   s = x + residual        y = s / sqrt(mean(s^2) + eps) w
 * All matrices hold one element type; s is rounded to it once, as it is kept,
 * and the norm is that of the rounded s.  Sums are float32; of rows whose
 * squares add up to 2^120 or more s is first multiplied by 2^-80.
 *
 * Codes of a row, every step one IEEE binary32 operation:
 *   t = s w (of rows without a norm t = x)      m = max(max |t|, 2^-100)
 *   code = rint(t (127 / m))                    scale = (m / 127) / sqrt(mean(s^2) + eps)
 * (without a norm scale = m / 127).  A row with a NaN or an infinity in t has
 * the codes 0 and the scale NaN.  No output overlaps an input. */
typedef struct carl_norm {
    int64_t rows;               /* at most 2^40 */
    int32_t width;              /* 1 to CARL_NORM_MAX_DIM */
    int32_t type;
    float eps;                  /* at least CARL_NORM_MIN_EPS */
    const void* x;              /* [rows, width], rows x_row elements apart */
    int64_t x_row;
    const void* residual;       /* likewise, or NULL */
    int64_t residual_row;
    const void* weight;         /* [width] */
    void* sum;                  /* written where there is a residual: [rows, width] */
    void* y;                    /* [rows, width] */
    int8_t* codes;              /* [rows, width], rows codes_row apart */
    int64_t codes_row;
    float* scale;               /* [rows] */
    /* backward: s (x where there is no residual) is read from `sum`, rows sum_row apart */
    int64_t sum_row;
    const void* dy;
    int64_t dy_row;
    const void* d_sum;          /* gradient of s from elsewhere, or NULL */
    int64_t d_sum_row;
    void* d_x;                  /* of x and of the residual alike, or NULL */
    void* d_weight;             /* or NULL */
    void* workspace;            /* carl_rms_norm_workspace bytes, or NULL for 0 */
} carl_norm;

enum { CARL_NORM_MAX_DIM = 16384 };
#define CARL_NORM_MIN_EPS 1e-30f

int carl_rms_norm(const carl_norm* n, void* stream);
int carl_rms_norm_workspace(const carl_norm* n, int64_t* bytes);        /* of the backward pass */
int carl_rms_norm_backward(const carl_norm* n, void* stream);
int carl_rms_norm_int8(const carl_norm* n, void* stream);
int carl_quantize_int8(const carl_norm* n, void* stream);               /* of x: no weight, no eps */

/* ---- products in 8 bits ----------------------------------------------------------
 *   acc = sum over k of x[row][k] w[column][k], exact
 *   y = (acc x_scale[row]) w_scale[column] + bias[column]
 *   gated: y = act(gate) up, both of them such products
 * in float32, rounded to y's type once.  All int8 values are allowed, -128
 * among them. */
typedef struct carl_int8_linear {
    int64_t rows;               /* at most CARL_INT8_MAX_ROWS; by columns at most CARL_INT8_MAX_TILES tiles of 128 x 128 */
    int32_t width, columns;     /* 1 to CARL_INT8_MAX_DIM */
    int32_t type;               /* of y and the bias */
    int32_t activation;         /* of the gated form: CARL_SILU or CARL_GELU */
    const int8_t* x;            /* [rows, width], rows x_row apart */
    int64_t x_row;
    const float* x_scale;       /* [rows] */
    const int8_t* w;            /* [columns, width], rows w_row apart */
    int64_t w_row;
    const float* w_scale;       /* [columns] */
    const int8_t* w_up;         /* gated: w is the gate's; or NULL */
    int64_t w_up_row;
    const float* w_up_scale;
    const void* bias;           /* [columns], or NULL (gated: NULL) */
    void* y;                    /* [rows, columns] */
} carl_int8_linear;

enum { CARL_INT8_MAX_DIM = 65536, CARL_INT8_MAX_ROWS = 1 << 28, CARL_INT8_MAX_TILES = 1 << 22 };

int carl_int8_linear_forward(const carl_int8_linear* p, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CARL_AMD_OPS_H */

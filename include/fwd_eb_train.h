/*
 * fwd_eb_train.h — training operators around the EmbeddingBag path (C ABI).
 *
 * The pooled lookup's way back: the gradient of an fwd_eb_forward call, layer norm of
 * the pooled rows with its gradients, and an AdamW step over many tensors at once.  The
 * reference is an inference framework and has no counterpart of these; its layer norm
 * plugin (source/trt_engine/trt_network_crt/plugins/layer_norm_plugin/) is forward only.
 *
 * Conventions are those of fwd_eb.h: device pointers of the current CUDA device, launches
 * on `stream` only, no allocation, no synchronisation, 0 / FWD_EB_E* / cudaError_t as
 * status.  Every result is deterministic: the same call on the same inputs gives the same
 * bits.  Calls that write the same buffer (two gradients accumulated into one) go one behind the
 * other; at the same time they have no defined result.  All launches can be captured into a graph.
 */
#ifndef FWD_EB_TRAIN_H_
#define FWD_EB_TRAIN_H_

#include "fwd_eb.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element type of layer norm rows and of AdamW's parameters and gradients, beside
 * FWD_EB_F32 and FWD_EB_F16.  Embedding tables have no such form. */
enum { FWD_EB_BF16 = 3 };

/* ---- gradient of the pooled lookup --------------------------------------------------- */

/* Flags (fwd_eb_backward_params.flags). */
enum {
  /* add to what grad_table holds instead of overwriting it: rows that no lookup names are
   * neither read nor written, so the cost goes by the lookups and not by the table.  In fp32 the
   * memory system adds, one atomic addition an element and call (so its order does not matter), which
   * takes subnormal values for zero; in fp16 the row is read, added to in fp32 and rounded */
  FWD_EB_BACKWARD_ACCUMULATE = 1
};

/*
 * The gradient of out = fwd_eb_forward(fwd) with respect to the table rows and the
 * per-sample weights, given grad_out = d loss / d out.  With lookup j of bag b naming row r:
 *
 *   grad_table[r]  = sum over the lookups j of r of  c_j * grad_out[b]
 *   grad_weights[j] = < table[r], grad_out[b] >
 *
 *   SUM         c_j = per_sample_weights[j], or 1
 *   MEAN        c_j = 1 / (non-padding indices of the bag; its raw length with
 *                     FWD_EB_FLAG_MEAN_RAW_LENGTH)
 *   MAX         c_j = 1 in the columns that lookup j won, else 0 (`winners`)
 *   SQUARE_SUM  c_j = 2 * table[r]
 *   GATHER      every index is a bag of its own
 *
 * Lookups of padding_idx, outside the row window or before the first bag contribute nothing,
 * and their grad_weights entry is 0.  A row's lookups are added in fp32, in an order that the
 * call's sizes and indices alone determine, and rounded once to grad_table_dtype.
 *
 * grad_table covers the same row window as fwd.table: [num_rows, dim].  Without
 * FWD_EB_BACKWARD_ACCUMULATE every element of those rows is written (zeros where no lookup
 * falls); elements between rows (stride > dim) are left as they are.
 *
 * Limits: num_indices, num_bags < 2^31 - 65536 and dim <= 2^20 (FWD_EB_ETOOBIG); FWD_EB_FLAG_OFFSET_PAIRS
 * is not supported (FWD_EB_EUNSUPPORTED).  Offsets must not decrease; offsets that do give
 * an unspecified gradient but never an access outside the buffers.
 */
typedef struct fwd_eb_backward_params {
  fwd_eb_params fwd;          /* the forward call.  table is read for SQUARE_SUM and grad_weights
                                 only; out, out_dtype, out_stride, strategy and workspace are ignored */
  const void* grad_out;       /* device, [num_bags, dim] (GATHER: [num_indices, dim]) */
  int32_t grad_out_dtype;     /* FWD_EB_F32 / FWD_EB_F16 */
  int32_t grad_table_dtype;   /* FWD_EB_F32 / FWD_EB_F16 */
  int64_t grad_out_stride;    /* elements between rows; 0 = dim */
  void* grad_table;           /* device, [num_rows, dim], or NULL: not wanted */
  int64_t grad_table_stride;  /* elements between rows; 0 = dim */
  float* grad_weights;        /* device, [num_indices], or NULL; mode SUM only */
  const void* winners;        /* MAX: the FWD_EB_F32_POS output of the forward call, 8-byte aligned */
  int64_t winners_stride;     /* pairs between rows; 0 = dim */
  void* workspace;            /* device, 256-byte aligned, contents neither read nor kept */
  size_t workspace_bytes;     /* at least fwd_eb_backward_workspace_size() */
  uint32_t flags;             /* FWD_EB_BACKWARD_* */
  int32_t reserved;
} fwd_eb_backward_params;

size_t fwd_eb_backward_params_size(void);

/* Scratch bytes fwd_eb_backward needs for `p` (0 for arguments it would refuse).  One
 * workspace serves one call at a time: calls that may overlap on the GPU need their own. */
size_t fwd_eb_backward_workspace_size(const fwd_eb_backward_params* p);

int fwd_eb_backward(const fwd_eb_backward_params* p, void* stream);

/* ---- layer norm ----------------------------------------------------------------------- */

/*
 * Forward:   mean = sum(x) / cols,  rstd = 1 / sqrt(sum((x - mean)^2) / cols + eps),
 *            y = (x - mean) * rstd * weight + bias          for each of `rows` rows.
 * Backward:  with h = (x - mean) * rstd and g = grad_y * weight,
 *            grad_x = rstd * (g - sum(g) / cols - h * sum(g * h) / cols)
 *            grad_weight = sum over the rows of grad_y * h,   grad_bias = sum of grad_y.
 * Sums and statistics are fp32; a result is rounded once to its type.  y may be x, and
 * grad_x may be grad_y or x (same stride); otherwise outputs must not overlap inputs.
 */
typedef struct fwd_eb_layer_norm_params {
  const void* x;              /* device, [rows, cols] */
  int32_t dtype;              /* FWD_EB_F32 / FWD_EB_F16 / FWD_EB_BF16, of x, y, grad_y and grad_x */
  int32_t weight_dtype;       /* of weight, bias, grad_weight and grad_bias */
  int64_t rows;               /* >= 0 */
  int64_t cols;               /* 1 .. 2^30 */
  int64_t x_stride;           /* elements between rows; 0 = cols */
  const void* weight;         /* device, [cols], or NULL: ones */
  const void* bias;           /* device, [cols], or NULL: zeros; forward only */
  double eps;                 /* >= 0 and finite; forward only */
  float* mean;                /* device, [rows]: written by the forward call (or NULL: not
                                 wanted), read by the backward call */
  float* rstd;                /* the same */
  void* y;                    /* forward: device, [rows, cols] */
  int64_t y_stride;           /* 0 = cols */
  const void* grad_y;         /* backward: device, [rows, cols] */
  int64_t grad_y_stride;
  void* grad_x;               /* backward: device, [rows, cols], or NULL: not wanted */
  int64_t grad_x_stride;
  void* grad_weight;          /* backward: device, [cols], or NULL.  Zeros when rows is 0 */
  void* grad_bias;            /* the same */
  void* workspace;            /* backward: device, 256-byte aligned; see the size function */
  size_t workspace_bytes;
} fwd_eb_layer_norm_params;

size_t fwd_eb_layer_norm_params_size(void);
int fwd_eb_layer_norm_forward(const fwd_eb_layer_norm_params* p, void* stream);

/* Scratch bytes of the backward call (the partial sums of grad_weight and grad_bias; 0 when
 * neither is wanted). */
size_t fwd_eb_layer_norm_workspace_size(const fwd_eb_layer_norm_params* p);
int fwd_eb_layer_norm_backward(const fwd_eb_layer_norm_params* p, void* stream);

/* ---- AdamW ---------------------------------------------------------------------------- */

/* Elements of a tensor that share one scale of an 8-bit state (the last block may be short). */
#define FWD_EB_ADAMW_BLOCK 256

/* One tensor of a step: n consecutive elements each of param, grad and the two states. */
typedef struct fwd_eb_adamw_tensor {
  void* param;
  const void* grad;
  float* master;              /* fp32 copy that the step works on, param being its rounded image;
                                 NULL: the step works on param itself */
  void* exp_avg;              /* m: fp32 [n], or e4m3 codes [n] */
  void* exp_avg_sq;           /* v: fp32 [n], or e4m3 codes of sqrt(v) [n] */
  float* exp_avg_scale;       /* 8-bit states: [ceil(n / FWD_EB_ADAMW_BLOCK)], else NULL */
  float* exp_avg_sq_scale;
  int64_t n;                  /* >= 0 */
  int32_t param_dtype;        /* FWD_EB_F32 / FWD_EB_F16 / FWD_EB_BF16 */
  int32_t grad_dtype;
  int32_t state_bits;         /* 32 or 8 */
  float weight_decay;
} fwd_eb_adamw_tensor;

/*
 * What all tensors of a step share.  With t = step:
 *   g = grad * grad_scale
 *   m = beta1 * m + (1 - beta1) * g,      v = beta2 * v + (1 - beta2) * g^2
 *   p = p * (1 - lr * weight_decay)
 *       - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 * in fp32.  8-bit states: each block of FWD_EB_ADAMW_BLOCK elements holds x as
 * scale * e4m3(x / scale), scale = max|x| / 448, rounded to nearest, for x = m and
 * x = sqrt(v); a sqrt(v) of 2^-63 and more never rounds to zero, and a block whose scale
 * would be below 2^-126 holds zeros.  m, v, sqrt(v), the scale and x * (1 / scale) are rounded an operation at a
 * time, so that the codes are those of the formulas in plain fp32 (root and reciprocal: but for a few in a
 * million).  The update itself uses the
 * unrounded m and v; a v near 2^-126 and below may count as less than it is where
 * eps * sqrt(1 - beta2) >= 2^-38, which moves no update by more than half an ulp.  An 8-bit v only follows changes larger than half a code (about 6 %
 * of sqrt(v)) within a step relative to its block's largest: it suits beta2 of 0.95 or so.
 * A gradient that is not finite makes the states of its element NaN or infinite, and the
 * parameter from then on; in 8 bits an infinity does that to its whole block.  d_skip is there to
 * leave such a step out.
 *
 * The d_* pointers are for captured graphs, which replay launches with the numbers they were
 * captured with: where one is not NULL, the kernel reads the value from the device and the
 * host's is ignored.
 */
typedef struct fwd_eb_adamw_config {
  double lr;                  /* >= 0, finite in fp32 */
  double beta1, beta2;        /* [0, 1) */
  double eps;                 /* 0, or 2^-126 .. 2^126 */
  double grad_scale;          /* finite in fp32 */
  int64_t step;               /* t of this step, from 1 */
  const float* d_lr;
  const float* d_grad_scale;
  const int64_t* d_step;      /* t of this step */
  const int32_t* d_skip;      /* != 0: the call changes nothing */
} fwd_eb_adamw_config;

size_t fwd_eb_adamw_tensor_size(void);
size_t fwd_eb_adamw_config_size(void);

/* One step over `count` tensors (a host array, read before the call returns; it needs not
 * outlive it).  No two tensors may overlap.  Everything is checked before the first launch;
 * one launch covers up to 256 tensors of one kind (state width; with 8-bit states also the
 * widths of values and gradients). */
int fwd_eb_adamw_step(const fwd_eb_adamw_tensor* tensors, int32_t count,
                      const fwd_eb_adamw_config* cfg, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* FWD_EB_TRAIN_H_ */

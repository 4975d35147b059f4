/*
 * muon_train_sm100.h -- C ABI of the training-step operators around the Muon
 * update on B200 (sm_100a): the distillation loss over a teacher's top logits
 * with its gradient, the norms before and after a residual block with its gate
 * and residual scale, and the routing of tokens to experts.
 *
 * They live in the library of muon_polar_sm100.h and follow its rules.  Every
 * entry point
 *   - takes plain device pointers, sizes and a cudaStream_t passed as void*,
 *   - allocates nothing (the caller owns every buffer),
 *   - launches asynchronously on `stream` of the current device and returns
 *     0, a negative MUON_POLAR_ERR_* code (nothing was launched) or the
 *     cudaError_t of the launch.
 * Sums, maxima and statistics are held in 32 bits or more, and each stored
 * value is rounded once.  All results are deterministic.
 */
#ifndef MUON_TRAIN_SM100_H
#define MUON_TRAIN_SM100_H

#include <stddef.h>
#include <stdint.h>

#include "muon_polar_sm100.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the tensors below. */
#define MUON_TRAIN_F32 0
#define MUON_TRAIN_BF16 1
#define MUON_TRAIN_F16 2

/* Longest list of teacher logits of one row. */
#define MUON_TRAIN_MAX_TOP 1024
/* Most experts of one router, and most experts a token is sent to. */
#define MUON_TRAIN_MAX_EXPERTS 1024
#define MUON_TRAIN_MAX_ROUTES 64

/* Kernels launched by the entry points of this header. */
uint64_t muon_train_launch_count(void);

/* Device status word (zero: no trouble).  Every wait inside a kernel is
 * bounded; a kernel that gives up a wait sets a bit here, runs on without
 * waiting and returns, its results void.  Synchronises the device.  The PyTorch
 * operators read it after each call when MUON_POLAR_DEBUG_SYNC is set. */
#define MUON_TRAIN_STATUS_WAIT 0x1u
int muon_train_read_device_status(int device, uint32_t* flags, int clear);

/* The limit of these kernels' waits on the current device (the largest, where
 * a setting was cut short).  muon_polar_set_wait_limit_ns sets it, with that of
 * the library's other kernels.  Waits for the device's default stream. */
int muon_train_wait_limit_ns(uint64_t* limit_ns);

/* ---- distillation from a teacher's top logits ------------------------------
 * One row has student logits z[vocab] and a list of `top` teacher logits t
 * with their vocabulary indices i.  An entry counts when 0 <= i < vocab and
 * t > -inf; others are left out (padding of shorter lists).  With
 * tau = temperature,
 *   q_j  = exp(t_j / tau) / sum over the counted entries, or
 *          exp(t_j / tau - teacher_lse) when teacher_lse is given: the
 *          teacher's own log-normaliser over its whole vocabulary at tau,
 *   loss = sum_j q_j (log q_j - z_{i_j} / tau + log sum_v exp(z_v / tau)),
 *   dz_v = row_scale / tau (sum_j q_j softmax(z / tau)_v - sum_{i_j = v} q_j).
 * A row without a counted entry has loss 0 and gradient 0, whatever its
 * logits; a row whose row_scale is 0 has gradient 0.
 */
typedef struct {
  const void* logits;          /* [rows][ld], element type dtype */
  int64_t rows, vocab, ld;     /* ld >= vocab (rows > 1), in elements */
  const void* teacher_logits;  /* [rows][top], contiguous */
  const void* teacher_indices; /* [rows][top], contiguous */
  const float* teacher_lse;    /* [rows] or NULL */
  const float* row_scale;      /* [rows] or NULL (1) */
  float* loss;                 /* [rows] */
  float* stats;                /* [rows][2]: the row's maximum and sum of exponentials */
  void* grad;                  /* [rows][ld_grad], element type dtype */
  int64_t ld_grad;
  int64_t top;                 /* 1 .. MUON_TRAIN_MAX_TOP */
  float temperature;           /* >= 2^-126: its reciprocal is taken */
  int dtype, teacher_dtype;    /* MUON_TRAIN_* */
  int index_bytes;             /* 4 or 8 */
} muon_train_distill_args;

/* loss, with stats (may be NULL without grad) for a later backward call, and
 * grad (may be NULL): the loss and its gradient in one launch, which reads the
 * logits once from memory where rows stay in registers or in L2. */
int muon_train_distill_sm100(const muon_train_distill_args* args, void* stream);

/* grad from the stats of an earlier call on the same inputs (loss unused). */
int muon_train_distill_backward_sm100(const muon_train_distill_args* args, void* stream);

/* ---- norms before and after a block, with its gate and residual scale -------
 * For rows y = block_out and x = residual of `width` elements:
 *   u = y * rsqrt(mean(y^2) + eps) * post_weight       (u = y without it)
 *   h = residual_scale * x + gate * u                  (hidden)
 *   n = h * rsqrt(mean(h^2) + eps) * pre_weight        (normed: optional)
 * n is computed from h before it is rounded.  gate has gate_rows rows; rows
 * [g * rows / gate_rows, (g + 1) * rows / gate_rows) use row g.
 */
typedef struct {
  const void* block_out;       /* [rows][width], element type dtype */
  const void* residual;        /* [rows][width] */
  const void* post_weight;     /* [width] or NULL */
  const void* pre_weight;      /* [width] or NULL: no normed */
  const void* gate;            /* [gate_rows][width] or NULL */
  const void* residual_scale;  /* [scale_count] or NULL */
  void* hidden;                /* [rows][width] */
  void* normed;                /* [rows][width], with pre_weight */
  float* rstd_post;            /* [rows], 1 without post_weight; may be NULL forward */
  float* rstd_pre;             /* [rows], 0 without pre_weight; may be NULL forward */
  int64_t rows, width;
  int64_t gate_rows;           /* divides rows; 0 without gate */
  int64_t scale_count;         /* 1 or width; 0 without residual_scale */
  float eps;
  int dtype;                   /* block_out, residual, hidden, normed and their gradients */
  int post_dtype, pre_dtype, gate_dtype, scale_dtype;
} muon_train_norm_args;

int muon_train_residual_norm_sm100(const muon_train_norm_args* args, void* stream);

/* Gradients of residual_norm.  grad_hidden or grad_normed may be NULL (zero),
 * not both; each output may be NULL (not wanted).  Gradients of gate,
 * residual_scale and the weights have their parameter's type. */
typedef struct {
  const void* grad_hidden;     /* [rows][width] */
  const void* grad_normed;     /* [rows][width] */
  void* grad_block_out;        /* [rows][width] */
  void* grad_residual;         /* [rows][width] */
  void* grad_post_weight;      /* [width] */
  void* grad_pre_weight;       /* [width] */
  void* grad_gate;             /* [gate_rows][width] */
  void* grad_residual_scale;   /* [scale_count] */
  void* workspace;             /* 16-byte aligned */
  size_t workspace_bytes;
} muon_train_norm_grads;

/* Bytes of workspace of a backward call on the current device (0 on error). */
size_t muon_train_residual_norm_workspace_bytes(const muon_train_norm_args* args);

/* args: the forward call's inputs with its rstd_post and rstd_pre (hidden and
 * normed are not read). */
int muon_train_residual_norm_backward_sm100(const muon_train_norm_args* args,
                                            const muon_train_norm_grads* grads, void* stream);

/* ---- routing to experts --------------------------------------------------------
 * For one token's logits l[experts]:
 *   s   = softmax(l) (score 0) or sigmoid(l) (score 1)
 *   key = s + bias; the logits themselves for a softmax without bias whose
 *         groups, if any, are ranked by one key (the same order)
 * The experts are `groups` equal runs.  A group's key is the sum of its
 * group_top (1 or 2) largest keys; the top_groups best groups stay, and the k
 * largest keys among their experts are chosen, in descending order.  Equal
 * keys go to the lowest index, and a NaN key counts as -inf.
 *   weight_j = scale * s_j / (sum of the chosen s + 1e-20)   (renormalize)
 *   weight_j = scale * s_j                                    (otherwise)
 * A softmax row without a logit above -inf has s = 0.  The bias only chooses:
 * it gets no gradient.  counts[e] is the number of tokens sent to expert e.
 */
typedef struct {
  const void* logits;          /* [tokens][ld], element type dtype */
  const float* bias;           /* [experts] or NULL */
  float* weights;              /* [tokens][k] */
  int64_t* indices;            /* [tokens][k] */
  int64_t* counts;             /* [experts] or NULL */
  int64_t tokens, experts, ld;
  int dtype;
  int score;                   /* 0 softmax, 1 sigmoid */
  int k, groups, top_groups, group_top;
  int renormalize;
  float scale;
} muon_train_route_args;

int muon_train_route_sm100(const muon_train_route_args* args, void* stream);

/* grad_logits[tokens][experts] (element type dtype, contiguous) from
 * grad_weights[tokens][k]; args: the forward call's logits, indices and
 * settings (weights, counts and bias are not used).  An index outside the
 * experts is left out. */
int muon_train_route_backward_sm100(const muon_train_route_args* args, const float* grad_weights,
                                    void* grad_logits, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MUON_TRAIN_SM100_H */

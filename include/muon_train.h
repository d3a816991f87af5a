/*
 * muon_train.h — C ABI of the operators of a training step around the Muon update
 * (same library as muon_polar.h: libmuon_polar.so).
 *
 *   norms    the norms before and after a block, with its gate and residual scale
 *   distill  the loss against a teacher's top logits
 *
 * All functions are asynchronous on the given HIP stream.  Pointers are device pointers
 * unless said otherwise; structs are read during the call only.  No function allocates
 * device memory or synchronises.  Return value: MUON_POLAR_OK (0) or a negative
 * muon_polar_status; muon_polar_last_error() gives the detail.  Results are the same
 * bits on every run: no sum depends on the order in which workgroups arrive.
 * No reference counterpart: the reference orthogonalises one matrix and leaves the
 * training step to its caller (README.md:130).
 */
#ifndef MUON_TRAIN_H_
#define MUON_TRAIN_H_

#include "muon_polar.h"

#ifdef __cplusplus
extern "C" {
#endif

enum muon_train_dtype { MUON_TRAIN_F32 = 0, MUON_TRAIN_BF16 = 1 };

/* ------------------------------------------------------------------- norms
 * Of each row (a token of `d` channels), in fp32:
 *
 *     n = y·ρ1,  ρ1 = 1/sqrt(mean(y²) + eps)       (post_norm; otherwise n = y)
 *     u = n·post_weight
 *     R = scale·residual + gate·u
 *     h = R·ρ2·pre_weight,  ρ2 = 1/sqrt(mean(R²) + eps)   (pre_norm; otherwise no h)
 *
 * residual_out = R and normed = h are rounded once; h is taken from the unrounded R. */
enum muon_train_gate {
    MUON_TRAIN_GATE_NONE = 0,
    MUON_TRAIN_GATE_CHANNEL = 1,  /* [d] */
    MUON_TRAIN_GATE_SEQUENCE = 2, /* [rows / rows_per_sequence, d] */
    MUON_TRAIN_GATE_TOKEN = 3,    /* [rows] */
    MUON_TRAIN_GATE_FULL = 4      /* [rows, d] */
};
enum muon_train_scale {
    MUON_TRAIN_SCALE_NUMBER = 0, /* scale_value */
    MUON_TRAIN_SCALE_SCALAR = 1, /* scale[0], fp32 */
    MUON_TRAIN_SCALE_VECTOR = 2  /* scale[d], fp32 */
};

typedef struct muon_train_norms_args {
    int64_t rows, d;           /* d at most 16384 */
    int64_t rows_per_sequence; /* of a sequence gate: divides rows */
    int64_t ld_y, ld_residual; /* elements from row to row of y and residual (>= d); every
                                  other tensor is contiguous */
    const void *y, *residual;
    const void *post_weight, *pre_weight; /* [d], or null: 1 */
    const void *gate;
    const float *scale;
    double scale_value, eps;
    int y_dtype;        /* of y, normed and their gradients */
    int residual_dtype; /* of residual, residual_out and their gradients */
    int weight_dtype;   /* of post_weight, pre_weight and their gradients */
    int gate_dtype;     /* of gate and its gradient */
    int gate_kind, scale_kind, post_norm, pre_norm;
    /* forward */
    void *residual_out;
    void *normed; /* null without pre_norm */
    float *stats; /* [rows, 2]: ρ1, ρ2, which the backward pass reads; forward: may be null */
    /* backward: gradients of the outputs (null: zero) */
    const void *d_residual_out, *d_normed;
    void *d_y, *d_residual;                /* written */
    void *d_post_weight, *d_pre_weight;    /* [d], or null: not wanted */
    void *d_gate;                          /* of the gate's shape, or null */
    float *d_scale;                        /* [1] or [d], or null */
} muon_train_norms_args;

int muon_train_norms_forward(const muon_train_norms_args *args, hipStream_t stream);
/* Bytes of workspace the backward pass of these sizes and kinds needs (host call). */
int muon_train_norms_workspace(const muon_train_norms_args *args, size_t *bytes);
int muon_train_norms_backward(const muon_train_norms_args *args, void *workspace,
                              size_t workspace_bytes, hipStream_t stream);

/* ----------------------------------------------------------------- distill
 * Of each row (a token with `vocab` student logits z and k teacher logits t at the
 * indices i), in fp32:
 *
 *     p = softmax(t / τ) over the row's entries with 0 <= i < vocab (others are absent)
 *     loss = (1 − λ)·τ²·Σ_j p_j·(log p_j − log softmax(z / τ)[i_j]) + λ·CE(z, label)
 *     grad = g·[(1 − λ)·τ·(softmax(z / τ) − p) + λ·(softmax(z) − onehot(label))]
 *
 * with λ = label_weight.  A row whose entries are all absent or −inf has no first term, a
 * row whose label is outside [0, vocab) no second.  An index that occurs twice counts
 * twice.  `grad` may be `logits` itself (same address and row length); otherwise the two
 * must not overlap. */
typedef struct muon_train_distill_args {
    int64_t rows, vocab, k; /* k: 1 to 1024 */
    int64_t ld_logits, ld_grad; /* elements from row to row, >= vocab */
    const void *logits;         /* [rows, vocab] */
    const void *teacher_logits; /* [rows, k] */
    const void *teacher_indices; /* [rows, k], int32 or int64 */
    const int64_t *labels;      /* [rows], or null: no second term */
    const float *grad_loss;     /* [rows], or null: grad_value for every row */
    double temperature, label_weight, grad_value;
    int logits_dtype, teacher_dtype, index_bytes; /* index_bytes: 4 or 8 */
    float *loss;  /* [rows] */
    float *stats; /* [rows, 4]: max z, 1 / Σ exp((z − max) / τ), 1 / Σ exp(z − max), 0 */
    void *grad;   /* [rows, vocab], logits' dtype */
} muon_train_distill_args;

/* loss, and where they are not null stats and (in the same pass over the logits) grad. */
int muon_train_distill_forward(const muon_train_distill_args *args, hipStream_t stream);
/* grad from the stats of a forward pass. */
int muon_train_distill_backward(const muon_train_distill_args *args, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* MUON_TRAIN_H_ */

/*
 * muon_train.h — C ABI of the operators of a training step around the Muon update
 * (same library as muon_polar.h: libmuon_polar.so).
 *
 *   norms    the norms before and after a block, with its gate and residual scale
 *   distill  the loss against a teacher's top logits
 *   fp8      products in 8-bit floating point with a scale for each block of 128
 *
 * All functions are asynchronous on the given HIP stream.  Pointers are device pointers
 * unless said otherwise; structs are read during the call only.  No function allocates
 * device memory or synchronises.  Return value: MUON_POLAR_OK (0) or a negative
 * muon_polar_status; muon_polar_last_error() gives the detail.  Outputs must not overlap
 * inputs or each other but where that is said; the large ones are checked.  Results are the
 * same bits on every run: no sum depends on the order in which workgroups arrive.
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
/* Bytes of workspace the backward pass of these sizes and kinds needs (host call): 2·d fp32 (3·d
 * with a scale vector) for each workgroup that the card holds at once, and for each sequence at
 * least with a sequence gate. */
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
 * row whose label is outside [0, vocab) no second, whatever its logits are.  An index that
 * occurs twice counts twice.  `grad` may be `logits` itself (same address and row length); otherwise the two
 * must not overlap. */
typedef struct muon_train_distill_args {
    int64_t rows, vocab, k; /* k: 1 to 1024 */
    int64_t ld_logits, ld_grad; /* elements from row to row, >= vocab */
    const void *logits;         /* [rows, vocab] */
    const void *teacher_logits; /* [rows, k] */
    const void *teacher_indices; /* [rows, k], int32 or int64 */
    const int64_t *labels;      /* [rows], or null: no second term */
    const float *grad_loss;     /* [rows], or null: grad_value for every row */
    double temperature, label_weight, grad_value; /* temperature: normal in fp32, below 1e30 */
    int logits_dtype, teacher_dtype, index_bytes; /* index_bytes: 4 or 8 */
    float *loss;  /* [rows] */
    float *stats; /* [rows, 4]: max z, 1 / Σ exp((z − max) / τ), 1 / Σ exp(z − max) (labels),
                     1 / Σ exp((t − max t) / τ) (0 without entries); 1 / Σ is NaN of a
                     row that is all −inf */
    void *grad;   /* [rows, vocab], logits' dtype */
} muon_train_distill_args;

/* loss, and where they are not null stats and (in the same pass over the logits) grad. */
int muon_train_distill_forward(const muon_train_distill_args *args, hipStream_t stream);
/* grad from the stats of a forward pass. */
int muon_train_distill_backward(const muon_train_distill_args *args, hipStream_t stream);

/* --------------------------------------------------------------------- fp8
 * A matrix [rows, cols] held as e4m3 values (OCP, no infinities, largest 448) and one fp32
 * scale for each block of block_rows x 128 elements, block_rows 1 (activations and
 * gradients) or 128 (weights):
 *
 *     s = max(amax·(1/448), 2^-126)       amax: largest |x| of the block
 *     value = round_to_nearest_even_e4m3(x·(1/s))
 *
 * in fp32 (1/448 the nearest fp32).  A block with an infinity or a NaN has no finite
 * element back.  The rows of values lie `ld` bytes apart, a multiple of 128 at least cols,
 * and are zero past cols (operands of products: a multiple of 16).  Scale (i, j), of row block i and column block j, is at
 * scales[i·scale_row + j·scale_col]. */
typedef struct muon_train_fp8_quantize_args {
    int64_t rows, cols, ld_x; /* elements from row to row of x (>= cols) */
    const void *x;
    int x_dtype, block_rows;
    void *values;    /* [rows, roundup(cols, 128)], or null */
    float *scales;   /* block_rows 1: [ceil(cols / 128)][rows] (scale_row 1);
                        block_rows 128: [ceil(rows / 128)][ceil(cols / 128)] */
    void *values_t;  /* of the transposed matrix: [cols, roundup(rows, 128)], or null */
    float *scales_t; /* block_rows 1: [ceil(rows / 128)][cols]; block_rows 128: the
                        transposed matrix's scales are the same ones, scales with scale_row
                        and scale_col changed over (scales_t unused, scales written) */
} muon_train_fp8_quantize_args;
int muon_train_fp8_quantize(const muon_train_fp8_quantize_args *args, hipStream_t stream);

/* c[m][n] = Σ_blocks a_scale·b_scale·Σ_{k in block} a[m][k]·b[n][k], both operands with k
 * running along their rows, blocks summed in fp32, rounded once.  A block's own sum is in fp32
 * for a c of fp32.  For one of bf16 the matrix unit adds eight products (k = 8i .. 8i + 7) at a
 * time and cuts each off below 2^-13 of their largest: at most 7·2^-13 of the sum of |a·b|,
 * 1.5e-5 to 7e-5 of a result's 2-norm measured.  a_scale·b_scale may leave fp32's range where
 * the result does not. */
enum { MUON_TRAIN_FP8_MAX_LD = 1 << 22, MUON_TRAIN_FP8_MAX_SCALES = 1 << 28 };
typedef struct muon_train_fp8_operand {
    const void *values; /* [rows, k], 16-byte aligned */
    const float *scales;
    int64_t ld, scale_row, scale_col; /* ld at most MAX_LD, scale_col·(k / 128 + 1) MAX_SCALES */
    int block_rows; /* 1 (scale_row must be 1) or 128 */
} muon_train_fp8_operand;
typedef struct muon_train_fp8_matmul_args {
    int64_t m, n, k; /* k a multiple of 128 (values padded with zeros); 0: c is zeros */
    muon_train_fp8_operand a, b;
    void *c; /* [m, n] */
    int64_t ldc;
    int c_dtype;
} muon_train_fp8_matmul_args;
int muon_train_fp8_matmul(const muon_train_fp8_matmul_args *args, hipStream_t stream);
/* The same with a workspace (16-byte aligned): a product of few tiles and a long k is then
 * split along k over the compute units, its parts added up in order.  Bytes that it takes, 0 if
 * it is not split (host call; a null workspace: not split). */
int muon_train_fp8_matmul_workspace(const muon_train_fp8_matmul_args *args, size_t *bytes);
int muon_train_fp8_matmul_in(const muon_train_fp8_matmul_args *args, void *workspace,
                             size_t workspace_bytes, hipStream_t stream);

/* c = held(x) · wᵀ for up to 16 rows of x [m, cols], quantised in blocks of 1 x 128 in the
 * same kernel: the bits of muon_train_fp8_quantize and muon_train_fp8_matmul.  w: rows of
 * roundup(cols, 128) values, block_rows 128. */
typedef struct muon_train_fp8_decode_args {
    int64_t m, n, cols, ld_x; /* m: 0 to 16 */
    const void *x;
    int x_dtype;
    muon_train_fp8_operand w;
    void *c; /* [m, n] */
    int64_t ldc;
    int c_dtype;
} muon_train_fp8_decode_args;
int muon_train_fp8_decode(const muon_train_fp8_decode_args *args, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* MUON_TRAIN_H_ */

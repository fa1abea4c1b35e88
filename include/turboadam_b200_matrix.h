/*
 * turboadam_b200_matrix.h -- C ABI of the matrix operators beside the packed
 * optimizer step (turboadam_b200.h), in the same library and with the same
 * conventions: plain pointers and sizes, every pointer named *_dev is device
 * memory of the caller, `stream` is a cudaStream_t passed as void*, calls are
 * asynchronous on it and return host-side validation and launch errors
 * (ta_last_error has the message). A call enqueues kernels (and one memset)
 * only, so it can be captured into a CUDA graph. A workspace needs no set-up
 * and holds nothing between calls; calls that can overlap need workspaces of
 * their own. status_dev is a 4-byte word the caller zeroes once and may share
 * between calls, in device memory (ta_read_status takes its address) or in
 * pinned host memory: a bounded wait that ran out sets TA_STATUS_WAIT_TIMEOUT
 * in it, and the call's results are void.
 *
 * None of the three has a counterpart in the reference (davidkny22/turboadam),
 * which updates every tensor elementwise.
 */
#ifndef TURBOADAM_B200_MATRIX_H
#define TURBOADAM_B200_MATRIX_H

#include "turboadam_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* a third element type, for the matrix operators only */
enum { TA_F16 = 2 };

/* activations of ta_linear_forward */
enum {
  TA_ACT_NONE = 0,
  TA_ACT_RELU = 1,
  TA_ACT_GELU = 2,      /* z Phi(z)                                        */
  TA_ACT_GELU_TANH = 3, /* z (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3))) / 2 */
  TA_ACT_SILU = 4       /* z / (1 + exp(-z))                               */
};

/* ta_ortho_tensor.flags */
enum {
  TA_ORTHO_UPDATE = 1u << 0, /* out <- keep * out - gain * O instead of out <- O */
  TA_ORTHO_PAIR = 1u << 1    /* hold a 32-bit input as a pair of fp16 numbers
                                (22 bits) instead of rounding it to one         */
};

/*
 * A stack of `batch` matrices [rows][cols], contiguous, row-major.
 * With u the input (no momentum), the momentum m <- mu m + (1 - mu) in, or
 * with nesterov mu m + (1 - mu) in:
 *   X <- u / (|u|_F + eps);  `steps` times, with that step's (a, b, c):
 *   A <- X X^T (X^T X if rows > cols);  X <- (a I + b A + c A^2) X
 *   O <- X
 * The products run on fp16 operands (X, A and the polynomial, each scaled by
 * a power of two) with fp32 sums; X enters unrounded (16-bit inputs) or to 22
 * bits, of which the first A sees 11 (TA_ORTHO_PAIR), and the
 * first two steps (of large long matrices all steps) act in pairs, X <- P' P X
 * with the second Gram matrix formed from the first. The relative error is
 * 0.8e-3 to 2e-3 of O (Frobenius norm; 1.5e-3 to 5e-3 in the 2-norm; more for
 * matrices of a few rows close to singular); bf16 operands would leave 1e-2
 * to 3e-2. Coefficients have to keep singular values below 8 (the quintic: 1.3)
 * and a step's polynomial and the product of a pair's below 255 (the quintic:
 * 12), or fp16 overflows and O is NaN. A
 * zero matrix gives zero; a NaN or an infinity in a matrix makes all of that
 * matrix's O NaN.
 */
typedef struct ta_ortho_tensor {
  const void* in_dev;
  void* momentum_dev; /* NULL: orthogonalise `in` itself   */
  void* out_dev;      /* result or (UPDATE) parameter      */
  int64_t batch, rows, cols;
  int32_t in_dtype, momentum_dtype, out_dtype; /* TA_F32, TA_BF16 or TA_F16 */
  uint32_t flags;
  double keep, gain; /* TA_ORTHO_UPDATE */
} ta_ortho_tensor;

typedef struct ta_ortho_options {
  const double* coefficients; /* host, [steps][3] */
  int32_t steps;              /* 1 .. 32          */
  int32_t nesterov;
  double eps;
  double momentum;
} ta_ortho_options;

/* Workspace bytes of ta_orthogonalize for this list (0: an invalid list). */
TA_API size_t ta_ortho_workspace_size(const ta_ortho_tensor* tensors, int32_t n_tensors,
                                      const ta_ortho_options* options);

/* Orthogonalises (and, with TA_ORTHO_UPDATE, applies) the whole list: three or more small kernels
 * (tables, momentum and norm, scaling), then one cooperative kernel for every 8 distinct shapes. */
TA_API ta_status ta_orthogonalize(const ta_ortho_tensor* tensors, int32_t n_tensors,
                                  const ta_ortho_options* options, void* workspace_dev,
                                  size_t workspace_bytes, uint32_t* status_dev, void* stream);

/*
 * y = act(x w^T + bias) + residual, in one product with that epilogue.
 * x is [tokens][fan_in], w [fan_out][fan_in], each with one unit stride;
 * residual and y have unit column stride. Sums, bias, activation and residual
 * are in fp32, rounded once. deriv_dev (optional): receives act' of the
 * unrounded argument in 16-bit codes for ta_linear_backward of the same dtype,
 * in rows of fan_out rounded up to 8. A code is off by at most 2^-15, and
 * relative to act' by at most 2^-9 (bf16, down to 2^-93) or 2^-12 (fp16, down
 * to 2^-13, 2^-25 absolute beyond).
 */
typedef struct ta_linear {
  const void* x_dev;
  const void* w_dev;
  const void* bias_dev;     /* NULL: none */
  const void* residual_dev; /* NULL: none */
  void* y_dev;
  int16_t* deriv_dev;
  int64_t tokens, fan_in, fan_out;
  int64_t x_strides[2], w_strides[2]; /* elements */
  int64_t residual_stride, y_stride;  /* elements between rows */
  int32_t dtype;                      /* TA_BF16 or TA_F16: x, w, residual, y */
  int32_t bias_dtype;                 /* TA_F32, TA_BF16 or TA_F16            */
  int32_t activation;
  int32_t reserved0;
} ta_linear;

TA_API size_t ta_linear_workspace_size(const ta_linear* op);
TA_API ta_status ta_linear_forward(const ta_linear* op, void* workspace_dev,
                                   size_t workspace_bytes, uint32_t* status_dev, void* stream);

/*
 * Gradients of ta_linear_forward: dz = dy act', dx = dz w, dw = dz^T x,
 * db = column sums of dz (the residual's gradient is dy). Each output may be
 * NULL. dz is rounded once to the operand type for the two products; db sums
 * it unrounded, in a fixed order. dw has one unit stride.
 */
typedef struct ta_linear_grad {
  const void* dy_dev;
  const int16_t* deriv_dev; /* from the forward pass; NULL: no activation */
  const void* x_dev;        /* needed for dw */
  const void* w_dev;        /* needed for dx */
  void* dx_dev;             /* [tokens][fan_in], contiguous */
  void* dw_dev;
  void* db_dev;
  int64_t tokens, fan_in, fan_out;
  int64_t dy_stride;
  int64_t x_strides[2], w_strides[2], dw_strides[2];
  int32_t dtype;      /* TA_BF16 or TA_F16: dy, x, w, dx, dw */
  int32_t bias_dtype; /* of db */
} ta_linear_grad;

TA_API size_t ta_linear_backward_workspace_size(const ta_linear_grad* op);
TA_API ta_status ta_linear_backward(const ta_linear_grad* op, void* workspace_dev,
                                    size_t workspace_bytes, uint32_t* status_dev, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TURBOADAM_B200_MATRIX_H */

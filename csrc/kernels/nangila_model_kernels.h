/* C launchers of the kernels that a decoder's training step runs next to its products: RMS norm, rotary positions, and the
 * orthogonalisation of updates. Types are NANGILA_F32 / NANGILA_F16 / NANGILA_BF16. Every function queues on `stream` and returns a
 * cudaError_t as int. */
#ifndef NANGILA_MODEL_KERNELS_H
#define NANGILA_MODEL_KERNELS_H
#include <cuda_runtime.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NANGILA_NORM_MAX_D 32768

/* h = x + residual (rounded to the type of x; h = x without a residual), y = h * rstd * weight with rstd = (mean(h^2) + eps)^-1/2.
 * Rows of x and residual are `*_stride` elements apart; everything else is packed. */
typedef struct {
  const void* x;
  const void* residual; /* NULL: none */
  const void* weight;
  void* h;              /* NULL without a residual */
  void* y;              /* NULL with q */
  float* rstd;          /* rows; NULL: not kept */
  uint8_t* q;           /* e4m3 output in place of y; NULL: none */
  float* scale;         /* with q: rows, or rows x d / group */
  int64_t rows, x_stride, residual_stride;
  int32_t d, group;     /* group: 0 (one scale a row) or 128 */
  int32_t dtype, weight_dtype;
  float eps;
} NangilaNormParams;
int nangila_rms_norm_forward(const NangilaNormParams* p, cudaStream_t stream);

/* dx = dh + rstd * (dy w - xhat mean(dy w xhat)) with xhat = h rstd; dw = sum over rows of dy xhat. */
typedef struct {
  const void* h;        /* the normalised rows, h_stride apart */
  const void* dy;       /* NULL: no gradient arrived at y */
  const void* dh;       /* NULL: no gradient arrived at h */
  const void* weight;
  const float* rstd;
  void* dx;             /* packed; NULL: not wanted */
  void* dw;             /* d values of the weight's type; NULL: not wanted */
  float* partial;       /* scratch: nangila_rms_norm_partials() x d floats, with dw */
  int64_t rows, h_stride, dy_stride, dh_stride;
  int32_t d, dtype, weight_dtype;
} NangilaNormGradParams;
int nangila_rms_norm_partials(int64_t rows, int32_t d, int32_t dtype, int32_t* count);
int nangila_rms_norm_backward(const NangilaNormGradParams* p, cudaStream_t stream);

/* Turns pairs of columns of one or two tensors [batch, seq, heads, d] by the angles of their positions. */
typedef struct {
  const void* in[2];    /* in[1] NULL: one tensor */
  void* out[2];         /* packed [batch, seq, heads, d] */
  int64_t stride_b[2], stride_t[2], stride_h[2]; /* of the inputs, in elements; columns are adjacent */
  int32_t heads[2];
  int64_t batch, seq;
  int32_t d, rot;       /* the first `rot` columns are turned */
  int32_t half;         /* 0: pairs (2i, 2i + 1), 1: pairs (i, i + rot / 2) */
  int32_t inverse;      /* 1: by the negative angles (the gradient) */
  const float* table;   /* [table_rows, rot / 2, 2]: cosine and sine */
  int64_t table_rows;
  const void* positions; /* NULL: 0 .. seq - 1 */
  int32_t positions_64;  /* 1: int64, 0: int32 */
  int64_t pos_stride_b, pos_stride_t;
  int32_t dtype;
} NangilaRotaryParams;
int nangila_rotary(const NangilaRotaryParams* p, cudaStream_t stream);

/* Newton-Schulz steps on `count` matrices of rows x cols, all of them together. */
#define NANGILA_ORTH_MAX_COUNT 64
#define NANGILA_ORTH_MAX_STEPS 32
typedef struct {
  const void* grad[NANGILA_ORTH_MAX_COUNT]; /* packed rows x cols */
  float* momentum[NANGILA_ORTH_MAX_COUNT];  /* NULL in [0]: none */
  void* param[NANGILA_ORTH_MAX_COUNT];      /* NULL in [0]: the result goes to `out` */
  void* out;                                /* bf16, count x rows x cols */
  int32_t count, rows, cols;
  int32_t grad_dtype, param_dtype;
  int32_t steps, nesterov;
  float coefficients[NANGILA_ORTH_MAX_STEPS][3];
  float eps, mu, decay, rate;               /* param = param * decay - rate * result */
  void* workspace;                          /* nangila_orth_workspace() bytes, 256-byte aligned */
} NangilaOrthParams;
int64_t nangila_orth_workspace(int32_t count, int32_t rows, int32_t cols);
int nangila_orth(const NangilaOrthParams* p, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
#endif

/* C launchers of the kernels at a language model's two ends: token embeddings, dropout, and the loss of a head whose logits are not kept.
 * Types are NANGILA_F32 / NANGILA_F16 / NANGILA_BF16. Every function queues on `stream` and returns a cudaError_t as int. */
#ifndef NANGILA_VOCAB_KERNELS_H
#define NANGILA_VOCAB_KERNELS_H
#include <cuda_runtime.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* out[i] = residual[i] + (kept(i) ? x[i] * scale : 0), without a residual 0 in its place; kept(i): the 32-bit number of element i reaches
 * `least`, 0 to 2^32. */
typedef struct {
  const void* x;
  const void* residual;    /* NULL: none */
  void* out;
  const int64_t* seed_ptr; /* on the device, read when the kernel runs; NULL: `seed` */
  int64_t n;               /* adjacent elements */
  uint64_t seed;
  uint64_t least;
  uint32_t draw;
  int32_t dtype;
  float scale;
} NangilaDropoutParams;
int nangila_dropout(const NangilaDropoutParams* p, cudaStream_t stream);

/* out[i] = scale * weight[ids[i]], rows of d adjacent elements; an id outside 0 .. rows - 1 makes its row not a number. */
typedef struct {
  const void* ids;         /* n adjacent int64 (ids_64) or int32 */
  const void* weight;      /* rows weight_stride elements apart */
  void* out;               /* packed, 16-byte aligned */
  int64_t n, rows, weight_stride;
  int32_t d, dtype, ids_64;
  float scale;
} NangilaEmbeddingParams;
int nangila_embedding(const NangilaEmbeddingParams* p, cudaStream_t stream);

/* dw[v] = scale * sum of dy[i] over the i with ids[i] = v, in the order of i; zero for the other rows and for `padding`. */
typedef struct {
  const void* ids;
  const void* dy;          /* rows dy_stride elements apart */
  void* dw;                /* packed, 32-byte aligned */
  void* workspace;         /* nangila_embedding_workspace() bytes, 256-byte aligned */
  int64_t n, rows, dy_stride, padding; /* padding: -1 for none */
  int32_t d, dtype, ids_64;
  float scale;
} NangilaEmbeddingGradParams;
int64_t nangila_embedding_workspace(int64_t n, int64_t rows, int32_t d);
int nangila_embedding_backward(const NangilaEmbeddingGradParams* p, cudaStream_t stream);

#define NANGILA_EMBEDDING_MAX_TOKENS 0x7fffff00
#define NANGILA_EMBEDDING_MAX_ROWS 0x7fffff00
#define NANGILA_EMBEDDING_MAX_WIDTH (1 << 20)

/* Softmax cross entropy of z = x w^T + bias over the first `classes` rows of w, rows of z that are never kept whole.
 *   loss_i = log sum_v exp(z_iv) - z_i,target(i);   0 where the target is `ignore`, not a number where it lies outside 0 .. classes - 1
 * and, for the gradients, with u_i = *upstream (over the count of targets that are not ignored if mean) or upstream[i]:
 *   G_iv = u_i (exp(z_iv - lse_i) - [v = target(i)]),  dx = G w,  dw = G^T x,  dbias = sum_i G_i;  rows whose loss is 0 or not a number by the
 * rule above add nothing, whatever they hold. */
#define NANGILA_CE_LOSSES 0     /* losses and lse; `loss` if it is there */
#define NANGILA_CE_BOTH 1       /* losses, and the gradients for u_i = 1 (over the count if mean); bf16 only */
#define NANGILA_CE_GRADIENTS 2  /* the gradients, from the losses and lse of a call before */
typedef struct {
  const void* x;           /* n rows of d, x_stride elements apart; 16-byte aligned, strides multiples of 8 elements */
  const void* w;           /* rows x d, w_stride elements apart; the same */
  const void* bias;        /* rows; NULL: none */
  const int64_t* targets;  /* n */
  int64_t n, x_stride, w_stride, ignore;
  int32_t d;               /* a multiple of 8 */
  int32_t rows, classes;
  int32_t dtype;           /* NANGILA_F16 or NANGILA_BF16 */
  int32_t bias_dtype;      /* any of the three */
  int32_t mean;            /* u_i is divided by the count of targets that are not ignored */
  float* losses;           /* n */
  float* losses_too;       /* n: the same once more; NULL: not wanted */
  float* lse;              /* n */
  float* loss;             /* 1: the sum of the losses, or their mean; NULL: not wanted */
  void* dx;                /* packed, of the type of x; NULL: not wanted */
  void* dw;                /* rows x d, packed; NULL: not wanted */
  void* dbias;             /* rows, of the bias's type, NANGILA_CE_BOTH: float32; NULL: not wanted */
  const float* upstream;   /* NANGILA_CE_GRADIENTS: 1 value, or n */
  int32_t upstream_rows;   /* whether there are n */
  void* workspace;         /* nangila_linear_ce_workspace() bytes, 256-byte aligned */
} NangilaLinearCeParams;
int64_t nangila_linear_ce_workspace(const NangilaLinearCeParams* p, int what);
int nangila_linear_ce(const NangilaLinearCeParams* p, int what, cudaStream_t stream);

/* The arrays (NULL: none) multiplied by *factor, rounded to their types; nothing of them is read or written where it is one. And `narrow`, the values of `wide` times
 * *factor. */
typedef struct {
  void* array[2];
  int64_t count[2];
  int32_t dtype[2];
  const float* wide;       /* NULL: none */
  void* narrow;
  int64_t narrow_count;
  int32_t narrow_dtype;
  const float* factor;
} NangilaRescaleParams;
int nangila_rescale(const NangilaRescaleParams* p, cudaStream_t stream);

#define NANGILA_CE_MAX_WIDTH 65536
#define NANGILA_CE_MAX_CLASSES (1 << 24)

#ifdef __cplusplus
}
#endif
#endif

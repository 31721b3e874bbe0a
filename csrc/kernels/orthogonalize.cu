// Updates made orthogonal by Newton-Schulz steps, as the Muon optimiser does, for several matrices of one shape at a time (sm_100a).
//
//   X = U / max(|U|_F, eps), and `steps` times:   A = X X^T,   B = b A + c A^2,   X <- a X + B X
//
// X has m rows and n >= m columns; a matrix that is taller than wide is kept as it lies, and its transpose is what the formulas speak of.
// The three products are one tcgen05 kernel with different operands and epilogues: operands come through TMA (128-byte swizzle, K-major or
// MN-major, so that nothing is transposed in memory), one thread issues the products with the accumulator in tensor memory, four warps read
// it back and write results. Of the symmetric A and A^2 only the tiles that reach the lower triangle are computed; their epilogue writes both halves.
//
// Roundings. The products' operands are rounded to fp16 (11 bits; the values are bounded, so that bf16's range is not needed and its 8 bits
// would cost a factor of eight), the accumulator is fp32. A and B multiply X: their errors, and those of X inside the products, come out as relative
// errors of a few 2^-12 of directions that are large already. The term a X is another matter: it alone carries the small singular values up, by
// a^5 = 485 with the usual coefficients, and what is lost of them in X's rounding grows along. So the state X is kept in two halves, hi + lo / 2048, both fp16
// (22 bits), hi being the operand of the products, and a X is formed from both in fp32.
//
// X is kept times a power of two near sqrt(n), so that an orthogonal matrix has elements near one and fp16's subnormals are far away.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <mutex>

#include "follow.cuh"
#include "nangila_kernels.h"
#include "nangila_model_kernels.h"
#include "ptx_sm100.cuh"
#include "quant.cuh"

namespace nangila {
namespace {

using namespace sm100;

constexpr int kTileM = 128;
constexpr int kSlabK = 64;                       // one 128-byte swizzle row of fp16
constexpr int kABytes = kTileM * kSlabK * 2;
constexpr int kGemmThreads = 192;                // warp 0: TMA, warp 1: products, warps 2 to 5: epilogue
constexpr uint64_t kTimeoutNs = 10ull * 1000 * 1000 * 1000;
constexpr float kLoScale = 2048.0f;
template <int TN>
struct Tile {
  static constexpr int kBBytes = TN * kSlabK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = 196608 / kStageBytes;         // 4 or 6
  static constexpr int kSmem = kStages * kStageBytes + 1024 + 256;
};

enum Kind { kGram, kPoly, kUpdate, kFinal };

struct Product {
  int M, N, K;             // D is M x N
  int tiles_m, tiles_n, per, total;  // tiles of one matrix, of all
  int lower;               // only tiles that reach the lower triangle
  float alpha, beta;       // gram: D alpha;  poly: alpha A + beta D;  update: alpha X + D
  float unscale;           // final: result = (alpha X + D) unscale
  const __half* in;        // poly: A;  update: hi
  __half* lo;              // update: read and written in place
  __half* out;             // gram, poly, update
  int64_t ld, matrix;      // of `in`, `lo` and `out`, in elements
  __nv_bfloat16* result;   // final: packed M x N, or NULL
  int param_dtype, vector; // final: the parameters' type; runs of eight elements can be written
  float decay, rate;
  void* param[NANGILA_ORTH_MAX_COUNT];
};

struct TileAt {
  int batch, m0, n0;
};
template <int TN>
__device__ __forceinline__ TileAt tile_at(const Product& p, int i) {
  TileAt t;
  t.batch = i / p.per;
  int r = i - t.batch * p.per;
  int rb, cb;
  if (!p.lower) {
    cb = r / p.tiles_m;  // neighbours share the columns of the wide operand
    rb = r - cb * p.tiles_m;
  } else if (TN == 128) {
    rb = int((sqrtf(8.0f * r + 1.0f) - 1.0f) * 0.5f);
    while (rb * (rb + 1) / 2 > r) --rb;
    while ((rb + 1) * (rb + 2) / 2 <= r) ++rb;
    cb = r - rb * (rb + 1) / 2;
  } else {  // two rows of tiles at a time, with h + 1 tiles each
    int h = int((sqrtf(4.0f * r + 1.0f) - 1.0f) * 0.5f);
    while (h * (h + 1) > r) --h;
    while ((h + 1) * (h + 2) <= r) ++h;
    r -= h * (h + 1);
    rb = 2 * h + (r > h ? 1 : 0);
    cb = r > h ? r - h - 1 : r;
  }
  t.m0 = rb * kTileM;
  t.n0 = cb * TN;
  return t;
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// x = hi + lo / 2048
__device__ __forceinline__ void split8(const float (&x)[8], uint4& hi, uint4& lo) {
  hi = pack8(x);
  float h[8], l[8];
  unpack8(hi, h);
#pragma unroll
  for (int k = 0; k < 8; ++k) l[k] = (x[k] - h[k]) * kLoScale;
  lo = pack8(l);
}
template <typename T>
__device__ __forceinline__ void update_param(T* p, int n, bool vector, const float (&r)[8], float decay, float rate) {
  if (vector) {
    float v[8];
    dev::Vec8<T>::load(p, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = v[k] * decay - rate * r[k];
    dev::Vec8<T>::store(p, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) p[k] = dev::Vec16<T>::from_float(dev::Vec16<T>::to_float(p[k]) * decay - rate * r[k]);
  }
}

// Eight results of one row, D[row][col .. col + 7], taken to where they belong. The row is inside the matrix, col < N.
template <int KIND>
__device__ __forceinline__ void finish8(const Product& p, int batch, int row, int col, float (&v)[8]) {
  const int64_t at = batch * p.matrix + int64_t(row) * p.ld + col;
  if constexpr (KIND == kGram || KIND == kPoly) {
    if (col > row) return;  // the other half is written from below the diagonal
    if constexpr (KIND == kGram) {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= p.alpha;
    } else {
      float a[8];
      unpack8(*reinterpret_cast<const uint4*>(p.in + at), a);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = __fmaf_rn(p.alpha, a[k], p.beta * v[k]);
    }
    __half* mirror = p.out + batch * p.matrix + int64_t(col) * p.ld + row;
    if (col + 7 <= row) {
      *reinterpret_cast<uint4*>(p.out + at) = pack8(v);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (col + k <= row) p.out[at + k] = __float2half_rn(v[k]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (col + k < row) mirror[k * p.ld] = __float2half_rn(v[k]);
  } else {
    float hi[8], lo[8];
    unpack8(*reinterpret_cast<const uint4*>(p.in + at), hi);
    unpack8(*reinterpret_cast<const uint4*>(p.lo + at), lo);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __fmaf_rn(p.alpha, __fmaf_rn(lo[k], 1.0f / kLoScale, hi[k]), v[k]);
    if constexpr (KIND == kUpdate) {
      uint4 h, l;
      split8(v, h, l);
      *reinterpret_cast<uint4*>(p.out + at) = h;
      *reinterpret_cast<uint4*>(p.lo + at) = l;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= p.unscale;
      const int left = p.N - col;
      const int64_t to = int64_t(row) * p.N + col;
      if (p.result != nullptr) {
        __nv_bfloat16* o = p.result + int64_t(batch) * p.M * p.N + to;
        if (p.vector) {
          dev::Vec8<__nv_bfloat16>::store(o, v);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < left) o[k] = __float2bfloat16_rn(v[k]);
        }
      } else if (p.param_dtype == NANGILA_F32) {
        update_param(static_cast<float*>(p.param[batch]) + to, left, p.vector != 0, v, p.decay, p.rate);
      } else if (p.param_dtype == NANGILA_BF16) {
        update_param(static_cast<__nv_bfloat16*>(p.param[batch]) + to, left, p.vector != 0, v, p.decay, p.rate);
      } else {
        update_param(static_cast<__half*>(p.param[batch]) + to, left, p.vector != 0, v, p.decay, p.rate);
      }
    }
  }
}

// D = A B for tiles of kTileM x TN of all matrices, walked over by CTAs that stay. A_MN / B_MN: the operand lies with its rows (columns of B)
// adjacent in memory, not its K. The accumulators of two tiles share tensor memory: the epilogue of one runs under the products of the next.
// A wait that runs out makes every result of this CTA from there on not a number.
template <int KIND, bool A_MN, bool B_MN, int TN>
__global__ void __launch_bounds__(kGemmThreads, 1) orth_product_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                                                                      const __grid_constant__ Product p) {
  using T = Tile<TN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + T::kStages * T::kStageBytes);
  uint64_t* empty = full + T::kStages;
  uint64_t* acc_full = empty + T::kStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;       // [2]
  uint64_t* drained = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile uint32_t* failed = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slabs = (p.K + kSlabK - 1) / kSlabK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < T::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 4);
    }
    mbar_init(drained, 1);
    *failed = 0;
    fence_barrier_init();
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
  }
  if (warp == 1) tmem_alloc(tmem_slot, 2 * TN);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  may_follow();
  follow();

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA ----------------
      int i = 0;  // slabs so far
      bool ok = true;
      for (int tile = blockIdx.x; tile < p.total && ok; tile += gridDim.x) {
        const TileAt at = tile_at<TN>(p, tile);
        for (int k = 0; k < slabs; ++k, ++i) {
          const int s = i % T::kStages;
          if (i >= T::kStages && !mbar_wait(&empty[s], uint32_t((i / T::kStages - 1) & 1), kTimeoutNs)) {
            *failed = 1;
            ok = false;
            break;
          }
          uint8_t* a = smem + s * T::kStageBytes;
          uint8_t* b = a + kABytes;
          const int k0 = k * kSlabK;
          mbar_arrive_expect_tx(&full[s], T::kStageBytes);
          if (A_MN) {
#pragma unroll
            for (int g = 0; g < kTileM / 64; ++g) tma_load_3d(a + g * 8192, &tmA, at.m0 + g * 64, k0, at.batch, &full[s]);
          } else {
            tma_load_3d(a, &tmA, k0, at.m0, at.batch, &full[s]);
          }
          if (B_MN) {
#pragma unroll
            for (int g = 0; g < TN / 64; ++g) tma_load_3d(b + g * 8192, &tmB, at.n0 + g * 64, k0, at.batch, &full[s]);
          } else {
            tma_load_3d(b, &tmB, k0, at.n0, at.batch, &full[s]);
          }
        }
      }
      // the copies that are still under way, if somebody has given up on them
      if (*failed != 0)
        for (int j = max(0, i - T::kStages); j < i; ++j) mbar_wait(&full[j % T::kStages], uint32_t((j / T::kStages) & 1), kTimeoutNs);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------- products ----------------
      constexpr uint32_t idesc = (1u << 4) | (uint32_t(A_MN) << 15) | (uint32_t(B_MN) << 16) | (uint32_t(TN >> 3) << 17) | (uint32_t(kTileM >> 4) << 24);
      int i = 0, n = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < p.total && ok; tile += gridDim.x, ++n) {
        const int acc = n & 1;
        if (n >= 2 && !mbar_wait(&acc_empty[acc], uint32_t((n / 2 - 1) & 1), kTimeoutNs)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t d = tmem + uint32_t(acc * TN);
        for (int k = 0; k < slabs; ++k, ++i) {
          const int s = i % T::kStages;
          if (!mbar_wait(&full[s], uint32_t((i / T::kStages) & 1), kTimeoutNs)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t a = smem_u32(smem + s * T::kStageBytes), b = a + kABytes;
#pragma unroll
          for (int kk = 0; kk < kSlabK / 16; ++kk) {
            // K-major: 16 elements along K are 32 bytes of a swizzle row; MN-major: 16 K-rows are two groups of eight rows of 128 bytes
            const uint64_t ad = A_MN ? make_smem_desc(a + kk * 2048, 8192, 1024) : make_smem_desc(a + kk * 32, 16, 1024);
            const uint64_t bd = B_MN ? make_smem_desc(b + kk * 2048, 8192, 1024) : make_smem_desc(b + kk * 32, 16, 1024);
            umma_f16(d, ad, bd, idesc, (k > 0 || kk > 0) ? 1u : 0u);
          }
          umma_commit(&empty[s]);
        }
        if (ok) umma_commit(&acc_full[acc]);
      }
      if (!ok) {
        *failed = 1;
        umma_commit(drained);
        mbar_wait(drained, 0, kTimeoutNs);
      }
    }
  } else {
    // ---------------- epilogue ----------------
    const int quad = warp & 3;  // the lanes of tensor memory that this warp may read
    int n = 0;
    for (int tile = blockIdx.x; tile < p.total; tile += gridDim.x, ++n) {
      const TileAt at = tile_at<TN>(p, tile);
      const int acc = n & 1;
      bool ok = *failed == 0 && mbar_wait(&acc_full[acc], uint32_t((n / 2) & 1), kTimeoutNs);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) *failed = 1;
      tc_fence_after_sync();
      const int row = at.m0 + quad * 32 + lane;
#pragma unroll 1
      for (int c = 0; c < TN; c += 16) {
        if (at.n0 + c >= p.N) break;
        __syncwarp();  // the reads of tensor memory are the whole warp's
        float v[16];
        if (ok) {
          tmem_ld_32x32b_x16(tmem + (uint32_t(quad * 32) << 16) + uint32_t(acc * TN + c), v);
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) v[k] = __uint_as_float(0x7fc00000u);
        }
        if (row < p.M) {
#pragma unroll
          for (int g = 0; g < 16; g += 8) {
            float w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = v[g + k];
            if (at.n0 + c + g < p.N) finish8<KIND>(p, at.batch, row, at.n0 + c + g, w);
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 2 * TN);
}

// ---- from the gradients to X -------------------------------------------------------------------------------------------------
// Two passes over the gradients, which are small next to the products: the sum of squares, in 64 bits and in an order that the sizes determine,
// then X. With momentum the first pass also advances it: M <- mu M + G, U = G + mu M (Nesterov) or M.
constexpr int kPrepT = 256;
constexpr int kMaxChunks = 512;
struct Prep {
  const void* grad[NANGILA_ORTH_MAX_COUNT];
  float* momentum[NANGILA_ORTH_MAX_COUNT];
  double* partial;   // [count][chunks]
  __half* hi;
  __half* lo;
  int64_t numel, ld, matrix;
  int cols, chunks, nesterov, vector;
  float mu, eps, scale;
};
__device__ __forceinline__ double block_sum(double v, double* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < kPrepT / 32; ++i) v += s[i];
  return v;
}
template <typename T>
__global__ void __launch_bounds__(kPrepT) orth_norm_kernel(const __grid_constant__ Prep p) {
  __shared__ double s[kPrepT / 32];
  const T* g = static_cast<const T*>(p.grad[blockIdx.y]);
  float* m = p.momentum[blockIdx.y];
  const int64_t stride = int64_t(gridDim.x) * kPrepT, first = int64_t(blockIdx.x) * kPrepT + threadIdx.x;
  double sum = 0.0;
  may_follow();
  const int64_t runs = p.vector ? p.numel / 8 : 0;
  for (int64_t i = first; i < runs; i += stride) {
    float u[8];
    dev::Vec8<T>::load(g + i * 8, u);
    if (m != nullptr) {
      float v[8];
      dev::Vec8<float>::load(m + i * 8, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = __fmaf_rn(p.mu, v[k], u[k]);
        u[k] = p.nesterov ? __fmaf_rn(p.mu, v[k], u[k]) : v[k];
      }
      dev::Vec8<float>::store(m + i * 8, v);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sum = fma(double(u[k]), double(u[k]), sum);
  }
  for (int64_t i = runs * 8 + first; i < p.numel; i += stride) {
    float u = dev::Vec16<T>::to_float(g[i]);
    if (m != nullptr) {
      const float v = __fmaf_rn(p.mu, m[i], u);
      u = p.nesterov ? __fmaf_rn(p.mu, v, u) : v;
      m[i] = v;
    }
    sum = fma(double(u), double(u), sum);
  }
  sum = block_sum(sum, s);
  if (threadIdx.x == 0) p.partial[int64_t(blockIdx.y) * p.chunks + blockIdx.x] = sum;
}
template <typename T>
__global__ void __launch_bounds__(kPrepT) orth_start_kernel(const __grid_constant__ Prep p) {
  __shared__ double s[kPrepT / 32];
  const T* g = static_cast<const T*>(p.grad[blockIdx.y]);
  const float* m = p.momentum[blockIdx.y];
  follow();
  double sum = 0.0;
  for (int i = threadIdx.x; i < p.chunks; i += kPrepT) sum += p.partial[int64_t(blockIdx.y) * p.chunks + i];
  sum = sqrt(block_sum(sum, s));
  const double scale = double(p.scale) / (sum < double(p.eps) ? double(p.eps) : sum);
  const float f = float(scale);
  may_follow();
  const int64_t stride = int64_t(gridDim.x) * kPrepT, first = int64_t(blockIdx.x) * kPrepT + threadIdx.x;
  __half* hi = p.hi + blockIdx.y * p.matrix;
  __half* lo = p.lo + blockIdx.y * p.matrix;
  if (p.vector) {  // packed like the gradient
    for (int64_t i = first; i < p.numel / 8; i += stride) {
      float u[8];
      dev::Vec8<T>::load(g + i * 8, u);
      if (m != nullptr) {
        float v[8];
        dev::Vec8<float>::load(m + i * 8, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = p.nesterov ? __fmaf_rn(p.mu, v[k], u[k]) : v[k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] *= f;
      uint4 h, l;
      split8(u, h, l);
      *reinterpret_cast<uint4*>(hi + i * 8) = h;
      *reinterpret_cast<uint4*>(lo + i * 8) = l;
    }
  } else {
    for (int64_t i = first; i < p.numel; i += stride) {
      float u = dev::Vec16<T>::to_float(g[i]);
      if (m != nullptr) u = p.nesterov ? __fmaf_rn(p.mu, m[i], u) : m[i];
      u *= f;
      const int64_t row = i / p.cols, at = row * p.ld + (i - row * p.cols);
      const __half h = __float2half_rn(u);
      hi[at] = h;
      lo[at] = __float2half_rn((u - __half2float(h)) * kLoScale);
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}
// count matrices of outer x inner, rows `ld` elements apart, copied in boxes of 64 x box_outer; what lies outside reads as zero
bool make_map(CUtensorMap* map, const __half* base, int64_t inner, int64_t outer, int64_t ld, int64_t matrix, int count, uint32_t box_outer) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {cuuint64_t(inner), cuuint64_t(outer), cuuint64_t(count)};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, cuuint64_t(matrix) * 2};
  const cuuint32_t box[3] = {64, box_outer, 1}, step[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Matrix {  // an operand as it lies in memory
  const __half* base;
  int64_t rows, cols, ld, matrix;
};

int sm_count() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  return sms[dev];
}

template <int KIND, bool A_MN, bool B_MN, int TN>
int launch_product(const Matrix& a, const Matrix& b, Product p, int count, cudaStream_t stream) {
  CUtensorMap ta, tb;
  if (!make_map(&ta, a.base, a.cols, a.rows, a.ld, a.matrix, count, A_MN ? 64 : kTileM) || !make_map(&tb, b.base, b.cols, b.rows, b.ld, b.matrix, count, B_MN ? 64 : TN))
    return int(cudaErrorNotSupported);
  p.tiles_m = (p.M + kTileM - 1) / kTileM;
  p.tiles_n = (p.N + TN - 1) / TN;
  p.per = p.tiles_m * p.tiles_n;
  if (p.lower) {
    p.per = 0;
    for (int r = 0; r < p.tiles_m; ++r) p.per += r * kTileM / TN + 1;
  }
  p.total = p.per * count;
  auto* kernel = orth_product_kernel<KIND, A_MN, B_MN, TN>;
  static std::mutex mu;
  static uint64_t opted_in = 0;  // by device
  {
    int dev = 0;
    if (const cudaError_t e = cudaGetDevice(&dev)) return int(e);
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 64 || !((opted_in >> dev) & 1)) {
      if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<TN>::kSmem)) return int(e);
      if (dev < 64) opted_in |= uint64_t(1) << dev;
    }
  }
  return int(launch_following(kernel, dim3(unsigned(std::min(p.total, sm_count()))), kGemmThreads, size_t(Tile<TN>::kSmem), stream, ta, tb, p));
}
// 256 columns a tile, or 128 where the wider tiles would leave SMs idle
template <int KIND, bool A_MN, bool B_MN>
int product(const Matrix& a, const Matrix& b, const Product& p, int count, cudaStream_t stream) {
  const int64_t tm = (p.M + kTileM - 1) / kTileM, n128 = (p.N + 127) / 128, n256 = (p.N + 255) / 256;
  const int64_t narrow = (p.lower ? tm * (tm + 1) / 2 : tm * n128) * count, wide = (p.lower ? (tm / 2) * (tm / 2 + 1) + (tm % 2) * (tm / 2 + 1) : tm * n256) * count;
  const int sms = sm_count();
  // a wide tile takes about 1.7 times as long as a narrow one
  const double cost_narrow = double((narrow + sms - 1) / sms), cost_wide = 1.7 * double((wide + sms - 1) / sms);
  return cost_wide < cost_narrow ? launch_product<KIND, A_MN, B_MN, 256>(a, b, p, count, stream) : launch_product<KIND, A_MN, B_MN, 128>(a, b, p, count, stream);
}

struct Layout {
  int64_t m, n, ld, ldm, x, s;  // x: elements of one X, s: of one symmetric matrix
  int64_t hi[2], lo, gram, poly, partial, total;
};
Layout layout(int64_t count, int64_t rows, int64_t cols) {
  auto up8 = [](int64_t v) { return (v + 7) / 8 * 8; };
  auto up256 = [](int64_t v) { return (v + 255) / 256 * 256; };
  Layout l;
  l.m = std::min(rows, cols);
  l.n = std::max(rows, cols);
  l.ld = up8(cols);
  l.ldm = up8(l.m);
  l.x = rows * l.ld;
  l.s = l.m * l.ldm;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at = up256(at + bytes);
    return o;
  };
  l.hi[0] = take(count * l.x * 2);
  l.hi[1] = take(count * l.x * 2);
  l.lo = take(count * l.x * 2);
  l.gram = take(count * l.s * 2);
  l.poly = take(count * l.s * 2);
  l.partial = take(count * kMaxChunks * 8);
  l.total = at;
  return l;
}
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T>
int start(const Prep& p, int count, cudaStream_t stream) {
  const dim3 grid(unsigned(p.chunks), unsigned(count));
  orth_norm_kernel<T><<<grid, kPrepT, 0, stream>>>(p);
  if (const cudaError_t e = cudaGetLastError()) return int(e);
  return int(launch_following(orth_start_kernel<T>, grid, kPrepT, 0, stream, p));
}

}  // namespace
}  // namespace nangila

extern "C" int64_t nangila_orth_workspace(int32_t count, int32_t rows, int32_t cols) { return nangila::layout(count, rows, cols).total; }

extern "C" int nangila_orth(const NangilaOrthParams* p, cudaStream_t stream) {
  using namespace nangila;
  if (!p || p->count < 1 || p->count > NANGILA_ORTH_MAX_COUNT || p->rows < 1 || p->cols < 1 || p->rows > 65536 || p->cols > 65536 || p->steps < 1 ||
      p->steps > NANGILA_ORTH_MAX_STEPS || !p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 255u) || (p->out == nullptr && p->param[0] == nullptr))
    return int(cudaErrorInvalidValue);
  for (int i = 0; i < p->count; ++i)
    if (!p->grad[i] || (p->param[0] != nullptr && !p->param[i]) || (p->momentum[0] != nullptr && !p->momentum[i])) return int(cudaErrorInvalidValue);
  const Layout l = layout(p->count, p->rows, p->cols);
  auto* ws = static_cast<uint8_t*>(p->workspace);
  __half* hi[2] = {reinterpret_cast<__half*>(ws + l.hi[0]), reinterpret_cast<__half*>(ws + l.hi[1])};
  __half* lo = reinterpret_cast<__half*>(ws + l.lo);
  __half* gram = reinterpret_cast<__half*>(ws + l.gram);
  __half* poly = reinterpret_cast<__half*>(ws + l.poly);
  const bool tall = p->rows > p->cols;
  float scale = 1.0f;
  while (scale * scale < float(l.n)) scale *= 2.0f;

  Prep prep;
  std::memset(&prep, 0, sizeof prep);
  prep.vector = p->cols % 8 == 0;
  for (int i = 0; i < p->count; ++i) {
    prep.grad[i] = p->grad[i];
    prep.momentum[i] = p->momentum[0] != nullptr ? p->momentum[i] : nullptr;
    if (!aligned(p->grad[i]) || !aligned(prep.momentum[i])) prep.vector = 0;
  }
  prep.partial = reinterpret_cast<double*>(ws + l.partial);
  prep.hi = hi[0];
  prep.lo = lo;
  prep.numel = int64_t(p->rows) * p->cols;
  prep.ld = l.ld;
  prep.matrix = l.x;
  prep.cols = p->cols;
  prep.chunks = int(std::max<int64_t>(1, std::min<int64_t>(kMaxChunks, (prep.numel + kPrepT * 16 - 1) / (kPrepT * 16))));
  prep.nesterov = p->nesterov;
  prep.mu = p->mu;
  prep.eps = p->eps;
  prep.scale = scale;
  int e = 0;
  switch (p->grad_dtype) {
    case NANGILA_F32: e = start<float>(prep, p->count, stream); break;
    case NANGILA_F16: e = start<__half>(prep, p->count, stream); break;
    case NANGILA_BF16: e = start<__nv_bfloat16>(prep, p->count, stream); break;
    default: return int(cudaErrorInvalidValue);
  }
  const Matrix A{gram, l.m, l.m, l.ldm, l.s}, B{poly, l.m, l.m, l.ldm, l.s};
  for (int step = 0; step < p->steps && e == 0; ++step) {
    const float* c = p->coefficients[step];
    const bool last = step == p->steps - 1;
    const Matrix X{hi[step & 1], p->rows, p->cols, l.ld, l.x};
    Product q;
    std::memset(&q, 0, sizeof q);
    q.M = q.N = int(l.m);
    q.lower = 1;
    q.ld = l.ldm;
    q.matrix = l.s;
    q.K = int(l.n);
    q.alpha = 1.0f / (scale * scale);
    q.out = gram;
    e = tall ? product<kGram, true, true>(X, X, q, p->count, stream) : product<kGram, false, false>(X, X, q, p->count, stream);
    if (e != 0) break;
    q.K = int(l.m);
    q.alpha = c[1];
    q.beta = c[2];
    q.in = gram;
    q.out = poly;
    e = product<kPoly, false, false>(A, A, q, p->count, stream);
    if (e != 0) break;
    q.lower = 0;
    q.M = p->rows;
    q.N = p->cols;
    q.ld = l.ld;
    q.matrix = l.x;
    q.alpha = c[0];
    q.in = hi[step & 1];
    q.lo = lo;
    q.out = hi[(step & 1) ^ 1];
    if (last) {
      q.unscale = 1.0f / scale;
      q.vector = p->cols % 8 == 0;
      if (p->param[0] != nullptr) {
        for (int i = 0; i < p->count; ++i) {
          q.param[i] = p->param[i];
          if (!aligned(p->param[i])) q.vector = 0;
        }
        q.param_dtype = p->param_dtype;
        q.decay = p->decay;
        q.rate = p->rate;
      } else {
        q.result = static_cast<__nv_bfloat16*>(p->out);
        if (!aligned(p->out)) q.vector = 0;
      }
      e = tall ? product<kFinal, false, false>(X, B, q, p->count, stream) : product<kFinal, false, true>(B, X, q, p->count, stream);
    } else {
      e = tall ? product<kUpdate, false, false>(X, B, q, p->count, stream) : product<kUpdate, false, true>(B, X, q, p->count, stream);
    }
  }
  return e;
}

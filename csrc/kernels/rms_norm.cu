// RMS norm of rows, with the residual's addition before it, with its gradients, and with an output in 8 bits.
//
//   h = x + r (rounded to the rows' type, as a sum of its own would be),   rstd = (mean(h^2) + eps)^-1/2,   y = h rstd w
//   8 bits: f = h rstd w in fp32; scale = max |f| / 448 over the row or over 128 columns; q = e4m3(f / scale)
//   xhat = h rstd;   dx = dr = dh + rstd (dy w - xhat mean(dy w xhat));   dw = sum over rows of dy xhat
//
// All of it is bound by HBM: every value is read once and written once, and a row stays in the registers of the threads that read it
// between the sums and the results. (bf16, 8192 x 2048: x + r -> h, y in 22 us, 6.1 TB/s; the gradients in 29 us, 4.7 TB/s, and 6 for the weight's parts. 8191 x 5632
// in 8 bits with groups 62 us, 5.2 TB/s: there the conversions keep the SMs two thirds busy.) A row belongs to a warp, or where it is too long for one to 256, 512 or 1024 threads (gradients: 64 and 128 too; `by_width` and the others below). Sums and rstd
// are fp32 and added up in an order that only the sizes determine. The gradient of the weight is summed in registers by CTAs
// that walk over the rows, and a second kernel adds up the CTAs' parts in order: no atomics.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "follow.cuh"
#include "nangila_kernels.h"
#include "nangila_model_kernels.h"
#include "quant.cuh"
#include "raw8.cuh"

namespace nangila {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kMinAmax = 1e-12f;  // a row of zeros gets a scale that can be divided by

using dev::Raw8;
using dev::fetch;
using dev::pack;
using dev::put;
using dev::unpack;

// Which columns a thread holds in a run of eight: G adjacent ones, the next G of the row being the next thread's (8: runs as a whole, 16-byte loads; 4, 2 and 1 for
// rows whose width and place allow no more). Neighbouring threads read neighbouring addresses whatever G is. 20000 x 1002 bf16 with a residual: one
// by one 53 us, in twos 29.
template <int TPR, int G>
__device__ __forceinline__ int column(int v, int k, int t) { return ((v * (8 / G) + k / G) * TPR + t) * G + k % G; }
// Whether a warp has nothing in its run `v` (rows that fill fewer runs than the threads have).
template <int TPR, int G>
__device__ __forceinline__ bool beyond(int v, int t, int d) { return column<TPR, G>(v, 0, t & ~31) >= d; }

template <typename T>
__device__ __forceinline__ void words_of(const Raw8<T>& r, uint32_t (&w)[2 * sizeof(T)]) {
  w[0] = r.a.x; w[1] = r.a.y; w[2] = r.a.z; w[3] = r.a.w;
  if constexpr (sizeof(T) == 4) { w[4] = r.b.x; w[5] = r.b.y; w[6] = r.b.z; w[7] = r.b.w; }
}
template <typename T>
__device__ __forceinline__ void of_words(const uint32_t (&w)[2 * sizeof(T)], Raw8<T>& r) {
  r.a = make_uint4(w[0], w[1], w[2], w[3]);
  if constexpr (sizeof(T) == 4) r.b = make_uint4(w[4], w[5], w[6], w[7]);
}
// Bytes of `BYTES` to and from memory, at the low end of the words.
template <int BYTES>
__device__ __forceinline__ void read_piece(const void* p, uint32_t* w) {
  if constexpr (BYTES == 2) w[0] = *static_cast<const uint16_t*>(p);
  if constexpr (BYTES == 4) w[0] = *static_cast<const uint32_t*>(p);
  if constexpr (BYTES == 8) {
    const uint2 u = *static_cast<const uint2*>(p);
    w[0] = u.x; w[1] = u.y;
  }
  if constexpr (BYTES == 16) {
    const uint4 u = *static_cast<const uint4*>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  }
}
template <int BYTES>
__device__ __forceinline__ void write_piece(void* p, const uint32_t* w) {
  if constexpr (BYTES == 1) *static_cast<uint8_t*>(p) = uint8_t(w[0]);
  if constexpr (BYTES == 2) *static_cast<uint16_t*>(p) = uint16_t(w[0]);
  if constexpr (BYTES == 4) *static_cast<uint32_t*>(p) = w[0];
  if constexpr (BYTES == 8) *static_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  if constexpr (BYTES == 16) *static_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T, int TPR, int G>
__device__ __forceinline__ void load_row8(const T* row, int v, int t, int d, Raw8<T>& raw) {
  if constexpr (G == 8) {
    if (column<TPR, G>(v, 0, t) < d) fetch(row + column<TPR, G>(v, 0, t), raw);
    else raw = Raw8<T>{};
  } else {
    constexpr int kBytes = G * int(sizeof(T));
    uint32_t w[2 * sizeof(T)] = {};
    if constexpr (kBytes == 2) {  // two values a word
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        uint32_t lo = 0u, hi = 0u;
        const int c0 = column<TPR, G>(v, k, t), c1 = column<TPR, G>(v, k + 1, t);
        if (c0 < d) read_piece<2>(row + c0, &lo);
        if (c1 < d) read_piece<2>(row + c1, &hi);
        w[k / 2] = lo | hi << 16;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; k += G) {
        const int c = column<TPR, G>(v, k, t);
        if (c < d) read_piece<kBytes>(row + c, w + k * int(sizeof(T)) / 4);
      }
    }
    of_words(w, raw);
  }
}
template <typename T, int TPR, int G>
__device__ __forceinline__ void store_row8(T* row, int v, int t, int d, const float (&f)[8]) {
  Raw8<T> raw;
  pack(f, raw);
  if constexpr (G == 8) {
    if (column<TPR, G>(v, 0, t) < d) put(row + column<TPR, G>(v, 0, t), raw);
  } else {
    constexpr int kBytes = G * int(sizeof(T));
    uint32_t w[2 * sizeof(T)];
    words_of(raw, w);
#pragma unroll
    for (int k = 0; k < 8; k += G) {
      const int c = column<TPR, G>(v, k, t);
      if constexpr (kBytes == 2) {
        const uint32_t one = w[k / 2] >> (k % 2 * 16);
        if (c < d) write_piece<2>(row + c, &one);
      } else {
        if (c < d) write_piece<kBytes>(row + c, w + k * int(sizeof(T)) / 4);
      }
    }
  }
}
template <int TPR, int G>
__device__ __forceinline__ void store_bytes8(uint8_t* row, int v, int t, int d, const uint32_t (&word)[2]) {
#pragma unroll
  for (int k = 0; k < 8; k += G) {
    const int c = column<TPR, G>(v, k, t);
    const uint32_t w[2] = {word[k / 4] >> (k % 4 * 8), word[1]};
    if (c < d) write_piece<G>(row + c, w);
  }
}
template <typename W, int TPR, int G>
__device__ __forceinline__ void load_weight_as(const W* w, int v, int t, int d, float (&f)[8]) {
  Raw8<W> r;
  if constexpr (G == 8) {
    const int c = column<TPR, G>(v, 0, t);
    r = Raw8<W>{};
    if (c < d) {
      r.a = __ldg(reinterpret_cast<const uint4*>(w + c));
      if constexpr (sizeof(W) == 4) r.b = __ldg(reinterpret_cast<const uint4*>(w + c) + 1);
    }
  } else {
    load_row8<W, TPR, G>(w, v, t, d, r);
  }
  unpack(r, f);
}
template <int TPR, int G>
__device__ __forceinline__ void load_weight8(const void* w, int dtype, int v, int t, int d, float (&f)[8]) {
  if (dtype == NANGILA_BF16) load_weight_as<__nv_bfloat16, TPR, G>(static_cast<const __nv_bfloat16*>(w), v, t, d, f);
  else if (dtype == NANGILA_F16) load_weight_as<__half, TPR, G>(static_cast<const __half*>(w), v, t, d, f);
  else load_weight_as<float, TPR, G>(static_cast<const float*>(w), v, t, d, f);
}

// The threads of a row meet. Rows of a CTA have barriers of their own: one may have a row more to do than the others. The instruction needs whole warps, and
// its callers come from a branch that one lane took.
template <int TPR>
__device__ __forceinline__ void meet() {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"r"(1 + int(threadIdx.x) / TPR), "n"(TPR) : "memory");
}
// The sum over the threads of a row, in all of them. `s`: TPR / 32 floats of this row, given again only after the row's threads
// have met in between (the sums of a kernel take turns with two of them).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) s[(threadIdx.x % TPR) >> 5] = v;
    meet<TPR>();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) v += s[i];
  }
  return v;
}
// The larger of two magnitudes, and not a number where either is not one.
__device__ __forceinline__ float larger(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
template <int TPR>
__device__ __forceinline__ float row_max(float v, float* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = larger(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) s[(threadIdx.x % TPR) >> 5] = v;
    meet<TPR>();
    v = s[0];
#pragma unroll
    for (int i = 1; i < TPR / 32; ++i) v = larger(v, s[i]);
  }
  return v;
}

// Threads of a CTA, forward: four rows of a warp each, or one row. Backward: 256, three CTAs an SM (two in fp32), which keeps
// enough loads on their way and leaves few parts of the weight's gradient to add up.
template <int TPR>
constexpr int kThreads = TPR < 128 ? 128 : TPR;
template <int TPR>
constexpr int kThreadsBackward = TPR < 256 ? 256 : TPR;

template <typename T, int TPR, int NV, int G, bool FP8>
__global__ void __launch_bounds__(kThreads<TPR>) norm_forward_kernel(const __grid_constant__ NangilaNormParams p) {
  constexpr int kRows = kThreads<TPR> / TPR;
  __shared__ float s_sums[kThreads<TPR> / 32], s_maxima[kThreads<TPR> / 32];  // of each of the CTA's rows
  const int t = threadIdx.x % TPR;
  const int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / TPR;
  if (row >= p.rows) return;  // all threads of a row
  float* s_sum = s_sums + threadIdx.x / TPR * (TPR / 32);
  float* s_max = s_maxima + threadIdx.x / TPR * (TPR / 32);
  const int d = p.d;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  Raw8<T> raw[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) load_row8<T, TPR, G>(x, v, t, d, raw[v]);
  if (p.residual != nullptr) {
    const T* r = static_cast<const T*>(p.residual) + row * p.residual_stride;
    Raw8<T> more[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) load_row8<T, TPR, G>(r, v, t, d, more[v]);
    T* h = static_cast<T*>(p.h) + row * d;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (beyond<TPR, G>(v, t, d)) continue;
      float a[8], b[8];
      unpack(raw[v], a);
      unpack(more[v], b);
#pragma unroll
      for (int k = 0; k < 8; ++k) a[k] += b[k];
      store_row8<T, TPR, G>(h, v, t, d, a);
      pack(a, raw[v]);  // what is normalised is the sum as it is kept
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (beyond<TPR, G>(v, t, d)) continue;
    float a[8];
    unpack(raw[v], a);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum = __fmaf_rn(a[k], a[k], sum);
  }
  sum = row_sum<TPR>(sum, s_sum);
  const float rstd = rsqrtf(__fdiv_rn(sum, float(d)) + p.eps);
  if (p.rstd != nullptr && t == 0) p.rstd[row] = rstd;
  if constexpr (!FP8) {
    T* y = static_cast<T*>(p.y) + row * d;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (beyond<TPR, G>(v, t, d)) continue;
      float a[8], w[8];
      unpack(raw[v], a);
      load_weight8<TPR, G>(p.weight, p.weight_dtype, v, t, d, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) a[k] = a[k] * rstd * w[k];
      store_row8<T, TPR, G>(y, v, t, d, a);
    }
  } else {
    uint8_t* q = p.q + row * d;
    float amax = 0.0f;  // of the row; with groups each run of 16 threads has one of its own below
    if (p.group == 0) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (beyond<TPR, G>(v, t, d)) continue;
        float a[8], w[8];
        unpack(raw[v], a);
        load_weight8<TPR, G>(p.weight, p.weight_dtype, v, t, d, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) amax = larger(amax, fabsf(a[k] * rstd * w[k]));
      }
      amax = row_max<TPR>(amax, s_max);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (beyond<TPR, G>(v, t, d)) continue;
      float a[8], w[8];
      unpack(raw[v], a);
      load_weight8<TPR, G>(p.weight, p.weight_dtype, v, t, d, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) a[k] = a[k] * rstd * w[k];
      if (p.group != 0) {
        amax = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) amax = larger(amax, fabsf(a[k]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) amax = larger(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      }
      // a row or group with a value that is not finite has no scale: all of it is not a number
      const float scale = amax <= 3.4028234e38f ? __fdiv_rn(fmaxf(amax, kMinAmax), kE4m3Max) : __uint_as_float(0x7fc00000u);
      // A reciprocal and a product where the definition divides: a value within 2^-23 of the middle between two of e4m3's may go to the other one. Against torch operations in 32 bits, 8191 x 5632
      // in groups of 128, 1.2e-4 of the values do; 1.0e-4 would with divisions, for most of them go with the last bit of rstd and the scale; and divisions take 78 us for 65.5.
      const float inverse = __frcp_rn(scale);
      const int c0 = column<TPR, G>(v, 0, t);
      if (p.group != 0) {
        if ((t & 15) == 0 && c0 < d) p.scale[row * (d / 128) + c0 / 128] = scale;
      } else if (v == 0 && t == 0) {
        p.scale[row] = scale;
      }
      uint32_t word[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {  // (not a number times anything is not one, and stays so in e4m3)
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a[4 * k] * inverse, a[4 * k + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(a[4 * k + 2] * inverse, a[4 * k + 3] * inverse), __NV_SATFINITE, __NV_E4M3);
        word[k] = lo | hi << 16;
      }
      store_bytes8<TPR, G>(q, v, t, d, word);
    }
  }
}

template <typename T, int TPR, int NV, int G>
__global__ void __launch_bounds__(kThreadsBackward<TPR>, TPR > 256 ? 1 : sizeof(T) == 2 ? 3 : 2) norm_backward_kernel(const __grid_constant__ NangilaNormGradParams p) {
  constexpr int kRows = kThreadsBackward<TPR> / TPR;
  __shared__ float s_sum[2][kThreadsBackward<TPR> / 32];
  extern __shared__ float s_dw[];  // d, where a CTA has several rows at a time
  const int t = threadIdx.x % TPR, mine = threadIdx.x / TPR;
  const int d = p.d;
  float acc[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[v][k] = 0.0f;
  may_follow();
  int turn = 0;
  for (int64_t row = int64_t(blockIdx.x) * kRows + mine; row < p.rows; row += int64_t(gridDim.x) * kRows) {
    Raw8<T> h[NV], g[NV], more[NV];
    float mean = 0.0f, rstd = 0.0f;
    if (p.dy != nullptr) {
      const T* hr = static_cast<const T*>(p.h) + row * p.h_stride;
      const T* gr = static_cast<const T*>(p.dy) + row * p.dy_stride;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        load_row8<T, TPR, G>(hr, v, t, d, h[v]);
        load_row8<T, TPR, G>(gr, v, t, d, g[v]);
      }
      rstd = p.rstd[row];
    }
    if (p.dh != nullptr && p.dx != nullptr) {
      const T* dr = static_cast<const T*>(p.dh) + row * p.dh_stride;
#pragma unroll
      for (int v = 0; v < NV; ++v) load_row8<T, TPR, G>(dr, v, t, d, more[v]);
    }
    if (p.dy != nullptr) {
      float sum = 0.0f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (beyond<TPR, G>(v, t, d)) continue;
        float a[8], b[8], w[8];
        unpack(h[v], a);
        unpack(g[v], b);
        load_weight8<TPR, G>(p.weight, p.weight_dtype, v, t, d, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float unit = a[k] * rstd;
          acc[v][k] = __fmaf_rn(b[k], unit, acc[v][k]);
          sum = __fmaf_rn(b[k] * w[k], unit, sum);
        }
      }
      mean = __fdiv_rn(row_sum<TPR>(sum, s_sum[turn] + mine * (TPR / 32)), float(d));
      turn ^= 1;
    }
    if (p.dx != nullptr) {
      T* dx = static_cast<T*>(p.dx) + row * d;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (beyond<TPR, G>(v, t, d)) continue;
        float o[8];
        if (p.dh != nullptr) {
          unpack(more[v], o);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] = 0.0f;
        }
        if (p.dy != nullptr) {
          float a[8], b[8], w[8];
          unpack(h[v], a);
          unpack(g[v], b);
          load_weight8<TPR, G>(p.weight, p.weight_dtype, v, t, d, w);
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] += rstd * (b[k] * w[k] - a[k] * rstd * mean);
        }
        store_row8<T, TPR, G>(dx, v, t, d, o);
      }
    }
  }
  if (p.dw == nullptr) return;
  // the CTA's part: its rows' sums added up one after the other
  float* part = p.partial + int64_t(blockIdx.x) * d;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = column<TPR, G>(v, k, t);
        if (c < d) part[c] = acc[v][k];
      }
  } else {
    for (int r = 0; r < kRows; ++r) {
      if (mine == r) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int c = column<TPR, G>(v, k, t);
            if (c < d) s_dw[c] = r == 0 ? acc[v][k] : s_dw[c] + acc[v][k];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < d; c += kThreadsBackward<TPR>) part[c] = s_dw[c];
  }
}

// dw: 32 columns of a CTA, 32 threads for each add up every 32nd part in order, then the 32 in order.
constexpr int kDwY = 32;
__global__ void __launch_bounds__(32 * kDwY) norm_dw_kernel(const float* partial, int parts, int d, void* dw, int dtype) {
  __shared__ float s[kDwY][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
  follow();
  float sum = 0.0f;
  if (c < d) {
#pragma unroll 8
    for (int i = y; i < parts; i += kDwY) sum += partial[int64_t(i) * d + c];
  }
  s[y][x] = sum;
  __syncthreads();
  if (y == 0 && c < d) {
#pragma unroll
    for (int i = 1; i < kDwY; ++i) sum += s[i][x];
    if (dtype == NANGILA_BF16) static_cast<__nv_bfloat16*>(dw)[c] = __float2bfloat16_rn(sum);
    else if (dtype == NANGILA_F16) static_cast<__half*>(dw)[c] = __float2half_rn(sum);
    else static_cast<float*>(dw)[c] = sum;
  }
}

template <typename F>
int by_type(int dtype, const F& f) {
  switch (dtype) {
    case NANGILA_F32: return f(float{});
    case NANGILA_F16: return f(__half{});
    case NANGILA_BF16: return f(__nv_bfloat16{});
    default: return int(cudaErrorInvalidValue);
  }
}
template <int A, int B>
struct Shape {
  static constexpr int tpr = A, nv = B;
};
// Threads for a row, and runs of eight columns for a thread. Forward: a warp up to 2048 columns, which meets nobody else, then 256 threads and more. Measured (bf16,
// residual, 8 bits in groups): 16384 x 2048 45 us with a warp, 68 with 128 threads; 8192 x 4096 58 us with 128 threads, 48 with 256; 8191 x 5632 64 us with 256
// threads in four runs, 68 with 512 in two, 76 with 128 in eight.
template <typename F>
int by_width(int d, const F& f) {
  const int units = (d + 7) / 8;
  if (units <= 64) return f(Shape<32, 2>{});
  if (units <= 128) return f(Shape<32, 4>{});
  if (units <= 256) return f(Shape<32, 8>{});
  if (units <= 512) return f(Shape<256, 2>{});
  if (units <= 1024) return f(Shape<256, 4>{});
  if (units <= 2048) return f(Shape<512, 4>{});
  return f(Shape<1024, 4>{});
}
// Backward: two runs, for a thread also holds its columns of the weight's gradient. Measured, both kernels, ten in a graph, one, two and four runs a thread (us): bf16 32768 x 512 33, 31, 44;
// 16384 x 1024 32, 34, 61; 8192 x 2048 35, 30, 55; 8192 x 4096 93, 59, 82; 4096 x 8192 78, 75, 74; fp32 8192 x 2048 58, 51, 74; 8192 x 4096 144, 96, 117; 4096 x 8192 124, 118, 111. So two, or
// what is left of them for short rows. Above 8192 columns a row's h, dy, dh and sums do not fit into the 64 registers of 1024 threads and part of them goes through local memory: 2048 x 16384
// bf16 74 us (3.6 TB/s), fp32 152 (four runs a thread 134), 1024 x 32768 130 and 237.
template <typename F>
int by_width_backward(int d, const F& f) {
  const int units = (d + 7) / 8;
  if (units <= 32) return f(Shape<32, 1>{});
  if (units <= 64) return f(Shape<32, 2>{});
  if (units <= 128) return f(Shape<64, 2>{});
  if (units <= 256) return f(Shape<128, 2>{});
  if (units <= 512) return f(Shape<256, 2>{});
  if (units <= 1024) return f(Shape<512, 2>{});
  if (units <= 2048) return f(Shape<1024, 2>{});
  return f(Shape<1024, 4>{});
}
// Forward, where columns are read one by one and a thread's loads are eight times as many: fewer runs for each. Measured (bf16, 8 bits, residual): 10000 x 2047 a warp
// 87 us, 128 threads 68, 256 60; 5000 x 4099 512 threads in two runs 84, 1024 in one 102; 100000 x 77 one run 49, two 64; but 20000 x 1001 a warp 57, 64 threads 68.
template <typename F>
int by_width_singly(int d, const F& f) {
  const int units = (d + 7) / 8;
  if (units <= 32) return f(Shape<32, 1>{});
  if (units <= 64) return f(Shape<32, 2>{});
  if (units <= 128) return f(Shape<32, 4>{});
  if (units <= 256) return f(Shape<256, 1>{});
  if (units <= 512) return f(Shape<512, 1>{});
  if (units <= 1024) return f(Shape<512, 2>{});
  if (units <= 2048) return f(Shape<1024, 2>{});
  return f(Shape<1024, 4>{});
}
// How many adjacent columns go together: all of 8, 4, 2 that divide the width and the strides, at addresses that fit.
struct Adjacent {
  int g;
  void width(int64_t n) {
    while (n % g != 0) g /= 2;
  }
  void address(const void* p, int size) {
    while (g > 1 && reinterpret_cast<uintptr_t>(p) % std::min<uintptr_t>(16, uintptr_t(g) * size) != 0) g /= 2;
  }
};
int size_of(int dtype) { return dtype == NANGILA_F32 ? 4 : 2; }
template <typename F>
int by_adjacent(int g, const F& f) {
  return g == 8 ? f(std::integral_constant<int, 8>{}) : g == 4 ? f(std::integral_constant<int, 4>{}) : g == 2 ? f(std::integral_constant<int, 2>{}) : f(std::integral_constant<int, 1>{});
}

// CTAs an SM, backward
template <typename T, int TPR>
constexpr int kPerSm = TPR > 256 ? 1 : sizeof(T) == 2 ? 3 : 2;
int sm_count() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  return sms[dev];
}
template <typename T, int TPR>
int backward_ctas(int64_t rows) {
  constexpr int kRows = kThreadsBackward<TPR> / TPR;
  return int(std::max<int64_t>(1, std::min<int64_t>((rows + kRows - 1) / kRows, int64_t(sm_count()) * kPerSm<T, TPR>)));
}

}  // namespace
}  // namespace nangila

extern "C" int nangila_rms_norm_forward(const NangilaNormParams* p, cudaStream_t stream) {
  using namespace nangila;
  if (!p || !p->x || !p->weight || p->rows < 1 || p->d < 1 || p->d > NANGILA_NORM_MAX_D || (p->residual != nullptr && p->h == nullptr) ||
      (p->q == nullptr ? p->y == nullptr : p->scale == nullptr) || (p->group != 0 && (p->group != 128 || p->d % 128 != 0)) || p->weight_dtype < 0 ||
      p->weight_dtype > 2)
    return int(cudaErrorInvalidValue);
  Adjacent adjacent{8};
  for (const int64_t n : {int64_t(p->d), p->x_stride, p->residual_stride}) adjacent.width(n);
  for (const void* q : {p->x, p->residual, static_cast<const void*>(p->h), static_cast<const void*>(p->y)}) adjacent.address(q, size_of(p->dtype));
  adjacent.address(p->weight, size_of(p->weight_dtype));
  adjacent.address(p->q, 1);
  if (p->group != 0 && adjacent.g != 8) return int(cudaErrorMisalignedAddress);
  return by_type(p->dtype, [&](auto type) {
    using T = decltype(type);
    auto run = [&](auto shape, auto how) {
      using S = decltype(shape);
      constexpr int G = decltype(how)::value, kT = kThreads<S::tpr>, kRows = kT / S::tpr;
      const int64_t ctas = (p->rows + kRows - 1) / kRows;
      if (ctas > 0x7fffffff) return int(cudaErrorInvalidValue);
      if (p->q != nullptr) norm_forward_kernel<T, S::tpr, S::nv, G, true><<<unsigned(ctas), kT, 0, stream>>>(*p);
      else norm_forward_kernel<T, S::tpr, S::nv, G, false><<<unsigned(ctas), kT, 0, stream>>>(*p);
      return int(cudaGetLastError());
    };
    if (adjacent.g == 1) return by_width_singly(p->d, [&](auto shape) { return run(shape, std::integral_constant<int, 1>{}); });
    return by_width(p->d, [&](auto shape) {
      return adjacent.g == 8   ? run(shape, std::integral_constant<int, 8>{})
             : adjacent.g == 4 ? run(shape, std::integral_constant<int, 4>{})
                               : run(shape, std::integral_constant<int, 2>{});
    });
  });
}

extern "C" int nangila_rms_norm_partials(int64_t rows, int32_t d, int32_t dtype, int32_t* count) {
  using namespace nangila;
  if (!count || rows < 1 || d < 1 || d > NANGILA_NORM_MAX_D) return int(cudaErrorInvalidValue);
  return by_type(dtype, [&](auto type) {
    using T = decltype(type);
    return by_width_backward(d, [&](auto shape) {
      using S = decltype(shape);
      *count = backward_ctas<T, S::tpr>(rows);
      return 0;
    });
  });
}

extern "C" int nangila_rms_norm_backward(const NangilaNormGradParams* p, cudaStream_t stream) {
  using namespace nangila;
  if (!p || !p->weight || p->rows < 1 || p->d < 1 || p->d > NANGILA_NORM_MAX_D || (p->dy != nullptr && (!p->h || !p->rstd)) || (p->dw != nullptr && !p->partial) ||
      p->weight_dtype < 0 || p->weight_dtype > 2)
    return int(cudaErrorInvalidValue);
  Adjacent adjacent{8};
  for (const int64_t n : {int64_t(p->d), p->h_stride, p->dy_stride, p->dh_stride}) adjacent.width(n);
  for (const void* q : {p->h, p->dy, p->dh, static_cast<const void*>(p->dx)}) adjacent.address(q, size_of(p->dtype));
  adjacent.address(p->weight, size_of(p->weight_dtype));
  return by_type(p->dtype, [&](auto type) {
    using T = decltype(type);
    return by_width_backward(p->d, [&](auto shape) {
      using S = decltype(shape);
      constexpr int kT = kThreadsBackward<S::tpr>;
      return by_adjacent(adjacent.g, [&](auto how) {
        constexpr int G = decltype(how)::value;
        const int ctas = backward_ctas<T, S::tpr>(p->rows);
        const size_t smem = kT > S::tpr ? size_t(p->d) * 4 : 0;  // below the default limit: such rows are short
        norm_backward_kernel<T, S::tpr, S::nv, G><<<unsigned(ctas), kT, smem, stream>>>(*p);
        if (const cudaError_t e = cudaGetLastError()) return int(e);
        if (p->dw == nullptr) return 0;
        return int(launch_following(norm_dw_kernel, dim3(unsigned((p->d + 31) / 32)), 32 * kDwY, 0, stream, static_cast<const float*>(p->partial), ctas, int(p->d),
                                    static_cast<void*>(p->dw), int(p->weight_dtype)));
      });
    });
  });
}

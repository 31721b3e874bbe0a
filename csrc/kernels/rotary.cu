// Rotary positions: pairs of columns of q and k turned by the angles of their positions, (a, b) -> (a c - b s, a s + b c), with c and s
// from a table in fp32. The gradient is the same with -s. Pairs are neighbours (2i, 2i + 1) or half the turned columns apart
// (i, i + rot / 2); columns from `rot` on are copied. Products in fp32, one rounding.
//
// Bound by HBM: each value is read once and written once, q and k in one launch. A thread takes eight adjacent columns (and the eight
// that they are paired with), of kHeads heads at a time so that all its loads are on their way before the first is used; the table's rows
// are shared by the heads of a token and come out of L1 and L2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "nangila_kernels.h"
#include "nangila_model_kernels.h"
#include "quant.cuh"

namespace nangila {
namespace {

constexpr int kT = 256;
constexpr int kHeads = 4;  // (token, head) pairs of a thread

struct Where {
  int which;       // q or k
  int64_t in, out; // first column of the head
  int64_t row;     // of the table; -1: outside of it
};

// Pair `g` of (token, head); the heads of both tensors follow one another.
__device__ __forceinline__ Where locate(const NangilaRotaryParams& p, int64_t g) {
  const int all = p.heads[0] + p.heads[1];
  const int64_t token = g / all;
  int head = int(g - token * all);
  const int64_t b = token / p.seq, t = token - b * p.seq;
  Where w;
  w.which = head >= p.heads[0] ? 1 : 0;
  if (w.which) head -= p.heads[0];
  w.in = b * p.stride_b[w.which] + t * p.stride_t[w.which] + head * p.stride_h[w.which];
  w.out = (token * p.heads[w.which] + head) * p.d;
  int64_t pos = t;
  if (p.positions != nullptr) {
    const int64_t at = b * p.pos_stride_b + t * p.pos_stride_t;
    pos = p.positions_64 ? static_cast<const int64_t*>(p.positions)[at] : int64_t(static_cast<const int32_t*>(p.positions)[at]);
  }
  w.row = pos >= 0 && pos < p.table_rows ? pos : -1;
  return w;
}
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = __fmaf_rn(a, c, -(b * s)), y = __fmaf_rn(a, s, b * c);
  a = x;
  b = y;
}

// Items of a head: runs of eight columns. HALF: first those of the first half of the turned columns, each with its partner, then the rest.
template <typename T, bool HALF>
__global__ void __launch_bounds__(kT) rotary_vec_kernel(const __grid_constant__ NangilaRotaryParams p, int items, int slots, int64_t pairs) {
  const int item = threadIdx.x % items, slot = threadIdx.x / items;
  if (slot >= slots) return;
  const int half = p.rot / 2;
  const int turned = HALF ? half / 8 : p.rot / 8;   // items that are turned
  const bool turns = item < turned;
  const int col = HALF && !turns ? p.rot + (item - turned) * 8 : item * 8;
  const float sign = p.inverse ? -1.0f : 1.0f;
  const int64_t g0 = int64_t(blockIdx.x) * slots * kHeads + slot;
  Where w[kHeads];
  float a[kHeads][8], b[kHeads][8];
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    const int64_t g = g0 + int64_t(j) * slots;
    if (g >= pairs) break;
    w[j] = locate(p, g);
    const T* in = static_cast<const T*>(p.in[w[j].which]) + w[j].in + col;
    dev::Vec8<T>::load(in, a[j]);
    if (HALF && turns) dev::Vec8<T>::load(in + half, b[j]);
  }
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    if (g0 + int64_t(j) * slots >= pairs) break;
    T* out = static_cast<T*>(p.out[w[j].which]) + w[j].out + col;
    if (turns) {
      constexpr int kPairs = HALF ? 8 : 4;
      float cs[2 * kPairs];
      const float4* row = reinterpret_cast<const float4*>(p.table + (w[j].row < 0 ? 0 : w[j].row) * p.rot + (HALF ? 2 * col : col));
#pragma unroll
      for (int i = 0; i < kPairs / 2; ++i) {
        const float4 f = __ldg(row + i);
        cs[4 * i] = f.x; cs[4 * i + 1] = f.y; cs[4 * i + 2] = f.z; cs[4 * i + 3] = f.w;
      }
      if (w[j].row < 0) {  // no such position: not a number, and not another position's angles
#pragma unroll
        for (int i = 0; i < 2 * kPairs; ++i) cs[i] = __uint_as_float(0x7fc00000u);
      }
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        if (HALF) turn(a[j][i], b[j][i], cs[2 * i], sign * cs[2 * i + 1]);
        else turn(a[j][2 * i], a[j][2 * i + 1], cs[2 * i], sign * cs[2 * i + 1]);
      }
      if (HALF) dev::Vec8<T>::store(out + half, b[j]);
    }
    dev::Vec8<T>::store(out, a[j]);
  }
}

// One pair, or one column that is not turned, for a thread: for heads and strides that no run of eight fits.
template <typename T>
__global__ void __launch_bounds__(kT) rotary_any_kernel(const __grid_constant__ NangilaRotaryParams p, int items, int64_t total) {
  const int64_t i = int64_t(blockIdx.x) * kT + threadIdx.x;
  if (i >= total) return;
  const int64_t g = i / items;
  const int item = int(i - g * items), half = p.rot / 2;
  const Where w = locate(p, g);
  const T* in = static_cast<const T*>(p.in[w.which]) + w.in;
  T* out = static_cast<T*>(p.out[w.which]) + w.out;
  if (item >= half) {
    const int c = p.rot + item - half;
    out[c] = in[c];
    return;
  }
  const int c0 = p.half ? item : 2 * item, c1 = p.half ? item + half : 2 * item + 1;
  float a = dev::Vec16<T>::to_float(in[c0]), b = dev::Vec16<T>::to_float(in[c1]);
  float c = __uint_as_float(0x7fc00000u), s = c;
  if (w.row >= 0) {
    c = p.table[w.row * p.rot + 2 * item];
    s = p.table[w.row * p.rot + 2 * item + 1];
  }
  turn(a, b, c, p.inverse ? -s : s);
  out[c0] = dev::Vec16<T>::from_float(a);
  out[c1] = dev::Vec16<T>::from_float(b);
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T>
int launch(const NangilaRotaryParams& p, cudaStream_t stream) {
  const int64_t pairs = p.batch * p.seq * (p.heads[0] + p.heads[1]);
  bool vec = p.d % 8 == 0 && p.d / 8 <= kT && p.rot % (p.half ? 16 : 8) == 0 && aligned(p.table);
  for (int i = 0; i < 2; ++i)
    if (p.in[i] != nullptr)
      vec = vec && aligned(p.in[i]) && aligned(p.out[i]) && p.stride_b[i] % 8 == 0 && p.stride_t[i] % 8 == 0 && p.stride_h[i] % 8 == 0;
  const int64_t limit = 0x7fffffff;
  if (vec) {
    const int items = p.half ? p.rot / 16 + (p.d - p.rot) / 8 : p.d / 8;
    const int slots = kT / items;
    const int64_t ctas = (pairs + int64_t(slots) * kHeads - 1) / (int64_t(slots) * kHeads);
    if (ctas > limit) return int(cudaErrorInvalidValue);
    if (p.half) rotary_vec_kernel<T, true><<<unsigned(ctas), kT, 0, stream>>>(p, items, slots, pairs);
    else rotary_vec_kernel<T, false><<<unsigned(ctas), kT, 0, stream>>>(p, items, slots, pairs);
  } else {
    const int items = p.rot / 2 + (p.d - p.rot);
    const int64_t total = pairs * items, ctas = (total + kT - 1) / kT;
    if (ctas > limit) return int(cudaErrorInvalidValue);
    rotary_any_kernel<T><<<unsigned(ctas), kT, 0, stream>>>(p, items, total);
  }
  return int(cudaGetLastError());
}

}  // namespace
}  // namespace nangila

extern "C" int nangila_rotary(const NangilaRotaryParams* p, cudaStream_t stream) {
  using namespace nangila;
  if (!p || !p->in[0] || !p->out[0] || (p->in[1] != nullptr && (!p->out[1] || p->heads[1] < 1)) || (p->in[1] == nullptr && p->heads[1] != 0) || p->heads[0] < 1 ||
      p->batch < 1 || p->seq < 1 || p->d < 2 || p->rot < 2 || p->rot % 2 != 0 || p->rot > p->d || !p->table || p->table_rows < 1 ||
      (p->positions == nullptr && p->seq > p->table_rows))
    return int(cudaErrorInvalidValue);
  switch (p->dtype) {
    case NANGILA_F32: return launch<float>(*p, stream);
    case NANGILA_F16: return launch<__half>(*p, stream);
    case NANGILA_BF16: return launch<__nv_bfloat16>(*p, stream);
    default: return int(cudaErrorInvalidValue);
  }
}

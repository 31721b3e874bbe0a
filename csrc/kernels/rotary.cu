// Rotary positions: pairs of columns of q and k turned by the angles of their positions, (a, b) -> (a c - b s, a s + b c), with c and s
// from a table in fp32. The gradient is the same with -s. Pairs are neighbours (2i, 2i + 1) or half the turned columns apart
// (i, i + rot / 2); columns from `rot` on are copied. Products in fp32, one rounding.
//
// Bound by HBM: each value is read once and written once, q and k in one launch. A thread takes eight adjacent columns (and the eight
// that they are paired with), of four heads at a time so that all its loads are on their way before the first is used; it keeps the
// table's values from one head of a token to the next.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "launch_util.cuh"
#include "nangila_kernels.h"
#include "nangila_model_kernels.h"
#include "quant.cuh"
#include "raw8.cuh"

namespace nangila {
namespace {

constexpr int kT = 128;
constexpr int kAtOnce = 4;  // (token, head) pairs of a thread whose loads are on their way together

// A pair of (token, head), counted from the CTA's first token; the heads of both tensors follow one another.
struct Where {
  int which;       // q or k
  int64_t in, out; // first column of the head
  int64_t row;     // of the table; -1: outside of it
};
struct First {
  int64_t token, b, t;
};
__device__ __forceinline__ First first_token(const NangilaRotaryParams& p, int64_t token) {
  const int64_t b = token / p.seq;
  return {token, b, token - b * p.seq};
}
__device__ __forceinline__ Where locate(const NangilaRotaryParams& p, const First& f, uint32_t pair) {
  const uint32_t all = uint32_t(p.heads[0] + p.heads[1]);
  const uint32_t ahead = pair / all;
  int head = int(pair - ahead * all);
  int64_t b = f.b, t = f.t + ahead;
  while (t >= p.seq) {  // a CTA's tokens are few
    t -= p.seq;
    ++b;
  }
  Where w;
  w.which = head >= p.heads[0] ? 1 : 0;
  if (w.which) head -= p.heads[0];
  w.in = b * p.stride_b[w.which] + t * p.stride_t[w.which] + head * p.stride_h[w.which];
  w.out = ((f.token + ahead) * p.heads[w.which] + head) * p.d;
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

// A division of numbers below 2^31 by one that the host knows.
struct Divisor {
  uint32_t by, magic, shift;
};
Divisor divisor(uint32_t by) {
  Divisor d{by, 0, 0};
  while ((uint64_t(1) << d.shift) < by) ++d.shift;
  d.magic = uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << d.shift) - by)) / by + 1);
  return d;
}
__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor& d) { return (__umulhi(d.magic, n) + n) >> d.shift; }

// How the work is shared out. Items of a head are runs of eight columns (HALF: first those of the first half of the turned columns, each with its
// partner, then the rest). A thread keeps its item, and its kAtOnce pairs of (token of a group, head): where they lie is worked out once, and per
// group of tokens only the group's place is added.
struct Plan {
  int items, slots, tokens;  // slots: threads with the same item; tokens of a group
  uint32_t all_tokens, groups;
  Divisor seq;
};
template <typename T, bool HALF>
__global__ void __launch_bounds__(kT) rotary_vec_kernel(const __grid_constant__ NangilaRotaryParams p, const __grid_constant__ Plan plan) {
  const int item = threadIdx.x % plan.items, slot = threadIdx.x / plan.items;
  if (slot >= plan.slots) return;
  const int half = p.rot / 2;
  const int turned = HALF ? half / 8 : p.rot / 8;   // items that are turned
  const bool turns = item < turned;
  const int col = HALF && !turns ? p.rot + (item - turned) * 8 : item * 8;
  const float sign = p.inverse ? -1.0f : 1.0f;
  const int all = p.heads[0] + p.heads[1], pairs = plan.tokens * all;
  const T* in[kAtOnce];
  T* out[kAtOnce];
  int ahead[kAtOnce], which[kAtOnce];  // tokens after the group's first (a group that is never reached for a pair that there is not)
#pragma unroll
  for (int j = 0; j < kAtOnce; ++j) {
    const int g = int(blockIdx.y) * plan.slots * kAtOnce + slot + j * plan.slots;
    ahead[j] = g / all;
    int head = g - ahead[j] * all;
    which[j] = head >= p.heads[0] ? 1 : 0;
    if (which[j]) head -= p.heads[0];
    in[j] = static_cast<const T*>(p.in[which[j]]) + head * p.stride_h[which[j]] + col;
    out[j] = static_cast<T*>(p.out[which[j]]) + int64_t(head) * p.d + col;
    if (g >= pairs) ahead[j] = 0x7fffffff;
  }
  constexpr int kPairs = HALF ? 8 : 4;
  float cs[2 * kPairs];
  // Positions are read a group ahead: the table's values, which depend on them, would otherwise arrive two trips to memory after the group's data.
  auto row_of = [&](uint32_t token) {
    const uint32_t b = divide(token, plan.seq), t = token - b * plan.seq.by;
    if (p.positions == nullptr) return int32_t(t);
    const int64_t at = int64_t(b) * p.pos_stride_b + int64_t(t) * p.pos_stride_t;
    const int64_t row = p.positions_64 ? static_cast<const int64_t*>(p.positions)[at] : int64_t(static_cast<const int32_t*>(p.positions)[at]);
    return row < 0 || row >= p.table_rows ? -1 : int32_t(row);
  };
  int32_t next[kAtOnce];
#pragma unroll
  for (int j = 0; j < kAtOnce; ++j) {
    const uint32_t token = blockIdx.x * uint32_t(plan.tokens) + uint32_t(ahead[j]);
    next[j] = turns && token < plan.all_tokens ? row_of(token) : -1;
  }
  for (uint32_t group = blockIdx.x; group < plan.groups; group += gridDim.x) {
    const uint32_t first = group * uint32_t(plan.tokens);
    int32_t have = -2;  // the row of the table in `cs`; -1: none
    int32_t row[kAtOnce];
    dev::Raw8<T> raw[kAtOnce], partner[HALF ? kAtOnce : 1];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const uint32_t token = first + uint32_t(ahead[j]);  // below 2^32
      if (token >= plan.all_tokens) continue;
      const uint32_t b = divide(token, plan.seq), t = token - b * plan.seq.by;
      const T* from = in[j] + int64_t(b) * p.stride_b[which[j]] + int64_t(t) * p.stride_t[which[j]];
      dev::fetch(from, raw[j]);
      if (HALF && turns) dev::fetch(from + half, partner[j]);
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      row[j] = next[j];
      const uint64_t token = uint64_t(first) + uint64_t(gridDim.x) * uint32_t(plan.tokens) + uint32_t(ahead[j]);
      if (turns && token < plan.all_tokens) next[j] = row_of(uint32_t(token));
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const uint32_t token = first + uint32_t(ahead[j]);
      if (token >= plan.all_tokens) continue;
      T* to = out[j] + int64_t(token) * (int64_t(p.heads[which[j]]) * p.d);
      if (turns) {
        if (row[j] != have) {
          have = row[j];
          const float4* values = reinterpret_cast<const float4*>(p.table + int64_t(have < 0 ? 0 : have) * p.rot + (HALF ? 2 * col : col));
#pragma unroll
          for (int i = 0; i < kPairs / 2; ++i) {
            const float4 f = __ldg(values + i);
            cs[4 * i] = f.x; cs[4 * i + 1] = sign * f.y; cs[4 * i + 2] = f.z; cs[4 * i + 3] = sign * f.w;
          }
          if (have < 0) {  // no such position: not a number, and not another position's angles
#pragma unroll
            for (int i = 0; i < 2 * kPairs; ++i) cs[i] = __uint_as_float(0x7fc00000u);
          }
        }
        float a[8];
        dev::unpack(raw[j], a);
        if constexpr (HALF) {
          float b[8];
          dev::unpack(partner[j], b);
#pragma unroll
          for (int i = 0; i < 8; ++i) turn(a[i], b[i], cs[2 * i], cs[2 * i + 1]);
          dev::pack(b, partner[j]);
          dev::put(to + half, partner[j]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) turn(a[2 * i], a[2 * i + 1], cs[2 * i], cs[2 * i + 1]);
        }
        dev::pack(a, raw[j]);
      }
      dev::put(to, raw[j]);
    }
  }
}

// One pair, or one column that is not turned, for a thread: for heads and strides that no run of eight fits.
template <typename T>
__global__ void __launch_bounds__(kT) rotary_any_kernel(const __grid_constant__ NangilaRotaryParams p, int items, int64_t total) {
  const int64_t i = int64_t(blockIdx.x) * kT + threadIdx.x;
  if (i >= total) return;
  const int64_t g = i / items, token = g / (p.heads[0] + p.heads[1]);
  const int item = int(i - g * items), half = p.rot / 2;
  const Where w = locate(p, first_token(p, token), uint32_t(g - token * (p.heads[0] + p.heads[1])));
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
  bool vec = p.batch * p.seq < (int64_t(1) << 31) && p.table_rows < (int64_t(1) << 31) && p.d % 8 == 0 && p.d / 8 <= kT && p.rot % (p.half ? 16 : 8) == 0 && aligned(p.table);
  for (int i = 0; i < 2; ++i)
    if (p.in[i] != nullptr)
      vec = vec && aligned(p.in[i]) && aligned(p.out[i]) && p.stride_b[i] % 8 == 0 && p.stride_t[i] % 8 == 0 && p.stride_h[i] % 8 == 0;
  const int64_t limit = 0x7fffffff;
  if (vec) {
    const int items = p.half ? p.rot / 16 + (p.d - p.rot) / 8 : p.d / 8;
    const int all = p.heads[0] + p.heads[1], slots = kT / items;
    Plan plan;
    plan.items = items;
    plan.slots = slots;
    plan.tokens = std::max(1, slots * kAtOnce / all);
    plan.all_tokens = uint32_t(p.batch * p.seq);
    plan.groups = (plan.all_tokens + uint32_t(plan.tokens) - 1) / uint32_t(plan.tokens);
    plan.seq = divisor(uint32_t(p.seq));
    auto* kernel = p.half ? rotary_vec_kernel<T, true> : rotary_vec_kernel<T, false>;
    int resident = 0;
    if (const cudaError_t e = resident_ctas(reinterpret_cast<const void*>(kernel), kT, 0, &resident)) return int(e);
    const unsigned heads = unsigned((plan.tokens * all + slots * kAtOnce - 1) / (slots * kAtOnce));  // rounds that the heads of a token take
    const unsigned ctas = std::min(plan.groups, std::max(1u, unsigned(resident) / heads));
    if (heads > 65535) return int(cudaErrorInvalidValue);
    kernel<<<dim3(ctas, heads), kT, 0, stream>>>(p, plan);
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

// Rotary positions: pairs of columns of q and k turned by the angles of their positions, (a, b) -> (a c - b s, a s + b c), with c and s
// from a table in fp32. The gradient is the same with -s. Pairs are neighbours (2i, 2i + 1) or half the turned columns apart
// (i, i + rot / 2); columns from `rot` on are copied. Products in fp32, one rounding.
//
// Bound by HBM: each value is read once and written once, q and k in one launch. A thread takes a run of eight adjacent columns (four or two where the head or
// the strides ask for it), in the half layout two of them, of four heads at a time so that all its loads are on their way before the first is used; it
// keeps the table's values from one head of a token to the next, and reads positions a group of tokens ahead. CTAs stay: where a thread's heads lie is worked
// out once (with a CTA for each token, that arithmetic kept the SMs busy: 8192 tokens x 32 heads x 128 bf16 took 49 us, now 22, 6.1 TB/s). A prompt of 32749 tokens, 40 heads of
// 128 with 64 columns turned in the half layout, fp16: 131 us, 5.1 TB/s.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "launch_util.cuh"
#include "nangila_kernels.h"
#include "nangila_model_kernels.h"
#include "quant.cuh"
#include "raw8.cuh"

namespace nangila {
namespace {

constexpr int kT = 128;
constexpr int kAtOnce = 4;  // (token, head) pairs of a thread whose loads are on their way together

// Where pair `g` of (token, head) lies; the heads of both tensors follow one another.
struct Where {
  int which;       // q or k
  int64_t in, out; // first column of the head
  int64_t row;     // of the table; -1: outside of it
};
__device__ __forceinline__ Where locate(const NangilaRotaryParams& p, int64_t g) {
  const int64_t all = int64_t(p.heads[0]) + p.heads[1], token = g / all, b = token / p.seq, t = token - b * p.seq;
  int64_t head = g - token * all;
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

// A division of numbers below 2^31 by one that the host knows: a multiplication by its reciprocal, rounded up to 33 bits, of which the leading one is added apart
// (T. Granlund and P. Montgomery, Division by invariant integers using multiplication, 1994).
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

// A run of V adjacent columns, as it lies in memory: 4 to 32 bytes in one or two loads.
template <typename T, int V>
struct Run {
  static constexpr int kWords = V * int(sizeof(T)) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWords == 1) w[0] = *reinterpret_cast<const uint32_t*>(p);
    if constexpr (kWords == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x; w[1] = u.y;
    }
    if constexpr (kWords >= 4) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 u = dev::load_stream(reinterpret_cast<const uint32_t*>(p) + i);
        w[i] = u.x; w[i + 1] = u.y; w[i + 2] = u.z; w[i + 3] = u.w;
      }
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kWords == 1) *reinterpret_cast<uint32_t*>(p) = w[0];
    if constexpr (kWords == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    if constexpr (kWords >= 4) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(p) + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
  }
  __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(f[i]);
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
  }
};

// How the work is shared out. An item is a run of a head's columns, or with HALF two of them: a run of the first half of the turned columns with its
// partner, or two runs of the columns that are copied. A thread keeps its item, and its kAtOnce pairs of (token of a group, head): where they lie is
// worked out once, and per group of tokens only the group's place is added.
struct Plan {
  int items, slots, tokens;  // slots: threads with the same item; tokens of a group
  uint32_t all_tokens, groups;
  Divisor seq;
};
template <typename T, bool HALF, int V>
__global__ void __launch_bounds__(kT) rotary_vec_kernel(const __grid_constant__ NangilaRotaryParams p, const __grid_constant__ Plan plan) {
  const int item = threadIdx.x % plan.items, slot = threadIdx.x / plan.items;
  if (slot >= plan.slots) return;
  const int half = p.rot / 2;
  const int turned = HALF ? half / V : p.rot / V;   // items that are turned
  const bool turns = item < turned;
  const int col = HALF && !turns ? p.rot + (item - turned) * 2 * V : item * V;
  const int second = turns ? half : V;              // HALF: how far on the other run is
  const bool two = HALF && col + second < p.d;
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
    in[j] = static_cast<const T*>(p.in[which[j]]) + int64_t(head) * p.stride_h[which[j]] + col;
    out[j] = static_cast<T*>(p.out[which[j]]) + int64_t(head) * p.d + col;
    if (g >= pairs) ahead[j] = 0x7fffffff;
  }
  constexpr int kPairs = HALF ? V : V / 2;
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
    Run<T, V> run[kAtOnce], other[HALF ? kAtOnce : 1];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const uint32_t token = first + uint32_t(ahead[j]);  // below 2^32
      if (token >= plan.all_tokens) continue;
      const uint32_t b = divide(token, plan.seq), t = token - b * plan.seq.by;
      const T* from = in[j] + int64_t(b) * p.stride_b[which[j]] + int64_t(t) * p.stride_t[which[j]];
      run[j].load(from);
      if (HALF && two) other[j].load(from + second);
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
          const float* values = p.table + int64_t(have < 0 ? 0 : have) * p.rot + (HALF ? 2 * col : col);
          if constexpr (kPairs >= 2) {
#pragma unroll
            for (int i = 0; i < kPairs; i += 2) {
              const float4 f = __ldg(reinterpret_cast<const float4*>(values) + i / 2);
              cs[2 * i] = f.x; cs[2 * i + 1] = sign * f.y; cs[2 * i + 2] = f.z; cs[2 * i + 3] = sign * f.w;
            }
          } else {
            const float2 f = __ldg(reinterpret_cast<const float2*>(values));
            cs[0] = f.x; cs[1] = sign * f.y;
          }
          if (have < 0) {  // no such position: not a number, and not another position's angles
#pragma unroll
            for (int i = 0; i < 2 * kPairs; ++i) cs[i] = __uint_as_float(0x7fc00000u);
          }
        }
        float a[V];
        run[j].get(a);
        if constexpr (HALF) {
          float b[V];
          other[j].get(b);
#pragma unroll
          for (int i = 0; i < V; ++i) turn(a[i], b[i], cs[2 * i], cs[2 * i + 1]);
          other[j].set(b);
        } else {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) turn(a[2 * i], a[2 * i + 1], cs[2 * i], cs[2 * i + 1]);
        }
        run[j].set(a);
      }
      run[j].store(to);
      if (HALF && two) other[j].store(to + second);
    }
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

// Whether runs of V columns fit the head and the tensors' places.
template <typename T>
bool runs_of(const NangilaRotaryParams& p, int v) {
  const uintptr_t bytes = std::min<uintptr_t>(16, uintptr_t(v) * sizeof(T));
  bool ok = p.d % v == 0 && p.rot % (p.half ? 2 * v : v) == 0;
  for (int i = 0; i < 2; ++i)
    if (p.in[i] != nullptr)
      ok = ok && reinterpret_cast<uintptr_t>(p.in[i]) % bytes == 0 && reinterpret_cast<uintptr_t>(p.out[i]) % bytes == 0 && p.stride_b[i] % v == 0 && p.stride_t[i] % v == 0 &&
           p.stride_h[i] % v == 0;
  const int items = p.half ? p.rot / 2 / v + ((p.d - p.rot) / v + 1) / 2 : p.d / v;
  return ok && items <= kT && aligned(p.table) && (p.rot % 4 == 0 || v == 2);
}
template <typename T, bool HALF, int V>
int launch_runs(const NangilaRotaryParams& p, cudaStream_t stream) {
  const int all = p.heads[0] + p.heads[1];
  Plan plan;
  plan.items = HALF ? p.rot / 2 / V + ((p.d - p.rot) / V + 1) / 2 : p.d / V;
  plan.slots = kT / plan.items;
  // as many tokens together as leave the fewest threads without a pair
  const int at_once = plan.slots * kAtOnce;
  plan.tokens = 1;
  double best = 0.0;
  for (int tokens = 1; tokens <= std::max(4, at_once / all); ++tokens) {
    const double used = double(tokens * all) / double((tokens * all + at_once - 1) / at_once * at_once);
    if (used > best * 1.02) {
      best = used;
      plan.tokens = tokens;
    }
  }
  plan.all_tokens = uint32_t(p.batch * p.seq);
  plan.groups = (plan.all_tokens + uint32_t(plan.tokens) - 1) / uint32_t(plan.tokens);
  plan.seq = divisor(uint32_t(p.seq));
  auto* kernel = rotary_vec_kernel<T, HALF, V>;
  int resident = 0;
  if (const cudaError_t e = resident_ctas(reinterpret_cast<const void*>(kernel), kT, 0, &resident)) return int(e);
  const unsigned rounds = unsigned((plan.tokens * all + at_once - 1) / at_once);  // that the heads of a group take
  if (rounds > 65535) return int(cudaErrorInvalidValue);
  kernel<<<dim3(std::min(plan.groups, std::max(1u, unsigned(resident) / rounds)), rounds), kT, 0, stream>>>(p, plan);
  return int(cudaGetLastError());
}
template <typename T>
int launch(const NangilaRotaryParams& p, cudaStream_t stream) {
  // (numbers of tokens, rows and pairs that 32 bits hold)
  const int64_t limit = 0x7fffffff;
  if (p.batch * p.seq <= limit && p.table_rows <= limit && int64_t(p.heads[0]) + p.heads[1] <= 65536) {
    if (runs_of<T>(p, 8)) return p.half ? launch_runs<T, true, 8>(p, stream) : launch_runs<T, false, 8>(p, stream);
    if (runs_of<T>(p, 4)) return p.half ? launch_runs<T, true, 4>(p, stream) : launch_runs<T, false, 4>(p, stream);
    if (runs_of<T>(p, 2)) return p.half ? launch_runs<T, true, 2>(p, stream) : launch_runs<T, false, 2>(p, stream);
  }
  const int64_t pairs = p.batch * p.seq * (int64_t(p.heads[0]) + p.heads[1]);
  const int items = p.rot / 2 + (p.d - p.rot);
  const int64_t total = pairs * items, ctas = (total + kT - 1) / kT;
  if (ctas > limit) return int(cudaErrorInvalidValue);
  rotary_any_kernel<T><<<unsigned(ctas), kT, 0, stream>>>(p, items, total);
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
  try {
    switch (p->dtype) {
      case NANGILA_F32: return launch<float>(*p, stream);
      case NANGILA_F16: return launch<__half>(*p, stream);
      case NANGILA_BF16: return launch<__nv_bfloat16>(*p, stream);
      default: return int(cudaErrorInvalidValue);
    }
  } catch (...) {  // (the host's table of occupancies allocates)
    return int(cudaErrorMemoryAllocation);
  }
}

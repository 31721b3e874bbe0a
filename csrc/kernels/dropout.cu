// Dropout with a mask that is never stored: out = residual + (kept ? x * scale : 0), and the same without a residual for the gradient.
//
// Element i is kept where its 32-bit number reaches `least` = round(p 2^32). The numbers come from Philox4x32 with ten rounds (J. Salmon, M. Moraes, R. Dror, D. Shaw, Parallel
// random numbers: as easy as 1, 2, 3, 2011), a bijection of a 128-bit counter under a 64-bit key: eight elements share a block of the counter (i / 8, draw, 0), whose 128 bits are the upper halves
// of their numbers; the lower halves are the block (i / 8, draw, 1), made only where an upper half equals that of `least`, one element in 65536. So the
// probability is held in 2^-32, at the cost of sixteen bits a value. A value that is not kept is not looked at: infinities and NaN go.
//
// One rounding: x * scale in fp32 (the residual added there too).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "launch_util.cuh"
#include "nangila_kernels.h"
#include "nangila_vocab_kernels.h"
#include "quant.cuh"
#include "raw8.cuh"

namespace nangila {
namespace {

constexpr int kT = 256;

__device__ __forceinline__ uint4 philox(uint64_t block, uint32_t draw, uint32_t which, uint2 key) {
  uint4 c = make_uint4(uint32_t(block), uint32_t(block >> 32), draw, which);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = uint64_t(0xD2511F53u) * c.x, b = uint64_t(0xCD9E8D57u) * c.z;
    c = make_uint4(uint32_t(b >> 32) ^ c.y ^ key.x, uint32_t(b), uint32_t(a >> 32) ^ c.w ^ key.y, uint32_t(a));
    key.x += 0x9E3779B9u;
    key.y += 0xBB67AE85u;
  }
  return c;
}
// A block's eight values: v * scale where they are kept, 0 where not. An element's upper half is compared where it lies in its word.
struct Limits {
  uint32_t upper, lower;  // of `least`; upper up to 2^16 - 1
  bool none;              // nothing is kept
};
__device__ __forceinline__ void drop8(float (&v)[8], float scale, uint64_t block, uint32_t draw, uint2 key, const Limits& limit) {
  const uint4 c = philox(block, draw, 0, key);
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  if (limit.lower != 0) {
    // a half that is equal leaves a zero half of x, which borrows into its top bit (one above a zero half may too: looked at for nothing)
    uint32_t tied = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = w[i] ^ (limit.upper * 0x10001u);
      tied |= (x - 0x00010001u) & ~x;
    }
    if ((tied & 0x80008000u) != 0) {
      const uint4 e = philox(block, draw, 1, key);
      const uint32_t l[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t u = (i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xffffu, d = (i & 1) ? l[i / 2] >> 16 : l[i / 2] & 0xffffu;
        if (u == limit.upper && d < limit.lower) v[i] = 0.0f;
      }
    }
  }
  const uint32_t least = limit.upper << 16;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = ((i & 1) ? w[i / 2] : w[i / 2] << 16) >= least && !limit.none ? v[i] * scale : 0.0f;
}

// Blocks of a thread on their way together. (One at a time, the way to memory and the generator's ten rounds took turns: 8192 x 2048 bf16 with a residual 24 us, the gradient 23.)
template <typename T>
constexpr int kAtOnce = sizeof(T) == 4 ? 2 : 4;

template <typename T, bool VECTOR>
__global__ void __launch_bounds__(kT) dropout_kernel(const __grid_constant__ NangilaDropoutParams p) {
  const uint64_t seed = p.seed_ptr != nullptr ? uint64_t(*p.seed_ptr) : p.seed;
  const uint2 key = make_uint2(uint32_t(seed), uint32_t(seed >> 32));
  const Limits limit{uint32_t(p.least >> 16) & 0xffffu, uint32_t(p.least) & 0xffffu, p.least >> 32 != 0};
  const T* x = static_cast<const T*>(p.x);
  const T* r = static_cast<const T*>(p.residual);
  T* out = static_cast<T*>(p.out);
  const int64_t step = int64_t(gridDim.x) * kT, first = int64_t(blockIdx.x) * kT + threadIdx.x;
  const int64_t whole = VECTOR ? p.n / 8 : 0;
  if (VECTOR) {
    for (int64_t b0 = first; b0 < whole; b0 += kAtOnce<T> * step) {
      dev::Raw8<T> raw[kAtOnce<T>], add[kAtOnce<T>];
#pragma unroll
      for (int j = 0; j < kAtOnce<T>; ++j) {
        const int64_t b = b0 + j * step;
        if (b >= whole) break;
        dev::fetch(x + b * 8, raw[j]);
        if (r != nullptr) dev::fetch(r + b * 8, add[j]);
      }
#pragma unroll
      for (int j = 0; j < kAtOnce<T>; ++j) {
        const int64_t b = b0 + j * step;
        if (b >= whole) break;
        float v[8], a[8];
        dev::unpack(raw[j], v);
        drop8(v, p.scale, uint64_t(b), p.draw, key, limit);
        if (r != nullptr) {
          dev::unpack(add[j], a);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += a[i];
        }
        dev::pack(v, raw[j]);
        dev::put(out + b * 8, raw[j]);
      }
    }
  }
  for (int64_t b = whole + first; b < (p.n + 7) / 8; b += step) {  // the last elements, or all of them one by one
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = b * 8 + i < p.n ? dev::Vec16<T>::to_float(x[b * 8 + i]) : 0.0f;
    drop8(v, p.scale, uint64_t(b), p.draw, key, limit);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t at = b * 8 + i;
      if (at < p.n) out[at] = dev::Vec16<T>::from_float(r != nullptr ? v[i] + dev::Vec16<T>::to_float(r[at]) : v[i]);
    }
  }
}

template <typename T>
int launch(const NangilaDropoutParams& p, cudaStream_t stream) {
  auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
  const bool vector = aligned(p.x) && aligned(p.residual) && aligned(p.out);
  auto* kernel = vector ? dropout_kernel<T, true> : dropout_kernel<T, false>;
  int resident = 0;
  if (const cudaError_t e = resident_ctas(reinterpret_cast<const void*>(kernel), kT, 0, &resident)) return int(e);
  const int64_t want = ((p.n + 7) / 8 + kT - 1) / kT;
  kernel<<<unsigned(std::min<int64_t>(want, resident)), kT, 0, stream>>>(p);
  return int(cudaGetLastError());
}

}  // namespace
}  // namespace nangila

extern "C" int nangila_dropout(const NangilaDropoutParams* p, cudaStream_t stream) {
  using namespace nangila;
  if (!p || !p->x || !p->out || p->n < 0 || p->least > (uint64_t(1) << 32)) return int(cudaErrorInvalidValue);
  if (p->n == 0) return 0;
  try {
    switch (p->dtype) {
      case NANGILA_F32: return launch<float>(*p, stream);
      case NANGILA_F16: return launch<__half>(*p, stream);
      case NANGILA_BF16: return launch<__nv_bfloat16>(*p, stream);
      default: return int(cudaErrorInvalidValue);
    }
  } catch (...) {  // (the host's tables of kernels that were set up allocate)
    return int(cudaErrorMemoryAllocation);
  }
}

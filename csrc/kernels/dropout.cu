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

// The keys of the ten rounds: in the kernel's parameters, where instructions take them from, or worked out by each thread from a seed in memory.
struct Keys {
  uint32_t x[10], y[10];
};
__host__ __device__ __forceinline__ void make_keys(uint64_t seed, Keys& k) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    k.x[r] = uint32_t(seed) + uint32_t(r) * 0x9E3779B9u;
    k.y[r] = uint32_t(seed >> 32) + uint32_t(r) * 0xBB67AE85u;
  }
}
struct Launch {
  NangilaDropoutParams p;
  Keys keys;
  uint32_t upper, lower;  // of `least`, which is below 2^32
};
__device__ __forceinline__ uint4 philox(uint64_t block, uint32_t draw, uint32_t which, const Keys& k) {
  uint4 c = make_uint4(uint32_t(block), uint32_t(block >> 32), draw, which);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = uint64_t(0xD2511F53u) * c.x, b = uint64_t(0xCD9E8D57u) * c.z;
    c = make_uint4(uint32_t(b >> 32) ^ c.y ^ k.x[r], uint32_t(b), uint32_t(a >> 32) ^ c.w ^ k.y[r], uint32_t(a));
  }
  return c;
}
// A block's eight values, c its numbers' upper halves: v * scale where they reach `upper`, 0 where not. An upper half is compared where it lies in its word.
__device__ __forceinline__ void drop8(float (&v)[8], float scale, const uint4& c, uint32_t upper) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w}, least = upper << 16;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = ((i & 1) ? w[i / 2] : w[i / 2] << 16) >= least ? __fmul_rn(v[i], scale) : 0.0f;
}
// Whether one of the upper halves may equal that of `least`: an equal one leaves a zero half of x, which borrows into its top bit (one above a zero half may too: looked at for nothing).
__device__ __forceinline__ bool tied8(const uint4& c, uint32_t upper) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint32_t tied = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = w[i] ^ (upper * 0x10001u);
    tied |= (x - 0x00010001u) & ~x;
  }
  return (tied & 0x80008000u) != 0;
}
// Of the block's elements that tied, those whose lower half is below that of `least`: written once more, as dropped.
template <typename T>
__device__ __noinline__ void settle8(const Launch& a, int64_t block, uint4 c, const Keys& keys) {
  const uint4 e = philox(uint64_t(block), a.p.draw, 1, keys);
  const uint32_t w[4] = {c.x, c.y, c.z, c.w}, l[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t at = block * 8 + i;
    const uint32_t u = (i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xffffu, d = (i & 1) ? l[i / 2] >> 16 : l[i / 2] & 0xffffu;
    if (at < a.p.n && u == a.upper && d < a.lower) static_cast<T*>(a.p.out)[at] = a.p.residual != nullptr ? static_cast<const T*>(a.p.residual)[at] : dev::Vec16<T>::from_float(0.0f);
  }
}

// Copies of a thread's own, in groups.
__device__ __forceinline__ void copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A thread's blocks are on their way through shared memory, four of them (in fp32 three) at a time: with 32 warps an SM, 64 KB (and as much of the residual). In registers, one or two at a time, the
// loads of all SMs did not cover the way to memory: 8192 x 2048 bf16 took 19 to 21 us, now 17 (4.0 TB/s; with a residual 19, 5.3 TB/s), floors 10 and 15. The numbers themselves
// take 5 of it (twenty 32 x 32 bit products a block), comparisons and conversions keep the SMs' integer pipe 60 % busy. fp32 4099 x 1001: 8 us, floor 5.
template <typename T>
constexpr int kAheadOf = sizeof(T) == 4 ? 3 : 4;

template <typename T, bool VECTOR, bool SEED_IN_MEMORY>
__global__ void __launch_bounds__(kT, 4) dropout_kernel(const __grid_constant__ Launch l) {
  constexpr int kAhead = kAheadOf<T>, kParts = sizeof(T) / 2;  // sixteen bytes each, of a block
  extern __shared__ uint4 ring[];        // [residual][kAhead][block of the thread][kParts]
  const NangilaDropoutParams& p = l.p;
  Keys made;
  if (SEED_IN_MEMORY) make_keys(uint64_t(*p.seed_ptr), made);
  const Keys& keys = SEED_IN_MEMORY ? made : l.keys;
  const T* x = static_cast<const T*>(p.x);
  const T* r = static_cast<const T*>(p.residual);
  T* out = static_cast<T*>(p.out);
  const int64_t step = int64_t(gridDim.x) * kT, first = int64_t(blockIdx.x) * kT + threadIdx.x;
  const int64_t whole = VECTOR ? p.n / 8 : 0;
  if (VECTOR) {
    // a warp's 32 blocks lie side by side, and its lanes copy neighbouring sixteen bytes: with kParts > 1 not all of them their own
    const int lane = threadIdx.x & 31;
    auto slot = [&](int which, int stage) { return ring + (which * kAhead + stage) * kParts * kT + (threadIdx.x - lane) * kParts; };
    auto fetch = [&](int64_t b0, int stage) {
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        const int64_t at = kParts > 1 ? b0 * kParts + k * 32 + lane : b0;
        if (at >= whole * kParts) continue;
        copy16(slot(0, stage) + k * 32 + lane, reinterpret_cast<const uint4*>(x) + at);
        if (r != nullptr) copy16(slot(1, stage) + k * 32 + lane, reinterpret_cast<const uint4*>(r) + at);
      }
      copies_commit();
    };
    auto read = [&](int which, int stage, float (&v)[8]) {
      dev::Raw8<T> raw;
      raw.a = slot(which, stage)[lane * kParts];
      if constexpr (kParts > 1) raw.b = slot(which, stage)[lane * kParts + 1];
      dev::unpack(raw, v);
    };
    // (each thread for itself where its copies are its own)
    const int64_t first0 = kParts > 1 ? first - lane : first;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) fetch(first0 + k * step, k);
    int stage = 0;
    for (int64_t b0 = first0; b0 < whole; b0 += step) {
      const int64_t b = kParts > 1 ? b0 + lane : b0;
      const uint4 c = philox(uint64_t(b), p.draw, 0, keys);
      copies_wait_but<kAhead - 1>();
      if (kParts > 1) __syncwarp();
      float v[8], a[8];  // (of a block behind the last: never written)
      read(0, stage, v);
      drop8(v, p.scale, c, l.upper);
      if (r != nullptr) {
        read(1, stage, a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += a[i];
      }
      if (kParts > 1) __syncwarp();
      fetch(b0 + kAhead * step, stage);
      stage = stage + 1 == kAhead ? 0 : stage + 1;
      if (kParts > 1 && b >= whole) continue;
      dev::Raw8<T> raw;
      dev::pack(v, raw);
      dev::put(out + b * 8, raw);
      if (tied8(c, l.upper) && l.lower != 0) settle8<T>(l, b, c, keys);
    }
    copies_wait_but<0>();
  }
  for (int64_t b = whole + first; b < (p.n + 7) / 8; b += step) {  // the last elements, or all of them one by one
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = b * 8 + i < p.n ? dev::Vec16<T>::to_float(x[b * 8 + i]) : 0.0f;
    const uint4 c = philox(uint64_t(b), p.draw, 0, keys);
    drop8(v, p.scale, c, l.upper);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t at = b * 8 + i;
      if (at < p.n) out[at] = dev::Vec16<T>::from_float(r != nullptr ? v[i] + dev::Vec16<T>::to_float(r[at]) : v[i]);
    }
    if (tied8(c, l.upper) && l.lower != 0) settle8<T>(l, b, c, keys);
  }
}

template <typename T>
int launch(const NangilaDropoutParams& p, cudaStream_t stream) {
  if (p.least >> 32 != 0) {  // nothing is kept
    const size_t bytes = size_t(p.n) * sizeof(T);
    return int(p.residual != nullptr ? cudaMemcpyAsync(p.out, p.residual, bytes, cudaMemcpyDeviceToDevice, stream) : cudaMemsetAsync(p.out, 0, bytes, stream));
  }
  Launch l;
  l.p = p;
  make_keys(p.seed, l.keys);
  l.upper = uint32_t(p.least >> 16);
  l.lower = uint32_t(p.least) & 0xffffu;
  auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
  const bool vector = aligned(p.x) && aligned(p.residual) && aligned(p.out);
  auto* kernel = p.seed_ptr != nullptr ? (vector ? dropout_kernel<T, true, true> : dropout_kernel<T, false, true>) : (vector ? dropout_kernel<T, true, false> : dropout_kernel<T, false, false>);
  constexpr size_t kRing = 2 * kAheadOf<T> * (sizeof(T) / 2) * kT * sizeof(uint4);  // with a residual
  int resident = 0;
  if (const cudaError_t e = resident_ctas(reinterpret_cast<const void*>(kernel), kT, kRing, &resident)) return int(e);
  const int64_t want = ((p.n + 7) / 8 + kT - 1) / kT;
  kernel<<<unsigned(std::min<int64_t>(want, resident)), kT, vector ? (p.residual != nullptr ? kRing : kRing / 2) : 0, stream>>>(l);
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

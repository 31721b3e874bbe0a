// Eight values of a tensor as they lie in memory, so that a thread can have many loads on their way without a register for each value.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace nangila {
namespace dev {

template <typename T>
struct Raw8;
template <> struct Raw8<float> { uint4 a, b; };
template <> struct Raw8<__nv_bfloat16> { uint4 a; };
template <> struct Raw8<__half> { uint4 a; };

__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// 16-byte aligned addresses
template <typename T>
__device__ __forceinline__ void fetch(const T* p, Raw8<T>& r) {
  r.a = load_stream(p);
  if constexpr (sizeof(T) == 4) r.b = load_stream(reinterpret_cast<const uint4*>(p) + 1);
}
template <typename T>
__device__ __forceinline__ void put(T* p, const Raw8<T>& r) {
  *reinterpret_cast<uint4*>(p) = r.a;
  if constexpr (sizeof(T) == 4) reinterpret_cast<uint4*>(p)[1] = r.b;
}
__device__ __forceinline__ void unpack(const Raw8<float>& r, float (&v)[8]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void unpack(const Raw8<__nv_bfloat16>& r, float (&v)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const Raw8<__half>& r, float (&v)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void pack(const float (&v)[8], Raw8<float>& r) {
  r.a = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  r.b = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
}
__device__ __forceinline__ void pack(const float (&v)[8], Raw8<__nv_bfloat16>& r) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  r.a = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void pack(const float (&v)[8], Raw8<__half>& r) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  r.a = make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace dev
}  // namespace nangila

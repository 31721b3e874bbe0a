// Token embeddings: out[i] = scale * weight[ids[i]], and the table's gradient dw[v] = scale * sum of dy[i] over ids[i] = v.
//
// The gradient goes by sorted tokens, so that every sum has a fixed order and no atomics decide it:
//   1. the gradient is filled with zeros, which is most of what is written: a batch has far fewer tokens than the table has rows. Meanwhile a cluster of eight CTAs sorts
//      the positions by id (radix sort, least significant digit first, stable);
//   2. the sorted positions are cut into pieces of a few dozen, and each piece adds up its runs of equal ids, in fp32; a run that lies in one piece is
//      a finished row, one that goes on in the next leaves partial sums;
//   3. the partial sums of each run that crosses pieces are added up. A token that fills half the batch is spread over all SMs that way.
// Ids outside the table and the padding id sort behind all others and are left out.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>

#include "follow.cuh"
#include "launch_util.cuh"
#include "nangila_kernels.h"
#include "nangila_vocab_kernels.h"
#include "ptx_sm100.cuh"
#include "quant.cuh"
#include "raw8.cuh"

namespace nangila {
namespace {

__device__ __forceinline__ int64_t id_at(const void* ids, int ids_64, int64_t i) {
  return ids_64 ? static_cast<const int64_t*>(ids)[i] : int64_t(static_cast<const int32_t*>(ids)[i]);
}

// Sixteen bytes from any address of a T, put together from the two aligned sixteen that hold them. An aligned sixteen that holds a byte of the tensor lies in the memory that
// was allocated for it; one that holds none, from `lo` to `hi`, is not read, and is zero.
struct Window {
  uint4 x, y;
};
__device__ __forceinline__ Window window_at(const void* p, const char* lo, const char* hi) {
  const char* a = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15));
  Window w;
  w.x = w.y = make_uint4(0, 0, 0, 0);
  if (a + 16 > lo && a < hi) w.x = __ldg(reinterpret_cast<const uint4*>(a));
  if (a + 32 > lo && a + 16 < hi) w.y = __ldg(reinterpret_cast<const uint4*>(a + 16));
  return w;
}
template <typename T>
__device__ __forceinline__ uint4 shifted(const Window& at, const void* p) {
  const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(p));
  uint32_t w[8] = {at.x.x, at.x.y, at.x.z, at.x.w, at.y.x, at.y.y, at.y.z, at.y.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = (off & 8u) ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = (off & 4u) ? w[i + 1] : w[i];
  if (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (off & 2u) * 8u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- lookup ------------------------------------------------------------------------------------------------------
constexpr int kLookupT = 256;
constexpr int kLookupAtOnce = 4;  // vectors of a lane on their way together

// A warp for each token, rows of whole vectors.
template <typename T>
__global__ void __launch_bounds__(kLookupT) embedding_kernel(const __grid_constant__ NangilaEmbeddingParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = int64_t(gridDim.x) * (kLookupT / 32);
  for (int64_t i = int64_t(blockIdx.x) * (kLookupT / 32) + (threadIdx.x >> 5); i < p.n; i += warps) {
    const int64_t id = id_at(p.ids, p.ids_64, i);
    const bool inside = id >= 0 && id < p.rows;
    const T* from = static_cast<const T*>(p.weight) + (inside ? id : 0) * p.weight_stride;
    T* to = static_cast<T*>(p.out) + i * p.d;
    for (int c = lane * 8; c < p.d; c += 256 * kLookupAtOnce) {
      dev::Raw8<T> raw[kLookupAtOnce];
#pragma unroll
      for (int k = 0; k < kLookupAtOnce; ++k)
        if (c + 256 * k < p.d) dev::fetch(from + c + 256 * k, raw[k]);
#pragma unroll
      for (int k = 0; k < kLookupAtOnce; ++k) {
        if (c + 256 * k >= p.d) continue;
        float v[8];
        dev::unpack(raw[k], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = inside ? v[e] * p.scale : __uint_as_float(0x7fc00000u);
        dev::pack(v, raw[k]);
        dev::put(to + c + 256 * k, raw[k]);
      }
    }
  }
}
// Rows that start anywhere: the packed output is cut into sixteen bytes each, and each of those is put together from its row, or from the two that meet in it (value by value
// where rows are shorter than that). (A value at a time, a warp for each token, 16381 x 769 fp16 took 24 us.)
template <typename T, typename Index>
__global__ void __launch_bounds__(kLookupT) embedding_any_kernel(const __grid_constant__ NangilaEmbeddingParams p, Index values) {
  constexpr int N = 16 / sizeof(T), kOnTheWay = 2;
  const char* lo = static_cast<const char*>(p.weight);
  const char* hi = lo + ((p.rows - 1) * p.weight_stride + p.d) * int64_t(sizeof(T));
  auto row_of = [&](Index i, bool& inside) {
    const int64_t id = id_at(p.ids, p.ids_64, i);
    inside = id >= 0 && id < p.rows;
    return static_cast<const T*>(p.weight) + (inside ? id : 0) * p.weight_stride;
  };
  auto put_scaled = [&](const uint4& raw, bool inside, float (&v)[N], int from) {  // the values from `from` on
    float u[8];
    dev::Raw8<T> r;
    r.a = raw;
    if constexpr (sizeof(T) == 4) r.b = make_uint4(0, 0, 0, 0);
    dev::unpack(r, u);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k >= from) v[k] = inside ? u[k] * p.scale : __uint_as_float(0x7fc00000u);
  };
  const Index step = Index(gridDim.x) * kLookupT * N;
  for (Index at0 = (Index(blockIdx.x) * kLookupT + threadIdx.x) * N; at0 < values; at0 += step * kOnTheWay) {
    const T *row[kOnTheWay], *next[kOnTheWay];  // where the sixteen begin in their row, and would have begun in the one behind it
    bool inside[kOnTheWay], next_inside[kOnTheWay];
    int left[kOnTheWay];                        // values of the first row
    Window w[kOnTheWay], next_w[kOnTheWay];
#pragma unroll
    for (int j = 0; j < kOnTheWay; ++j) {
      const Index at = at0 + step * j;
      left[j] = 0;
      if (at >= values) continue;
      const Index i = at / Index(p.d);
      const int col = int(at - i * Index(p.d));
      left[j] = p.d - col;
      row[j] = row_of(i, inside[j]) + col;
      next[j] = row[j], next_inside[j] = false;
      if (left[j] < N && int64_t(i) + 1 < p.n) next[j] = row_of(i + 1, next_inside[j]) - left[j];
    }
#pragma unroll
    for (int j = 0; j < kOnTheWay; ++j) {
      if (left[j] == 0) continue;
      w[j] = window_at(row[j], lo, hi);
      if (left[j] < N) next_w[j] = window_at(next[j], lo, hi);
    }
#pragma unroll
    for (int j = 0; j < kOnTheWay; ++j) {
      if (left[j] == 0) continue;
      const Index at = at0 + step * j;
      float v[N];
      put_scaled(shifted<T>(w[j], row[j]), inside[j], v, 0);
      if (left[j] < N) {
        put_scaled(shifted<T>(next_w[j], next[j]), next_inside[j], v, left[j]);
        if (p.d < N) {
#pragma unroll
          for (int k = 0; k < N; ++k) {
            if (k < left[j] || at + Index(k) >= values) continue;
            const Index i = (at + Index(k)) / Index(p.d);
            bool in;
            const T* from = row_of(i, in);
            v[k] = in ? dev::Vec16<T>::to_float(from[at + Index(k) - i * Index(p.d)]) * p.scale : __uint_as_float(0x7fc00000u);
          }
        }
      }
      T* to = static_cast<T*>(p.out) + at;
      if (at + N <= values) {
        float u[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = v[k % N];
        dev::Raw8<T> r;
        dev::pack(u, r);
        *reinterpret_cast<uint4*>(to) = r.a;
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (at + Index(k) < values) to[k] = dev::Vec16<T>::from_float(v[k]);
      }
    }
  }
}

// ---- gradient ----------------------------------------------------------------------------------------------------
constexpr int kSortT = 1024;
constexpr int kSortCtas = 8;       // one cluster: 13 us for 8192 positions, hidden by the zeros; of long lists of narrow rows it is the most (262144 x 64 of 32000 103 us, of 180 with the lookup)
constexpr int kSortWarps = kSortCtas * kSortT / 32;
constexpr int kMaxDigit = 10;      // bits
constexpr int kSortSmem = ((kSortT / 32) + 1) * (4 << kMaxDigit) + 256;
constexpr int kSumT = 128;
constexpr int kJoinT = 512;
constexpr int kFew = 4;            // further pieces of a run that a warp adds up by itself (65536 tokens x 1024, lookup and gradient: 119.5 us, with up to 32 122.2, with up to 256 126.3)
constexpr int kFillT = 512;
constexpr int kMaxPiece = 64;

struct Sorted {
  uint32_t *key[2], *at[2];        // ids and positions, there and back
  uint32_t* crossing;              // runs that begin in one piece and go on behind it. [0], [1]: how many of up to kFew pieces more, and of more than that
  uint2* run;                      // [pieces] each the first piece and how many more: the short ones from the front, the long ones from the back
  float* partial;                  // [2 * pieces][pitch]
  int passes, digit;               // bits of a digit
  int last;                        // which of the two buffers the sorted ones are in
  int per_warp;                    // positions of a warp of the sort, a multiple of 32
  int piece, pieces, pitch;
};

__device__ __forceinline__ uint32_t load_cluster(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// Zeros in all of dw, two CTAs on each SM that stay. The sort is set up beside them. (In CTAs of the sort's own launch, whose clusters of eight do not all fit at a time, 131 MB took
// 35 us, for 24.)
__global__ void __launch_bounds__(kFillT) embedding_fill_kernel(uint8_t* dw, int64_t bytes) {
  may_follow();
  const int64_t step = int64_t(gridDim.x) * kFillT, first = int64_t(blockIdx.x) * kFillT + threadIdx.x, wide = bytes / 32;
  for (int64_t i = first; i < wide; i += step) asm volatile("st.global.v8.b32 [%0], {%1, %1, %1, %1, %1, %1, %1, %1};" ::"l"(dw + i * 32), "r"(0) : "memory");
  if (first < (bytes & 31)) dw[wide * 32 + first] = 0;
}
// Ends behind the kernel before it, which it does not wait for until then: what follows finds the work of both.
template <int kBatch>  // of a lane's positions on their way together
__global__ void __launch_bounds__(kSortT, 1) embedding_sort_kernel(const __grid_constant__ NangilaEmbeddingGradParams p, const __grid_constant__ Sorted s) {
  extern __shared__ uint32_t smem[];
  uint32_t* count = smem;                                       // [warp][digit]
  uint32_t* total = count + (kSortT / 32) * (1 << kMaxDigit);   // of this CTA's positions, by digit
  uint32_t* scan = total + (1 << kMaxDigit);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, digits = 1 << s.digit;
  const uint32_t rank = blockIdx.x;
  const int64_t from = int64_t(int(rank) * (kSortT / 32) + warp) * s.per_warp, to = min(p.n, from + s.per_warp);
  if (rank == 0 && threadIdx.x < 2) s.crossing[threadIdx.x] = 0;
  for (int pass = 0; pass < s.passes; ++pass) {
    const uint32_t *src_key = s.key[(pass + 1) & 1], *src_at = s.at[(pass + 1) & 1];
    uint32_t *dst_key = s.key[pass & 1], *dst_at = s.at[pass & 1];
    const int shift = pass * s.digit;
    auto key_of = [&](int64_t i) -> uint32_t {
      if (pass > 0) return __ldcg(src_key + i);
      const int64_t id = id_at(p.ids, p.ids_64, i);
      return id >= 0 && id < p.rows && id != p.padding ? uint32_t(id) : uint32_t(p.rows);
    };
    for (int i = threadIdx.x; i < (kSortT / 32) * digits; i += kSortT) count[i] = 0;
    __syncthreads();
    uint32_t* mine = count + warp * digits;
    for (int64_t i0 = from; i0 < to; i0 += 32 * kBatch) {
      uint32_t k[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + 32 * j + lane < to) k[j] = key_of(i0 + 32 * j + lane);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + 32 * j + lane < to) atomicAdd(&mine[k[j] >> shift & uint32_t(digits - 1)], 1u);
    }
    __syncthreads();
    // where each (digit, CTA, warp) begins: before it come all smaller digits, and this digit's positions of the CTAs and warps before
    const int d = threadIdx.x;
    if (d < digits) {
      uint32_t run = 0;
#pragma unroll 8
      for (int w = 0; w < kSortT / 32; ++w) {
        const uint32_t t = count[w * digits + d];
        count[w * digits + d] = run;
        run += t;
      }
      total[d] = run;
    }
    sm100::cluster_sync();
    uint32_t before = 0, all = 0;
    if (d < digits) {
#pragma unroll
      for (uint32_t q = 0; q < kSortCtas; ++q) {
        const uint32_t v = load_cluster(sm100::cluster_address(total + d, q));
        all += v;
        before += q < rank ? v : 0u;
      }
    }
    uint32_t sum = all;  // up to this digit, in the warp
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += v;
    }
    if (lane == 31) scan[warp] = sum;
    __syncthreads();
    if (d < digits) {
      for (int w = 0; w < warp; ++w) before += scan[w];
      before += sum - all;
#pragma unroll 8
      for (int w = 0; w < kSortT / 32; ++w) count[w * digits + d] += before;
    }
    __syncthreads();
    for (int64_t i0 = from; i0 < to; i0 += 32 * kBatch) {
      uint32_t k[kBatch], a[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int64_t i = i0 + 32 * j + lane;
        if (i >= to) continue;
        k[j] = key_of(i);
        a[j] = pass > 0 ? __ldcg(src_at + i) : uint32_t(i);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (i0 + 32 * j >= to) break;
        const bool here = i0 + 32 * j + lane < to;
        const uint32_t digit = here ? k[j] >> shift & uint32_t(digits - 1) : uint32_t(digits);  // (those that are not here keep to themselves)
        const uint32_t same = __match_any_sync(0xffffffffu, digit);
        const uint32_t order = __popc(same & ((1u << lane) - 1u));
        uint32_t pos = 0;
        if (here) pos = mine[digit] + order;
        __syncwarp();
        if (here && order == 0) mine[digit] += __popc(same);
        __syncwarp();
        if (here) {
          dst_key[pos] = k[j];
          dst_at[pos] = a[j];
        }
      }
    }
    sm100::cluster_sync();  // what one CTA has written, all read in the next pass
  }
  follow();
}

// A thread takes eight adjacent columns of a piece; threadIdx.y: the piece of the CTA's. VECTOR: rows start on sixteen bytes and end with a whole eight.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(kSumT, (!VECTOR ? 512 : sizeof(T) == 4 ? 768 : 1024) / kSumT) embedding_sum_kernel(const __grid_constant__ NangilaEmbeddingGradParams p, const __grid_constant__ Sorted s) {
  // Rows on their way together. (Eight, with half as many threads an SM: 65536 tokens x 1024, lookup and gradient, 120 us, for 114.)
  constexpr int kAtOnce = !VECTOR && sizeof(T) == 2 ? 8 : 4;
  __shared__ uint32_t keys[kSumT / 32 * kMaxPiece], positions[kSumT / 32 * kMaxPiece];  // of the CTA's pieces
  const int piece = blockIdx.x * blockDim.y + threadIdx.y, col = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  follow();
  const uint32_t* key = s.key[s.last];
  const int64_t all0 = int64_t(blockIdx.x) * blockDim.y * s.piece;
  for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < int(blockDim.y) * s.piece && all0 + i < p.n; i += kSumT) {
    keys[i] = key[all0 + i];
    positions[i] = s.at[s.last][all0 + i];
  }
  __syncthreads();
  if (piece >= s.pieces || col >= p.d) return;
  const int64_t s0 = int64_t(piece) * s.piece;
  const int count = int(min(p.n, s0 + s.piece) - s0);
  const uint32_t *mine = keys + threadIdx.y * s.piece, *at = positions + threadIdx.y * s.piece;
  const T* dy = static_cast<const T*>(p.dy);
  const char* lo = reinterpret_cast<const char*>(dy);
  const char* hi = lo + ((p.n - 1) * p.dy_stride + p.d) * int64_t(sizeof(T));
  uint32_t current = mine[0];
  bool before = s0 > 0 && key[s0 - 1] == current;
  const uint32_t behind = s0 + count < p.n ? key[s0 + count] : uint32_t(p.rows);
  float acc[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] = 0.0f;
  auto finish = [&](bool goes_on) {
    if (current >= uint32_t(p.rows)) return;
    if (!before && !goes_on) {
      T* to = static_cast<T*>(p.dw) + int64_t(current) * p.d + col;
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = acc[k] * p.scale;
      if constexpr (VECTOR) {
        dev::Raw8<T> raw;
        dev::pack(v, raw);
        dev::put(to, raw);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (col + k < p.d) to[k] = dev::Vec16<T>::from_float(v[k]);
      }
    } else {
      float4* to = reinterpret_cast<float4*>(s.partial + (int64_t(2) * piece + (before ? 0 : 1)) * s.pitch + col);
      to[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      to[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (!before && col == 0) {
        // how many pieces more begin with this id: twice as far at a time, then halved
        auto begins = [&](int64_t j) { return (piece + j) * s.piece < p.n && key[(piece + j) * s.piece] == current; };
        int64_t in = 1, out = 2;  // the last that is known to, and one that may not
        while (begins(out)) in = out, out *= 2;
        while (out - in > 1) {
          const int64_t mid = (in + out) / 2;
          if (begins(mid)) in = mid;
          else out = mid;
        }
        // (in any order: each is summed by itself)
        if (in <= kFew) s.run[atomicAdd(s.crossing, 1u)] = make_uint2(uint32_t(piece), uint32_t(in));
        else s.run[s.pieces - 1 - atomicAdd(s.crossing + 1, 1u)] = make_uint2(uint32_t(piece), uint32_t(in));
      }
    }
  };
  for (int i0 = 0; i0 < count; i0 += kAtOnce) {
    uint32_t k[kAtOnce];
    dev::Raw8<T> raw[VECTOR ? kAtOnce : 1];
    const T* row[VECTOR ? 1 : kAtOnce];
    Window w[VECTOR ? 1 : kAtOnce][sizeof(T) / 2];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      k[j] = i0 + j < count ? mine[i0 + j] : uint32_t(p.rows);
      if (k[j] >= uint32_t(p.rows)) continue;
      const T* from = dy + int64_t(at[i0 + j]) * p.dy_stride + col;
      if constexpr (VECTOR) {
        dev::fetch(from, raw[j]);
      } else {
        row[j] = from;
#pragma unroll
        for (int h = 0; h < int(sizeof(T)) / 2; ++h) w[j][h] = window_at(from + 4 * h, lo, hi);
      }
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (i0 + j >= count) break;
      if (k[j] != current) {
        finish(false);
        current = k[j];
        before = false;
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c] = 0.0f;
      }
      if (current >= uint32_t(p.rows)) return;  // nothing but what is left out from here on
      float v[8];
      if constexpr (VECTOR) {
        dev::unpack(raw[j], v);
      } else {
        dev::Raw8<T> r;
        r.a = shifted<T>(w[j][0], row[j]);
        if constexpr (sizeof(T) == 4) r.b = shifted<T>(w[j][1], row[j]);
        dev::unpack(r, v);
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[c] += v[c];
    }
  }
  finish(behind == current);
}

// The runs that cross pieces, 128 columns at a time: a long one by the sixteen warps of a CTA, each with every sixteenth partial sum, added up in order; a short one by a warp.
template <typename T>
__global__ void __launch_bounds__(kJoinT) embedding_join_kernel(const __grid_constant__ NangilaEmbeddingGradParams p, const __grid_constant__ Sorted s) {
  constexpr int kGroups = kJoinT / 32;
  __shared__ float4 part[kGroups][32];
  follow();
  const uint32_t* key = s.key[s.last];
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
  const int blocks = (p.d + 127) / 128;
  auto sum_of = [&](const uint2 run, int col, int from, int step) {
    float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int j = from; j <= int(run.y); j += step) {
      const float4 v = *reinterpret_cast<const float4*>(s.partial + (int64_t(2) * (run.x + j) + (j == 0 ? 1 : 0)) * s.pitch + col);
      sum.x += v.x;
      sum.y += v.y;
      sum.z += v.z;
      sum.w += v.w;
    }
    return sum;
  };
  auto put = [&](const uint2 run, int col, const float4& sum) {
    const float v[4] = {sum.x, sum.y, sum.z, sum.w};
    T* to = static_cast<T*>(p.dw) + int64_t(key[int64_t(run.x + 1) * s.piece]) * p.d + col;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (col + k < p.d) to[k] = dev::Vec16<T>::from_float(v[k] * p.scale);
  };
  const int64_t few = int64_t(s.crossing[0]) * blocks, many = int64_t(s.crossing[1]) * blocks;
  for (int64_t task = blockIdx.x; task < many; task += gridDim.x) {
    const uint2 run = s.run[s.pieces - 1 - task / blocks];
    const int col = int(task % blocks) * 128 + lane * 4;
    float4 sum = make_float4(0, 0, 0, 0);
    if (col < p.d) sum = sum_of(run, col, group, kGroups);
    part[group][lane] = sum;
    __syncthreads();
    if (group == 0 && col < p.d) {
      for (int g = 1; g < kGroups; ++g) {
        const float4 v = part[g][lane];
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
      }
      put(run, col, sum);
    }
    __syncthreads();
  }
  for (int64_t task = int64_t(blockIdx.x) * kGroups + group; task < few; task += int64_t(gridDim.x) * kGroups) {
    const uint2 run = s.run[task / blocks];
    const int col = int(task % blocks) * 128 + lane * 4;
    if (col < p.d) put(run, col, sum_of(run, col, 0, 1));
  }
}

// ---- host --------------------------------------------------------------------------------------------------------
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T>
int lookup(const NangilaEmbeddingParams& p, cudaStream_t stream) {
  const bool vector = p.d % 8 == 0 && aligned16(p.weight) && aligned16(p.out) && p.weight_stride * int64_t(sizeof(T)) % 16 == 0;
  int resident = 0;
  if (vector) {
    if (const cudaError_t e = resident_ctas(reinterpret_cast<const void*>(embedding_kernel<T>), kLookupT, 0, &resident)) return int(e);
    const int64_t want = (p.n + kLookupT / 32 - 1) / (kLookupT / 32);
    embedding_kernel<T><<<unsigned(std::min<int64_t>(want, resident)), kLookupT, 0, stream>>>(p);
    return int(cudaGetLastError());
  }
  const int64_t values = p.n * p.d, each = kLookupT * 16 / int64_t(sizeof(T));
  const unsigned ctas = unsigned(std::min<int64_t>((values + each - 1) / each, 148 * 8));
  // (where a position and the step behind the last fit into 32 bits, divisions are short)
  if (values < (int64_t(1) << 31)) embedding_any_kernel<T, uint32_t><<<ctas, kLookupT, 0, stream>>>(p, uint32_t(values));
  else embedding_any_kernel<T, uint64_t><<<ctas, kLookupT, 0, stream>>>(p, uint64_t(values));
  return int(cudaGetLastError());
}

// How the work on n positions is cut up, and where it lies in the workspace.
Sorted layout(int64_t n, int64_t rows, int32_t d, uint8_t* base, int64_t* bytes) {
  Sorted s;
  int64_t used = 0;
  auto take = [&](int64_t size) {
    uint8_t* at = base + used;
    used += (size + 255) / 256 * 256;
    return at;
  };
  for (int i = 0; i < 2; ++i) {
    s.key[i] = reinterpret_cast<uint32_t*>(take(n * 4));
    s.at[i] = reinterpret_cast<uint32_t*>(take(n * 4));
  }
  int bits = 1;
  while (rows >> bits) ++bits;  // keys 0 .. rows
  s.passes = (bits + kMaxDigit - 1) / kMaxDigit;
  s.digit = (bits + s.passes - 1) / s.passes;
  s.last = (s.passes - 1) & 1;
  s.per_warp = int(((n + kSortWarps - 1) / kSortWarps + 31) / 32 * 32);
  // Pieces: no shorter than what a thread has on its way at a time, and longer where there are positions enough for a thousand of them. (Lookup and gradient, in pieces of 8, so, of 64:
  // 512 tokens x 1024 26.7, 26.7, 34.9 us; 8192 x 2048 63.7, 59.4, 61.5; 65536 x 1024 142.6, 122.2, 122.2.)
  s.piece = 8;
  while (s.piece < kMaxPiece && n >= int64_t(s.piece) * 1024) s.piece *= 2;
  s.pieces = int((n + s.piece - 1) / s.piece);
  s.pitch = (d + 7) / 8 * 8;
  s.crossing = reinterpret_cast<uint32_t*>(take(8));
  s.run = reinterpret_cast<uint2*>(take(int64_t(s.pieces) * 8));
  s.partial = reinterpret_cast<float*>(take(int64_t(2) * s.pieces * s.pitch * 4));
  *bytes = used;
  return s;
}

template <typename T>
int gradient(const NangilaEmbeddingGradParams& p, cudaStream_t stream) {
  int64_t bytes = 0;
  const Sorted s = layout(p.n, p.rows, p.d, static_cast<uint8_t*>(p.workspace), &bytes);
  // (One position of a lane at a time is less to fetch of the kernel itself: 8192 tokens 13 us, in batches of eight 15.7; 65536 x 1024, lookup and gradient, 114 and 112.8.)
  auto* sort = s.per_warp <= 64 ? embedding_sort_kernel<1> : embedding_sort_kernel<8>;
  int resident = 0;
  if (const cudaError_t e = resident_ctas(reinterpret_cast<const void*>(sort), kSortT, kSortSmem, &resident)) return int(e);
  const int64_t size = p.rows * p.d * int64_t(sizeof(T));
  embedding_fill_kernel<<<unsigned(std::min<int64_t>((size / 32 + kFillT) / kFillT, 2 * 148)), kFillT, 0, stream>>>(static_cast<uint8_t*>(p.dw), size);
  if (const cudaError_t e = cudaGetLastError()) return int(e);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kSortCtas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kSortCtas);
  cfg.blockDim = dim3(kSortT);
  cfg.dynamicSmemBytes = kSortSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (const cudaError_t e = cudaLaunchKernelEx(&cfg, sort, p, s)) return int(e);
  const bool vector = p.d % 8 == 0 && aligned16(p.dy) && aligned16(p.dw) && p.dy_stride * int64_t(sizeof(T)) % 16 == 0;
  const int threads = (p.d + 7) / 8;
  int x = 32;
  while (x < kSumT && x < threads) x *= 2;
  const int y = kSumT / x;
  auto* sum = vector ? embedding_sum_kernel<T, true> : embedding_sum_kernel<T, false>;
  cfg.gridDim = dim3(unsigned((s.pieces + y - 1) / y), unsigned((threads + x - 1) / x));
  cfg.blockDim = dim3(unsigned(x), unsigned(y));
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  if (const cudaError_t e = cudaLaunchKernelEx(&cfg, sum, p, s)) return int(e);
  if (s.pieces < 2) return 0;
  const int64_t tasks = int64_t(s.pieces - 1) * ((p.d + 127) / 128);
  return int(launch_following(embedding_join_kernel<T>, dim3(unsigned(std::min<int64_t>(tasks, 2 * 148))), kJoinT, 0, stream, p, s));
}

}  // namespace
}  // namespace nangila

extern "C" int nangila_embedding(const NangilaEmbeddingParams* p, cudaStream_t stream) {
  using namespace nangila;
  if (!p || !p->ids || !p->weight || !p->out || !aligned16(p->out) || p->n < 0 || p->rows < 1 || p->d < 1) return int(cudaErrorInvalidValue);
  if (p->n == 0) return 0;
  try {
    switch (p->dtype) {
      case NANGILA_F32: return lookup<float>(*p, stream);
      case NANGILA_F16: return lookup<__half>(*p, stream);
      case NANGILA_BF16: return lookup<__nv_bfloat16>(*p, stream);
      default: return int(cudaErrorInvalidValue);
    }
  } catch (...) {  // (the host's tables of kernels that were set up allocate)
    return int(cudaErrorMemoryAllocation);
  }
}

extern "C" int64_t nangila_embedding_workspace(int64_t n, int64_t rows, int32_t d) {
  int64_t bytes = 0;
  nangila::layout(n, rows, d, nullptr, &bytes);
  return bytes;
}

extern "C" int nangila_embedding_backward(const NangilaEmbeddingGradParams* p, cudaStream_t stream) {
  using namespace nangila;
  if (!p || !p->ids || !p->dy || !p->dw || !p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 255u) || (reinterpret_cast<uintptr_t>(p->dw) & 31u) || p->n < 1 || p->n > NANGILA_EMBEDDING_MAX_TOKENS || p->rows < 1 ||
      p->rows > NANGILA_EMBEDDING_MAX_ROWS || p->d < 1)
    return int(cudaErrorInvalidValue);
  try {
    switch (p->dtype) {
      case NANGILA_F32: return gradient<float>(*p, stream);
      case NANGILA_F16: return gradient<__half>(*p, stream);
      case NANGILA_BF16: return gradient<__nv_bfloat16>(*p, stream);
      default: return int(cudaErrorInvalidValue);
    }
  } catch (...) {
    return int(cudaErrorMemoryAllocation);
  }
}

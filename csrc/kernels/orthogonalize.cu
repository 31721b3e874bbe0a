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

constexpr int kTileM = 128;                      // rows of a CTA
constexpr int kSlabK = 64;                       // one 128-byte swizzle row of fp16
constexpr int kOperandBytes = 128 * kSlabK * 2;  // what a CTA holds of an operand's slab
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kStages = 5;
constexpr int kChunk = 64;                       // columns that a warp of the epilogue takes at a time
constexpr int kBoxBytes = 32 * kChunk * 2;       // 32 rows of them in fp16
constexpr int kSlotBytes = 2 * kBoxBytes;        // what comes in and goes out at a time, in place
constexpr int kEpilogueWarps = 8;                // two for each quarter of tensor memory, taking turns with the chunks
constexpr int kEpilogueBytes = kEpilogueWarps * kSlotBytes;
constexpr int kSmem = kStages * kStageBytes + kEpilogueBytes + 1024 + 256;
constexpr int kGemmThreads = 64 + 32 * kEpilogueWarps;  // warp 0: TMA, warp 1: products, the others: epilogue
constexpr uint64_t kTimeoutNs = 10ull * 1000 * 1000 * 1000;
constexpr float kLoScale = 2048.0f;

enum Kind { kGram, kPoly, kUpdate, kFinal };

struct Product {
  int M, N, K;             // D is M x N
  int tiles_m, per, total; // tiles along M; tiles of one matrix, of all
  int lower;               // only tiles that reach the lower triangle
  float alpha, beta;       // gram: D alpha;  poly: alpha A + beta D;  update: alpha X + D
  float unscale;           // final: result = (alpha X + D) unscale
  __nv_bfloat16* result;   // final: packed M x N, or NULL
  int param_dtype, vector; // final: the parameters' type; runs of four elements can be read and written
  float decay, rate;
  void* param[NANGILA_ORTH_MAX_COUNT];
};
struct Maps {
  CUtensorMap a, b;        // the operands
  CUtensorMap in, lo;      // poly: A;  update and final: hi and lo
  CUtensorMap out, mirror; // gram, poly: the result and its other half;  update: hi (lo goes back where it came from)
};

struct TileAt {
  int batch, m0, n0;
};
// Square tiles of SIDE x SIDE.
template <int SIDE>
__device__ __forceinline__ TileAt tile_at(const Product& p, int i) {
  TileAt t;
  t.batch = i / p.per;
  const int r = i - t.batch * p.per;
  int rb, cb;
  if (!p.lower) {
    cb = r / p.tiles_m;  // neighbours share the columns of the wide operand
    rb = r - cb * p.tiles_m;
  } else {
    rb = int((sqrtf(8.0f * r + 1.0f) - 1.0f) * 0.5f);
    while (rb * (rb + 1) / 2 > r) --rb;
    while ((rb + 1) * (rb + 2) / 2 <= r) ++rb;
    cb = r - rb * (rb + 1) / 2;
  }
  t.m0 = rb * SIDE;
  t.n0 = cb * SIDE;
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
// Sixteen bytes `j` of a lane's row in a box of 32 rows of 128 bytes, as TMA swizzles them (the box starts on 1024 bytes).
__device__ __forceinline__ uint4* box_at(uint8_t* box, int row, int j) { return reinterpret_cast<uint4*>(box + row * 128 + ((j ^ (row & 7)) << 4)); }

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]);
template <>
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
template <>
__device__ __forceinline__ void load4(const __half* p, float (&v)[4]) {
  const uint2 a = *reinterpret_cast<const uint2*>(p);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a.x)), y = __half22float2(*reinterpret_cast<const __half2*>(&a.y));
  v[0] = x.x; v[1] = x.y; v[2] = y.x; v[3] = y.y;
}
template <>
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 a = *reinterpret_cast<const uint2*>(p);
  v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xffff0000u); v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(__half* p, const float (&v)[4]) {
  const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&v)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
// A warp's 32 rows of results in a slot, fp32, taken to the parameters (T) or, with `fresh`, out. Two rows at a time, four columns a lane; the loads of
// sixteen rows are on their way before the first store.
template <typename T, bool fresh>
__device__ __forceinline__ void put_results(const Product& p, T* base, uint8_t* slot, int lane, int row0, int col0) {
  const int x = lane & 15, col = col0 + 4 * x, left = p.N - col;
  if (left <= 0) return;
  // four columns 4 x: group x / 4 of sixteen, its quarter x % 4
  uint8_t* box = slot + ((x & 2) ? kBoxBytes : 0);
  const int j = 2 * (x >> 2) + (x & 1);
#pragma unroll
  for (int half = 0; half < 32; half += 16) {
    float v[8][4];
    if (!fresh) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = row0 + half + 2 * i + (lane >> 4);
        if (row >= p.M) continue;
        const T* from = base + int64_t(row) * p.N + col;
        if (p.vector) {
          load4<T>(from, v[i]);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[i][k] = k < left ? dev::Vec16<T>::to_float(from[k]) : 0.0f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = half + 2 * i + (lane >> 4);
      if (row0 + at >= p.M) continue;
      const uint4 raw = *box_at(box, at, j);
      const float r[4] = {__uint_as_float(raw.x), __uint_as_float(raw.y), __uint_as_float(raw.z), __uint_as_float(raw.w)};
#pragma unroll
      for (int k = 0; k < 4; ++k) v[i][k] = fresh ? r[k] : v[i][k] * p.decay - p.rate * r[k];
      T* to = base + int64_t(row0 + at) * p.N + col;
      if (p.vector) {
        store4(to, v[i]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < left) to[k] = dev::Vec16<T>::from_float(v[i][k]);
      }
    }
  }
}

// Sixteen accumulators of a lane's row, columns 16 g to 16 g + 15 of the chunk in the slot, taken into the slot as what goes out.
template <int KIND>
__device__ __forceinline__ void into_slot(const Product& p, uint8_t* slot, int lane, int g, float (&v)[16]) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int j = 2 * g + e;
    float w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = v[8 * e + k];
    uint4* first = box_at(slot, lane, j);
    uint4* second = box_at(slot + kBoxBytes, lane, j);
    if constexpr (KIND == kGram || KIND == kPoly) {
      if constexpr (KIND == kGram) {
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] *= p.alpha;
      } else {
        float a[8];
        unpack8(*first, a);
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = __fmaf_rn(p.alpha, a[k], p.beta * w[k]);
      }
      *first = pack8(w);
      // the mirror: 64 rows of 32 values, one from each lane
      __half* t = reinterpret_cast<__half*>(slot + kBoxBytes) + lane;
#pragma unroll
      for (int k = 0; k < 8; ++k) t[(8 * j + k) * 32] = __float2half_rn(w[k]);
    } else {
      float hi[8], lo[8];
      unpack8(*first, hi);
      unpack8(*second, lo);
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = __fmaf_rn(p.alpha, __fmaf_rn(lo[k], 1.0f / kLoScale, hi[k]), w[k]);
      if constexpr (KIND == kUpdate) {
        uint4 h, l;
        split8(w, h, l);
        *first = h;
        *second = l;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[8 * e + k] = w[k] * p.unscale;
      }
    }
  }
}

// D = A B for square tiles of all matrices, walked over by CTAs that stay (PAIR: pairs of CTAs that share the tensor cores' work on 256 x 256, each
// with its 128 rows of A, half of B's columns, and 128 rows of the result; else one CTA and 128 x 128). A_MN / B_MN: the operand lies with its rows
// (columns of B) adjacent in memory, not its K. The accumulators of two tiles share tensor memory: the epilogue of one runs under the
// products of the next, and what it needs of X or A is on its way before they end. Each of its warps has a slot of shared memory of its own,
// filled and emptied by TMA, and meets no other warp.
// A wait that runs out makes every result of this CTA from there on not a number.
template <int KIND, bool A_MN, bool B_MN, bool PAIR>
__global__ void __launch_bounds__(kGemmThreads, 1) orth_product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Product p) {
  constexpr int kSide = PAIR ? 256 : 128;
  constexpr int kChunks = kSide / kChunk;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* slots = smem + kStages * kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(slots + kEpilogueBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;   // [2]
  uint64_t* acc_empty = acc_full + 2;     // [2]
  uint64_t* loaded = acc_empty + 2;       // [kEpilogueWarps]
  uint64_t* drained = loaded + kEpilogueWarps;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile uint32_t* failed = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slabs = (p.K + kSlabK - 1) / kSlabK;
  const uint32_t rank = PAIR ? cluster_rank() : 0u;   // 0: the CTA that issues the pair's products
  const int first = PAIR ? blockIdx.x / 2 : blockIdx.x, step = PAIR ? gridDim.x / 2 : gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], kEpilogueWarps * (PAIR ? 2 : 1));
    }
    for (int s = 0; s < kEpilogueWarps; ++s) mbar_init(&loaded[s], 1);
    mbar_init(drained, 1);
    *failed = 0;
    fence_barrier_init();
    prefetch_tensormap(&maps.a);
    prefetch_tensormap(&maps.b);
  }
  if (warp == 1) {
    if (PAIR) tmem_alloc_pair(tmem_slot, 2 * kSide);
    else tmem_alloc(tmem_slot, 2 * kSide);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync();  // the other CTA's barriers exist from here on
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  may_follow();
  follow();

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA: both CTAs of a pair, each its own halves; the bytes are counted where the products are issued ----------------
      int i = 0;  // slabs so far
      bool ok = true;
      for (int tile = first; tile < p.total && ok; tile += step) {
        const TileAt at = tile_at<kSide>(p, tile);
        const int row = at.m0 + int(rank) * kTileM, col = at.n0 + int(rank) * 128;
        for (int k = 0; k < slabs; ++k, ++i) {
          const int s = i % kStages;
          if (i >= kStages && !mbar_wait(&empty[s], uint32_t((i / kStages - 1) & 1), kTimeoutNs)) {
            *failed = 1;
            ok = false;
            break;
          }
          uint8_t* a = smem + s * kStageBytes;
          uint8_t* b = a + kOperandBytes;
          const int k0 = k * kSlabK;
          if (rank == 0) mbar_arrive_expect_tx(&full[s], kStageBytes * (PAIR ? 2 : 1));
          const uint32_t bar = PAIR ? rank0_address(&full[s]) : smem_u32(&full[s]);
          if (A_MN) {
            tma_operand<PAIR>(a, &maps.a, row, k0, at.batch, bar);
            tma_operand<PAIR>(a + 8192, &maps.a, row + 64, k0, at.batch, bar);
          } else {
            tma_operand<PAIR>(a, &maps.a, k0, row, at.batch, bar);
          }
          if (B_MN) {
            tma_operand<PAIR>(b, &maps.b, col, k0, at.batch, bar);
            tma_operand<PAIR>(b + 8192, &maps.b, col + 64, k0, at.batch, bar);
          } else {
            tma_operand<PAIR>(b, &maps.b, k0, col, at.batch, bar);
          }
        }
      }
      // the copies that are still under way: all have arrived when the products that read them are done; if somebody has given up, as
      // much as can be waited for (the bytes of a pair are counted by rank 0, the stages of rank 1 are given back by its products)
      for (int j = max(0, i - kStages); j < i; ++j) {
        if (*failed == 0 || rank != 0) mbar_wait(&empty[j % kStages], uint32_t((j / kStages) & 1), kTimeoutNs);
        else mbar_wait(&full[j % kStages], uint32_t((j / kStages) & 1), kTimeoutNs);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      // ---------------- products ----------------
      constexpr uint32_t idesc = (1u << 4) | (uint32_t(A_MN) << 15) | (uint32_t(B_MN) << 16) | (uint32_t(kSide >> 3) << 17) | (uint32_t(kSide >> 4) << 24);
      int i = 0, n = 0;
      bool ok = true;
      for (int tile = first; tile < p.total && ok; tile += step, ++n) {
        const int acc = n & 1;
        if (n >= 2 && !mbar_wait(&acc_empty[acc], uint32_t((n / 2 - 1) & 1), kTimeoutNs)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t d = tmem + uint32_t(acc * kSide);
        for (int k = 0; k < slabs; ++k, ++i) {
          const int s = i % kStages;
          if (!mbar_wait(&full[s], uint32_t((i / kStages) & 1), kTimeoutNs)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t a = smem_u32(smem + s * kStageBytes), b = a + kOperandBytes;
#pragma unroll
          for (int kk = 0; kk < kSlabK / 16; ++kk) {
            // K-major: 16 elements along K are 32 bytes of a swizzle row; MN-major: 16 K-rows are two groups of eight rows of 128 bytes
            const uint64_t ad = A_MN ? make_smem_desc(a + kk * 2048, 8192, 1024) : make_smem_desc(a + kk * 32, 16, 1024);
            const uint64_t bd = B_MN ? make_smem_desc(b + kk * 2048, 8192, 1024) : make_smem_desc(b + kk * 32, 16, 1024);
            if (PAIR) umma_f16_pair(d, ad, bd, idesc, (k > 0 || kk > 0) ? 1u : 0u);
            else umma_f16(d, ad, bd, idesc, (k > 0 || kk > 0) ? 1u : 0u);
          }
          if (PAIR) umma_commit_pair(&empty[s]);
          else umma_commit(&empty[s]);
        }
        if (ok) {
          if (PAIR) umma_commit_pair(&acc_full[acc]);
          else umma_commit(&acc_full[acc]);
        }
      }
      if (!ok) {
        *failed = 1;
        if (PAIR) umma_commit_pair(drained);
        else umma_commit(drained);
        mbar_wait(drained, 0, kTimeoutNs);
      }
    }
  } else {
    // ---------------- epilogue ----------------
    const int quad = warp & 3;  // the lanes of tensor memory that this warp may read
    const int turn = (warp - 2) >> 2;
    uint8_t* slot = slots + (warp - 2) * kSlotBytes;
    uint64_t* my_loaded = loaded + (warp - 2);
    const uint32_t acc_empty_at = PAIR ? rank0_address(&acc_empty[0]) : smem_u32(&acc_empty[0]);
    constexpr bool kLoads = KIND != kGram;
    constexpr uint32_t kLoadBytes = KIND == kPoly ? kBoxBytes : kSlotBytes;
    int n = 0;
    uint32_t chunks = 0;  // so far
    for (int tile = first; tile < p.total; tile += step, ++n) {
      const TileAt at = tile_at<kSide>(p, tile);
      const int acc = n & 1;
      const int row0 = at.m0 + int(rank) * kTileM + quad * 32;
      const int mine = row0 < p.M ? min(kChunks, (p.N - at.n0 + kChunk - 1) / kChunk) : 0;
      auto fetch = [&](int c) {  // lane 0: chunk c into the slot, once nothing goes out of it any more
        bulk_wait_read();
        mbar_arrive_expect_tx(my_loaded, kLoadBytes);
        tma_load_3d(slot, &maps.in, at.n0 + c * kChunk, row0, at.batch, my_loaded);
        if (KIND != kPoly) tma_load_3d(slot + kBoxBytes, &maps.lo, at.n0 + c * kChunk, row0, at.batch, my_loaded);
      };
      if (kLoads && turn < mine && lane == 0) fetch(turn);
      bool ok = *failed == 0 && mbar_wait(&acc_full[acc], uint32_t((n / 2) & 1), kTimeoutNs);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) *failed = 1;
      tc_fence_after_sync();
#pragma unroll 1
      for (int c = turn; c < mine; c += 2, ++chunks) {
        if (kLoads) {
          if (c != turn && lane == 0) fetch(c);
          const bool here = mbar_wait(my_loaded, chunks & 1, kTimeoutNs);
          if (!__all_sync(0xffffffffu, here)) ok = false;
          if (!ok) *failed = 1;
        } else {
          if (lane == 0) bulk_wait_read();  // the slot's last stores
          __syncwarp();
        }
#pragma unroll
        for (int g = 0; g < kChunk / 16; ++g) {
          float v[16];
          tmem_ld_32x32b_x16(tmem + (uint32_t(quad * 32) << 16) + uint32_t(acc * kSide + c * kChunk + g * 16), v);
          if (!ok) {
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = __uint_as_float(0x7fc00000u);
          }
          into_slot<KIND>(p, slot, lane, g, v);
          if constexpr (KIND == kFinal) {
            // columns 16 g and on are 32 bytes of each of the boxes that came in; they are 64 bytes of results, which stay in this lane's rows of both
            *box_at(slot, lane, 2 * g) = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            *box_at(slot, lane, 2 * g + 1) = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
            *box_at(slot + kBoxBytes, lane, 2 * g) = make_uint4(__float_as_uint(v[8]), __float_as_uint(v[9]), __float_as_uint(v[10]), __float_as_uint(v[11]));
            *box_at(slot + kBoxBytes, lane, 2 * g + 1) = make_uint4(__float_as_uint(v[12]), __float_as_uint(v[13]), __float_as_uint(v[14]), __float_as_uint(v[15]));
          }
        }
        if constexpr (KIND == kFinal) {
          __syncwarp();
          const int col0 = at.n0 + c * kChunk;
          if (p.result != nullptr) put_results<__nv_bfloat16, true>(p, p.result + int64_t(at.batch) * p.M * p.N, slot, lane, row0, col0);
          else if (p.param_dtype == NANGILA_F32) put_results<float, false>(p, static_cast<float*>(p.param[at.batch]), slot, lane, row0, col0);
          else if (p.param_dtype == NANGILA_BF16) put_results<__nv_bfloat16, false>(p, static_cast<__nv_bfloat16*>(p.param[at.batch]), slot, lane, row0, col0);
          else put_results<__half, false>(p, static_cast<__half*>(p.param[at.batch]), slot, lane, row0, col0);
          // the slot is filled by TMA again: what was read and written here comes first
          fence_async_proxy();
          __syncwarp();
        } else {
          fence_async_proxy();
          __syncwarp();
          if (lane == 0) {
            const int col = at.n0 + c * kChunk;
            tma_store_3d(&maps.out, slot, col, row0, at.batch);
            if (KIND == kUpdate) tma_store_3d(&maps.lo, slot + kBoxBytes, col, row0, at.batch);
            else if (at.m0 != at.n0) tma_store_3d(&maps.mirror, slot + kBoxBytes, row0, col, at.batch);
            bulk_commit();
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_at(acc_empty_at + uint32_t(acc) * 8);
    }
    if (lane == 0) bulk_wait_read();  // the stores have left shared memory; the end of the kernel is what others wait for
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync();  // neither CTA's barriers and tensor memory go while the other may still use them
  if (warp == 1) {
    if (PAIR) tmem_dealloc_pair(tmem, 2 * kSide);
    else tmem_dealloc(tmem, 2 * kSide);
  }
}

// ---- from the gradients to X -------------------------------------------------------------------------------------------------
// Two passes over the gradients, which are small next to the products: the sum of squares, in 64 bits and in an order that the sizes determine,
// then X. With momentum the first pass also advances it: M <- mu M + G, U = G + mu M (Nesterov) or M.
constexpr int kPrepT = 256;
constexpr int kMaxChunks = 1024;
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
    // eight squares in fp32 where they fit into its range, else in 64 bits
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) q = __fmaf_rn(u[k], u[k], q);
    if (q > 1e-28f && q < 1e38f) {
      sum += double(q);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) sum = fma(double(u[k]), double(u[k]), sum);
    }
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
struct Matrix {  // `count` matrices as they lie in memory
  const __half* base;
  int64_t rows, cols, ld, matrix;
};
// copied in boxes of box_inner x box_outer; what lies outside reads as zero and is not written
bool make_map(CUtensorMap* map, const Matrix& m, int count, uint32_t box_inner, uint32_t box_outer, bool swizzle = true) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {cuuint64_t(m.cols), cuuint64_t(m.rows), cuuint64_t(count)};
  const cuuint64_t strides[2] = {cuuint64_t(m.ld) * 2, cuuint64_t(m.matrix) * 2};
  const cuuint32_t box[3] = {box_inner, box_outer, 1}, step[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(m.base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int sm_count() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  return sms[dev];
}
int64_t tiles_of(const Product& p, int side, int count) {
  const int64_t tm = (p.M + side - 1) / side, tn = (p.N + side - 1) / side;
  return (p.lower ? tm * (tm + 1) / 2 : tm * tn) * count;
}

template <int KIND, bool A_MN, bool B_MN, bool PAIR>
int launch_product(const Maps& maps, Product p, int count, cudaStream_t stream) {
  constexpr int kSide = PAIR ? 256 : 128;
  const int64_t total = tiles_of(p, kSide, count);
  if (total > 0x7fffffff) return int(cudaErrorInvalidValue);
  p.tiles_m = (p.M + kSide - 1) / kSide;
  p.total = int(total);
  p.per = int(total / count);
  auto* kernel = orth_product_kernel<KIND, A_MN, B_MN, PAIR>;
  static std::mutex mu;
  static uint64_t opted_in = 0;  // by device
  {
    int dev = 0;
    if (const cudaError_t e = cudaGetDevice(&dev)) return int(e);
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 64 || !((opted_in >> dev) & 1)) {
      if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem)) return int(e);
      if (dev < 64) opted_in |= uint64_t(1) << dev;
    }
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = PAIR ? 2 : 1;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  const int sms = sm_count();
  cfg.gridDim = dim3(unsigned(PAIR ? 2 * std::min(p.total, sms / 2) : std::min(p.total, sms)));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return int(cudaLaunchKernelEx(&cfg, kernel, maps, p));
}
// D of the operands a and b; `in` and `lo` are what the epilogue reads, `out` what it writes.
template <int KIND, bool A_MN, bool B_MN>
int product(const Matrix& a, const Matrix& b, const Matrix* in, const Matrix* lo, const Matrix* out, const Product& p, int count, cudaStream_t stream) {
  Maps maps;
  bool ok = make_map(&maps.a, a, count, 64, A_MN ? 64 : 128) && make_map(&maps.b, b, count, 64, B_MN ? 64 : 128);
  ok = ok && make_map(&maps.in, in != nullptr ? *in : a, count, kChunk, 32) && make_map(&maps.lo, lo != nullptr ? *lo : a, count, kChunk, 32);
  ok = ok && make_map(&maps.out, out != nullptr ? *out : a, count, kChunk, 32) && make_map(&maps.mirror, out != nullptr ? *out : a, count, 32, kChunk, false);
  if (!ok) return int(cudaErrorNotSupported);
  // A tile of a pair takes hardly longer than a small one, which is bound by what L2 delivers to an SM (twice the bytes for each product); only its
  // epilogue is longer. So it is the number of rounds that decides.
  const int sms = sm_count();
  const int64_t small = tiles_of(p, 128, count), large = tiles_of(p, 256, count);
  const double cost_small = double((small + sms - 1) / sms), cost_large = 1.2 * double((large + sms / 2 - 1) / (sms / 2));
  return cost_large <= cost_small ? launch_product<KIND, A_MN, B_MN, true>(maps, p, count, stream) : launch_product<KIND, A_MN, B_MN, false>(maps, p, count, stream);
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
  const Matrix A{gram, l.m, l.m, l.ldm, l.s}, B{poly, l.m, l.m, l.ldm, l.s}, Lo{lo, p->rows, p->cols, l.ld, l.x};
  for (int step = 0; step < p->steps && e == 0; ++step) {
    const float* c = p->coefficients[step];
    const bool last = step == p->steps - 1;
    const Matrix X{hi[step & 1], p->rows, p->cols, l.ld, l.x}, Next{hi[(step & 1) ^ 1], p->rows, p->cols, l.ld, l.x};
    Product q;
    std::memset(&q, 0, sizeof q);
    q.M = q.N = int(l.m);
    q.lower = 1;
    q.K = int(l.n);
    q.alpha = 1.0f / (scale * scale);
    e = tall ? product<kGram, true, true>(X, X, nullptr, nullptr, &A, q, p->count, stream) : product<kGram, false, false>(X, X, nullptr, nullptr, &A, q, p->count, stream);
    if (e != 0) break;
    q.K = int(l.m);
    q.alpha = c[1];
    q.beta = c[2];
    e = product<kPoly, false, false>(A, A, &A, nullptr, &B, q, p->count, stream);
    if (e != 0) break;
    q.lower = 0;
    q.M = p->rows;
    q.N = p->cols;
    q.alpha = c[0];
    if (last) {
      q.unscale = 1.0f / scale;
      q.vector = p->cols % 4 == 0;
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
      e = tall ? product<kFinal, false, false>(X, B, &X, &Lo, nullptr, q, p->count, stream) : product<kFinal, false, true>(B, X, &X, &Lo, nullptr, q, p->count, stream);
    } else {
      e = tall ? product<kUpdate, false, false>(X, B, &X, &Lo, &Next, q, p->count, stream) : product<kUpdate, false, true>(B, X, &X, &Lo, &Next, q, p->count, stream);
    }
  }
  return e;
}

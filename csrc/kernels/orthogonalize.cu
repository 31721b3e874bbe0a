// Updates made orthogonal by Newton-Schulz steps, as the Muon optimiser does, for several matrices of one shape at a time (sm_100a).
//
//   X = U / max(|U|_F, eps), and `steps` times:   A = X X^T,   B = b A + c A^2,   X <- a X + B X
//
// X has m rows and n >= m columns; a matrix that is taller than wide is kept as it lies, and its transpose is what the formulas speak of.
// The three products are one tcgen05 kernel with different operands and epilogues: operands come through TMA (128-byte swizzle, K-major or
// MN-major, so that nothing is transposed in memory), one thread issues the products with the accumulator in tensor memory, four or eight warps
// read it back and write results. Of the symmetric A and A^2 only the tiles that reach the lower triangle are computed; their epilogue writes both halves.
//
// Roundings. The products' operands are rounded to fp16 (11 bits; the values are bounded, so that bf16's range is not needed and its 8 bits
// would cost a factor of eight), the accumulator is fp32. A and B multiply X: their errors, and those of X inside the products, come out as relative
// errors of a few 2^-12 of directions that are large already. The term a X is another matter: it alone carries the small singular values up, by
// a^5 = 485 with the usual coefficients, and what is lost of them in X's rounding grows along. So the state X is kept in two halves, hi + lo / 2048, both fp16
// (22 bits), hi being the operand of the products, and a X is formed from both in fp32.
//
// In the last step nothing grows any more, and what is left is the rounding of B and of X in B X, with B near b + c = -2.7 where the singular values have come near
// one. There the same polynomial is taken as (a + b + c) X + (B - (b + c) I) X, whose second factor is near zero. The result's error against exact
// arithmetic, without its rounding to bf16 (1.7e-3): 768 x 768 noise 1.46e-3 -> 1.20e-3, 300 x 3000 1.77e-3 -> 1.66e-3, 128 x 128 1.76e-3 -> 1.53e-3; a matrix of
// rank 8, where most directions have not come near one, goes from 3.0e-4 to 6.1e-4.
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
#include <set>
#include <type_traits>
#include <utility>

#include "follow.cuh"
#include "nangila_kernels.h"
#include "nangila_model_kernels.h"
#include "ptx_sm100.cuh"
#include "quant.cuh"
#include "raw8.cuh"

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
constexpr int kEpilogueSlots = 8;
constexpr int kEpilogueBytes = kEpilogueSlots * kSlotBytes;
constexpr int kSmem = kStages * kStageBytes + kEpilogueBytes + 1024 + 256;
constexpr uint64_t kTimeoutNs = 10ull * 1000 * 1000 * 1000;
constexpr float kLoScale = 2048.0f;
constexpr int kMaxCluster = 8;

enum Kind { kGram, kPoly, kUpdate, kFinal };

// Warps of the epilogue for each quarter of tensor memory, and slots of each. Two warps with a slot each take turns with a tile's chunks, which ends small tiles
// sooner; where the results go under the next tile's products anyhow, one warp with two slots disturbs those less (update of 4096 x 16384 376 us, for 397; of sixteen
// 2048 x 2048 204 us, for 219), but for the last one, which reads and writes parameters (sixteen 2048 x 2048: 409 us with one warp, 228 with two
// and the parameters fetched ahead).
template <int KIND, bool PAIR>
constexpr int kTurns = PAIR && KIND != kFinal ? 1 : 2;
template <int KIND, bool PAIR>
constexpr int kGemmThreads = 64 + 32 * 4 * kTurns<KIND, PAIR>;  // warp 0: TMA, warp 1: products, the others: epilogue

struct Product {
  int M, N, K;             // D is M x N
  int tiles_m, per, total; // tiles along M; tiles of one matrix, of all
  int lower;               // only tiles that reach the lower triangle
  float alpha, beta;       // gram: D alpha;  poly: alpha A + beta D;  update: alpha X + D
  float shift;             // poly: added on the diagonal
};
// Where the last update goes: result = (alpha X + D) unscale.
struct Target {
  __nv_bfloat16* result;   // packed, one matrix behind the other, or NULL
  int param_dtype, vector; // the parameters' type; runs of four elements can be read and written
  float unscale, decay, rate;
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
__device__ __forceinline__ void put_results(const Product& p, const Target& to_where, T* base, uint8_t* slot, int lane, int row0, int col0) {
  const int x = lane & 15, col = col0 + 4 * x, left = p.N - col;
  if (left <= 0) return;
  // four columns 4 x: group x / 4 of sixteen, its quarter x % 4
  uint8_t* box = slot + ((x & 2) ? kBoxBytes : 0);
  const int j = 2 * (x >> 2) + (x & 1);
#pragma unroll 1
  for (int half = 0; half < 32; half += 16) {
    float v[8][4];
    if (!fresh) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = row0 + half + 2 * i + (lane >> 4);
        if (row >= p.M) continue;
        const T* from = base + int64_t(row) * p.N + col;
        if (to_where.vector) {
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
      for (int k = 0; k < 4; ++k) v[i][k] = fresh ? r[k] : v[i][k] * to_where.decay - to_where.rate * r[k];
      T* to = base + int64_t(row0 + at) * p.N + col;
      if (to_where.vector) {
        store4(to, v[i]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < left) to[k] = dev::Vec16<T>::from_float(v[i][k]);
      }
    }
  }
}

// Sixteen accumulators of a lane's row, columns 16 g to 16 g + 15 of the chunk in the slot, taken into the slot as what goes out. `diagonal`: which of them
// lies on the matrix's diagonal, if one does.
template <int KIND>
__device__ __forceinline__ void into_slot(const Product& p, float unscale, uint8_t* slot, int lane, int g, int diagonal, float (&v)[16]) {
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
        for (int k = 0; k < 8; ++k) w[k] = __fmaf_rn(p.alpha, a[k], __fmaf_rn(p.beta, w[k], 8 * e + k == diagonal ? p.shift : 0.0f));
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
        for (int k = 0; k < 8; ++k) v[8 * e + k] = w[k] * unscale;
      }
    }
  }
}

// What a CTA's roles share, in shared memory.
struct Shared {
  uint8_t *stages, *slots;
  uint64_t *full, *empty;          // [kStages]
  uint64_t *acc_full, *acc_empty;  // [2]
  uint64_t *loaded;                // [kEpilogueSlots]
  uint64_t *drained;
  uint32_t* tmem_slot;
  volatile uint32_t* failed;       // a wait has run out
};
__device__ __forceinline__ Shared shared_parts(uint8_t* raw) {
  Shared s;
  s.stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  s.slots = s.stages + kStages * kStageBytes;
  s.full = reinterpret_cast<uint64_t*>(s.slots + kEpilogueBytes);
  s.empty = s.full + kStages;
  s.acc_full = s.empty + kStages;
  s.acc_empty = s.acc_full + 2;
  s.loaded = s.acc_empty + 2;
  s.drained = s.loaded + kEpilogueSlots;
  s.tmem_slot = reinterpret_cast<uint32_t*>(s.drained + 1);
  s.failed = s.tmem_slot + 1;
  return s;
}
template <int KIND, bool PAIR>
__device__ __forceinline__ void init_barriers(const Shared& s) {
  for (int i = 0; i < kStages; ++i) {
    mbar_init(&s.full[i], 1);
    mbar_init(&s.empty[i], 1);
  }
  for (int i = 0; i < 2; ++i) {
    mbar_init(&s.acc_full[i], 1);
    mbar_init(&s.acc_empty[i], 4 * kTurns<KIND, PAIR> * (PAIR ? 2 : 1));
  }
  for (int i = 0; i < kEpilogueSlots; ++i) mbar_init(&s.loaded[i], 1);
  mbar_init(s.drained, 1);
  *s.failed = 0;
  fence_barrier_init();
}

// TMA of a tile's slabs, `i` of which have gone before: both CTAs of a pair, each its own halves; the bytes are counted where the products are issued.
// False when a wait has run out.
template <bool PAIR>
__device__ __forceinline__ bool load_tile(const Shared& s, const CUtensorMap* a_map, const CUtensorMap* b_map, bool a_mn, bool b_mn, const TileAt& at, uint32_t rank, int slabs, int& i, int slab0 = 0) {
  const int row = at.m0 + int(rank) * kTileM, col = at.n0 + int(rank) * 128;
  for (int k = 0; k < slabs; ++k, ++i) {
    const int st = i % kStages;
    if (i >= kStages && !mbar_wait(&s.empty[st], uint32_t((i / kStages - 1) & 1), kTimeoutNs)) {
      *s.failed = 1;
      return false;
    }
    uint8_t* a = s.stages + st * kStageBytes;
    uint8_t* b = a + kOperandBytes;
    const int k0 = (slab0 + k) * kSlabK;
    if (rank == 0) mbar_arrive_expect_tx(&s.full[st], kStageBytes * (PAIR ? 2 : 1));
    const uint32_t bar = PAIR ? rank0_address(&s.full[st]) : smem_u32(&s.full[st]);
    if (a_mn) {
      tma_operand<PAIR>(a, a_map, row, k0, at.batch, bar);
      tma_operand<PAIR>(a + 8192, a_map, row + 64, k0, at.batch, bar);
    } else {
      tma_operand<PAIR>(a, a_map, k0, row, at.batch, bar);
    }
    if (b_mn) {
      tma_operand<PAIR>(b, b_map, col, k0, at.batch, bar);
      tma_operand<PAIR>(b + 8192, b_map, col + 64, k0, at.batch, bar);
    } else {
      tma_operand<PAIR>(b, b_map, k0, col, at.batch, bar);
    }
  }
  return true;
}
// The copies that are still under way when the loads end: all have arrived when the products that read them are done; if somebody has given up, as
// much as can be waited for (the bytes of a pair are counted by rank 0, the stages of rank 1 are given back by its products).
__device__ __forceinline__ void drain_loads(const Shared& s, uint32_t rank, int i) {
  for (int j = max(0, i - kStages); j < i; ++j) {
    if (*s.failed == 0 || rank != 0) mbar_wait(&s.empty[j % kStages], uint32_t((j / kStages) & 1), kTimeoutNs);
    else mbar_wait(&s.full[j % kStages], uint32_t((j / kStages) & 1), kTimeoutNs);
  }
}
// The products of a tile, the n-th, into its accumulator. False when a wait has run out.
template <bool PAIR>
__device__ __forceinline__ bool multiply_tile(const Shared& s, uint32_t tmem, bool a_mn, bool b_mn, int slabs, int n, int& i) {
  constexpr int kSide = PAIR ? 256 : 128;
  const uint32_t idesc = (1u << 4) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) | (uint32_t(kSide >> 3) << 17) | (uint32_t(kSide >> 4) << 24);
  const int acc = n & 1;
  if (n >= 2 && !mbar_wait(&s.acc_empty[acc], uint32_t((n / 2 - 1) & 1), kTimeoutNs)) return false;
  tc_fence_after_sync();
  const uint32_t d = tmem + uint32_t(acc * kSide);
  for (int k = 0; k < slabs; ++k, ++i) {
    const int st = i % kStages;
    if (!mbar_wait(&s.full[st], uint32_t((i / kStages) & 1), kTimeoutNs)) return false;
    tc_fence_after_sync();
    const uint32_t a = smem_u32(s.stages + st * kStageBytes), b = a + kOperandBytes;
#pragma unroll
    for (int kk = 0; kk < kSlabK / 16; ++kk) {
      // K-major: 16 elements along K are 32 bytes of a swizzle row; MN-major: 16 K-rows are two groups of eight rows of 128 bytes
      const uint64_t ad = a_mn ? make_smem_desc(a + kk * 2048, 8192, 1024) : make_smem_desc(a + kk * 32, 16, 1024);
      const uint64_t bd = b_mn ? make_smem_desc(b + kk * 2048, 8192, 1024) : make_smem_desc(b + kk * 32, 16, 1024);
      if (PAIR) umma_f16_pair(d, ad, bd, idesc, (k > 0 || kk > 0) ? 1u : 0u);
      else umma_f16(d, ad, bd, idesc, (k > 0 || kk > 0) ? 1u : 0u);
    }
    if (PAIR) umma_commit_pair(&s.empty[st]);
    else umma_commit(&s.empty[st]);
  }
  if (PAIR) umma_commit_pair(&s.acc_full[acc]);
  else umma_commit(&s.acc_full[acc]);
  return true;
}
template <bool PAIR>
__device__ __forceinline__ void drain_products(const Shared& s) {
  *s.failed = 1;
  if (PAIR) umma_commit_pair(s.drained);
  else umma_commit(s.drained);
  mbar_wait(s.drained, 0, kTimeoutNs);
}
// The n-th tile's accumulator taken to where it belongs, by one of the epilogue's warps; `chunks`: how many it has done so far.
template <int KIND, bool PAIR>
__device__ __forceinline__ void finish_tile(const Shared& s, uint32_t tmem, const Product& p, const Target& target, const CUtensorMap* in, const CUtensorMap* lo, const CUtensorMap* out,
                                            const CUtensorMap* mirror, const TileAt& at, uint32_t rank, int n, uint32_t& chunks) {
  constexpr int kSide = PAIR ? 256 : 128;
  constexpr int kChunks = kSide / kChunk;
  constexpr bool kLoads = KIND != kGram;
  constexpr uint32_t kLoadBytes = KIND == kPoly ? kBoxBytes : kSlotBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = warp & 3;  // the lanes of tensor memory that this warp may read
  const int turn = (warp - 2) >> 2;
  constexpr int kWarps = kTurns<KIND, PAIR>, kSlots = 2 / kWarps;
  const int acc = n & 1;
  const int row0 = at.m0 + int(rank) * kTileM + quad * 32;
  const int mine = row0 < p.M ? min(kChunks, (p.N - at.n0 + kChunk - 1) / kChunk) : 0;
  auto slot_of = [&](uint32_t turn_no) { return s.slots + ((warp - 2) * kSlots + turn_no % kSlots) * kSlotBytes; };
  auto loaded_of = [&](uint32_t turn_no) { return s.loaded + (warp - 2) * kSlots + turn_no % kSlots; };
  auto fetch = [&](int c, uint32_t turn_no) {  // lane 0: chunk c into the slot whose turn it is, once nothing goes out any more
    uint8_t* to = slot_of(turn_no);
    uint64_t* bar = loaded_of(turn_no);
    bulk_wait_read();
    mbar_arrive_expect_tx(bar, kLoadBytes);
    tma_load_3d(to, in, at.n0 + c * kChunk, row0, at.batch, bar);
    if (KIND != kPoly) tma_load_3d(to + kBoxBytes, lo, at.n0 + c * kChunk, row0, at.batch, bar);
  };
  if (kLoads && turn < mine && lane == 0) fetch(turn, chunks);
  if constexpr (KIND == kFinal) {
    // the parameters that this tile is going to change: on their way from memory while its products are made
    if (target.result == nullptr && row0 + lane < p.M) {
      const int size = target.param_dtype == NANGILA_F32 ? 4 : 2;
      const char* at_row = static_cast<const char*>(target.param[at.batch]) + (int64_t(row0 + lane) * p.N + at.n0) * size;
      for (int c = turn; c < mine; c += kWarps)
        for (int x = c * kChunk; x < min((c + 1) * kChunk, p.N - at.n0); x += 128 / size) asm volatile("prefetch.global.L2 [%0];" ::"l"(at_row + int64_t(x) * size));
    }
  }
  bool ok = *s.failed == 0 && mbar_wait(&s.acc_full[acc], uint32_t((n / 2) & 1), kTimeoutNs);
  ok = __all_sync(0xffffffffu, ok);
  if (!ok) *s.failed = 1;
  tc_fence_after_sync();
#pragma unroll 1
  for (int c = turn; c < mine; c += kWarps, ++chunks) {
    uint8_t* slot = slot_of(chunks);
    if (kLoads) {
      if (kSlots > 1) {
        if (c + kWarps < mine && lane == 0) fetch(c + kWarps, chunks + 1);
      } else {
        if (c != turn && lane == 0) fetch(c, chunks);
      }
      const bool here = mbar_wait(loaded_of(chunks), (chunks / kSlots) & 1, kTimeoutNs);
      if (!__all_sync(0xffffffffu, here)) ok = false;
      if (!ok) *s.failed = 1;
    } else {
      if (lane == 0) {  // the slot's last stores
        if (kSlots > 1) bulk_wait_read_but_one();
        else bulk_wait_read();
      }
      __syncwarp();
    }
    // (In small tiles a loop, not four copies of it: the only tile of a launch is bound by fetching this code. 256 x 256 in all: 97 us unrolled, 91 so.)
    constexpr int kCopies = PAIR ? kChunk / 16 : 1;
#pragma unroll kCopies
    for (int g = 0; g < kChunk / 16; ++g) {
      float v[16];
      tmem_ld_32x32b_x16(tmem + (uint32_t(quad * 32) << 16) + uint32_t(acc * kSide + c * kChunk + g * 16), v);
      if (!ok) {
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = __uint_as_float(0x7fc00000u);
      }
      into_slot<KIND>(p, target.unscale, slot, lane, g, row0 + lane - (at.n0 + c * kChunk + g * 16), v);
      if constexpr (KIND == kFinal) {
        // columns 16 g and on are 32 bytes of each of the boxes that came in; they are 64 bytes of results, which stay in this lane's rows of both
        *box_at(slot, lane, 2 * g) = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        *box_at(slot, lane, 2 * g + 1) = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
        *box_at(slot + kBoxBytes, lane, 2 * g) = make_uint4(__float_as_uint(v[8]), __float_as_uint(v[9]), __float_as_uint(v[10]), __float_as_uint(v[11]));
        *box_at(slot + kBoxBytes, lane, 2 * g + 1) = make_uint4(__float_as_uint(v[12]), __float_as_uint(v[13]), __float_as_uint(v[14]), __float_as_uint(v[15]));
      }
    }
    const int col0 = at.n0 + c * kChunk;
    if constexpr (KIND == kFinal) {
      // the slot is filled by TMA again: what was written here comes first (a fence after the stores to memory below would wait for them)
      fence_async_proxy();
      __syncwarp();
      if (target.result != nullptr) put_results<__nv_bfloat16, true>(p, target, target.result + int64_t(at.batch) * p.M * p.N, slot, lane, row0, col0);
      else if (target.param_dtype == NANGILA_F32) put_results<float, false>(p, target, static_cast<float*>(target.param[at.batch]), slot, lane, row0, col0);
      else if (target.param_dtype == NANGILA_BF16) put_results<__nv_bfloat16, false>(p, target, static_cast<__nv_bfloat16*>(target.param[at.batch]), slot, lane, row0, col0);
      else put_results<__half, false>(p, target, static_cast<__half*>(target.param[at.batch]), slot, lane, row0, col0);
      __syncwarp();  // all have read the slot
    } else {
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) {
        tma_store_3d(out, slot, col0, row0, at.batch);
        if (KIND == kUpdate) tma_store_3d(lo, slot + kBoxBytes, col0, row0, at.batch);
        else if (at.m0 != at.n0) tma_store_3d(mirror, slot + kBoxBytes, row0, col0, at.batch);
        bulk_commit();
      }
    }
  }
  tc_fence_before_sync();
  __syncwarp();
  if (lane == 0) mbar_arrive_at((PAIR ? rank0_address(&s.acc_empty[0]) : smem_u32(&s.acc_empty[0])) + uint32_t(acc) * 8);
}

// The sum of a few squares: in fp32 where they fit into its range, else in 64 bits.
template <int N>
__device__ __forceinline__ double square_sum(const float (&u)[N]) {
  float q = 0.0f;
#pragma unroll
  for (int k = 0; k < N; ++k) q = __fmaf_rn(u[k], u[k], q);
  if (q > 1e-28f && q < 1e38f) return double(q);
  double d = 0.0;
#pragma unroll
  for (int k = 0; k < N; ++k) d = fma(double(u[k]), double(u[k]), d);
  return d;
}

// D = A B for square tiles of all matrices, walked over by CTAs that stay (PAIR: pairs of CTAs that share the tensor cores' work on 256 x 256, each
// with its 128 rows of A, half of B's columns, and 128 rows of the result; else one CTA and 128 x 128). A_MN / B_MN: the operand lies with its rows
// (columns of B) adjacent in memory, not its K. The accumulators of two tiles share tensor memory: the epilogue of one runs under the
// products of the next, and what it needs of X or A is on its way before they end. Each of its warps has one or two slots of shared memory of its own,
// filled and emptied by TMA, and meets no other warp.
// A wait that runs out makes every result of this CTA from there on not a number.
// Bound: large ones by the tensor cores, and by power in a long run (update of 4096 x 16384: 376 us, 1.46 PFLOP/s on its own; five steps of it 4.0 ms at the 1000 W limit, where
// a library's fp16 product of this shape runs at 1.27). Alone, a CTA's 128 x 128 tile is bound by the 64 bytes a cycle that L2 delivers to an SM (32 KB a slab,
// 0.27 us); with 128 x 256 tiles of one CTA the update took 469 us. Small ones by the way from launch to launch: 768 x 768 about 8 us for each of 15 products, of which
// 3.2 are the 12 slabs, 1.4 the first load, 1.2 the results, 1.9 the end of a kernel until the next one sees its data.
template <int KIND, bool A_MN, bool B_MN, bool PAIR>
__global__ void __launch_bounds__(kGemmThreads<KIND, PAIR>, 1) orth_product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Product p, const __grid_constant__ Target target) {
  constexpr int kSide = PAIR ? 256 : 128;
  extern __shared__ uint8_t smem_raw[];
  const Shared s = shared_parts(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slabs = (p.K + kSlabK - 1) / kSlabK;
  const uint32_t rank = PAIR ? cluster_rank() : 0u;   // 0: the CTA that issues the pair's products
  const int first = PAIR ? blockIdx.x / 2 : blockIdx.x, step = PAIR ? gridDim.x / 2 : gridDim.x;

  if (threadIdx.x == 0) {
    init_barriers<KIND, PAIR>(s);
    prefetch_tensormap(&maps.a);
    prefetch_tensormap(&maps.b);
  }
  if (threadIdx.x == 64) {
    if (KIND != kGram) prefetch_tensormap(&maps.in);
    if (KIND == kUpdate || KIND == kFinal) prefetch_tensormap(&maps.lo);
    if (KIND != kFinal) prefetch_tensormap(&maps.out);
    if (KIND == kGram || KIND == kPoly) prefetch_tensormap(&maps.mirror);
  }
  if (warp == 1) {
    if (PAIR) tmem_alloc_pair(s.tmem_slot, 2 * kSide);
    else tmem_alloc(s.tmem_slot, 2 * kSide);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync();  // the other CTA's barriers exist from here on
  tc_fence_after_sync();
  const uint32_t tmem = *s.tmem_slot;
  TileAt at = tile_at<kSide>(p, first);  // (before the wait: every role needs it first of all)
  may_follow();
  follow();

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      for (int tile = first; tile < p.total; tile += step) {
        if (tile != first) at = tile_at<kSide>(p, tile);
        if (!load_tile<PAIR>(s, &maps.a, &maps.b, A_MN, B_MN, at, rank, slabs, i)) break;
      }
      drain_loads(s, rank, i);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int i = 0, n = 0;
      bool ok = true;
      for (int tile = first; tile < p.total && ok; tile += step, ++n) ok = multiply_tile<PAIR>(s, tmem, A_MN, B_MN, slabs, n, i);
      if (!ok) drain_products<PAIR>(s);
    }
  } else {
    int n = 0;
    uint32_t chunks = 0;
    for (int tile = first; tile < p.total; tile += step, ++n) {
      if (tile != first) at = tile_at<kSide>(p, tile);
      finish_tile<KIND, PAIR>(s, tmem, p, target, &maps.in, &maps.lo, &maps.out, &maps.mirror, at, rank, n, chunks);
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

// The Gram matrix where few tiles share a long K: a cluster takes a tile, each CTA a part of K and, in the end, 128 / S columns of the result. The parts
// meet through shared memory, in the order of the ranks. Three of 2051 x 517 (45 tiles, 33 slabs, two CTAs a tile): five steps 243 -> 219 us.
template <bool MN>
__global__ void __launch_bounds__(kGemmThreads<kGram, false>, 1) orth_gram_split_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Product p, __half* __restrict__ out, int64_t ld, int64_t matrix) {
  extern __shared__ uint8_t smem_raw[];
  const Shared s = shared_parts(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int slabs = (p.K + kSlabK - 1) / kSlabK;
  const int slab0 = int(rank) * slabs / int(ranks), mine = (int(rank) + 1) * slabs / int(ranks) - slab0;  // one at least
  const TileAt at = tile_at<128>(p, int(blockIdx.x / ranks));
  const int width = 128 / int(ranks), pitch = width * 4;   // columns of a CTA; bytes of a row of theirs, fp32
  auto part_at = [&](uint32_t from, int row, int j) {      // sixteen bytes `j` of what rank `from` sends, in the slots of the CTA whose columns they are
    return s.slots + from * uint32_t(128 * pitch) + row * pitch + ((j ^ (row & (pitch / 16 - 1))) << 4);
  };

  if (threadIdx.x == 0) {
    init_barriers<kGram, false>(s);
    prefetch_tensormap(&maps.a);
    prefetch_tensormap(&maps.b);
  }
  if (warp == 1) tmem_alloc(s.tmem_slot, 256);
  tc_fence_before_sync();
  cluster_sync();
  tc_fence_after_sync();
  const uint32_t tmem = *s.tmem_slot;
  may_follow();
  follow();

  const int quad = warp & 3, turn = (warp - 2) >> 2, row = quad * 32 + lane;
  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      load_tile<false>(s, &maps.a, &maps.b, MN, MN, at, 0, mine, i, slab0);
      drain_loads(s, 0, i);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int i = 0;
      if (!multiply_tile<false>(s, tmem, MN, MN, mine, 0, i)) drain_products<false>(s);
    }
  } else {
    bool ok = mbar_wait(&s.acc_full[0], 0, kTimeoutNs);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) *s.failed = 1;
    tc_fence_after_sync();
    // sixteen columns at a time: to whom they belong, the groups shared out between the two warps of a quarter
    for (int g = turn; g < 8; g += 2) {
      const uint32_t owner = uint32_t(g * 16 / width);
      if (owner == rank) continue;
      float v[16];
      tmem_ld_32x32b_x16(tmem + (uint32_t(quad * 32) << 16) + uint32_t(g * 16), v);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float4 f = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        if (!ok) f.x = f.y = f.z = f.w = __uint_as_float(0x7fc00000u);
        store_cluster(cluster_address(part_at(rank, row, (g * 16 % width) / 4 + q), owner), *reinterpret_cast<const uint4*>(&f));
      }
    }
  }
  __syncwarp();
  cluster_sync();
  if (warp >= 2) {
    const bool ok = *s.failed == 0;
    // this CTA's columns, eight at a time
    for (int c = turn * 8; c < width; c += 16) {
      float v[8], own[8];
      tmem_ld_32x32b_x8(tmem + (uint32_t(quad * 32) << 16) + uint32_t(int(rank) * width + c), own);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.0f;
      for (uint32_t from = 0; from < ranks; ++from) {
        float4 x, y;
        if (from == rank) {
          x = make_float4(own[0], own[1], own[2], own[3]);
          y = make_float4(own[4], own[5], own[6], own[7]);
        } else {
          x = *reinterpret_cast<const float4*>(part_at(from, row, c / 4));
          y = *reinterpret_cast<const float4*>(part_at(from, row, c / 4 + 1));
        }
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w; v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = ok ? v[k] * p.alpha : __uint_as_float(0x7fc00000u);
      const int r = at.m0 + row, col = at.n0 + int(rank) * width + c;
      if (r < p.M && col < p.N) {  // rows of `out` are padded to eight
        __half* to = out + at.batch * matrix;
        *reinterpret_cast<uint4*>(to + int64_t(r) * ld + col) = pack8(v);
        if (at.m0 != at.n0) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (col + k < p.N) to[int64_t(col + k) * ld + r] = __float2half_rn(v[k]);
        }
      }
      __syncwarp();
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 256);
}

// ---- from the gradients to X -------------------------------------------------------------------------------------------------
// Two passes over the gradients, which are small next to the products (16 of 2048 x 2048, momentum and all: 98 us each, 6.8 TB/s): the sum of squares, in 64 bits and in an order that the sizes determine,
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
  int cols, chunks, nesterov, vector, flat; // vector: runs of eight that X has too; flat: of the gradient alone
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
template <typename T, bool MOM>
__global__ void __launch_bounds__(kPrepT) orth_norm_kernel(const __grid_constant__ Prep p) {
  __shared__ double s[kPrepT / 32];
  const T* g = static_cast<const T*>(p.grad[blockIdx.y]);
  float* m = p.momentum[blockIdx.y];
  const int64_t stride = int64_t(gridDim.x) * kPrepT, first = int64_t(blockIdx.x) * kPrepT + threadIdx.x;
  double sum = 0.0;
  may_follow();
  const int64_t runs = p.flat ? p.numel / 8 : 0;
  constexpr int kAhead = MOM ? 1 : 4;  // runs of eight on their way (with momentum, 16 of 2048 x 2048: one 98 us, four 121: fewer threads fit)
  for (int64_t i0 = first; i0 < runs; i0 += kAhead * stride) {
    dev::Raw8<T> raw[kAhead];
    dev::Raw8<float> old[MOM ? kAhead : 1];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = i0 + k * stride;
      if (i >= runs) break;
      dev::fetch(g + i * 8, raw[k]);
      if constexpr (MOM) dev::fetch(m + i * 8, old[k]);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = i0 + k * stride;
      if (i >= runs) break;
      float u[8];
      dev::unpack(raw[k], u);
      if constexpr (MOM) {
        float v[8];
        dev::unpack(old[k], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] = __fmaf_rn(p.mu, v[j], u[j]);
          u[j] = p.nesterov ? __fmaf_rn(p.mu, v[j], u[j]) : v[j];
        }
        dev::pack(v, old[k]);
        dev::put(m + i * 8, old[k]);
      }
      sum += square_sum(u);
    }
  }
  for (int64_t i = runs * 8 + first; i < p.numel; i += stride) {
    float u = dev::Vec16<T>::to_float(g[i]);
    if (MOM) {
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
  } else {  // a warp takes a row, 128 columns at a time
    const int lane = threadIdx.x & 31;
    const int64_t rows = p.numel / p.cols;
    for (int64_t row = (int64_t(blockIdx.x) * kPrepT + threadIdx.x) >> 5; row < rows; row += stride >> 5) {
      for (int c0 = lane; c0 < p.cols; c0 += 128) {
        float u[4], v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (c0 + 32 * k >= p.cols) break;
          const int64_t i = row * p.cols + c0 + 32 * k;
          u[k] = dev::Vec16<T>::to_float(g[i]);
          if (m != nullptr) v[k] = m[i];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (c0 + 32 * k >= p.cols) break;
          if (m != nullptr) u[k] = p.nesterov ? __fmaf_rn(p.mu, v[k], u[k]) : v[k];
          u[k] *= f;
          const int64_t at = row * p.ld + c0 + 32 * k;
          const __half h = __float2half_rn(u[k]);
          hi[at] = h;
          lo[at] = __float2half_rn((u[k] - __half2float(h)) * kLoScale);
        }
      }
    }
  }
}

// ---- matrices with a side of at most 128 ---------------------------------------------------------------------------------------------------
// Such a matrix stays on the SMs from the gradient to the parameter, in one launch: a CTA keeps up to 384 of its rows (of the longer side) in
// fp32 in tensor memory, and rounded to fp16 in shared memory as the products' operand; longer ones are shared out over a cluster, whose
// CTAs add up their parts of the Gram matrix through one another's shared memory, in the order of their ranks. Every product is a few instructions of
// 128 x 128, so what bounds this is the way from one to the next: two thirds of a step are waits for a product and the pass over its results.
// 128 x 128: 25 us in all, 2.6 a step; 352 x 128, 24 of them: 39 us (product by product 117); 1024 x 128 in a cluster of four: 52 us (95).
//   D = X^T X (n long, from X by rows of n: MN-major),  A = D;   D = A A,  B = b A + c D;   X <- a X + X B, accumulated onto a X in tensor memory.
constexpr int kSmallT = 256;
constexpr int kRuns = 8;                         // of elements that a thread has on their way, to and from memory
constexpr int kBlocks = 3;                       // of 128 rows in a CTA
constexpr int kBlockBytes = 32768;               // 128 x 128 in fp16, two swizzled halves of 64 columns
constexpr int kHalfBytes = 16384;
constexpr int kSmallSmem = (kBlocks + 2) * kBlockBytes + 65536 + 1024 + 256;
struct Small {
  const void* grad[NANGILA_ORTH_MAX_COUNT];
  float* momentum[NANGILA_ORTH_MAX_COUNT];
  float coefficients[NANGILA_ORTH_MAX_STEPS][3];
  int steps, m, n, nesterov, blocks, per; // blocks of 128 along n, of a CTA
  int vector, vector_out; // runs of four elements can be read, and written
  float mu, eps, scale, shift;
};
// Four fp32 of row r in the staging area, columns 4 c to 4 c + 3: neighbouring rows, and every fourth, in different banks.
__device__ __forceinline__ float4* stage_at(uint8_t* stage, int r, int c) { return reinterpret_cast<float4*>(stage + r * 512 + ((c ^ ((r ^ (r >> 2)) & 31)) << 4)); }
__device__ __forceinline__ float* stage_one(uint8_t* stage, int r, int i) { return reinterpret_cast<float*>(stage_at(stage, r, i >> 2)) + (i & 3); }
__device__ __forceinline__ void products_128(uint32_t d, uint32_t a, uint32_t b, bool mn, uint32_t first_accumulates) {
  const uint32_t idesc = (1u << 4) | (uint32_t(mn) << 15) | (uint32_t(mn) << 16) | (uint32_t(128 >> 3) << 17) | (uint32_t(128 >> 4) << 24);
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) {
    const uint32_t off = mn ? kk * 2048 : (kk >> 2) * kHalfBytes + (kk & 3) * 32;
    const uint64_t ad = make_smem_desc(a + off, mn ? kHalfBytes : 16, 1024), bd = make_smem_desc(b + off, mn ? kHalfBytes : 16, 1024);
    umma_f16(d, ad, bd, idesc, kk > 0 ? 1u : first_accumulates);
  }
}
template <typename T, bool TALL>
__global__ void __launch_bounds__(kSmallT, 1) orth_small_kernel(const __grid_constant__ Small p, const __grid_constant__ Target target) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* hi = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* a_mat = hi + kBlocks * kBlockBytes;
  uint8_t* b_mat = a_mat + kBlockBytes;
  uint8_t* stage = b_mat + kBlockBytes;
  uint64_t* done = reinterpret_cast<uint64_t*>(stage + 65536);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile uint32_t* failed = tmem_slot + 1;
  double* sums = reinterpret_cast<double*>(done + 2);            // [kMaxCluster], then a warp's each
  double* warp_sums = sums + kMaxCluster;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = warp & 3, half = warp >> 2;                   // of tensor memory's lanes; of 128 columns
  const int row = quad * 32 + lane;                              // this thread's, wherever results are passed over
  const uint32_t lanes = uint32_t(quad * 32) << 16;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int batch = int(blockIdx.x / ranks);
  const int block0 = int(rank) * p.per, mine = max(0, min(p.per, p.blocks - block0));

  if (threadIdx.x == 0) {
    mbar_init(done, 1);
    *failed = 0;
    fence_barrier_init();
  }
  if (warp == 0) tmem_alloc(tmem_slot, 512);
  tc_fence_before_sync();
  cluster_sync();  // all CTAs of the cluster have started
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  uint32_t phase = 0;
  // All wait for the products that thread 0 has just issued.
  auto finish = [&]() {
    if (!mbar_wait(done, phase & 1, kTimeoutNs)) *failed = 1;
    ++phase;
    __syncwarp();
    tc_fence_after_sync();
  };
  // What the threads have written to shared and tensor memory is there for thread 0's products.
  auto ready = [&]() {
    fence_async_proxy();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
  };
  // A block's elements are passed over in runs of V = 4, neighbours in memory, or one by one; the threads take turns with the runs, kRuns of a thread
  // being a round. With the longer side outermost (TALL) a block is one stretch of memory; else a thread keeps its rows and goes down the columns.
  // All of this is a chain of waits in a kernel that runs once, so there are no divisions in it and no branches around a run.
  struct Walk {
    int r, i;  // row (along n) and column of a thread's run in a block
  };
  auto first_of = [&](auto run) {
    constexpr int V = decltype(run)::value;
    const int e = int(threadIdx.x) * V;
    if (TALL) return Walk{e / p.m, e % p.m};
    return Walk{e & 127, e >> 7};
  };
  auto advance = [&](auto run, Walk& w, int dr, int di) {  // dr, di: kSmallT runs further on
    constexpr int V = decltype(run)::value;
    if (TALL) {
      w.i += di;
      w.r += dr + (w.i >= p.m ? 1 : 0);
      w.i -= w.i >= p.m ? p.m : 0;
    } else {
      w.i += kSmallT * V / 128;
    }
  };
  auto runs_of = [&](auto run, int b, const Walk& first) {  // that a thread has in block b
    constexpr int V = decltype(run)::value;
    const int rows = min(128, p.n - (block0 + b) * 128);
    if (TALL) return max(0, (rows * p.m / V - int(threadIdx.x) + kSmallT - 1) / kSmallT);
    return first.r < rows ? max(0, (p.m - first.i + 2 * V - 1) / (2 * V)) : 0;
  };
  auto start_of = [&](auto run, int b, const Walk& first) {  // where the first of them lies
    constexpr int V = decltype(run)::value;
    const int base = (block0 + b) * 128;
    return TALL ? int64_t(base) * p.m + int64_t(threadIdx.x) * V : int64_t(first.i) * p.n + base + first.r;
  };
  auto step_of = [&](auto run) {
    constexpr int V = decltype(run)::value;
    return TALL ? int64_t(kSmallT * V) : int64_t(2 * V) * p.n;
  };

  // ---- the gradient, with its momentum: into tensor memory as it is, and its norm. A round is on its way while the one before it is worked on. ----
  const T* g = static_cast<const T*>(p.grad[batch]);
  float* mom = p.momentum[batch];
  double sum = 0.0;
  auto take = [&](auto run) {
    constexpr int V = decltype(run)::value;
    const int last = (128 * p.m / V + kSmallT - 1) / kSmallT;  // runs of a thread in a whole block
    const int64_t step = step_of(run);
    const Walk first = first_of(run);
    const int dr = TALL ? kSmallT * V / p.m : 0, di = TALL ? kSmallT * V - dr * p.m : 0;
    float u[kRuns][V], v[kRuns][V], next_u[kRuns][V], next_v[kRuns][V];
    auto fetch = [&](int b, int k0) {
      const int runs = runs_of(run, b, first);
      const int64_t at = start_of(run, b, first) + k0 * step;
#pragma unroll
      for (int k = 0; k < kRuns; ++k) {
        if (k0 + k < runs) {
          if constexpr (V == 4) load4<T>(g + at + k * step, next_u[k]);
          else next_u[k][0] = dev::Vec16<T>::to_float(g[at + k * step]);
        }
      }
      if (mom == nullptr) return;
#pragma unroll
      for (int k = 0; k < kRuns; ++k) {
        if (k0 + k < runs) {
          if constexpr (V == 4) load4<float>(mom + at + k * step, next_v[k]);
          else next_v[k][0] = mom[at + k * step];
        }
      }
    };
    if (mine > 0) fetch(0, 0);
    for (int b = 0; b < mine; ++b) {
      const int runs = runs_of(run, b, first);
      const int64_t start = start_of(run, b, first);
      Walk w = first;
      if (p.m < 128 || (block0 + b + 1) * 128 > p.n) {  // what lies outside of the matrix
        for (int c = threadIdx.x; c < 128 * 32; c += kSmallT) *stage_at(stage, c >> 5, c & 31) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        __syncthreads();
      }
      for (int k0 = 0; k0 < last; k0 += kRuns) {
#pragma unroll
        for (int k = 0; k < kRuns; ++k)
#pragma unroll
          for (int x = 0; x < V; ++x) {
            u[k][x] = k0 + k < runs ? next_u[k][x] : 0.0f;
            v[k][x] = next_v[k][x];
          }
        if (k0 + kRuns < last) fetch(b, k0 + kRuns);
        else if (b + 1 < mine) fetch(b + 1, 0);
        if (mom != nullptr) {
#pragma unroll
          for (int k = 0; k < kRuns; ++k) {
#pragma unroll
            for (int x = 0; x < V; ++x) {
              v[k][x] = __fmaf_rn(p.mu, v[k][x], u[k][x]);
              u[k][x] = k0 + k >= runs ? 0.0f : p.nesterov ? __fmaf_rn(p.mu, v[k][x], u[k][x]) : v[k][x];
            }
            if (k0 + k < runs) {
              if constexpr (V == 4) store4(mom + start + (k0 + k) * step, v[k]);
              else mom[start + (k0 + k) * step] = v[k][0];
            }
          }
        }
        float squares = 0.0f;
#pragma unroll
        for (int k = 0; k < kRuns; ++k) {
          if (k0 + k < runs) {
            if constexpr (V == 4 && TALL) {
              *stage_at(stage, w.r, w.i >> 2) = make_float4(u[k][0], u[k][1], u[k][2], u[k][3]);
            } else {
#pragma unroll
              for (int x = 0; x < V; ++x) *stage_one(stage, w.r + x, w.i) = u[k][x];
            }
          }
          advance(run, w, dr, di);
#pragma unroll
          for (int x = 0; x < V; ++x) squares = __fmaf_rn(u[k][x], u[k][x], squares);
        }
        if (squares > 1e-28f && squares < 1e38f) {
          sum += double(squares);
        } else {  // where fp32's range does not hold them
#pragma unroll
          for (int k = 0; k < kRuns; ++k)
#pragma unroll
            for (int x = 0; x < V; ++x) sum = fma(double(u[k][x]), double(u[k][x]), sum);
        }
      }
      __syncthreads();
#pragma unroll 1
      for (int c = 0; c < 64; c += 16) {
        float f16[16];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float4 f = *stage_at(stage, row, (half * 64 + c) / 4 + x);
          f16[4 * x] = f.x; f16[4 * x + 1] = f.y; f16[4 * x + 2] = f.z; f16[4 * x + 3] = f.w;
        }
        tmem_st_32x32b_x16(tmem + lanes + uint32_t(128 * (1 + b) + half * 64 + c), f16);
      }
      __syncthreads();
    }
  };
  if (p.vector) take(std::integral_constant<int, 4>{});
  else take(std::integral_constant<int, 1>{});
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) warp_sums[warp] = sum;
  __syncthreads();
  if (threadIdx.x < ranks) {
    sum = 0.0;
    for (int i = 0; i < kSmallT / 32; ++i) sum += warp_sums[i];
    store_cluster(cluster_address(sums + rank, threadIdx.x), sum);  // to every CTA of the cluster
  }
  cluster_sync();
  sum = 0.0;
  for (uint32_t i = 0; i < ranks; ++i) sum += sums[i];
  sum = sqrt(sum);
  const float norm = float(double(p.scale) / (sum < double(p.eps) ? double(p.eps) : sum));

  // X (times `f`) from tensor memory: rounded into shared memory, and a X back
  auto round_x = [&](float f, float a) {
    for (int b = 0; b < mine; ++b) {
#pragma unroll 1
      for (int c = 0; c < 64; c += 16) {
        const uint32_t at = tmem + lanes + uint32_t(128 * (1 + b) + half * 64 + c);
        float v[16];
        tmem_ld_32x32b_x16(at, v);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float w[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = v[8 * e + k] *= f;
          *box_at(hi + b * kBlockBytes + half * kHalfBytes, row, c / 8 + e) = pack8(w);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] *= a;
        tmem_st_32x32b_x16(at, v);
      }
    }
  };
  auto linear = [&](int step) { return p.coefficients[step][0] - (step + 1 == p.steps ? p.shift : 0.0f); };
  round_x(norm, linear(0));
  const float unscale2 = 1.0f / (p.scale * p.scale);

  for (int step = 0; step < p.steps; ++step) {
    ready();
    // ---- A ----
    if (threadIdx.x == 0) {
      for (int b = 0; b < mine; ++b) products_128(tmem, smem_u32(hi + b * kBlockBytes), smem_u32(hi + b * kBlockBytes), true, b > 0 ? 1u : 0u);
      umma_commit(done);
    }
    finish();
    if (ranks == 1) {
#pragma unroll 1
      for (int c = 0; c < 64; c += 16) {
        float v[16];
        tmem_ld_32x32b_x16(tmem + lanes + uint32_t(half * 64 + c), v);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float w[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = v[8 * e + k] * unscale2;
          *box_at(a_mat + half * kHalfBytes, row, c / 8 + e) = pack8(w);
        }
      }
    } else {
      // 128 / ranks rows are each CTA's to add up, for all: the others' parts of them go into its staging area, [rank][row]. A CTA without rows sends zeros.
      auto add_up = [&](auto of) {
        constexpr int R = decltype(of)::value, kRows = 128 / R;
        const float mul = *failed != 0 ? __uint_as_float(0x7fc00000u) : mine > 0 ? unscale2 : 0.0f;
        const uint32_t owner = uint32_t(row / kRows);
        const int at = int(rank) * kRows + row % kRows;
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          float v[16];
          tmem_ld_32x32b_x16(tmem + lanes + uint32_t(half * 64 + c), v);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float4 f = make_float4(v[4 * q] * mul, v[4 * q + 1] * mul, v[4 * q + 2] * mul, v[4 * q + 3] * mul);
            if (mine == 0) f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // (its accumulator holds nothing, not even numbers)
            store_cluster(cluster_address(stage_at(stage, at, (half * 64 + c) / 4 + q), owner), *reinterpret_cast<const uint4*>(&f));
          }
        }
        tc_fence_before_sync();
        cluster_sync();
#pragma unroll
        for (int e = 0; e < kRows * 16 / kSmallT; ++e) {  // eight columns at a time
          const int own = (int(threadIdx.x) >> 4) + e * (kSmallT / 16), r = int(rank) * kRows + own, c = threadIdx.x & 15;
          float v[8] = {};
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const float4 x = *stage_at(stage, i * kRows + own, 2 * c), y = *stage_at(stage, i * kRows + own, 2 * c + 1);
            v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w; v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
          }
          const uint4 packed = pack8(v);
          const void* to = box_at(a_mat + (c >> 3) * kHalfBytes, r, c & 7);
#pragma unroll
          for (int i = 0; i < R; ++i) store_cluster(cluster_address(to, uint32_t(i)), packed);
        }
      };
      if (ranks == 2) add_up(std::integral_constant<int, 2>{});
      else if (ranks == 4) add_up(std::integral_constant<int, 4>{});
      else add_up(std::integral_constant<int, 8>{});
      cluster_sync();
    }
    ready();
    // ---- B ----
    if (threadIdx.x == 0) {
      products_128(tmem, smem_u32(a_mat), smem_u32(a_mat), false, 0u);
      umma_commit(done);
    }
    finish();
    const float fb = p.coefficients[step][1], fc = p.coefficients[step][2], shift = step + 1 == p.steps ? p.shift : 0.0f;
#pragma unroll 1
    for (int c = 0; c < 64; c += 16) {
      float v[16];
      tmem_ld_32x32b_x16(tmem + lanes + uint32_t(half * 64 + c), v);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float a[8], w[8];
        unpack8(*box_at(a_mat + half * kHalfBytes, row, c / 8 + e), a);
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = __fmaf_rn(fb, a[k], __fmaf_rn(fc, v[8 * e + k], half * 64 + c + 8 * e + k == row ? shift : 0.0f));
        *box_at(b_mat + half * kHalfBytes, row, c / 8 + e) = pack8(w);
      }
    }
    ready();
    // ---- X ----
    if (threadIdx.x == 0) {
      for (int b = 0; b < mine; ++b) products_128(tmem + uint32_t(128 * (1 + b)), smem_u32(hi + b * kBlockBytes), smem_u32(b_mat), false, 1u);
      umma_commit(done);
    }
    finish();
    if (step + 1 < p.steps) round_x(1.0f, linear(step + 1));
  }

  // ---- out, the parameters read a round ahead ----
  const float unscale = *failed != 0 ? __uint_as_float(0x7fc00000u) : target.unscale;
  auto write = [&](auto* to, auto fresh, auto run) {
    using P = std::remove_pointer_t<decltype(to)>;
    constexpr int V = decltype(run)::value;
    constexpr bool kFresh = decltype(fresh)::value;
    const int last = (128 * p.m / V + kSmallT - 1) / kSmallT;
    const int64_t step = step_of(run);
    const Walk first = first_of(run);
    const int dr = TALL ? kSmallT * V / p.m : 0, di = TALL ? kSmallT * V - dr * p.m : 0;
    float v[kRuns][V], next[kRuns][V];
    auto fetch = [&](int b, int k0) {
      const int runs = runs_of(run, b, first);
      const int64_t at = start_of(run, b, first) + k0 * step;
#pragma unroll
      for (int k = 0; k < kRuns; ++k) {
        if (k0 + k < runs) {
          if constexpr (V == 4) load4<P>(to + at + k * step, next[k]);
          else next[k][0] = dev::Vec16<P>::to_float(to[at + k * step]);
        }
      }
    };
    if (!kFresh && mine > 0) fetch(0, 0);
    for (int b = 0; b < mine; ++b) {
      const int runs = runs_of(run, b, first);
      const int64_t start = start_of(run, b, first);
      Walk w = first;
      __syncthreads();
#pragma unroll 1
      for (int c = 0; c < 64; c += 16) {
        float f16[16];
        tmem_ld_32x32b_x16(tmem + lanes + uint32_t(128 * (1 + b) + half * 64 + c), f16);
#pragma unroll
        for (int x = 0; x < 4; ++x)
          *stage_at(stage, row, (half * 64 + c) / 4 + x) = make_float4(f16[4 * x] * unscale, f16[4 * x + 1] * unscale, f16[4 * x + 2] * unscale, f16[4 * x + 3] * unscale);
      }
      __syncthreads();
      for (int k0 = 0; k0 < last; k0 += kRuns) {
        if constexpr (!kFresh) {
#pragma unroll
          for (int k = 0; k < kRuns; ++k)
#pragma unroll
            for (int x = 0; x < V; ++x) v[k][x] = next[k][x];
          if (k0 + kRuns < last) fetch(b, k0 + kRuns);
          else if (b + 1 < mine) fetch(b + 1, 0);
        }
        float x[kRuns][V];
#pragma unroll
        for (int k = 0; k < kRuns; ++k) {
          if (k0 + k < runs) {
            if constexpr (V == 4 && TALL) {
              const float4 f = *stage_at(stage, w.r, w.i >> 2);
              x[k][0] = f.x; x[k][1] = f.y; x[k][2] = f.z; x[k][3] = f.w;
            } else {
#pragma unroll
              for (int y = 0; y < V; ++y) x[k][y] = *stage_one(stage, w.r + y, w.i);
            }
          }
          advance(run, w, dr, di);
        }
#pragma unroll
        for (int k = 0; k < kRuns; ++k) {
          if constexpr (!kFresh) {
#pragma unroll
            for (int y = 0; y < V; ++y) x[k][y] = v[k][y] * target.decay - target.rate * x[k][y];
          }
          if (k0 + k < runs) {
            if constexpr (V == 4) store4(to + start + (k0 + k) * step, x[k]);
            else to[start + (k0 + k) * step] = dev::Vec16<P>::from_float(x[k][0]);
          }
        }
      }
    }
  };
  auto write_all = [&](auto* to, auto fresh) {
    if (p.vector_out) write(to, fresh, std::integral_constant<int, 4>{});
    else write(to, fresh, std::integral_constant<int, 1>{});
  };
  if (target.result != nullptr) write_all(target.result + int64_t(batch) * p.m * p.n, std::true_type{});
  else if (target.param_dtype == NANGILA_F32) write_all(static_cast<float*>(target.param[batch]), std::false_type{});
  else if (target.param_dtype == NANGILA_BF16) write_all(static_cast<__nv_bfloat16*>(target.param[batch]), std::false_type{});
  else write_all(static_cast<__half*>(target.param[batch]), std::false_type{});
  tc_fence_before_sync();
  cluster_sync();  // nobody's shared memory goes while another may read it
  if (warp == 0) tmem_dealloc(tmem, 512);
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

// Shared memory above the default limit, asked for once for each kernel and device.
int allow_smem(const void* kernel, int bytes) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> asked;
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return int(e);
  std::lock_guard<std::mutex> lock(mu);
  if (asked.count({kernel, dev})) return 0;
  if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return int(e);
  asked.insert({kernel, dev});
  return 0;
}

template <int KIND, bool A_MN, bool B_MN, bool PAIR>
int launch_product(const Maps& maps, Product p, const Target& target, int count, cudaStream_t stream) {
  constexpr int kSide = PAIR ? 256 : 128;
  const int64_t total = tiles_of(p, kSide, count);
  if (total > 0x7fffffff) return int(cudaErrorInvalidValue);
  p.tiles_m = (p.M + kSide - 1) / kSide;
  p.total = int(total);
  p.per = int(total / count);
  auto* kernel = orth_product_kernel<KIND, A_MN, B_MN, PAIR>;
  if (const int e = allow_smem(reinterpret_cast<const void*>(kernel), kSmem)) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = PAIR ? 2 : 1;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  const int sms = sm_count();
  cfg.gridDim = dim3(unsigned(PAIR ? 2 * std::min(p.total, sms / 2) : std::min(p.total, sms)));
  cfg.blockDim = dim3(kGemmThreads<KIND, PAIR>);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  return int(cudaLaunchKernelEx(&cfg, kernel, maps, p, target));
}
template <bool MN>
int launch_gram_split(const Maps& maps, Product p, const Matrix& out, int total, int per, int split, cudaStream_t stream) {
  auto* kernel = orth_gram_split_kernel<MN>;
  if (const int e = allow_smem(reinterpret_cast<const void*>(kernel), kSmem)) return e;
  p.tiles_m = (p.M + 127) / 128;
  p.total = total;
  p.per = per;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(split);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(total * split));
  cfg.blockDim = dim3(kGemmThreads<kGram, false>);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return int(cudaLaunchKernelEx(&cfg, kernel, maps, p, const_cast<__half*>(out.base), out.ld, out.matrix));
}
// D of the operands a and b; `in` and `lo` are what the epilogue reads, `out` what it writes.
template <int KIND, bool A_MN, bool B_MN>
int product(const Matrix& a, const Matrix& b, const Matrix* in, const Matrix* lo, const Matrix* out, const Product& p, const Target& target, int count, cudaStream_t stream) {
  Maps maps;
  bool ok = make_map(&maps.a, a, count, 64, A_MN ? 64 : 128) && make_map(&maps.b, b, count, 64, B_MN ? 64 : 128);
  ok = ok && make_map(&maps.in, in != nullptr ? *in : a, count, kChunk, 32) && make_map(&maps.lo, lo != nullptr ? *lo : a, count, kChunk, 32);
  ok = ok && make_map(&maps.out, out != nullptr ? *out : a, count, kChunk, 32) && make_map(&maps.mirror, out != nullptr ? *out : a, count, 32, kChunk, false);
  if (!ok) return int(cudaErrorNotSupported);
  // A tile of a pair takes hardly longer than a small one, which is bound by what L2 delivers to an SM (twice the bytes for each product); only its
  // epilogue is longer. So it is the number of rounds that decides. Measured, all products of five steps with small tiles, and with those of pairs: as many rounds of either, 768 x 768 157 us and
  // 202, thirty of 384 x 300 195 and 237; two rounds or one, eight of 768 x 768 250 and 220; three and seven or two and four, twenty of 700 x 900 506 and 464; two and three or one and two,
  // 2305 x 2177 651 and 481. Each product by its rounds, 2048 x 2048: 322, 316, and 288 so.
  const int sms = sm_count();
  const int64_t small = tiles_of(p, 128, count), large = tiles_of(p, 256, count);
  if constexpr (KIND == kGram) {
    // A CTA's share of K is 8 slabs (2 us) at least: what the meeting costs. Three quarters of the SMs: clusters of eight do not fit into all of them.
    const int64_t slabs = (p.K + kSlabK - 1) / kSlabK;
    int split = 1;
    while (split < kMaxCluster && small * split * 2 <= sms * 3 / 4 && slabs >= split * 2 * 8) split *= 2;
    if (split > 1) return launch_gram_split<A_MN>(maps, p, *out, int(small), int(small / count), split, stream);
  }
  const double cost_small = double((small + sms - 1) / sms), cost_large = 1.2 * double((large + sms / 2 - 1) / (sms / 2));
  return cost_large <= cost_small ? launch_product<KIND, A_MN, B_MN, true>(maps, p, target, count, stream) : launch_product<KIND, A_MN, B_MN, false>(maps, p, target, count, stream);
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

// Whether a matrix stays on the SMs for all its steps, and how many CTAs it takes.
int small_cluster(int64_t m, int64_t n) {
  if (m > 128 || n > 128 * kBlocks * kMaxCluster) return 0;
  const int64_t blocks = (n + 127) / 128;
  int ctas = 1;
  while (ctas * kBlocks < blocks) ctas *= 2;
  return ctas;
}
template <typename T>
int launch_small(const Small& p, const Target& target, bool tall, int count, int cluster, cudaStream_t stream) {
  auto* kernel = tall ? orth_small_kernel<T, true> : orth_small_kernel<T, false>;
  if (const int e = allow_smem(reinterpret_cast<const void*>(kernel), kSmallSmem)) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(cluster * count));
  cfg.blockDim = dim3(kSmallT);
  cfg.dynamicSmemBytes = kSmallSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return int(cudaLaunchKernelEx(&cfg, kernel, p, target));
}

template <typename T>
int start(const Prep& p, int count, cudaStream_t stream) {
  const dim3 grid(unsigned(p.chunks), unsigned(count));
  if (p.momentum[0] != nullptr) orth_norm_kernel<T, true><<<grid, kPrepT, 0, stream>>>(p);
  else orth_norm_kernel<T, false><<<grid, kPrepT, 0, stream>>>(p);
  if (const cudaError_t e = cudaGetLastError()) return int(e);
  return int(launch_following(orth_start_kernel<T>, grid, kPrepT, 0, stream, p));
}

}  // namespace
}  // namespace nangila

extern "C" int64_t nangila_orth_workspace(int32_t count, int32_t rows, int32_t cols) {
  using namespace nangila;
  return small_cluster(std::min(rows, cols), std::max(rows, cols)) != 0 ? 256 : layout(count, rows, cols).total;
}

namespace nangila {
namespace {
int orth(const NangilaOrthParams* p, cudaStream_t stream) {
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

  // what the last step moves from a X to B X
  const float* final_step = p->coefficients[p->steps - 1];
  const float shift = -(final_step[1] + final_step[2]);

  Target target;
  std::memset(&target, 0, sizeof target);
  target.unscale = 1.0f / scale;
  target.vector = p->cols % 4 == 0;
  if (p->param[0] != nullptr) {
    for (int i = 0; i < p->count; ++i) {
      target.param[i] = p->param[i];
      if (!aligned(p->param[i])) target.vector = 0;
    }
    target.param_dtype = p->param_dtype;
    target.decay = p->decay;
    target.rate = p->rate;
  } else {
    target.result = static_cast<__nv_bfloat16*>(p->out);
    if (!aligned(p->out)) target.vector = 0;
  }
  if (p->grad_dtype < 0 || p->grad_dtype > 2 || (p->param[0] != nullptr && (p->param_dtype < 0 || p->param_dtype > 2))) return int(cudaErrorInvalidValue);
  if (const int cluster = small_cluster(l.m, l.n)) {
    Small s;
    std::memset(&s, 0, sizeof s);
    s.vector = p->cols % 4 == 0;
    s.vector_out = target.vector;
    for (int i = 0; i < p->count; ++i) {
      s.grad[i] = p->grad[i];
      s.momentum[i] = p->momentum[0] != nullptr ? p->momentum[i] : nullptr;
      if (!aligned(p->grad[i]) || !aligned(s.momentum[i])) s.vector = 0;
    }
    std::memcpy(s.coefficients, p->coefficients, sizeof s.coefficients);
    s.steps = p->steps;
    s.m = int(l.m);
    s.n = int(l.n);
    s.nesterov = p->nesterov;
    s.blocks = int((l.n + 127) / 128);
    s.per = (s.blocks + cluster - 1) / cluster;
    s.mu = p->mu;
    s.eps = p->eps;
    s.scale = scale;
    s.shift = shift;
    return p->grad_dtype == NANGILA_F32   ? launch_small<float>(s, target, tall, p->count, cluster, stream)
           : p->grad_dtype == NANGILA_F16 ? launch_small<__half>(s, target, tall, p->count, cluster, stream)
                                          : launch_small<__nv_bfloat16>(s, target, tall, p->count, cluster, stream);
  }

  Prep prep;
  std::memset(&prep, 0, sizeof prep);
  prep.flat = 1;
  for (int i = 0; i < p->count; ++i) {
    prep.grad[i] = p->grad[i];
    prep.momentum[i] = p->momentum[0] != nullptr ? p->momentum[i] : nullptr;
    if (!aligned(p->grad[i]) || !aligned(prep.momentum[i])) prep.flat = 0;
  }
  prep.vector = prep.flat != 0 && p->cols % 8 == 0;
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
  if (e != 0) return e;
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
    e = tall ? product<kGram, true, true>(X, X, nullptr, nullptr, &A, q, target, p->count, stream) : product<kGram, false, false>(X, X, nullptr, nullptr, &A, q, target, p->count, stream);
    if (e != 0) break;
    q.K = int(l.m);
    q.alpha = c[1];
    q.beta = c[2];
    q.shift = last ? shift : 0.0f;
    e = product<kPoly, false, false>(A, A, &A, nullptr, &B, q, target, p->count, stream);
    if (e != 0) break;
    q.lower = 0;
    q.M = p->rows;
    q.N = p->cols;
    q.alpha = c[0] - (last ? shift : 0.0f);
    if (last) {
      e = tall ? product<kFinal, false, false>(X, B, &X, &Lo, nullptr, q, target, p->count, stream) : product<kFinal, false, true>(B, X, &X, &Lo, nullptr, q, target, p->count, stream);
    } else {
      e = tall ? product<kUpdate, false, false>(X, B, &X, &Lo, &Next, q, target, p->count, stream) : product<kUpdate, false, true>(B, X, &X, &Lo, &Next, q, target, p->count, stream);
    }
  }
  return e;
}

}  // namespace
}  // namespace nangila

extern "C" int nangila_orth(const NangilaOrthParams* p, cudaStream_t stream) {
  try {
    return nangila::orth(p, stream);
  } catch (...) {  // (the host's tables of kernels that were set up allocate)
    return int(cudaErrorMemoryAllocation);
  }
}

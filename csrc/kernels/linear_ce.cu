// The loss of a language model's head without its logits: z = x w^T + b, loss_i = log sum_v exp(z_iv) - z_it, and the gradients of x, w, b (sm_100a).
//
// Losses alone: the tiles of z stay in tensor memory. Their epilogue takes each row's largest value and the sum of its exponentials over 128 classes, and those
// are all that is written; a last kernel joins them to lse and loss. The target's own logit is a dot product in fp32 by itself and is left out of the sums:
// loss = log(1 + sum over the others of exp(z_v - z_t)) keeps its digits where the model is sure.
//
// Gradients need G = exp(z - lse) - [v = t] twice: dx = G w and dw = G^T x. A group of tokens at a time (as many as fit into a gigabyte of 16-bit values) the tiles' epilogue
// writes exponentials E, and two products read them. The exponent's reference need not be lse, which is known only when the whole row is: in bf16, whose range is that of
// fp32, E = exp(z - z_t) is as good. Its row sums give lse, and the factor f = exp(z_t - lse) of each row is applied to the rows of dx, and to those of x
// on their way into dw. So the losses and the gradients take three products (6 n d V operations), where logits that are formed again for the gradients take four. A row in which some z is above z_t by more than
// 60 (exp(60) = 1e26) is formed again with its largest value as the reference. fp16 has no such range, and gradients weighted row by row need their weights: there the
// losses come first, and the gradients form z again with lse as the reference.
//
// Roundings: products of 16-bit operands, summed in fp32; E once to the type of x (with fp16 as 2^15 exp(z - lse), which keeps 11 bits down to 2^-29); f x once;
// results once. dx and dw that are formed along with the loss are rounded once more where the upstream gradient, which is known in the backward pass only, is no power of two: kept in fp32 until
// then they would be on their way some 100 us longer at 8192 x 2048 x 32000, whatever the upstream gradient is (the second rounding: 59 us, and none for one). The target's element of E is minus the sum of all others, in fp32, before its rounding: no 1 - p where p is near one.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <mutex>
#include <set>
#include <utility>

#include "follow.cuh"
#include "launch_util.cuh"
#include "nangila_kernels.h"
#include "nangila_vocab_kernels.h"
#include "ptx_sm100.cuh"
#include "quant.cuh"
#include "raw8.cuh"
#include "warp_sums.cuh"

namespace nangila {
namespace {

using namespace sm100;

constexpr int kTileM = 128;                      // rows of a CTA
constexpr int kSlabK = 64;                       // one 128-byte swizzle row of 16-bit values
constexpr int kOperandBytes = 128 * kSlabK * 2;  // what a CTA holds of an operand's slab
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kStages = 5;
constexpr int kSlotBytes = 32 * 128;             // 32 rows of 64 values in 16 bits, or of 32 in fp32
constexpr int kEpilogueWarps = 8;                // two for each quarter of tensor memory, each with one half of a tile's columns
constexpr int kSlots = 2;                        // of each
constexpr int kBiasBytes = 32 * 4;               // of 32 columns, for each of the epilogue's warps
constexpr int kSmem = kStages * kStageBytes + kEpilogueWarps * (kSlots * kSlotBytes + kBiasBytes) + 1024 + 256;
static_assert(kSmem <= 227 * 1024, "what a CTA can have");
constexpr int kThreads = 64 + 32 * kEpilogueWarps;  // warp 0: TMA, warp 1: products, the others: epilogue
constexpr int kTasks = 4;                           // tiles that a pair of CTAs has taken and not all of its warps have read
constexpr int kTaskReaders = 2 * (kEpilogueWarps + 1);  // the epilogues, the products of rank 0, the copies of rank 1
constexpr uint64_t kTimeoutNs = 10ull * 1000 * 1000 * 1000;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kMostAbove = 60.0f * kLog2e;     // how far a logit may lie above a row's reference

// What becomes of a tile of logits. kStats: the largest one and the sum of exponentials of each row over half a tile's columns. kExp: the same, and E. kWeighted: E, its rows weighted
// and with their elements at the target.
enum Kind { kStats, kExp, kWeighted };

// What is known of a group's rows when their tiles are made, and what comes out.
struct Rows {
  const int64_t* targets;
  const float* ref;     // exponents' reference, times log2(e)
  const float* mul;     // kWeighted: factors of E's rows
  const float* value;   // and E's element at the target (kExp: 0, to be filled in)
  const float* bias;    // padded to whole tiles; NULL: none
  float2* parts;        // [half tiles][stride]: largest z log2(e), sum of exp
  const int32_t* again; // for each 32 rows, whether they are to be formed again; NULL: all tiles are made
  int64_t stride, ignore;
  int n, classes;
};
struct Maps {
  CUtensorMap a, b, out;
};
// One result of the gradients' products, M x N, its K cut into `split` parts of `slabs` slabs (the last may have fewer).
struct Result {
  int M, N, K;
  int tiles_n, total;   // tiles along N; of all parts
  int split, slabs, per; // per: tiles of a part
  int wide;             // 0: alpha f_row D in 16 bits; 1: D in fp32; 2: added to what is there
  const float* factor;  // of D's rows; NULL: one
  int live;             // rows from here on get zeros (`wide` 0)
};
// Columns of E, each row times its factor, added up: 256 columns and a share of the rows a warp, the shares' sums one behind the other.
struct Columns {
  const void* e;
  const float* factor;
  float* partial;       // [shares][e_stride]; NULL: not wanted
  int64_t e_stride;
  int n, blocks, shares, share;
};
struct Gradients {
  Result x, w;          // dx = E w, dw = E^T x'
  Columns columns;
  const float* alpha;
  int* next;            // the next tile that nobody has taken
  int w_again;          // where along dw's K the rows of E begin once more, for the rests of x'
};
struct GradientMaps {
  CUtensorMap e_rows, w, out_x;      // dx
  CUtensorMap e_columns, xs, out_w;  // dw
};

template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&f)[8]) {
  dev::Raw8<T> r;
  dev::pack(f, r);
  return r.a;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Sixteen bytes `j` of a lane's row in a box of 32 rows of 128 bytes, as TMA swizzles them (the box starts on 1024 bytes).
__device__ __forceinline__ uint4* box_at(uint8_t* box, int row, int j) { return reinterpret_cast<uint4*>(box + row * 128 + ((j ^ (row & 7)) << 4)); }

struct TileAt {
  int m0, n0;
};

// What a CTA's roles share, in shared memory.
struct Shared {
  uint8_t *stages, *slots;
  float* bias;                     // [kEpilogueWarps][32]
  uint64_t *full, *empty;          // [kStages]
  uint64_t *acc_full, *acc_empty;  // [2]
  uint64_t* drained;
  uint64_t *task_full, *task_empty;  // [kTasks]
  volatile int* task;              // [kTasks]
  uint32_t* tmem_slot;
  volatile uint32_t* failed;       // a wait has run out
};
__device__ __forceinline__ Shared shared_parts(uint8_t* raw) {
  Shared s;
  s.stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  s.slots = s.stages + kStages * kStageBytes;
  s.bias = reinterpret_cast<float*>(s.slots + kEpilogueWarps * kSlots * kSlotBytes);
  s.full = reinterpret_cast<uint64_t*>(s.bias + kEpilogueWarps * 32);
  s.empty = s.full + kStages;
  s.acc_full = s.empty + kStages;
  s.acc_empty = s.acc_full + 2;
  s.drained = s.acc_empty + 2;
  s.task_full = s.drained + 1;
  s.task_empty = s.task_full + kTasks;
  s.task = reinterpret_cast<int*>(s.task_empty + kTasks);
  s.tmem_slot = reinterpret_cast<uint32_t*>(s.task_empty + kTasks) + kTasks;
  s.failed = s.tmem_slot + 1;
  return s;
}
template <bool PAIR>
__device__ __forceinline__ void init_barriers(const Shared& s) {
  for (int i = 0; i < kStages; ++i) {
    mbar_init(&s.full[i], 1);
    mbar_init(&s.empty[i], 1);
  }
  for (int i = 0; i < 2; ++i) {
    mbar_init(&s.acc_full[i], 1);
    mbar_init(&s.acc_empty[i], kEpilogueWarps * (PAIR ? 2 : 1));
  }
  mbar_init(s.drained, 1);
  for (int i = 0; i < kTasks; ++i) {
    mbar_init(&s.task_full[i], 1);
    mbar_init(&s.task_empty[i], kTaskReaders);
  }
  *s.failed = 0;
  fence_barrier_init();
}

// The copies and the products are each issued by one lane of a warp, but all of its lanes go through the loops: what the instructions take is then the same for the warp, and stays in the
// registers that they take it from. (With one lane in the loops, each of its instructions moved its operands there first: 640 cycles a slab, whose products take 512. 8192 x 768 x 50304's
// logits, half of them at a time, 245 us.)
__device__ __forceinline__ bool elected() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
// A wait of a whole warp, with one answer for all of it. CLUSTER: for what the other CTA did before it arrived, too.
template <bool CLUSTER = false>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  auto done = [&] { return __all_sync(0xffffffffu, CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) != 0; };
  if (done()) return true;
  const uint64_t t0 = timer_ns();
  uint32_t spins = 0;
  while (!done()) {
    if ((++spins & 255u) == 0u && __any_sync(0xffffffffu, timer_ns() - t0 > kTimeoutNs)) return false;
  }
  return true;
}
// Where a role is in the ring of stages.
struct Ring {
  int stage = 0;
  uint32_t round = 0;  // how often the ring has been gone round
  __device__ __forceinline__ void next(int stages) {
    if (++stage == stages) stage = 0, ++round;
  }
};

// TMA of a tile's slabs: both CTAs of a pair, each its own halves; the bytes are counted where the products are issued. By a whole warp. False when a wait has run out.
// before(k) comes before slab k's wait. `again`: where along K operand A begins once more.
template <bool PAIR, typename Before>
__device__ __forceinline__ bool load_tile(const Shared& s, const CUtensorMap* a_map, const CUtensorMap* b_map, bool a_mn, bool b_mn, const TileAt& at, uint32_t rank, int slab0, int slabs, int again,
                                          Ring& ring, const Before& before) {
  const int row = at.m0 + int(rank) * kTileM, col = at.n0 + int(rank) * 128;
  for (int k = 0; k < slabs; ++k, ring.next(kStages)) {
    if (!before(k)) {
      *s.failed = 1;
      return false;
    }
    const int st = ring.stage;
    if (ring.round > 0 && !warp_wait(&s.empty[st], (ring.round - 1) & 1)) {
      *s.failed = 1;
      return false;
    }
    if (elected()) {
      uint8_t* a = s.stages + st * kStageBytes;
      uint8_t* b = a + kOperandBytes;
      const int k0 = (slab0 + k) * kSlabK, a_k0 = k0 < again ? k0 : k0 - again;
      if (rank == 0) mbar_arrive_expect_tx(&s.full[st], kStageBytes * (PAIR ? 2 : 1));
      const uint32_t bar = PAIR ? rank0_address(&s.full[st]) : smem_u32(&s.full[st]);
      if (a_mn) {
        tma_operand<PAIR>(a, a_map, row, a_k0, 0, bar);
        tma_operand<PAIR>(a + 8192, a_map, row + 64, a_k0, 0, bar);
      } else {
        tma_operand<PAIR>(a, a_map, a_k0, row, 0, bar);
      }
      if (b_mn) {
        tma_operand<PAIR>(b, b_map, col, k0, 0, bar);
        tma_operand<PAIR>(b + 8192, b_map, col + 64, k0, 0, bar);
      } else {
        tma_operand<PAIR>(b, b_map, k0, col, 0, bar);
      }
    }
    __syncwarp();
  }
  return true;
}
// The copies that are still under way when the loads end: all have arrived when the products that read them are done; if somebody has given up, as
// much as can be waited for (the bytes of a pair are counted by rank 0, the stages of rank 1 are given back by its products).
__device__ __forceinline__ void drain_loads(const Shared& s, uint32_t rank, Ring ring) {
  const int under_way = ring.round > 0 ? kStages : ring.stage;
  for (int j = 0; j < under_way; ++j) {
    // backwards from the last one
    if (ring.stage == 0) ring.stage = kStages, --ring.round;
    --ring.stage;
    if (*s.failed == 0 || rank != 0) warp_wait(&s.empty[ring.stage], ring.round & 1);
    else warp_wait(&s.full[ring.stage], ring.round & 1);
  }
}
// The products of a tile, the n-th, into its accumulator, by a whole warp. False when a wait has run out.
template <bool PAIR, bool BF16, typename Before>
__device__ __forceinline__ bool multiply_tile(const Shared& s, uint32_t tmem, bool a_mn, bool b_mn, int slabs, int n, Ring& ring, const Before& before) {
  constexpr int kSide = PAIR ? 256 : 128;
  const uint32_t idesc = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) | (uint32_t(kSide >> 3) << 17) | (uint32_t(kSide >> 4) << 24);
  const int acc = n & 1;
  if (n >= 2 && !warp_wait(&s.acc_empty[acc], uint32_t((n / 2 - 1) & 1))) return false;
  tc_fence_after_sync();
  const uint32_t d = tmem + uint32_t(acc * kSide);
  // K-major: 16 elements along K are 32 bytes of a swizzle row; MN-major: 16 K-rows are two groups of eight rows of 128 bytes
  const uint64_t a0 = make_smem_desc(smem_u32(s.stages), a_mn ? 8192 : 16, 1024), b0 = make_smem_desc(smem_u32(s.stages) + kOperandBytes, b_mn ? 8192 : 16, 1024);
  const uint64_t a_step = (a_mn ? 2048 : 32) >> 4, b_step = (b_mn ? 2048 : 32) >> 4;
  for (int k = 0; k < slabs; ++k, ring.next(kStages)) {
    if (!before(k) || !warp_wait(&s.full[ring.stage], ring.round & 1)) return false;
    tc_fence_after_sync();
    if (elected()) {
      const uint64_t from = uint64_t(uint32_t(ring.stage * (kStageBytes >> 4)));  // (addresses of 18 bits: nothing is carried out of their field)
#pragma unroll
      for (int kk = 0; kk < kSlabK / 16; ++kk) {
        if (PAIR) umma_f16_pair(d, a0 + from + kk * a_step, b0 + from + kk * b_step, idesc, (k > 0 || kk > 0) ? 1u : 0u);
        else umma_f16(d, a0 + from + kk * a_step, b0 + from + kk * b_step, idesc, (k > 0 || kk > 0) ? 1u : 0u);
      }
      if (PAIR) umma_commit_pair(&s.empty[ring.stage]);
      else umma_commit(&s.empty[ring.stage]);
      if (k + 1 == slabs) {
        if (PAIR) umma_commit_pair(&s.acc_full[acc]);
        else umma_commit(&s.acc_full[acc]);
      }
    }
    __syncwarp();
  }
  return true;
}
// What has been issued ends, when a wait has run out.
template <bool PAIR>
__device__ __forceinline__ void drain_products(const Shared& s) {
  *s.failed = 1;
  if (elected()) {
    if (PAIR) umma_commit_pair(s.drained);
    else umma_commit(s.drained);
  }
  __syncwarp();
  warp_wait(s.drained, 0);
}

__device__ __forceinline__ void nan16(float (&v)[16]) {
#pragma unroll
  for (int k = 0; k < 16; ++k) v[k] = __uint_as_float(0x7fc00000u);
}
// The wait of an epilogue's warp for the n-th accumulator; false if it, or somebody's, has run out.
__device__ __forceinline__ bool accumulator_here(const Shared& s, int n) {
  const bool ok = *s.failed == 0 && mbar_wait(&s.acc_full[n & 1], uint32_t((n / 2) & 1), kTimeoutNs);
  const bool all = __all_sync(0xffffffffu, ok);
  if (!all) *s.failed = 1;
  tc_fence_after_sync();
  return all;
}
// (With an arrival that also waits for the warp's stores, 2400 cycles a tile.)
template <bool PAIR>
__device__ __forceinline__ void accumulator_read(const Shared& s, int n) {
  tc_fence_before_sync();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive_only((PAIR ? rank0_address(&s.acc_empty[0]) : smem_u32(&s.acc_empty[0])) + uint32_t(n & 1) * 8);
}
// A slot of this warp's that nothing goes out of any more, and its way out; `used`: how many have been filled.
__device__ __forceinline__ uint8_t* free_slot(const Shared& s, uint32_t used) {
  if ((threadIdx.x & 31) == 0) bulk_wait_read_but_one();
  __syncwarp();
  return s.slots + (((threadIdx.x >> 5) - 2) * kSlots + used % kSlots) * kSlotBytes;
}
__device__ __forceinline__ void send_slot(const uint8_t* slot, const CUtensorMap* map, int col, int row, int part, bool add) {
  fence_async_proxy();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    if (add) tma_add_3d(map, slot, col, row, part);
    else tma_store_3d(map, slot, col, row, part);
    bulk_commit();
  }
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void halves_of(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}

// What an epilogue's warp knows of the rows of a tile of logits, a lane each, and finds out about them.
struct LogitRow {
  int target;               // -1: none
  bool dead;                // adds nothing
  float ref, mul, value;
  float most;               // raw logits
  uint64_t sum[2];
};
// 32 columns from `first` on: their part of the row's sums, and with E its 64 bytes of the slot from sixteen bytes `at` on.
template <typename T, int KIND>
__device__ __forceinline__ void take_logits(const Rows& rows, LogitRow& r, uint32_t (&raw)[32], bool ok, int first, float bias, float* biases, uint8_t* slot, int lane, int at) {
  float v[32];
#pragma unroll
  for (int k = 0; k < 32; ++k) v[k] = ok ? __uint_as_float(raw[k]) : __uint_as_float(0x7fc00000u);
  if (rows.bias != nullptr) {  // each lane's column to all lanes
    __syncwarp();
    biases[lane] = bias;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 32; k += 4) {
      const float4 b = *reinterpret_cast<const float4*>(biases + k);
      v[k] += b.x, v[k + 1] += b.y, v[k + 2] += b.z, v[k + 3] += b.w;
    }
  }
  const bool here = r.target >= first && r.target < first + 32, any = __any_sync(0xffffffffu, here);
  if (any || first + 32 > rows.classes) {  // what is no class, and the target, stay out of the sums
#pragma unroll
    for (int k = 0; k < 32; ++k)
      if (first + k >= rows.classes || first + k == r.target) v[k] = -INFINITY;
  }
  float base = r.ref;
  if constexpr (KIND != kWeighted) {
    float top[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) top[k] = fmaxf(v[k], v[k + 4]);
#pragma unroll
    for (int k = 8; k < 32; ++k) top[k & 3] = fmaxf(top[k & 3], v[k]);
    const float now = fmaxf(fmaxf(r.most, fmaxf(top[0], top[1])), fmaxf(top[2], top[3]));
    if constexpr (KIND == kStats) {
      // the sums so far, relative to the largest logit so far
      const float to = now == -INFINITY ? 0.0f : now, by = exp2_fast((r.most - to) * kLog2e);
      const uint64_t by2 = pair_of(by, by), none = pair_of(-0.0f, -0.0f);
      r.sum[0] = fma_pair(r.sum[0], by2, none);
      r.sum[1] = fma_pair(r.sum[1], by2, none);
      base = to * kLog2e;
    }
    r.most = now;
  }
  const uint64_t scale = pair_of(kLog2e, kLog2e), from = pair_of(-base, -base);
#pragma unroll
  for (int k = 0; k < 32; k += 2) {
    float a, b;
    halves_of(fma_pair(pair_of(v[k], v[k + 1]), scale, from), a, b);
    v[k] = exp2_fast(a), v[k + 1] = exp2_fast(b);
    if constexpr (KIND != kWeighted) r.sum[(k / 2) & 1] = add_pair(r.sum[(k / 2) & 1], pair_of(v[k], v[k + 1]));
  }
  if constexpr (KIND == kWeighted) {
#pragma unroll
    for (int k = 0; k < 32; ++k) v[k] *= r.mul;
    if (any) {
#pragma unroll
      for (int k = 0; k < 32; ++k)
        if (first + k == r.target) v[k] = r.value;
    }
  }
  if constexpr (KIND != kStats) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = v[8 * e + k];
      uint4 packed = pack16<T>(w);
      if (r.dead) packed = make_uint4(0, 0, 0, 0);
      *box_at(slot, lane, at + e) = packed;
    }
  }
}
// What the epilogue's lanes read from memory for a tile: their row's, and one column's of each 32.
template <int HALF>
struct LogitInputs {
  int64_t target;
  float ref, mul, value, bias[HALF / 32];
};
// The warp's first row and column in a tile.
template <bool PAIR>
__device__ __forceinline__ TileAt warp_at(const TileAt& at, uint32_t rank) {
  const int warp = threadIdx.x >> 5;  // (lanes 32 (warp & 3) and on of tensor memory are the ones that it may read; half of the columns)
  return {at.m0 + int(rank) * kTileM + (warp & 3) * 32, at.n0 + ((warp - 2) >> 2) * (PAIR ? 128 : 64)};
}
template <int KIND, int HALF>
__device__ __forceinline__ void fetch_inputs(const Rows& rows, const TileAt& at, LogitInputs<HALF>& in) {
  const int lane = threadIdx.x & 31, row = at.m0 + lane;
  in.target = -1;
  in.ref = 0.0f, in.mul = 1.0f, in.value = 0.0f;
  if (row < rows.n) {
    in.target = rows.targets[row];
    if (KIND != kStats) in.ref = rows.ref[row];
    if (KIND == kWeighted) in.mul = rows.mul[row], in.value = rows.value[row];
  }
  if (rows.bias != nullptr) {
#pragma unroll
    for (int k = 0; k < HALF / 32; ++k) in.bias[k] = at.n0 + k * 32 < rows.classes ? rows.bias[at.n0 + k * 32 + lane] : 0.0f;
  }
}
// A tile of logits, the n-th, by one of the epilogue's warps: 32 columns at a time, the next on their way out of tensor memory, what memory has to give for the tile after this one
// on its way too. (Columns sixteen at a time and each waited for, rows and bias read when they were needed, which takes 2000 cycles while the operands' copies fill the way from L2, the epilogue
// took longer than the products for K up to 1024: 1229 x 1024 x 30592 75 us.)
template <typename T, int KIND, bool PAIR>
__device__ __forceinline__ void finish_logits(const Shared& s, uint32_t tmem, const Rows& rows, const CUtensorMap* out, const TileAt& at, const TileAt* next, uint32_t rank, int n,
                                              LogitInputs<(PAIR ? 128 : 64)>& in, uint32_t& used) {
  constexpr int kSide = PAIR ? 256 : 128, kHalf = kSide / 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TileAt mine_at = warp_at<PAIR>(at, rank);
  const int row0 = mine_at.m0, row = row0 + lane, col0 = mine_at.n0;
  const bool mine = row0 < rows.n && col0 < rows.classes;
  LogitRow r;
  r.dead = in.target < 0 || in.target >= rows.classes || in.target == rows.ignore;  // (what is ignored may be a class)
  r.target = r.dead ? -1 : int(in.target);
  r.ref = in.ref, r.mul = in.mul, r.value = in.value;
  r.most = -INFINITY;
  r.sum[0] = r.sum[1] = 0;
  float bias[kHalf / 32];
#pragma unroll
  for (int k = 0; k < kHalf / 32; ++k) bias[k] = in.bias[k];
  if (next != nullptr) fetch_inputs<KIND, kHalf>(rows, warp_at<PAIR>(*next, rank), in);
  const bool ok = accumulator_here(s, n);
  if (mine) {
    const uint32_t from = tmem + (uint32_t((warp & 3) * 32) << 16) + uint32_t((n & 1) * kSide + ((warp - 2) >> 2) * kHalf);
    float* biases = s.bias + (warp - 2) * 32;
    uint32_t left[32], right[32];
    tmem_ld_32x32b_x32_start(from, left);
#pragma unroll
    for (int c = 0; c < kHalf; c += 64) {
      if (col0 + c >= rows.classes) break;
      uint8_t* slot = KIND != kStats ? free_slot(s, used) : nullptr;
      tmem_ld_wait(left);
      tmem_ld_32x32b_x32_start(from + c + 32, right);
      take_logits<T, KIND>(rows, r, left, ok, col0 + c, bias[c / 32], biases, slot, lane, 0);
      tmem_ld_wait(right);
      if (c + 64 < kHalf) tmem_ld_32x32b_x32_start(from + c + 64, left);
      take_logits<T, KIND>(rows, r, right, ok, col0 + c + 32, bias[c / 32 + 1], biases, slot, lane, 4);
      if (KIND != kStats) {
        send_slot(slot, out, col0 + c, row0, 0, false);
        ++used;
      }
    }
    tmem_ld_wait(left);
  }
  accumulator_read<PAIR>(s, n);
  if (KIND != kWeighted && mine && row < rows.n) {
    float a, b;
    halves_of(add_pair(r.sum[0], r.sum[1]), a, b);
    rows.parts[int64_t(col0 / kHalf) * rows.stride + row] = make_float2(r.most * kLog2e, a + b);
  }
}

// A tile of a gradient, the n-th, by one of the epilogue's warps: `wide` 0 in 16 bits, each row times `scale`; else in fp32, written (1) or added (2), as part `part`.
template <typename T>
__device__ __forceinline__ void finish_result(const Shared& s, uint32_t tmem, const Result& r, const float* alpha_at, const CUtensorMap* out, const TileAt& at, int part, uint32_t rank, int n,
                                              uint32_t& used) {
  constexpr int kSide = 256, kHalf = 128;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = warp & 3, half = (warp - 2) >> 2;
  const int row0 = at.m0 + int(rank) * kTileM + quad * 32, row = row0 + lane, col0 = at.n0 + half * kHalf;
  const bool mine = row0 < r.M && col0 < r.N;
  float scale = 1.0f;
  bool dead = false;  // a row that adds nothing gets nothing either, whatever the rest holds
  if (r.wide == 0) {
    scale = *alpha_at;
    dead = row >= r.live;
    if (r.factor != nullptr && mine && row < r.M) {
      const float f = r.factor[row];
      dead = dead || f == 0.0f;
      scale *= f;
    }
  }
  const bool ok = accumulator_here(s, n);
  if (mine) {
    const int chunk = r.wide != 0 ? 32 : 64;  // columns of a slot
#pragma unroll 1
    for (int c = 0; c < kHalf && col0 + c < r.N; c += chunk) {
      uint8_t* slot = free_slot(s, used);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (g * 16 >= chunk) break;
        float v[16];
        tmem_ld_32x32b_x16(tmem + (uint32_t(quad * 32) << 16) + uint32_t((n & 1) * kSide + half * kHalf + c + g * 16), v);
        if (!ok) nan16(v);
        if (r.wide == 0) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = dead ? 0.0f : v[8 * e + k] * scale;
            *box_at(slot, lane, 2 * g + e) = pack16<T>(w);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *box_at(slot, lane, 4 * g + e) = make_uint4(__float_as_uint(v[4 * e]), __float_as_uint(v[4 * e + 1]), __float_as_uint(v[4 * e + 2]), __float_as_uint(v[4 * e + 3]));
        }
      }
      send_slot(slot, out, col0 + c, row0, part, r.wide == 2);
      ++used;
    }
  }
  accumulator_read<true>(s, n);
}

// What all roles of a kernel of products begin and end with.
template <bool PAIR>
__device__ __forceinline__ uint32_t products_begin(const Shared& s) {
  constexpr int kSide = PAIR ? 256 : 128;
  if (threadIdx.x == 0) init_barriers<PAIR>(s);
  if (threadIdx.x >> 5 == 1) {
    if (PAIR) tmem_alloc_pair(s.tmem_slot, 2 * kSide);
    else tmem_alloc(s.tmem_slot, 2 * kSide);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync();  // the other CTA's barriers exist from here on
  tc_fence_after_sync();
  return *s.tmem_slot;
}
template <bool PAIR>
__device__ __forceinline__ void products_end(uint32_t tmem) {
  constexpr int kSide = PAIR ? 256 : 128;
  tc_fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync();  // neither CTA's barriers and tensor memory go while the other may still use them
  if (threadIdx.x >> 5 == 1) {
    if (PAIR) tmem_dealloc_pair(tmem, 2 * kSide);
    else tmem_dealloc(tmem, 2 * kSide);
  }
}

// z = x w^T, walked over tile by tile by CTAs that stay (PAIR: pairs of CTAs that share the tensor cores' work on 256 x 256, each with its 128 rows of x, half of
// the classes, and 128 rows of the result; else one CTA and 128 x 128). The accumulators of two tiles share tensor memory: the epilogue of one runs under the products of the next.
// Neighbouring tiles share classes: w is read once, x stays in L2.
// A wait that runs out makes every result of this CTA from there on not a number.
template <typename T, int KIND, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) ce_logits_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Rows rows, int tiles_m, int total, int slabs) {
  constexpr int kSide = PAIR ? 256 : 128;
  extern __shared__ uint8_t smem_raw[];
  const Shared s = shared_parts(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0u;   // 0: the CTA that issues the pair's products
  const int first = PAIR ? blockIdx.x / 2 : blockIdx.x, step = PAIR ? gridDim.x / 2 : gridDim.x;
  auto tile_at = [&](int i) { return TileAt{i % tiles_m * kSide, i / tiles_m * kSide}; };
  // rows to be formed again: their tiles alone
  const bool some = KIND == kExp && rows.again != nullptr;
  if (some) {
    follow();
    bool any = false;
    for (int i = threadIdx.x; i < (rows.n + 31) / 32; i += kThreads) any = any || rows.again[i] != 0;
    if (__syncthreads_or(any) == 0) return;
  }
  auto skip = [&](const TileAt& at) {
    if constexpr (KIND == kExp) {
      if (!some) return false;
      for (int i = at.m0 / 32; i < min((at.m0 + kSide) / 32, (rows.n + 31) / 32); ++i)
        if (rows.again[i] != 0) return false;
      return true;
    } else {
      return false;
    }
  };
  if (threadIdx.x == 0) {
    prefetch_tensormap(&maps.a);
    prefetch_tensormap(&maps.b);
    if (KIND != kStats) prefetch_tensormap(&maps.out);
  }
  const uint32_t tmem = products_begin<PAIR>(s);
  follow();
  may_follow();  // (the next kernel reads x and w before it waits for this one: they are complete)

  if (warp == 0) {
    Ring ring;
    for (int tile = first; tile < total; tile += step) {
      const TileAt at = tile_at(tile);
      if (skip(at)) continue;
      if (!load_tile<PAIR>(s, &maps.a, &maps.b, false, false, at, rank, 0, slabs, INT_MAX, ring, [](int) { return true; })) break;
    }
    drain_loads(s, rank, ring);
  } else if (warp == 1) {
    if (rank == 0) {
      Ring ring;
      int n = 0;
      bool ok = true;
      for (int tile = first; tile < total && ok; tile += step) {
        if (some && skip(tile_at(tile))) continue;
        ok = multiply_tile<PAIR, std::is_same<T, __nv_bfloat16>::value>(s, tmem, false, false, slabs, n, ring, [](int) { return true; });
        ++n;
      }
      if (!ok) drain_products<PAIR>(s);
    }
  } else {
    int n = 0;
    uint32_t used = 0;
    LogitInputs<(PAIR ? 128 : 64)> in;
    auto from = [&](int tile) {  // the first one that is made
      while (some && tile < total && skip(tile_at(tile))) tile += step;
      return tile;
    };
    int tile = from(first);
    TileAt at = tile_at(tile);
    if (tile < total) fetch_inputs<KIND, (PAIR ? 128 : 64)>(rows, warp_at<PAIR>(at, rank), in);
    for (; tile < total; ++n) {
      const int then = from(tile + step);
      const TileAt next = tile_at(then);
      finish_logits<T, KIND, PAIR>(s, tmem, rows, &maps.out, at, then < total ? &next : nullptr, rank, n, in, used);
      tile = then;
      at = next;
    }
    if (lane == 0) bulk_wait_read();  // the stores have left shared memory; the end of the kernel is what others wait for
  }
  products_end<PAIR>(tmem);
}

// The same sums for few tokens, TOKENS at most: bound by reading w once, so w's rows are what fills the products' 128 rows, and as many of its slabs as fit into shared memory are on
// their way. A tile's columns are tokens, its rows classes: each warp of the epilogue joins the 32 classes that its lanes hold, token by token, and keeps lane t's running pair for token t.
// (With the tokens as rows, 16 of 128 of them there, 16 x 2048 x 32000 took 39 us.)
template <int TOKENS>
struct Few {
  static constexpr int kStage = kOperandBytes + TOKENS * 128;
  static constexpr int kCount = TOKENS <= 16 ? 12 : TOKENS <= 32 ? 10 : 9;
  static constexpr int kBytes = kCount * kStage + 1024 + 256;
};
constexpr int kFewThreads = 64 + 128;
template <typename T, int TOKENS>
__global__ void __launch_bounds__(kFewThreads, 1) ce_few_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Rows rows, int total, int slabs) {
  using F = Few<TOKENS>;
  constexpr int kColumns = TOKENS <= 16 ? 32 : 2 * TOKENS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int targets[TOKENS];
  __shared__ float2 joined[4][TOKENS];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(stages + F::kCount * F::kStage);
  uint64_t *empty = full + F::kCount, *acc_full = empty + F::kCount, *acc_empty = acc_full + 2, *drained = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile uint32_t* failed = tmem_slot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < F::kCount; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4);
    }
    mbar_init(drained, 1);
    *failed = 0;
    fence_barrier_init();
    prefetch_tensormap(&maps.a);
    prefetch_tensormap(&maps.b);
  }
  if (warp == 1) tmem_alloc(tmem_slot, kColumns);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  follow();
  may_follow();  // (the next kernel reads x and w before it waits for this one: they are complete)
  if (warp == 0) {
    Ring ring;
    bool ok = true;
    for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x)
      for (int k = 0; k < slabs; ++k, ring.next(F::kCount)) {
        const int st = ring.stage;
        if (ring.round > 0 && !warp_wait(&empty[st], (ring.round - 1) & 1)) {
          *failed = 1;
          ok = false;
          break;
        }
        if (elected()) {
          uint8_t* a = stages + st * F::kStage;
          mbar_arrive_expect_tx(&full[st], F::kStage);
          tma_operand<false>(a, &maps.a, k * kSlabK, tile * kTileM, 0, smem_u32(&full[st]));
          tma_operand<false>(a + kOperandBytes, &maps.b, k * kSlabK, 0, 0, smem_u32(&full[st]));
        }
        __syncwarp();
      }
    const int under_way = ring.round > 0 ? F::kCount : ring.stage;
    for (int j = 0; j < under_way; ++j) {
      if (ring.stage == 0) ring.stage = F::kCount, --ring.round;
      --ring.stage;
      warp_wait(*failed == 0 ? &empty[ring.stage] : &full[ring.stage], ring.round & 1);
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = (1u << 4) | (std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u) | (uint32_t(TOKENS >> 3) << 17) | (uint32_t(kTileM >> 4) << 24);
    const uint64_t a0 = make_smem_desc(smem_u32(stages), 16, 1024), b0 = make_smem_desc(smem_u32(stages) + kOperandBytes, 16, 1024);
    Ring ring;
    int n = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x, ++n) {
      if (n >= 2 && !warp_wait(&acc_empty[n & 1], uint32_t((n / 2 - 1) & 1))) ok = false;
      tc_fence_after_sync();
      for (int k = 0; k < slabs && ok; ++k, ring.next(F::kCount)) {
        if (!warp_wait(&full[ring.stage], ring.round & 1)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        if (elected()) {
          const uint64_t from = uint64_t(uint32_t(ring.stage * (F::kStage >> 4)));
#pragma unroll
          for (int kk = 0; kk < kSlabK / 16; ++kk) umma_f16(tmem + uint32_t((n & 1) * TOKENS), a0 + from + kk * 2, b0 + from + kk * 2, idesc, (k > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&empty[ring.stage]);
          if (k + 1 == slabs) umma_commit(&acc_full[n & 1]);
        }
        __syncwarp();
      }
    }
    if (!ok) {
      *failed = 1;
      if (elected()) umma_commit(drained);
      __syncwarp();
      warp_wait(drained, 0);
    }
  } else {
    const int quad = warp & 3;
    for (int t = threadIdx.x - 64; t < TOKENS; t += 128) {
      const int64_t v = t < rows.n ? rows.targets[t] : -1;
      targets[t] = v >= 0 && v < rows.classes ? int(v) : -1;
    }
    asm volatile("" ::: "memory");
    __syncwarp();
    asm volatile("bar.sync 1, 128;" ::: "memory");
    float most[(TOKENS + 31) / 32], sum[(TOKENS + 31) / 32];
#pragma unroll
    for (int j = 0; j < (TOKENS + 31) / 32; ++j) most[j] = -INFINITY, sum[j] = 0.0f;
    int n = 0;
    for (int tile = blockIdx.x; tile < total; tile += gridDim.x, ++n) {
      const int row = tile * kTileM + quad * 32 + lane;  // the lane's class
      const bool here = row < rows.classes;
      const float bias = rows.bias != nullptr && here ? rows.bias[row] : 0.0f;
      bool ok = *failed == 0 && mbar_wait(&acc_full[n & 1], uint32_t((n / 2) & 1), kTimeoutNs);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) *failed = 1;
      tc_fence_after_sync();
      float tops[(TOKENS + 31) / 32], sums[(TOKENS + 31) / 32];
#pragma unroll
      for (int g = 0; g < TOKENS / 16; ++g) {
        float v[16];
        tmem_ld_32x32b_x16(tmem + (uint32_t(quad * 32) << 16) + uint32_t((n & 1) * TOKENS + g * 16), v);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int t = g * 16 + k;
          float z = ok ? (v[k] + bias) * kLog2e : __uint_as_float(0x7fc00000u);
          if (!here || row == targets[t]) z = -INFINITY;
          float top = z;
#pragma unroll
          for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          const float e = exp2_fast(z - (top == -INFINITY ? 0.0f : top));
          v[k] = e;
          if (lane == (t & 31)) tops[t / 32] = top;
        }
        const float total16 = warp_sums_of_power<16>(v);  // of token g * 16 + lane / 2
        const float mine = __shfl_sync(0xffffffffu, total16, (lane & 15) * 2);
        if (lane / 16 == (g & 1) || TOKENS <= 16) sums[g / 2] = mine;
      }
#pragma unroll
      for (int j = 0; j < (TOKENS + 31) / 32; ++j) {
        if (TOKENS <= 16 && lane >= 16) continue;
        const float now = fmaxf(most[j], tops[j]), base = now == -INFINITY ? 0.0f : now;
        sum[j] = sum[j] * exp2_fast(most[j] - base) + sums[j] * exp2_fast(tops[j] - base);
        most[j] = now;
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_only(smem_u32(&acc_empty[n & 1]));
    }
    // the four warps' pairs, for one part a CTA
#pragma unroll
    for (int j = 0; j < (TOKENS + 31) / 32; ++j)
      if (j * 32 + lane < TOKENS) joined[quad][j * 32 + lane] = make_float2(most[j], sum[j]);
    __syncwarp();
    asm volatile("bar.sync 1, 128;" ::: "memory");
    const int t = threadIdx.x - 64;
    if (t < TOKENS && t < rows.n) {
      float2 all = joined[0][t];
#pragma unroll
      for (int q = 1; q < 4; ++q) {
        const float2 v = joined[q][t];
        const float now = fmaxf(all.x, v.x), base = now == -INFINITY ? 0.0f : now;
        all = make_float2(now, all.y * exp2_fast(all.x - base) + v.y * exp2_fast(v.x - base));
      }
      rows.parts[int64_t(blockIdx.x) * rows.stride + t] = all;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, kColumns);
}

// dx = E w and dw = E^T x' in one launch of pairs of CTAs. A tile of dx has all classes as its K, one of dw all tokens of the group, and there may be fewer tiles of dx than pairs: those
// are taken first, by whoever comes for the next tile, and those of dw fill up what is left, so that all end together. dx's K is cut in parts where a
// single tile would take longer than that. (Shared out beforehand by their slabs, 4096 x 768 x 50304 took 417 to 428 us, for 407 to 414.)
struct Task {
  bool x;
  TileAt at;
  int part, slab0, slabs;
};
__device__ __forceinline__ bool task_of(const Gradients& g, int i, Task& t) {
  t.x = i < g.x.total;
  if (!t.x) i -= g.x.total;
  const Result& r = t.x ? g.x : g.w;
  if (i >= r.total) return false;
  t.part = i / r.per;
  i -= t.part * r.per;
  t.slab0 = t.part * r.slabs;
  t.slabs = min(r.slabs, (r.K + kSlabK - 1) / kSlabK - t.slab0);
  t.at.m0 = i / r.tiles_n * 256;
  t.at.n0 = i % r.tiles_n * 256;
  return true;
}
// Rank 0's copies take the pair's next tile, and tell all of its warps (both CTAs'). A slot is written again when all have read it: they give it back with what orders their reads before
// that, rank 0's warps in their CTA, rank 1's in the cluster. (The latter takes much longer: by rank 0's products and epilogue too, loss and gradients of 1229 x 1024 x 30592 took 244 us, for
// 236. Rank 1's slots given back by a warp that does nothing else: the same.)
__device__ __forceinline__ bool tell_task(const Shared& s, Ring& ring, int id) {
  const int lane = threadIdx.x & 31;
  if (ring.round > 0 && !warp_wait<true>(&s.task_empty[ring.stage], (ring.round - 1) & 1)) return false;
  if (lane < 2) {
    store_cluster(cluster_address(const_cast<const int*>(&s.task[ring.stage]), uint32_t(lane)), id);
    mbar_arrive_at(cluster_address(&s.task_full[ring.stage], uint32_t(lane)));
  }
  __syncwarp();
  ring.next(kTasks);
  return true;
}
__device__ __forceinline__ bool read_task(const Shared& s, uint32_t rank, Ring& ring, int& id) {
  if (!warp_wait<true>(&s.task_full[ring.stage], ring.round & 1)) return false;
  id = s.task[ring.stage];
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    if (rank == 0) mbar_arrive(&s.task_empty[ring.stage]);
    else mbar_arrive_at(rank0_address(&s.task_empty[ring.stage]));
  }
  ring.next(kTasks);
  return true;
}
template <typename T>
__device__ __forceinline__ void add_columns(const Columns& c, int warp, int warps) {
  const int lane = threadIdx.x & 31;
  for (int task = warp; task < c.blocks * c.shares; task += warps) {
    const int share = task / c.blocks, from = share * c.share, to = min(c.n, from + c.share);
    const int64_t col = int64_t(task - share * c.blocks) * 256 + lane * 8;
    if (col >= c.e_stride) continue;
    const T* e = static_cast<const T*>(c.e) + col;
    float acc[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.0f;
#pragma unroll 8
    for (int r = from; r < to; ++r) {
      dev::Raw8<T> raw;
      dev::fetch(e + r * c.e_stride, raw);
      const float f = c.factor[r];
      float v[8];
      dev::unpack(raw, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] = __fmaf_rn(v[k], f, acc[k]);
    }
    float4* out = reinterpret_cast<float4*>(c.partial + share * c.e_stride + col);
    out[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    out[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
  }
}
// (The epilogue's warps have the bias's gradient to add up while the first tiles are made: 1229 x 30592 in a kernel of its own took 18 us.)
template <typename T>
__global__ void __launch_bounds__(kThreads, 1) ce_gradients_kernel(const __grid_constant__ GradientMaps maps, const __grid_constant__ Gradients g) {
  extern __shared__ uint8_t smem_raw[];
  const Shared s = shared_parts(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  if (threadIdx.x == 0) {
    prefetch_tensormap(&maps.e_rows);
    prefetch_tensormap(&maps.w);
    prefetch_tensormap(&maps.e_columns);
    prefetch_tensormap(&maps.xs);
  }
  const uint32_t tmem = products_begin<true>(s);
  may_follow();
  follow();
  Task t;
  int id = 0;
  Ring tasks;
  // The next tile is asked for, told and worked out while this one's last slabs are on their way. (Behind them, the copies began 1200 to 2500 cycles after the products could have, and those
  // 500 later for theirs: 4096 x 768 x 50304 a tile of 64 slabs 37000 cycles, of them 33000 for products.)
  if (warp == 0) {
    Ring ring;
    int ahead = 0;  // in lane 0
    bool ok = true;
    if (rank == 0) {
      if (lane == 0) ahead = atomicAdd(g.next, 1);
      id = __shfl_sync(0xffffffffu, ahead, 0);
      ok = tell_task(s, tasks, id);
    } else {
      ok = read_task(s, rank, tasks, id);
    }
    while (ok && task_of(g, id, t)) {
      const Task now = t;
      const int ask = max(0, now.slabs - 14), tell = rank == 0 ? max(0, now.slabs - 7) : max(0, now.slabs - 3);
      ok = load_tile<true>(s, now.x ? &maps.e_rows : &maps.e_columns, now.x ? &maps.w : &maps.xs, !now.x, true, now.at, rank, now.slab0, now.slabs, now.x ? INT_MAX : g.w_again, ring, [&](int k) {
        if (rank == 0) {
          if (k == ask && lane == 0) ahead = atomicAdd(g.next, 1);
          if (k != tell) return true;
          id = __shfl_sync(0xffffffffu, ahead, 0);
          return tell_task(s, tasks, id);
        }
        return k != tell || read_task(s, rank, tasks, id);
      });
    }
    if (!ok) *s.failed = 1;
    drain_loads(s, rank, ring);
  } else if (warp == 1) {
    if (rank == 0) {
      Ring ring;
      bool ok = read_task(s, rank, tasks, id);
      for (int k = 0; ok && task_of(g, id, t); ++k) {
        const Task now = t;
        ok = multiply_tile<true, std::is_same<T, __nv_bfloat16>::value>(s, tmem, !now.x, true, now.slabs, k, ring, [&](int slab) { return slab + 1 != now.slabs || read_task(s, rank, tasks, id); });
      }
      if (!ok) drain_products<true>(s);
    }
  } else {
    uint32_t used = 0;
    if (g.columns.partial != nullptr) add_columns<T>(g.columns, int(blockIdx.x) * kEpilogueWarps + warp - 2, int(gridDim.x) * kEpilogueWarps);
    for (int k = 0;; ++k) {
      auto finish = [&](int n) { finish_result<T>(s, tmem, t.x ? g.x : g.w, g.alpha, t.x ? &maps.out_x : &maps.out_w, t.at, t.part, rank, n, used); };
      if (!read_task(s, rank, tasks, id)) {  // nobody knows what is missing: all of it is not a number
        *s.failed = 1;
        for (int i = 0; task_of(g, i, t); ++i) finish(i);
        break;
      }
      if (!task_of(g, id, t)) break;
      finish(k);
    }
    if (lane == 0) bulk_wait_read();
  }
  products_end<true>(tmem);
}

// ---- what goes before, between and behind the products -----------------------------------------------------------------------

constexpr int kBeginT = 256;
constexpr int kRowsT = 1024;
constexpr int kRowsAtOnce = 32;   // rows of a CTA, one for each lane, and one for each warp
constexpr int kWeightsT = 256;
constexpr int kTops = kWeightsT;  // CTAs that look at x (Begin), one for each thread of who joins them

// Of the whole call. alpha: what G's rows are multiplied by in the end; unit: the largest finite weight of a row, by which the weights are divided (1 where all are 0); plain: alpha for rows of
// x as they are.
struct Scales {
  float alpha, unit, plain;
};

struct Begin {
  NangilaLinearCeParams p;
  int what;
  float *zt, *ref; // [n] the targets' logits, and as references; NULL: not wanted
  float* bias;    // padded to whole tiles
  int bias_count;
  Scales* scales;
  int* next;      // [groups] of the gradients' tiles; set to 0
  int64_t groups;
  float e_scale;  // power of two by which E is larger
  float* tops;    // [top_ctas] the largest |upstream x| of the rows that a CTA has looked at; NULL: not wanted
  int top_ctas;
};
__device__ __forceinline__ float bias_value(const void* b, int dtype, int i) {
  return dtype == NANGILA_F32 ? static_cast<const float*>(b)[i] : dtype == NANGILA_F16 ? __half2float(static_cast<const __half*>(b)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(b)[i]);
}
__device__ __forceinline__ void put_bias_value(void* b, int dtype, int64_t i, float v) {
  if (dtype == NANGILA_F32) static_cast<float*>(b)[i] = v;
  else if (dtype == NANGILA_F16) static_cast<__half*>(b)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(b)[i] = __float2bfloat16_rn(v);
}
// Row i's logit at its target, by a warp; 0 where that is no class or ignored.
template <typename T>
__device__ __forceinline__ float target_logit(const NangilaLinearCeParams& p, int64_t i) {
  const int64_t t = p.targets[i];
  if (t < 0 || t >= p.classes || t == p.ignore) return 0.0f;
  const int lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(p.x) + i * p.x_stride;
  const T* w = static_cast<const T*>(p.w) + t * p.w_stride;
  float z = 0.0f;
  constexpr int kAtOnce = 4;
  for (int c0 = lane * 8; c0 < p.d; c0 += 256 * kAtOnce) {
    dev::Raw8<T> rx[kAtOnce], rw[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (c0 + 256 * j >= p.d) continue;
      dev::fetch(x + c0 + 256 * j, rx[j]);
      dev::fetch(w + c0 + 256 * j, rw[j]);
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (c0 + 256 * j >= p.d) continue;
      float u[8], v[8];
      dev::unpack(rx[j], u);
      dev::unpack(rw[j], v);
#pragma unroll
      for (int k = 0; k < 8; ++k) z = __fmaf_rn(u[k], v[k], z);
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) z += __shfl_xor_sync(0xffffffffu, z, off);
  return z + (p.bias != nullptr ? bias_value(p.bias, p.bias_dtype, int(t)) : 0.0f);
}
// The largest |upstream x| of row i, by a warp; 0 where the row adds nothing or either is not finite.
template <typename T>
__device__ __forceinline__ float weighted_top(const NangilaLinearCeParams& p, int64_t i) {
  const int64_t t = p.targets[i];
  const float u = fabsf(p.upstream[i]);
  if (t < 0 || t >= p.classes || t == p.ignore || !(u < INFINITY)) return 0.0f;
  const T* x = static_cast<const T*>(p.x) + i * p.x_stride;
  float top = 0.0f;
#pragma unroll 4
  for (int c = (threadIdx.x & 31) * 8; c < p.d; c += 256) {
    dev::Raw8<T> raw;
    dev::fetch(x + c, raw);
    float v[8];
    dev::unpack(raw, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(v[k]));
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  return top < INFINITY ? fminf(top * u, 3e38f) : 0.0f;
}
// CTA 0: how many targets are not ignored, the largest weight, and the factors that follow. The others: the targets' logits, a warp for each row; the bias in fp32; the largest |upstream x|.
template <typename T>
__global__ void __launch_bounds__(kBeginT) ce_begin_kernel(const __grid_constant__ Begin a) {
  const NangilaLinearCeParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.x == 0) {
    __shared__ int64_t counts[kBeginT / 32];
    __shared__ float tops[kBeginT / 32];
    if (a.what != NANGILA_CE_LOSSES)
      for (int64_t i = threadIdx.x; i < a.groups; i += kBeginT) a.next[i] = 0;
    int64_t count = 0;
    float top = 0.0f;
    for (int64_t i = threadIdx.x; i < p.n; i += kBeginT) {
      const int64_t t = p.targets[i];
      count += t != p.ignore ? 1 : 0;
      if (p.upstream_rows && t >= 0 && t < p.classes && t != p.ignore) {
        const float u = fabsf(p.upstream[i]);
        if (u < INFINITY) top = fmaxf(top, u);  // (the others' rows alone are not finite: row_weight)
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      count += __shfl_xor_sync(0xffffffffu, count, off);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    }
    if (lane == 0) counts[warp] = count, tops[warp] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kBeginT / 32; ++w) {
        count += counts[w];
        top = fmaxf(top, tops[w]);
      }
      if (top == 0.0f) top = 1.0f;
      float u = 1.0f;
      if (a.what == NANGILA_CE_GRADIENTS) u = p.upstream_rows ? top : *p.upstream;
      if (p.mean) u = count > 0 ? u / float(count) : 0.0f;
      a.scales->alpha = a.scales->plain = u / a.e_scale;
      a.scales->unit = p.upstream_rows ? top : 1.0f;
    }
    return;
  }
  const int64_t thread = int64_t(blockIdx.x - 1) * kBeginT + threadIdx.x, threads = int64_t(gridDim.x - 1) * kBeginT;
  if (p.bias != nullptr)
    for (int64_t i = thread; i < a.bias_count; i += threads) a.bias[i] = i < p.classes ? bias_value(p.bias, p.bias_dtype, int(i)) : 0.0f;
  if (a.tops != nullptr && int(blockIdx.x) <= a.top_ctas) {
    __shared__ float largest[kBeginT / 32];
    float top = 0.0f;
    for (int64_t i = thread / 32; i < p.n; i += int64_t(a.top_ctas) * (kBeginT / 32)) top = fmaxf(top, weighted_top<T>(p, i));
    if (lane == 0) largest[warp] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kBeginT / 32; ++w) top = fmaxf(top, largest[w]);
      a.tops[blockIdx.x - 1] = top;
    }
  }
  if (a.zt == nullptr) return;
  for (int64_t i = thread / 32; i < p.n; i += threads / 32) {
    const float z = target_logit<T>(p, i);
    if (lane == 0) {
      a.zt[i] = z;
      a.ref[i] = z * kLog2e;
    }
  }
}

// The rows of a group, before their tiles are made (gradients from lse) or behind them.
struct Group {
  NangilaLinearCeParams p;   // of the whole call
  int64_t row0, stride;      // the group's first row; of `parts`
  int n, parts_count;
  const float* zt;           // [n] of the group, as are the following
  const float2* parts;
  float *ref, *mul, *value, *factor;
  int32_t* again;            // [groups of 32 rows]; both passes of NANGILA_CE_BOTH
  void* e;                   // [n][e_stride]
  void* xs;                  // [n][d]: rows of x as dw's product takes them
  int rests;                 // not 0: xs has so many rows, zeros behind n, and as many again of what their rounding left over
  int64_t e_stride;
  Scales* scales;
  float e_scale;
  const float* tops;         // as in Begin
  int top_ctas;
};
// Eight values of a row of x', and with rests what their rounding left over. What would round to an infinity is rounded to the largest value: the rest has the difference.
template <typename T>
__device__ __forceinline__ void put_scaled(const Group& a, int64_t at, float (&v)[8]) {
  dev::Raw8<T> raw;
  if (a.rests != 0) {
    float left[8];
    if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int k = 0; k < 8; ++k) left[k] = v[k], v[k] = isfinite(v[k]) ? fminf(fmaxf(v[k], -65504.0f), 65504.0f) : v[k];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) left[k] = v[k];
    }
    dev::pack(v, raw);
    dev::put(static_cast<T*>(a.xs) + at, raw);
    dev::unpack(raw, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = isfinite(v[k]) ? left[k] - v[k] : 0.0f;
    at += int64_t(a.rests) * a.p.d;
  }
  dev::pack(v, raw);
  dev::put(static_cast<T*>(a.xs) + at, raw);
}
// The factor with which a row's element at the target, as it was rounded, comes out as `value`; where that is too small to tell, the factor it had. (The target's element is half
// of a row's gradient, and often all that a class gets from it: its rounding goes into the factor, where it moves each of the others by as much as
// their own roundings do. The encoder's loss: dx 1.4 -> 1.1 times the error that the results' rounding alone has, dw 1.7 -> 1.4.)
__device__ __forceinline__ float folded(float value, float rounded, float factor) {
  return fabsf(rounded) > 1e-4f && fabsf(rounded) < 1e30f ? value / rounded : factor;
}
// A CTA's rows: losses and lse of the joined sums; with E also the element at the target and the rows' factors.
template <typename T>
__device__ __forceinline__ void join_rows(const Group& a, int pass, const float* logit) {
  constexpr int kWarps = kRowsT / 32;
  __shared__ float2 joined[kWarps][kRowsAtOnce];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * kRowsAtOnce + lane;
  const bool here = row < a.n;
  const float ref = pass != 0 && here ? a.ref[row] : 0.0f;
  float most = -INFINITY, sum = 0.0f;
  auto add = [&](const float2 v) {
    if (pass == 0) {
      const float now = fmaxf(most, v.x), base = now == -INFINITY ? 0.0f : now;
      sum = sum * exp2_fast(most - base) + v.y * exp2_fast(v.x - base);
      most = now;
    } else {
      most = fmaxf(most, v.x);
      sum += v.y;
    }
  };
  if (here) {
#pragma unroll 8
    for (int i = warp; i < a.parts_count; i += kWarps) add(a.parts[int64_t(i) * a.stride + row]);
  }
  joined[warp][lane] = make_float2(most, sum);
  __syncthreads();
  if (warp != 0) return;
  for (int w = 1; w < kWarps; ++w) add(joined[w][lane]);
  bool above = false;
  if (here) {
    const int64_t i = a.row0 + row, t = a.p.targets[i];
    const bool ignored = t == a.p.ignore, outside = !ignored && (t < 0 || t >= a.p.classes);
    const float zt2 = (pass == 0 ? logit[lane] : a.zt[row]) * kLog2e;
    float loss, lse2, factor = 0.0f;
    if (pass == 0) {
      // sum of exp2(z - most) over the others; the target's own on top
      const float base = fmaxf(most, zt2);
      const float rest = sum * exp2_fast(most - base), own = exp2_fast(zt2 - base);
      lse2 = base + log2f(rest + own);
      loss = zt2 >= most ? log1pf(sum * exp2_fast(most - zt2)) : (base - zt2) * kLn2 + logf(rest + own);
    } else {
      const float own = exp2_fast(zt2 - ref), whole = sum + own;
      above = pass == 1 && !ignored && !outside && most - ref > kMostAbove;
      factor = 1.0f / whole;
      lse2 = ref + log2f(whole);
      loss = ref == zt2 ? log1pf(sum) : (ref - zt2) * kLn2 + logf(whole);
      if (above) a.ref[row] = most;  // (more than z_t: the largest of the row)
      if (!ignored && !outside) {
        const T element = dev::Vec16<T>::from_float(-sum);
        static_cast<T*>(a.e)[int64_t(row) * a.e_stride + t] = element;
        factor = folded(sum / whole, -dev::Vec16<T>::to_float(element), factor);
      }
    }
    if (ignored || outside) {
      loss = ignored ? 0.0f : __uint_as_float(0x7fc00000u);
      factor = 0.0f;
    }
    a.p.losses[i] = loss;
    if (a.p.losses_too != nullptr) a.p.losses_too[i] = loss;
    a.p.lse[i] = lse2 * kLn2;
    if (pass != 0) a.factor[row] = factor;
  }
  if (pass == 1) {
    const bool any = __any_sync(0xffffffffu, above);
    if (lane == 0) a.again[blockIdx.x] = any ? 1 : 0;
  }
}
// NANGILA_CE_LOSSES (pass 0), and NANGILA_CE_BOTH's first pass over all rows (1).
template <typename T>
__global__ void __launch_bounds__(kRowsT) ce_rows_kernel(const __grid_constant__ Group a, int pass) {
  __shared__ float logit[kRowsAtOnce];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x * kRowsAtOnce + warp;
  if (pass == 0 && row < a.n) {
    const float z = target_logit<T>(a.p, a.row0 + row);
    if (lane == 0) logit[warp] = z;
  }
  follow();
  if (pass == 0) __syncthreads();
  join_rows<T>(a, pass, logit);
}
// NANGILA_CE_BOTH: the rows of tiles that were formed again once more, and the rows of x times their factors, as dw's product takes them; blockIdx.y: a share of those. (Each share
// joins the rows for itself, and writes the same.)
template <typename T>
__global__ void __launch_bounds__(kRowsT) ce_scale_kernel(const __grid_constant__ Group a, int tile_rows) {
  follow();
  const int all = (a.n + kRowsAtOnce - 1) / kRowsAtOnce, tile = tile_rows / kRowsAtOnce, first = int(blockIdx.x) / tile * tile;
  bool any = false;
  for (int i = first; i < min(first + tile, all); ++i) any = any || a.again[i] != 0;
  if (any) {
    join_rows<T>(a, 2, nullptr);
    __syncthreads();
  }
  if (a.xs == nullptr) return;
  const int per = a.p.d / 8, row0 = blockIdx.x * kRowsAtOnce, last = blockIdx.x + 1 == gridDim.x, rows = last ? max(a.n, a.rests) - row0 : kRowsAtOnce;
#pragma unroll 4
  for (int i = blockIdx.y * kRowsT + threadIdx.x; i < rows * per; i += kRowsT * gridDim.y) {
    const int r = i / per, row = row0 + r;
    const float f = row < a.n ? a.factor[row] : 0.0f;
    dev::Raw8<T> raw;
    dev::fetch(static_cast<const T*>(a.p.x) + (a.row0 + min(row, a.n - 1)) * a.p.x_stride + (i - r * per) * 8, raw);
    float v[8];
    dev::unpack(raw, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = f == 0.0f ? 0.0f : v[k] * f;
    put_scaled<T>(a, int64_t(row0) * a.p.d + int64_t(i) * 8, v);
  }
}
// A row's weight, upstream over the largest one, as share * 2^power with a share above 1/2, up to 1: the share goes into E, where it is rounded with the rest, the power into the row of x and the row's
// factor, which it does not round. A single upstream gradient is alpha, and its rows' weight one.
// In fp16 all rows of x' are as much larger, by a power of two that alpha takes back (`lift`), as the largest |upstream x| of the call lets them be: what x' loses below 2^-24 is then at most 2^-38 of
// that in dw, for each token and probability, and as much as the results' own subnormal steps where dw does not overflow. (As they were, a row of 2^-20 of the largest weight had four bits.) So a
// row of little weight keeps the digits of its own gradients in fp16 too. Looking at x costs 0.7 us at 1023 x 1000 (119.9 -> 120.6, loss and gradients).
struct RowWeight {
  float share;
  int power;
  bool lives;
};
__device__ __forceinline__ RowWeight row_weight(const Group& a, int64_t i, int lift) {
  const int64_t t = a.p.targets[i];
  RowWeight w{1.0f, 0, t != a.p.ignore && t >= 0 && t < a.p.classes};
  if (a.p.upstream_rows) {
    const float ratio = a.p.upstream[i] / a.scales->unit;
    // one that is not finite makes its row's share that, and touches no other row of dx
    w.share = isfinite(ratio) ? frexpf(ratio, &w.power) : __uint_as_float(0x7fc00000u);
    if (fabsf(w.share) == 0.5f) w.share *= 2.0f, --w.power;  // (the largest weight's row of x is not doubled: it may be near the type's largest value)
    w.power += lift;
  }
  if (!w.lives) w.share = 0.0f;
  return w;
}
// |x'| stays below 2^15: |x| 2^power is below twice the largest |upstream x| over the unit. By all threads of a CTA.
__device__ __forceinline__ int lift_of(const Group& a) {
  if (a.tops == nullptr) return 0;
  __shared__ float largest[kWeightsT / 32];
  const int lane = threadIdx.x & 31;
  float top = int(threadIdx.x) < a.top_ctas ? a.tops[threadIdx.x] : 0.0f;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  if (lane == 0) largest[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int w = 0; w < kWeightsT / 32; ++w) top = fmaxf(top, largest[w]);
  int power = 14;  // (all zeros, or weights so small that alpha would lose digits, where dw is zero in fp16 whatever x: as they are)
  if (top > 0.0f && a.scales->plain > 1e-28f) frexpf(top / a.scales->unit, &power);
  return max(0, min(30, 14 - power));
}
// NANGILA_CE_GRADIENTS: what the tiles' epilogue takes of each row, and the rows of x without those that add nothing.
template <typename T>
__global__ void __launch_bounds__(kWeightsT) ce_weights_kernel(const __grid_constant__ Group a) {
  follow();
  const int64_t thread = int64_t(blockIdx.x) * kWeightsT + threadIdx.x, threads = int64_t(gridDim.x) * kWeightsT;
  const int lift = lift_of(a);
  if (thread == 0 && a.tops != nullptr) a.scales->alpha = ldexpf(a.scales->plain, -lift);  // (by each group the same)
  auto value_of = [&](const RowWeight& w, int64_t i) { return expm1f(-a.p.losses[i]) * w.share * a.e_scale; };
  auto factor_of = [&](const RowWeight& w, float value) {
    return w.lives && w.share != 0.0f ? ldexpf(folded(value, dev::Vec16<T>::to_float(dev::Vec16<T>::from_float(value)), 1.0f), w.power) : 0.0f;
  };
  for (int64_t row = thread; row < a.n; row += threads) {
    const int64_t i = a.row0 + row;
    const RowWeight w = row_weight(a, i, lift);
    a.ref[row] = a.p.lse[i] * kLog2e;
    a.mul[row] = w.share * a.e_scale;
    const float value = value_of(w, i);
    a.value[row] = value;
    a.factor[row] = factor_of(w, value);
  }
  if (a.xs == nullptr) return;
  const int per = a.p.d / 8;
  if (a.rests != 0) {
    for (int64_t i = thread; i < int64_t(a.rests) * per; i += threads) {
      const int64_t row = i / per;
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.0f;
      const RowWeight w = row < a.n ? row_weight(a, a.row0 + row, lift) : RowWeight{0.0f, 0, false};
      if (w.lives) {
        const float f = factor_of(w, value_of(w, a.row0 + row));
        dev::Raw8<T> raw;
        dev::fetch(static_cast<const T*>(a.p.x) + (a.row0 + row) * a.p.x_stride + (i - row * per) * 8, raw);
        dev::unpack(raw, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= f;
      }
      put_scaled<T>(a, i * 8, v);
    }
    return;
  }
#pragma unroll 4
  for (int64_t i = thread; i < int64_t(a.n) * per; i += threads) {
    const int64_t row = i / per;
    const RowWeight w = row_weight(a, a.row0 + row, lift);
    dev::Raw8<T> raw;
    dev::fetch(static_cast<const T*>(a.p.x) + (a.row0 + row) * a.p.x_stride + (i - row * per) * 8, raw);
    if (w.power != 0) {
      float v[8];
      dev::unpack(raw, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = ldexpf(v[k], w.power);
      dev::pack(v, raw);
    }
    if (!w.lives) raw.a = make_uint4(0, 0, 0, 0);
    dev::put(static_cast<T*>(a.xs) + i * 8, raw);
  }
}
// What is left behind the products, each by its own CTAs of one launch.
struct Finish {
  const Scales* scales;
  // dx = alpha f_row times the sum of its parts
  const float *dx_parts, *factor;
  void* dx;
  int64_t dx_part, dx_count;    // values of a part, eights of dx
  int parts, per, dx_ctas;      // eights of a row
  // dw = alpha sums, zero behind the classes
  const float* dw_sums;
  void* dw;
  int64_t dw_count, dw_live;    // eights; of them the classes'
  int dw_ctas;
  // the bias's gradient out of the shares' sums of all groups
  const float* columns;
  void* dbias;
  int64_t columns_stride;
  int shares, classes, rows, dbias_dtype, bias_ctas;
  // the sum or mean of the losses
  const float* losses;
  const int64_t* targets;
  float* loss;
  int64_t n, ignore;
  int mean;
};
constexpr int kFinishT = 256;
// In a fixed order, in 64 bits.
__device__ __forceinline__ void total_loss(const Finish& a) {
  constexpr int kWarps = kFinishT / 32;
  __shared__ double part[kWarps], counted[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double sum = 0.0;
  int64_t count = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < a.n; i += kFinishT) {
    sum += double(a.losses[i]);
    count += a.targets[i] != a.ignore ? 1 : 0;
  }
  double counts = double(count);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, off);
    counts += __shfl_xor_sync(0xffffffffu, counts, off);
  }
  if (lane == 0) part[warp] = sum, counted[warp] = counts;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) sum += part[w], counts += counted[w];
    *a.loss = float(a.mean ? sum / counts : sum);
  }
}
template <typename T>
__global__ void __launch_bounds__(kFinishT) ce_finish_kernel(const __grid_constant__ Finish a) {
  follow();
  int cta = blockIdx.x;
  if (cta < a.dx_ctas) {
    const float alpha = a.scales->alpha;
    for (int64_t i = int64_t(cta) * kFinishT + threadIdx.x; i < a.dx_count; i += int64_t(a.dx_ctas) * kFinishT) {
      const float f = a.factor[i / a.per];
      float v[8], w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.0f;
#pragma unroll 4
      for (int j = 0; j < a.parts; ++j) {
        dev::Raw8<float> in;
        dev::fetch(a.dx_parts + j * a.dx_part + i * 8, in);
        dev::unpack(in, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += w[k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = f == 0.0f ? 0.0f : v[k] * (alpha * f);
      dev::Raw8<T> r;
      dev::pack(v, r);
      dev::put(static_cast<T*>(a.dx) + i * 8, r);
    }
    return;
  }
  cta -= a.dx_ctas;
  if (cta < a.dw_ctas) {
    const float alpha = a.scales->alpha;
#pragma unroll 4
    for (int64_t i = int64_t(cta) * kFinishT + threadIdx.x; i < a.dw_count; i += int64_t(a.dw_ctas) * kFinishT) {
      dev::Raw8<float> in;
      dev::fetch(a.dw_sums + i * 8, in);
      float v[8];
      dev::unpack(in, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = i < a.dw_live ? v[k] * alpha : 0.0f;
      dev::Raw8<T> r;
      dev::pack(v, r);
      dev::put(static_cast<T*>(a.dw) + i * 8, r);
    }
    return;
  }
  cta -= a.dw_ctas;
  if (cta < a.bias_ctas) {
    const int i = cta * kFinishT + threadIdx.x;
    if (i >= a.rows) return;
    float sum = 0.0f;
    if (i < a.classes) {
#pragma unroll 8
      for (int s = 0; s < a.shares; ++s) sum += a.columns[s * a.columns_stride + i];
      sum *= a.scales->alpha;
    }
    put_bias_value(a.dbias, a.dbias_dtype, i, sum);
    return;
  }
  total_loss(a);
}
// (What is zero stays so: rows that add nothing get nothing from a factor that is not finite either.)
__device__ __forceinline__ float rescaled(float v, float f) { return v == 0.0f ? v : v * f; }
template <typename T>
__device__ void rescale(T* a, int64_t n, float f) {
  const int64_t thread = int64_t(blockIdx.x) * blockDim.x + threadIdx.x, threads = int64_t(gridDim.x) * blockDim.x;
  const int64_t whole = (reinterpret_cast<uintptr_t>(a) & 15u) == 0 ? n / 8 : 0;
  for (int64_t i = thread; i < whole; i += threads) {
    dev::Raw8<T> raw;
    dev::fetch(a + i * 8, raw);
    float v[8];
    dev::unpack(raw, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = rescaled(v[k], f);
    dev::pack(v, raw);
    dev::put(a + i * 8, raw);
  }
  for (int64_t i = whole * 8 + thread; i < n; i += threads) a[i] = dev::Vec16<T>::from_float(rescaled(dev::Vec16<T>::to_float(a[i]), f));
}
__global__ void __launch_bounds__(256) rescale_kernel(const __grid_constant__ NangilaRescaleParams p) {
  const float f = *p.factor;
  if (p.wide != nullptr)
    for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < p.narrow_count; i += int64_t(gridDim.x) * blockDim.x) put_bias_value(p.narrow, p.narrow_dtype, i, rescaled(p.wide[i], f));
  if (f == 1.0f) return;
  for (int i = 0; i < 2; ++i) {
    if (p.array[i] == nullptr) continue;
    if (p.dtype[i] == NANGILA_F32) rescale(static_cast<float*>(p.array[i]), p.count[i], f);
    else if (p.dtype[i] == NANGILA_F16) rescale(static_cast<__half*>(p.array[i]), p.count[i], f);
    else rescale(static_cast<__nv_bfloat16*>(p.array[i]), p.count[i], f);
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
struct Matrix {
  const void* base;
  int64_t rows, cols, ld;
  CUtensorMapDataType type;
  int64_t parts = 1;  // one behind the other
};
// copied in boxes of box_inner x box_outer; what lies outside reads as zero and is not written
bool make_map(CUtensorMap* map, const Matrix& m, uint32_t box_inner, uint32_t box_outer) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const int size = m.type == CU_TENSOR_MAP_DATA_TYPE_FLOAT32 ? 4 : 2;
  const cuuint64_t dims[3] = {cuuint64_t(m.cols), cuuint64_t(m.rows), cuuint64_t(m.parts)};
  const cuuint64_t strides[2] = {cuuint64_t(m.ld) * size, cuuint64_t(m.ld) * size * cuuint64_t(m.rows)};
  const cuuint32_t box[3] = {box_inner, box_outer, 1}, step[3] = {1, 1, 1};
  return fn(map, m.type, 3, const_cast<void*>(m.base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
int sm_count() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  return sms[dev];
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

cudaLaunchConfig_t pairs_config(cudaLaunchAttribute (&attr)[2], int ctas, bool pair, cudaStream_t stream) {
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = pair ? 2 : 1;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pair ? 2 : 1;
  return cfg;
}
// The tiles of x w^T; e: where E goes.
template <typename T, int KIND, bool PAIR>
int launch_logits(const Matrix& x, const Matrix& w, const Matrix* e, const Rows& rows, cudaStream_t stream) {
  constexpr int kSide = PAIR ? 256 : 128;
  Maps maps;
  if (!make_map(&maps.a, x, 64, 128) || !make_map(&maps.b, w, 64, 128) || !make_map(&maps.out, e != nullptr ? *e : x, 64, 32)) return int(cudaErrorNotSupported);
  const int64_t tiles_m = (rows.n + kSide - 1) / kSide, total = tiles_m * ((rows.classes + kSide - 1) / kSide);
  if (total > 0x3fffffff) return int(cudaErrorInvalidValue);
  auto* kernel = ce_logits_kernel<T, KIND, PAIR>;
  if (const int err = allow_smem(reinterpret_cast<const void*>(kernel), kSmem)) return err;
  const int sms = sm_count();
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = pairs_config(attr, int(PAIR ? 2 * std::min<int64_t>(total, sms / 2) : std::min<int64_t>(total, sms)), PAIR, stream);
  return int(cudaLaunchKernelEx(&cfg, kernel, maps, rows, int(tiles_m), int(total), int((x.cols + kSlabK - 1) / kSlabK)));
}
// The sums of few tokens; a part of them for each CTA. (2048 x 32000, losses alone in a captured graph: 16 tokens 30.7 us and 43.0 with tokens as rows, 64 tokens 30.8 and 32.8; above that
// the accumulators' columns are as many as tokens' rows would be, 128 tokens 33.3.)
constexpr int kFewTokens = 64;
int few_ctas(int64_t classes) { return int(std::min<int64_t>((classes + kTileM - 1) / kTileM, sm_count())); }
template <typename T, int TOKENS>
int launch_few(const Matrix& x, const Matrix& w, const Rows& rows, cudaStream_t stream) {
  Maps maps;
  if (!make_map(&maps.a, w, 64, 128) || !make_map(&maps.b, x, 64, TOKENS) || !make_map(&maps.out, x, 64, TOKENS)) return int(cudaErrorNotSupported);
  auto* kernel = ce_few_kernel<T, TOKENS>;
  if (const int err = allow_smem(reinterpret_cast<const void*>(kernel), Few<TOKENS>::kBytes)) return err;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = pairs_config(attr, few_ctas(rows.classes), false, stream);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = Few<TOKENS>::kBytes;
  return int(cudaLaunchKernelEx(&cfg, kernel, maps, rows, int((rows.classes + kTileM - 1) / kTileM), int((x.cols + kSlabK - 1) / kSlabK)));
}
template <typename T>
int few(const Matrix& x, const Matrix& w, const Rows& rows, cudaStream_t stream) {
  return rows.n <= 16 ? launch_few<T, 16>(x, w, rows, stream) : rows.n <= 32 ? launch_few<T, 32>(x, w, rows, stream) : launch_few<T, 64>(x, w, rows, stream);
}
template <typename T, int KIND>
int logits(bool pair, const Matrix& x, const Matrix& w, const Matrix* e, const Rows& rows, cudaStream_t stream) {
  return pair ? launch_logits<T, KIND, true>(x, w, e, rows, stream) : launch_logits<T, KIND, false>(x, w, e, rows, stream);
}

Result result(int64_t M, int64_t N, int64_t K, int split) {
  Result r;
  std::memset(&r, 0, sizeof r);
  r.M = int(M);
  r.N = int(N);
  r.K = int(K);
  const int slabs = (r.K + kSlabK - 1) / kSlabK;
  r.slabs = (slabs + split - 1) / split;
  r.split = (slabs + r.slabs - 1) / r.slabs;
  r.tiles_n = (r.N + 255) / 256;
  r.per = (r.M + 255) / 256 * r.tiles_n;
  r.total = r.per * r.split;
  return r;
}
// Into how many parts dx's K is cut: as few as let a pair's tiles of dx end before its share of all work does. (Loss and gradients of n tokens at 2048 x 32000: n = 128 in one part 252 us,
// in two 187, in four 174, in eight 182; n = 1229 in one 440, in two 452, in four 463. These and the figures of kRestsTokens and of small tiles are of captured passes, which copy dx and dw
// once: some 40 us of each.)
int split_of(int64_t n, int64_t d, int64_t classes, int64_t rows, bool dw) {
  const int pairs = sm_count() / 2;
  const Result w = result(rows, d, n, 1);
  int best = 1;
  double least = 1e30;
  for (int split = 1; split <= 16; ++split) {
    const Result x = result(n, d, classes, split);
    if (split > 1 && x.slabs < 8) break;
    // (a tile of dw takes as long as eight slabs at least, what its results take; sums of a part go through memory: some three slabs' time a tile)
    const double share = (double(x.per) * ((x.K + kSlabK - 1) / kSlabK) + (dw ? double(w.total) * std::max(w.slabs, 8) : 0.0)) / pairs;
    const double busiest = double((x.total + pairs - 1) / pairs) * x.slabs;
    const double cost = std::max(share, busiest) + (split > 1 ? 3.0 * x.total / pairs : 0.0);
    if (cost < least * 0.99) least = cost, best = x.split;
  }
  return best;
}

// How a call is cut up, and where its parts lie in the workspace.
struct Plan {
  int64_t group;      // tokens at a time
  int64_t groups, e_stride, parts, shares, share;
  bool pair, few;     // tiles of the logits
  bool wide;          // dw is summed up over the groups
  int rests;          // rows of xs with their roundings' rests behind them; 0: without
  int split;          // parts of dx's K
  int64_t at_scales, at_next, at_tops, at_zt, at_bias, at_ref, at_mul, at_value, at_factor, at_again, at_parts, at_e, at_xs, at_sums, at_dx, at_columns, total;
  int64_t bias_count;
  int top_ctas;       // that look at x; 0: none
};
// Of E. (Each group more adds to dw in fp32: 8192 x 768 x 50304 with a quarter, a half and one gigabyte, four, two and one groups, 1780, 1660 and 1535 us.)
constexpr int64_t kGroupBytes = int64_t(1) << 30;
// Up to so many tokens dw's product has the rests of x' roundings too. A class's gradient is then often one token's, x times what is nearly -1: without them the rounding of x times the row's factor
// is its largest error, 1.4 times the one that the result's rounding alone makes and up to 28 times where that one is exact, with them 1.0 to 1.3. What it costs, bf16 x 2048 x 32000 with loss and dx:
// 16 tokens 166 -> 169 us, 128 tokens 165 -> 176, 256 tokens 182 -> 199; 512, where rounding shows less as classes have several tokens, would be 242 -> 286.
constexpr int kRestsTokens = 256;
Plan plan(const NangilaLinearCeParams& p, int what) {
  Plan l;
  std::memset(&l, 0, sizeof l);
  const int64_t classes = p.classes;
  l.e_stride = (classes + 63) / 64 * 64;
  // Tokens that one small tile has rows for take small tiles. (Loss and gradients at 2048 x 32000: 128 tokens 173.6 us, in pairs' tiles 174.2, losses alone 35 and 37; 200 tokens 209, and 198.)
  l.pair = p.n > 128;
  const int64_t side = l.pair ? 256 : 128, half = side / 2;
  l.few = what == NANGILA_CE_LOSSES && p.n <= kFewTokens;
  l.parts = l.few ? few_ctas(classes) : (classes + half - 1) / half;
  const int64_t row_bytes = what == NANGILA_CE_LOSSES ? l.parts * 8 : l.e_stride * 2;
  const int64_t most = std::max<int64_t>(256, (what == NANGILA_CE_LOSSES ? kGroupBytes / 16 : kGroupBytes) / row_bytes / 256 * 256);
  l.groups = (p.n + most - 1) / most;
  l.group = std::min(p.n, ((p.n + l.groups - 1) / l.groups + 255) / 256 * 256);
  l.groups = (p.n + l.group - 1) / l.group;
  l.wide = l.groups > 1 && p.dw != nullptr;
  l.bias_count = (classes + side - 1) / side * side;
  // rows of E that a warp adds up for the bias's gradient: a task for each of the epilogue's warps
  l.shares = std::max<int64_t>(1, std::min<int64_t>((l.group + 31) / 32, kEpilogueWarps * 148 / ((classes + 255) / 256)));
  l.share = (l.group + l.shares - 1) / l.shares;
  auto take = [&](int64_t bytes) {
    const int64_t at = l.total;
    l.total += (bytes + 255) / 256 * 256;
    return at;
  };
  l.at_scales = take(sizeof(Scales));
  l.at_next = take(l.groups * 4);
  l.top_ctas = what == NANGILA_CE_GRADIENTS && p.dtype == NANGILA_F16 && p.upstream_rows && p.dw != nullptr ? int(std::min<int64_t>((p.n + kBeginT / 32 - 1) / (kBeginT / 32), kTops)) : 0;
  l.at_tops = take(l.top_ctas * 4);
  l.at_zt = take(what == NANGILA_CE_BOTH ? p.n * 4 : 0);
  l.at_ref = take(what == NANGILA_CE_BOTH ? p.n * 4 : what == NANGILA_CE_GRADIENTS ? l.group * 4 : 0);
  l.at_bias = take(p.bias != nullptr ? l.bias_count * 4 : 0);
  l.at_parts = take(what == NANGILA_CE_GRADIENTS ? 0 : l.parts * l.group * 8);
  if (what == NANGILA_CE_LOSSES) return l;
  l.at_mul = take(what == NANGILA_CE_GRADIENTS ? l.group * 4 : 0);
  l.at_value = take(what == NANGILA_CE_GRADIENTS ? l.group * 4 : 0);
  l.at_factor = take(l.group * 4);
  l.at_again = take((l.group + 31) / 32 * 4);
  l.at_e = take(l.group * l.e_stride * 2);
  l.rests = p.dw != nullptr && p.n <= kRestsTokens ? int((p.n + kSlabK - 1) / kSlabK * kSlabK) : 0;
  l.at_xs = take(p.dw != nullptr ? std::max<int64_t>(l.group, 2 * l.rests) * p.d * 2 : 0);
  l.at_sums = take(l.wide ? int64_t(p.rows) * p.d * 4 : 0);
  l.split = p.dx != nullptr ? split_of(l.group, p.d, classes, p.rows, p.dw != nullptr) : 1;
  l.at_dx = take(l.split > 1 ? l.split * l.group * p.d * 4 : 0);
  l.at_columns = take(p.dbias != nullptr ? l.groups * l.shares * l.e_stride * 4 : 0);
  return l;
}

template <typename T>
int run(const NangilaLinearCeParams& p, int what, cudaStream_t stream) {
  const CUtensorMapDataType type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const Plan l = plan(p, what);
  auto* ws = static_cast<uint8_t*>(p.workspace);
  auto* scales = reinterpret_cast<Scales*>(ws + l.at_scales);
  auto* zt = reinterpret_cast<float*>(ws + l.at_zt);
  auto* bias = p.bias != nullptr ? reinterpret_cast<float*>(ws + l.at_bias) : nullptr;
  auto* sums = reinterpret_cast<float*>(ws + l.at_sums);
  auto* columns = reinterpret_cast<float*>(ws + l.at_columns);

  Begin begin;
  std::memset(&begin, 0, sizeof begin);
  begin.p = p;
  begin.what = what;
  begin.zt = what == NANGILA_CE_BOTH ? zt : nullptr;
  begin.ref = reinterpret_cast<float*>(ws + l.at_ref);
  begin.bias = bias;
  begin.bias_count = int(l.bias_count);
  begin.scales = scales;
  begin.next = reinterpret_cast<int*>(ws + l.at_next);
  begin.groups = l.groups;
  begin.tops = l.top_ctas != 0 ? reinterpret_cast<float*>(ws + l.at_tops) : nullptr;
  begin.top_ctas = l.top_ctas;
  begin.e_scale = what == NANGILA_CE_GRADIENTS && std::is_same<T, __half>::value ? 32768.0f : 1.0f;
  int e = 0;
  if (what != NANGILA_CE_LOSSES || p.bias != nullptr) {
    const int64_t work = std::max<int64_t>(what == NANGILA_CE_BOTH ? (p.n + kBeginT / 32 - 1) / (kBeginT / 32) : 0, p.bias != nullptr ? (l.bias_count + kBeginT - 1) / kBeginT : 0);
    ce_begin_kernel<T><<<unsigned(1 + std::max<int64_t>(std::min<int64_t>(work, 148 * 8), l.top_ctas)), kBeginT, 0, stream>>>(begin);
    e = int(cudaGetLastError());
  }

  auto losses_into = [&](Finish& f) {
    f.losses = p.losses;
    f.targets = p.targets;
    f.loss = p.loss;
    f.n = p.n;
    f.ignore = p.ignore;
    f.mean = p.mean;
  };

  for (int64_t g = 0; g < l.groups && e == 0; ++g) {
    Group a;
    std::memset(&a, 0, sizeof a);
    a.p = p;
    a.row0 = g * l.group;
    a.n = int(std::min(l.group, p.n - a.row0));
    a.stride = l.group;
    a.parts_count = int(l.parts);
    a.parts = reinterpret_cast<const float2*>(ws + l.at_parts);
    a.scales = scales;
    a.tops = begin.tops;
    a.top_ctas = begin.top_ctas;
    a.e_scale = begin.e_scale;
    Rows rows;
    std::memset(&rows, 0, sizeof rows);
    rows.targets = p.targets + a.row0;
    rows.bias = bias;
    rows.parts = what == NANGILA_CE_GRADIENTS ? nullptr : reinterpret_cast<float2*>(ws + l.at_parts);
    rows.stride = l.group;
    rows.ignore = p.ignore;
    rows.n = a.n;
    rows.classes = p.classes;
    const Matrix x{static_cast<const T*>(p.x) + a.row0 * p.x_stride, a.n, p.d, p.x_stride, type}, w{p.w, p.classes, p.d, p.w_stride, type};
    const unsigned row_ctas = unsigned((a.n + kRowsAtOnce - 1) / kRowsAtOnce);
    const int tile_rows = l.pair ? 256 : 128;
    if (what == NANGILA_CE_LOSSES) {
      e = l.few ? few<T>(x, w, rows, stream) : logits<T, kStats>(l.pair, x, w, nullptr, rows, stream);
      if (e == 0) e = int(launch_following(ce_rows_kernel<T>, dim3(row_ctas), kRowsT, 0, stream, a, 0));
      continue;
    }
    a.ref = reinterpret_cast<float*>(ws + l.at_ref) + (what == NANGILA_CE_BOTH ? a.row0 : 0);
    a.factor = reinterpret_cast<float*>(ws + l.at_factor);
    a.e = ws + l.at_e;
    a.e_stride = l.e_stride;
    a.xs = p.dw != nullptr ? ws + l.at_xs : nullptr;
    a.rests = l.rests;
    rows.ref = a.ref;
    const Matrix ex{a.e, a.n, p.classes, l.e_stride, type};
    if constexpr (!std::is_same<T, __half>::value) if (what == NANGILA_CE_BOTH) {
      a.zt = zt + a.row0;
      a.again = reinterpret_cast<int32_t*>(ws + l.at_again);
      e = logits<T, kExp>(l.pair, x, w, &ex, rows, stream);
      if (e == 0) e = int(launch_following(ce_rows_kernel<T>, dim3(row_ctas), kRowsT, 0, stream, a, 1));
      rows.again = a.again;
      if (e == 0) e = logits<T, kExp>(l.pair, x, w, &ex, rows, stream);
      // So many shares that there are CTAs for all SMs, if rows are long enough. (16 x 2048 x 32000 4.7 us, in one share 14.)
      const unsigned row_shares = a.xs == nullptr ? 1u : unsigned(std::max<int64_t>(1, std::min<int64_t>(2 * 148 / row_ctas, (int64_t(kRowsAtOnce) * p.d / 8 + kRowsT - 1) / kRowsT)));
      if (e == 0) e = int(launch_following(ce_scale_kernel<T>, dim3(row_ctas, row_shares), kRowsT, 0, stream, a, tile_rows));
    }
    if (what == NANGILA_CE_GRADIENTS) {
      a.mul = reinterpret_cast<float*>(ws + l.at_mul);
      a.value = reinterpret_cast<float*>(ws + l.at_value);
      e = int(launch_following(ce_weights_kernel<T>, dim3(unsigned(std::min<int64_t>((int64_t(a.n) * p.d / 8 + kWeightsT - 1) / kWeightsT, 148 * 8))), kWeightsT, 0, stream, a));
      rows.mul = a.mul;
      rows.value = a.value;
      if (e == 0) e = logits<T, kWeighted>(l.pair, x, w, &ex, rows, stream);
    }
    if (e == 0) {
      Gradients q;
      std::memset(&q, 0, sizeof q);
      q.alpha = &scales->alpha;
      if (p.dbias != nullptr) q.columns = {a.e, a.factor, columns + g * l.shares * l.e_stride, l.e_stride, a.n, int((p.classes + 255) / 256), int(l.shares), int(l.share)};
      GradientMaps maps;
      bool ok = make_map(&maps.e_rows, ex, 64, 128) && make_map(&maps.e_columns, ex, 64, 64) && make_map(&maps.w, w, 64, 64) && make_map(&maps.xs, x, 64, 64) && make_map(&maps.out_x, x, 64, 32) &&
                make_map(&maps.out_w, x, 64, 32);  // (those that are not wanted are not used)
      if (p.dx != nullptr) {
        q.x = result(a.n, p.d, p.classes, l.split);
        q.x.live = a.n;
        q.x.factor = a.factor;
        q.x.wide = q.x.split > 1 ? 1 : 0;
        const Matrix out{static_cast<T*>(p.dx) + a.row0 * p.d, a.n, p.d, p.d, type}, parts{ws + l.at_dx, a.n, p.d, p.d, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, q.x.split};
        ok = ok && (q.x.wide ? make_map(&maps.out_x, parts, 32, 32) : make_map(&maps.out_x, out, 64, 32));
      }
      if (p.dw != nullptr) {
        q.w = result(p.rows, p.d, l.rests != 0 ? 2 * l.rests : a.n, 1);
        q.w_again = l.rests != 0 ? l.rests : INT_MAX;
        q.w.live = p.classes;  // (zeros of E times what is not finite would not be zero)
        q.w.wide = !l.wide ? 0 : g == 0 ? 1 : 2;
        const Matrix xs{a.xs, l.rests != 0 ? 2 * l.rests : a.n, p.d, p.d, type}, out{p.dw, p.rows, p.d, p.d, type}, wide{sums, p.rows, p.d, p.d, CU_TENSOR_MAP_DATA_TYPE_FLOAT32};
        ok = ok && make_map(&maps.xs, xs, 64, 64) && (l.wide ? make_map(&maps.out_w, wide, 32, 32) : make_map(&maps.out_w, out, 64, 32));
      }
      if (!ok) return int(cudaErrorNotSupported);
      q.next = begin.next + g;
      auto* kernel = ce_gradients_kernel<T>;
      if (const int err = allow_smem(reinterpret_cast<const void*>(kernel), kSmem)) return err;
      cudaLaunchAttribute attr[2];
      const cudaLaunchConfig_t cfg = pairs_config(attr, 2 * (p.dbias != nullptr ? sm_count() / 2 : std::min(q.x.total + q.w.total, sm_count() / 2)), true, stream);
      e = int(cudaLaunchKernelEx(&cfg, kernel, maps, q));
      if (e == 0) {
        auto ctas_of = [](int64_t work) { return int(std::min<int64_t>((work + kFinishT - 1) / kFinishT, 148 * 8)); };
        const bool last = g + 1 == l.groups, total = last && what == NANGILA_CE_BOTH && p.loss != nullptr;
        Finish f;
        std::memset(&f, 0, sizeof f);
        f.scales = scales;
        if (q.x.wide) {
          f.dx_parts = reinterpret_cast<const float*>(ws + l.at_dx);
          f.factor = a.factor;
          f.dx = static_cast<T*>(p.dx) + a.row0 * p.d;
          f.dx_part = int64_t(a.n) * p.d;
          f.dx_count = f.dx_part / 8;
          f.parts = q.x.split;
          f.per = int(p.d / 8);
          f.dx_ctas = ctas_of(f.dx_count);
        }
        if (last && l.wide) {
          f.dw_sums = sums;
          f.dw = p.dw;
          f.dw_count = int64_t(p.rows) * p.d / 8;
          f.dw_live = int64_t(p.classes) * p.d / 8;
          f.dw_ctas = ctas_of(f.dw_count);
        }
        if (last && p.dbias != nullptr) {
          f.columns = columns;
          f.dbias = p.dbias;
          f.columns_stride = l.e_stride;
          f.shares = int(l.groups * l.shares);
          f.classes = p.classes;
          f.rows = p.rows;
          f.dbias_dtype = what == NANGILA_CE_BOTH ? NANGILA_F32 : p.bias_dtype;  // (rounded when the upstream gradient is known: nangila_rescale)
          f.bias_ctas = int((p.rows + kFinishT - 1) / kFinishT);
        }
        const int ctas = f.dx_ctas + f.dw_ctas + f.bias_ctas + (total ? 1 : 0);
        if (total) losses_into(f);
        if (ctas > 0) e = int(launch_following(ce_finish_kernel<T>, dim3(unsigned(ctas)), kFinishT, 0, stream, f));
      }
    }
  }
  if (e == 0 && what == NANGILA_CE_LOSSES && p.loss != nullptr) {
    Finish f;
    std::memset(&f, 0, sizeof f);
    losses_into(f);
    e = int(launch_following(ce_finish_kernel<T>, dim3(1), kFinishT, 0, stream, f));
  }
  return e;
}

bool aligned(const void* p, unsigned to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
bool sound(const NangilaLinearCeParams* p, int what) {
  if (!p || what < 0 || what > 2 || p->n < 1 || p->n > (int64_t(1) << 40) || p->d < 8 || p->d % 8 != 0 || p->d > NANGILA_CE_MAX_WIDTH || p->classes < 1 || p->rows < p->classes ||
      p->rows > NANGILA_CE_MAX_CLASSES)
    return false;
  if (p->dtype != NANGILA_BF16 && p->dtype != NANGILA_F16) return false;
  return what != NANGILA_CE_BOTH || p->dtype == NANGILA_BF16;
}

}  // namespace
}  // namespace nangila

extern "C" int64_t nangila_linear_ce_workspace(const NangilaLinearCeParams* p, int what) { return nangila::sound(p, what) ? nangila::plan(*p, what).total : -1; }

extern "C" int nangila_linear_ce(const NangilaLinearCeParams* p, int what, cudaStream_t stream) {
  using namespace nangila;
  if (!sound(p, what) || !p->x || !p->w || !p->targets || !p->losses || !p->workspace || !aligned(p->workspace, 256) || !aligned(p->x, 16) || !aligned(p->w, 16) || p->x_stride % 8 != 0 ||
      p->w_stride % 8 != 0 || p->x_stride < p->d || p->w_stride < p->d || !aligned(p->dx, 16) || !aligned(p->dw, 16) || (p->dbias != nullptr && p->bias == nullptr) ||
      !p->lse || (what == NANGILA_CE_GRADIENTS && !p->upstream))
    return int(cudaErrorInvalidValue);
  try {
    return p->dtype == NANGILA_BF16 ? run<__nv_bfloat16>(*p, what, stream) : run<__half>(*p, what, stream);
  } catch (...) {  // (the host's tables of kernels that were set up allocate)
    return int(cudaErrorMemoryAllocation);
  }
}

extern "C" int nangila_rescale(const NangilaRescaleParams* p, cudaStream_t stream) {
  using namespace nangila;
  if (!p || !p->factor || (p->wide && !p->narrow)) return int(cudaErrorInvalidValue);
  rescale_kernel<<<148 * 4, 256, 0, stream>>>(*p);
  return int(cudaGetLastError());
}

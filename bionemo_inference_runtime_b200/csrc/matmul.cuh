// The tensor-core products of the trainable dense layers (sm_100a): D[m, n] = sum_k A[m, k] B[n, k], finished in one of
// six forms, for bf16 or fp16 operands with accumulators in 32 bits.
//
//   kDense      y = act(D + bias) + residual, and D + bias itself where the backward pass is to have it
//   kGated      value and gate columns in one tile: y = (value + b) act(gate + b')
//   kDenseGrad  dz = dy act'(D + bias)                                  D computed again from the layer's input
//   kGatedGrad  dz = [dy act(gate) | dy value act'(gate)]
//   kPlain      D                                                       products of gradients
//   kPartial    D in 32 bits, over one of several parts of k            weight gradients, joined by another kernel
//
// An operand lies with k contiguous (K-major) or with its rows contiguous (MN-major): x and W as they are make the forward
// product, dz and W that of dx, dz and x that of dW; nothing is transposed in memory.  Sizes are free (tiles past the edge
// are zero-filled by the loads and clipped by the stores); base addresses and row pitches of what is read are multiples of 16
// bytes.
//
// A persistent block walks [128 x tile_n] tiles; with kPair two blocks of a cluster walk [256 x tile_n] tiles together,
// each with its 128 rows of A and half of B (cta_group::2), which halves what a tile of B costs in shared memory and from L2.
// Warp roles (576 threads): warps 0-15 finish tiles (TMEM lane = row, groups of 32 columns), warp 16
// loads [128 x 64] and [tile_n x 64] operand blocks by TMA into a ring, warp 17 issues tcgen05.mma into two accumulators of
// 256 columns (four of 128 for tiles of that width), one filled while others are finished.  Where all of a column tile of B fits in half of the ring (64 KiB: 128
// wide layers), it is loaded once and only A passes through the ring.  The finishing warps fetch what they read beside the
// accumulators (residual, dy) by TMA a group ahead and store by TMA: a lane's own accesses to 32 rows occupy the load-store
// unit for some 56 clocks.  Results whose rows TMA cannot address are stored from the same slabs, a row at a time.
//
// Measured (bf16): with long k the tensor cores bound it: 8192 rows, 1024 -> 4096 gated with silu 87 us (1580 TFLOP/s), 4096 -> 4096
// dense 190 us (1450, at the power limit).  With short k finishing does, or HBM: 147456 rows of 128 -> 512: dense without an
// activation 39 us (4.8 TB/s; a fill writes at 3.9), gated with relu 48, with silu 62, where a warp's loads from tensor memory, its
// exponentials (42 % of that unit's rate) and its stores follow one another.  With the finishing warps in two sets, out of step, a
// training step of the last took 330 us instead of 343; registers moved to them (setmaxnreg) gained nothing, and their code as a loop
// over halves of a group lost 5 %.
#pragma once

#include <type_traits>

#include "activation.cuh"
#include "common.cuh"
#include "slab_ring.h"

namespace b200ta {

enum MatmulForm { kDense, kGated, kDenseGrad, kGatedGrad, kPlain, kPartial };

struct MatmulParams {
  int tiles_m, tiles_n, splits, work;  // work = tiles_m * tiles_n * splits items
  int group_m;                         // row tiles that are walked together
  int tiles_m_inner;                   // row tiles of one outer index of A (MN-major A with two halves)
  int kblocks, kblocks_inner;          // blocks of 64 along k: in all, of one outer index
  int kblocks_split;                   // of one split
  int rows_inner;                      // valid rows of D for one outer index
  int columns;                         // valid result columns (kGated*: hidden units)
  int tile_n;                          // accumulator columns of a tile: 64, 128 or 256 (pairs: 128, 256)
  int stages;
  int pair;                            // two blocks on [256 x tile_n] tiles (tiles_m counts those)
  int resident;                        // blocks keep their column tile of B (and walk the row tiles in steps of resident)
  const void* bias;                    // [columns] (kGated*: value biases, then gate biases), or NULL
  int activation;
  int has_aux;                         // kDense: a residual
  int has_saved;                       // kDense, kGated: D + bias is stored as well, in 32 bits
  int accumulate;                      // kPartial: add to what the parts hold
  int sets, buffers;                   // logarithms: sets of finishing warps that take tiles in turn (1, 2, 4); accumulators (2, 4)
  int beside;                          // kBesideFirst, kBesideSecond: see there
  void* sums;                          // kPlain, kPartial with MN-major A, tiles of up to 128: sums of A over k, [outer][rows] in
                                       // the operands' type (kPartial: [split][outer][rows] in 32 bits), or NULL
  void* direct;                        // results that a TMA store cannot address: base, pitch and distance of the outer planes
  long long direct_pitch, direct_outer;
  int* status;
};

// Two products that read the same dz run beside each other: the first lets its successor start only when what came before both
// is complete, so the second does not wait for it, except at its end (whatever follows them waits for the second alone).
enum { kBesideNone = 0, kBesideFirst, kBesideSecond };

#ifdef __CUDACC__

namespace matmul {

constexpr int kThreads = 576, kFinishers = 16;
constexpr int kBM = 128, kBK = 64;
constexpr int kABytes = kBM * kBK * 2;
constexpr int kRingBytes = 131072;         // operand stages
constexpr int kResidentBytes = 65536;      // of them for a resident B
constexpr int kMaxStages = 7;
constexpr int kSlab = 2048;                // 32 rows of 64 bytes
constexpr int kSmSlabs = kRingBytes;       // three for each finishing warp
constexpr int kSmOnes = kSmSlabs + kFinishers * 3 * kSlab;  // an operand block of ones, [16 x 16]
constexpr int kSmBars = kSmOnes + 512;
enum Bar {
  FULL = 0, EMPTY = kMaxStages, ACC_FULL = 2 * kMaxStages, ACC_EMPTY = ACC_FULL + 4, B_FULL = ACC_EMPTY + 4, AUX = B_FULL + 1,
  NUM_BARS = AUX + kFinishers
};
constexpr int kSmTotal = kSmBars + NUM_BARS * 8 + 32;
constexpr int kSmDynamic = kSmTotal + 1024;
static_assert(kSmDynamic <= 232448, "shared memory of a block");

struct Item {
  int split, m_outer, m0, n0, kb0, kb1;
};
// Item i of a block (of a cluster with kPair): rows from m0, result columns from n0, blocks kb0 to kb1 along k.
template <bool kPair, bool kOuter>
__device__ __forceinline__ Item item_of(const MatmulParams& p, int i, int units) {
  constexpr int kRows = kPair ? 2 * kBM : kBM;
  const int block = kPair ? blockIdx.x >> 1 : blockIdx.x, blocks = kPair ? gridDim.x >> 1 : gridDim.x;
  Item r;
  r.m_outer = 0;
  if (p.resident) {
    r.split = 0, r.kb0 = 0, r.kb1 = p.kblocks;
    const int m = block / p.tiles_n;
    r.n0 = (block - m * p.tiles_n) * units;
    r.m0 = (m + i * p.resident) * kRows;
    return r;
  }
  int t = block + i * blocks;
  const int tiles = p.tiles_m * p.tiles_n;
  r.split = 0;
  if (p.splits > 1) r.split = t / tiles, t -= r.split * tiles;
  // groups of row tiles, all columns of a group before the next: what the blocks of a wave read stays in L2
  const int per_group = p.group_m * p.tiles_n, g = t / per_group, first = g * p.group_m;
  const int rows = p.tiles_m - first < p.group_m ? p.tiles_m - first : p.group_m;
  t -= g * per_group;
  const int nt = t / rows;
  int mt = first + (t - nt * rows);
  if (kOuter) r.m_outer = mt / p.tiles_m_inner, mt -= r.m_outer * p.tiles_m_inner;
  r.m0 = mt * kRows;
  r.n0 = nt * units;
  r.kb0 = r.split * p.kblocks_split;
  const int end = r.kb0 + p.kblocks_split;
  r.kb1 = end < p.kblocks ? end : p.kblocks;
  return r;
}
template <bool kPair>
__device__ __forceinline__ int items_of(const MatmulParams& p) {
  const int block = kPair ? blockIdx.x >> 1 : blockIdx.x, blocks = kPair ? gridDim.x >> 1 : gridDim.x;
  if (p.resident) return (p.tiles_m - 1 - block / p.tiles_n) / p.resident + 1;
  return (p.work - 1 - block) / blocks + 1;
}

__host__ __device__ constexpr uint32_t idesc(bool f16, int m, int n, bool a_mn, bool b_mn) {
  return make_idesc_bf16(m, n, a_mn, b_mn) & ~(f16 ? (1u << 7 | 1u << 10) : 0u);
}

// y / dz of kN of a group's 32 columns, from column kFirst, of one row, as 16-bit pairs.  v: accumulators (kGated*: of the
// values), g: of the gates, aux: residual (with has_aux) or dy; kGatedGrad: y the gradients of the values, yg those of the gates.
// dz is formed in 32 bits and rounded once to the operands' type, since the products behind it take 16 bits: dx and dW are off by
// two roundings instead of one (root mean square, bf16: 0.0023 of their size where a single rounding has 0.0017; fp16: 0.00029 and
// 0.00021).  As a sum of two 16-bit numbers it would cost both products twice, and its way through memory.
template <typename T, MatmulForm kForm, int kAct, int kFirst, int kN>
__device__ __forceinline__ void finish(const float (&v)[kN], const float (&g)[kN], bool has_aux, const uint32_t (&aux)[16],
                                       uint32_t (&y)[16], uint32_t (&yg)[16]) {
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) {
    const int j = kFirst / 2 + i;
    float a0, a1, s0, s1;
    const float v0 = v[2 * i], v1 = v[2 * i + 1], g0 = g[2 * i], g1 = g[2 * i + 1];
    if constexpr (kForm == kDense) {
      activate2<kAct, false>(v0, v1, a0, a1, s0, s1);
      if (has_aux) {
        const float2 x = unpack2<T>(aux[j]);
        (F2(a0, a1) + F2(x.x, x.y)).to(a0, a1);
      }
      y[j] = pack2<T>(a0, a1);
    } else if constexpr (kForm == kGated) {
      activate2<kAct, false>(g0, g1, a0, a1, s0, s1);
      (F2(v0, v1) * F2(a0, a1)).to(a0, a1);
      y[j] = pack2<T>(a0, a1);
    } else {
      const float2 x = unpack2<T>(aux[j]);
      const F2 d(x.x, x.y);
      activate2<kAct, true>(kForm == kDenseGrad ? v0 : g0, kForm == kDenseGrad ? v1 : g1, a0, a1, s0, s1);
      if constexpr (kForm == kDenseGrad) {
        (d * F2(s0, s1)).to(s0, s1);
        y[j] = pack2<T>(s0, s1);
      } else {
        (d * F2(a0, a1)).to(a0, a1);
        (d * F2(v0, v1) * F2(s0, s1)).to(s0, s1);
        y[j] = pack2<T>(a0, a1);
        yg[j] = pack2<T>(s0, s1);
      }
    }
  }
}
template <typename T, MatmulForm kForm, int kFirst, int kN>
__device__ __forceinline__ void finish_any(int activation, const float (&v)[kN], const float (&g)[kN], bool has_aux,
                                           const uint32_t (&aux)[16], uint32_t (&y)[16], uint32_t (&yg)[16]) {
  switch (activation) {
    case kActNone: return finish<T, kForm, kActNone, kFirst, kN>(v, g, has_aux, aux, y, yg);
    case kActRelu: return finish<T, kForm, kActRelu, kFirst, kN>(v, g, has_aux, aux, y, yg);
    case kActSilu: return finish<T, kForm, kActSilu, kFirst, kN>(v, g, has_aux, aux, y, yg);
    case kActGelu: return finish<T, kForm, kActGelu, kFirst, kN>(v, g, has_aux, aux, y, yg);
    case kActGeluTanh: return finish<T, kForm, kActGeluTanh, kFirst, kN>(v, g, has_aux, aux, y, yg);
    default: return finish<T, kForm, kActSigmoid, kFirst, kN>(v, g, has_aux, aux, y, yg);
  }
}

// Biases n .. n + kN - 1 as 16-bit pairs, zeros for those from `columns` on; every lane reads the same addresses.  The forward
// forms load them before the accumulators they are added to, whose way hides theirs.
template <typename T, int kN>
__device__ __forceinline__ void load_bias(uint32_t (&b)[kN / 2], const T* bias, int n, int columns) {
  const T* p = bias + n;
  if (n + kN <= columns && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
#pragma unroll
    for (int c = 0; c < kN / 8; ++c) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(p) + c);
      b[4 * c] = x.x, b[4 * c + 1] = x.y, b[4 * c + 2] = x.z, b[4 * c + 3] = x.w;
    }
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int j = 0; j < kN / 2; ++j) {
      const uint32_t lo = n + 2 * j < columns ? __ldg(q + 2 * j) : 0u, hi = n + 2 * j + 1 < columns ? __ldg(q + 2 * j + 1) : 0u;
      b[j] = lo | hi << 16;
    }
  }
}
template <typename T, int kN>
__device__ __forceinline__ void add_bias(float (&v)[kN], const uint32_t (&b)[kN / 2]) {
#pragma unroll
  for (int j = 0; j < kN / 2; ++j) {
    const float2 f = unpack2<T>(b[j]);
    (F2(v[2 * j], v[2 * j + 1]) + F2(f.x, f.y)).to(v[2 * j], v[2 * j + 1]);
  }
}
template <int kN>
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[kN]) {
  uint32_t r[kN];
  if constexpr (kN == 32) tmem_ld32(addr, r);
  else tmem_ld16(addr, r);
#pragma unroll
  for (int j = 0; j < kN; ++j) v[j] = __uint_as_float(r[j]);
}

__device__ __forceinline__ uint16_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void tma_add_3d(const CUtensorMap* m, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(m), "r"(src),
               "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}

// A warp's groups of bulk stores, which its first lane commits and waits for.
struct StoreGroups {
  int lane;
  template <int kNewest>
  __device__ __forceinline__ void wait_read() const {
    if (lane == 0) tma_store_wait_read<kNewest>();
    __syncwarp();
  }
  __device__ __forceinline__ void commit() const {
    if (lane == 0) tma_store_commit();
  }
};

// ---- two blocks on one tile -------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of the first block's copy of a shared-memory variable.
__device__ __forceinline__ uint32_t in_first_block(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t slot_smem, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot_smem), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
// A load into this block's shared memory that is counted by a barrier of either block.
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(m), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void umma_ss_pair_warp(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, e;\nsetp.ne.b32 p, %4, 0;\nelect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on the barrier at this address in both blocks once all MMAs issued so far have completed.
__device__ __forceinline__ void umma_commit_pair_warp(uint32_t bar) {
  asm volatile(
      "{\n.reg .pred e;\nelect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster_warp(uint32_t bar) {
  asm volatile(
      "{\n.reg .pred e;\nelect.sync _|e, 0xffffffff;\n"
      "@e mbarrier.arrive.shared::cluster.b64 _, [%0];\n}" ::"r"(bar)
      : "memory");
}

template <typename T, MatmulForm kForm, bool kAMn, bool kBMn, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
matmul_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
              const __grid_constant__ CUtensorMap tm_out, const __grid_constant__ CUtensorMap tm_aux,
              const __grid_constant__ CUtensorMap tm_saved, const MatmulParams p) {
  constexpr bool kTwo = kForm == kGated || kForm == kGatedGrad;  // value and gate columns in a tile
  constexpr bool kGrad = kForm == kDenseGrad || kForm == kGatedGrad;
  constexpr bool kAux = kGrad || kForm == kDense;                // a warp's first slab receives residual or dy
  constexpr int kRing = kAux ? 2 : 3;                            // the others hold results
  constexpr bool kSums = kAMn && !kPair;                         // sums of A over k may be wanted

  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + kSmBars;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + kSmBars + NUM_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + kSmBars + NUM_BARS * 8 + 8);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = kPair ? cluster_rank() : 0;

  if (threadIdx.x == 0) {
    abort_flag[0] = 0, abort_flag[1] = 0;
    for (int i = 0; i < kMaxStages; ++i) {
      mbar_init(bars + (FULL + i) * 8, 1);
      mbar_init(bars + (EMPTY + i) * 8, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bars + (ACC_FULL + i) * 8, 1);
      mbar_init(bars + (ACC_EMPTY + i) * 8, (kPair ? 2 * kFinishers : kFinishers) >> p.sets);
    }
    mbar_init(bars + B_FULL * 8, 1);
    for (int i = 0; i < kFinishers; ++i) mbar_init(bars + (AUX + i) * 8, 1);
    fence_mbar_init();
  }
  if (kSums && p.sums != nullptr && threadIdx.x < 128) {
    const uint32_t one = __is_same(T, __half) ? 0x3C003C00u : 0x3F803F80u;
    reinterpret_cast<uint32_t*>(gen + kSmOnes)[threadIdx.x] = one;
    fence_proxy_async_smem();
  }
  if (warp == 17) {
    if constexpr (kPair) tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    else tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    if (p.beside == kBesideFirst) pdl_wait();
    pdl_trigger();
  }
  tc_fence_before();
  if constexpr (kPair) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int items = items_of<kPair>(p);
  const int units = kTwo ? p.tile_n / 2 : p.tile_n;           // result columns of a tile
  const int b_rows = kPair ? p.tile_n / 2 : p.tile_n;         // rows of B that this block loads
  const int b_bytes = b_rows * kBK * 2;
  const int stage_bytes = p.resident ? kABytes : kABytes + b_bytes;
  const uint32_t ring = base + (p.resident ? kResidentBytes : 0);

  if (warp == 16) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&tm_a);
      tma_prefetch_desc(&tm_b);
      if (p.beside != kBesideSecond) pdl_wait();
      auto load = [&](uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2) {
        if constexpr (kPair) tma_load_3d_pair(dst, m, bar, c0, c1, c2);
        else tma_load_3d(dst, m, bar, c0, c1, c2);
      };
      auto load_b = [&](uint32_t sb, uint32_t bar, int n0, int k0, int ko) {
        if constexpr (kBMn) {
          for (int n = 0; n < b_rows; n += 64) load(sb + n * kBK * 2, &tm_b, bar, n0 + int(rank) * b_rows + n, k0, ko);
        } else if constexpr (kTwo && kPair) {
          load(sb, &tm_b, bar, k0, n0, int(rank));  // the first block has the values, the second the gates
        } else {
          load(sb, &tm_b, bar, k0, n0 + int(rank) * b_rows, 0);  // kTwo: a box of value rows and a box of gate rows in one
        }
      };
      if (p.resident) {
        const Item t = item_of<kPair, kAMn>(p, 0, units);
        mbar_expect_tx(bars + B_FULL * 8, p.kblocks * b_bytes);
        for (int kb = 0, ko = 0, ki = 0; kb < p.kblocks; ++kb) {
          load_b(base + kb * b_bytes, bars + B_FULL * 8, t.n0, ki * kBK, ko);
          if (++ki == p.kblocks_inner) ki = 0, ++ko;
        }
      }
      int stage = 0, issued = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int i = 0; ok && i < items; ++i) {
        Item t = item_of<kPair, kAMn>(p, i, units);
        t.m0 += int(rank) * kBM;
        int ko = t.kb0 / p.kblocks_inner, ki = t.kb0 - ko * p.kblocks_inner;
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          ok = mbar_wait(bars + (EMPTY + stage) * 8, phase, abort_flag);
          if (!ok) break;
          uint32_t full = bars + (FULL + stage) * 8;
          // the first block's barrier counts the loads of both
          if (kPair) {
            if (rank == 0) mbar_expect_tx(full, 2 * stage_bytes);
            full = in_first_block(full);
          } else {
            mbar_expect_tx(full, stage_bytes);
          }
          const uint32_t sa = ring + stage * stage_bytes;
          const int k0 = ki * kBK;
          if constexpr (kAMn) {
            load(sa, &tm_a, full, t.m0, k0, t.m_outer);
            load(sa + kABytes / 2, &tm_a, full, t.m0 + 64, k0, t.m_outer);
          } else {
            load(sa, &tm_a, full, k0, t.m0, ko);
          }
          if (!p.resident) load_b(sa + kABytes, full, t.n0, k0, ko);
          ++issued;
          if (++stage == p.stages) stage = 0, phase ^= 1u;
          if (++ki == p.kblocks_inner) ki = 0, ++ko;
        }
      }
      // If the loop was abandoned, give copies still in flight a bounded chance to land (of a pair's first block: those of
      // both; its second block's copies are waited for there).
      if (*abort_flag) {
        if (p.resident) mbar_wait(bars + B_FULL * 8, 0, abort_flag + 1);
        if (rank == 0)
          for (int j = issued > p.stages ? issued - p.stages : 0; j < issued; ++j)
            mbar_wait(bars + (FULL + j % p.stages) * 8, (j / p.stages) & 1, abort_flag + 1);
      }
    }
  } else if (warp == 17) {
    // ------------------------------------------------------------------ MMA issuer (whole warp, one lane issues)
    if (rank == 0) {
      const uint32_t id = idesc(__is_same(T, __half), kPair ? 2 * kBM : kBM, p.tile_n, kAMn, kBMn);
      const uint32_t tb = __shfl_sync(0xffffffffu, tmem_base, 0);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      if (p.resident) ok = mbar_wait_warp(bars + B_FULL * 8, 0, abort_flag);
      for (int i = 0; ok && i < items; ++i) {
        const Item t = item_of<kPair, kAMn>(p, i, units);
        const int buffer = i & ((1 << p.buffers) - 1);
        const uint32_t acc = tb + buffer * (512 >> p.buffers);
        ok = mbar_wait_warp(bars + (ACC_EMPTY + buffer) * 8, ((i >> p.buffers) & 1) ^ 1, abort_flag);
        for (int kb = t.kb0; ok && kb < t.kb1; ++kb) {
          ok = mbar_wait_warp(bars + (FULL + stage) * 8, phase, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = ring + stage * stage_bytes, sb = p.resident ? base + kb * b_bytes : sa + kABytes;
          // K-major: rows of 128 bytes, groups of 8 rows 1 KiB apart, a step of 16 k is 32 bytes.  MN-major: rows (k) of 64
          // elements, blocks of 64 elements 8 KiB apart, a step of 16 k is 2 KiB.
          const uint64_t da = kAMn ? smem_desc<8192, 1024, kLayoutSw128>(sa) : smem_desc<16, 1024, kLayoutSw128>(sa);
          const uint64_t db = kBMn ? smem_desc<8192, 1024, kLayoutSw128>(sb) : smem_desc<16, 1024, kLayoutSw128>(sb);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            const uint64_t dak = da + k * (kAMn ? 128 : 2), dbk = db + k * (kBMn ? 128 : 2);
            const uint32_t add = (kb > t.kb0 || k > 0) ? 1u : 0u;
            if constexpr (kPair) umma_ss_pair_warp(acc, dak, dbk, id, add);
            else umma_ss_warp(acc, dak, dbk, id, add);
          }
          if (kSums && p.sums != nullptr && t.n0 == 0) {  // A times a block of ones, into 16 columns of their own
            const uint32_t id_ones = idesc(__is_same(T, __half), kBM, 16, kAMn, false);
            const uint64_t ones = smem_desc<16, 256, kLayoutSw32>(base + kSmOnes);
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) umma_ss_warp(acc + 128, da + k * 128, ones, id_ones, (kb > t.kb0 || k > 0) ? 1u : 0u);
          }
          if constexpr (kPair) umma_commit_pair_warp(bars + (EMPTY + stage) * 8);
          else umma_commit_warp(bars + (EMPTY + stage) * 8);
          if (++stage == p.stages) stage = 0, phase ^= 1u;
        }
        if (!ok) break;
        if constexpr (kPair) umma_commit_pair_warp(bars + (ACC_FULL + buffer) * 8);
        else umma_commit_warp(bars + (ACC_FULL + buffer) * 8);
      }
    }
  } else {
    // ------------------------------------------------------------------ finishing warps
    if (p.beside != kBesideSecond) pdl_wait();
    // All of them on every tile, each with every fourth group of 32 result columns; or eight on the even tiles and eight on the
    // odd ones, with every second group; or four on every fourth tile, with all groups.
    const int first_i = warp >> (4 - p.sets), step_i = 1 << p.sets, step_g = 4 >> p.sets, first_g = (warp >> 2) & (step_g - 1);
    const int m = (warp & 3) * 32 + int(rank) * kBM;
    const uint32_t lane_acc = tmem_base + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t slabs = base + kSmSlabs + warp * 3 * kSlab, out_slabs = slabs + (kAux ? kSlab : 0);
    const uint32_t aux_bar = bars + (AUX + warp) * 8;
    const bool has_aux = kGrad || (kForm == kDense && p.has_aux);
    const T* bias = static_cast<const T*>(p.bias);
    // groups of 32 result columns of an item
    auto groups_of = [&](const Item& t) {
      if (t.m0 + m >= p.rows_inner) return 0;
      const int left = p.columns - t.n0;
      return ((left < units ? left : units) + 31) / 32;
    };
    // residual or dy: the load of the next group runs while this one is finished
    int next_i = first_i, next_g = first_g, next_groups = -1;
    Item next{};
    uint32_t loads = 0, taken = 0;
    auto load_aux = [&]() {
      for (; next_i < items; next_i += step_i, next_g = first_g, next_groups = -1) {
        if (next_groups < 0) next = item_of<kPair, kAMn>(p, next_i, units), next_groups = groups_of(next);
        if (next_g >= next_groups) continue;
        if (lane == 0) {
          mbar_expect_tx(aux_bar, kSlab);
          tma_load_3d(slabs, &tm_aux, aux_bar, next.n0 + next_g * 32, next.m0 + m, 0);
        }
        ++loads, next_g += step_g;
        return;
      }
    };
    if (has_aux) load_aux();

    SlabRing<kRing> ring_out;
    const StoreGroups store_groups{lane};
    // writes a slab (32 columns in 16 bits or 16 in 32 bits, of the 32 rows) and stores it
    auto store = [&](const CUtensorMap& map, const uint32_t (&x)[16], int column, int row, int outer) {
      const bool direct = (kForm == kDense || kForm == kGated || kForm == kPlain) && p.direct != nullptr && &map == &tm_out;
      ring_out.pass(
          store_groups,
          [&](uint32_t slot) {
            const uint32_t slab = out_slabs + slot * kSlab;
#pragma unroll
            for (int j = 0; j < 4; ++j) sts128(slab + sw64_offset(lane, j), make_uint4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]));
          },
          [&](uint32_t slot) {
            const uint32_t slab = out_slabs + slot * kSlab;
            if (direct) {
              __syncwarp();
              const int rows = p.rows_inner - row < 32 ? p.rows_inner - row : 32;
              T* to = static_cast<T*>(p.direct) + outer * p.direct_outer + (long long)row * p.direct_pitch + column + lane;
              if (column + lane < p.columns)
#pragma unroll 4
                for (int i = 0; i < rows; ++i, to += p.direct_pitch)
                  *reinterpret_cast<uint16_t*>(to) = lds16(slab + sw64_offset(i, lane >> 3) + (lane & 7) * 2);
              __syncwarp();
              return;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (kForm == kPartial && p.accumulate) tma_add_3d(&map, slab, column, row, outer);
              else tma_store_3d(&map, slab, column, row, outer);
            }
          });
    };
    auto release = [&](int i) {  // the accumulator is in registers
      tc_fence_before();
      __syncwarp();
      const uint32_t bar = bars + (ACC_EMPTY + (i & ((1 << p.buffers) - 1))) * 8;
      if (kPair) mbar_arrive_cluster_warp(in_first_block(bar));
      else mbar_arrive_warp(bar);
    };

    bool ok = true;
    for (int i = first_i; ok && i < items; i += step_i) {
      const Item t = item_of<kPair, kAMn>(p, i, units);
      const int groups = groups_of(t), row = t.m0 + m;
      const int buffer = i & ((1 << p.buffers) - 1);
      ok = mbar_wait_warp(bars + (ACC_FULL + buffer) * 8, (i >> p.buffers) & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = lane_acc + buffer * (512 >> p.buffers);
      if (kSums && p.sums != nullptr && t.n0 == 0 && first_g == 0 && groups > 0) {
        float sum[16];
        tmem_load(acc + 128, sum);
        tmem_ld_wait();
        if (row + lane < p.rows_inner) {
          if constexpr (kForm == kPartial) {
            const int outer = t.split * (p.tiles_m / p.tiles_m_inner) + t.m_outer;
            float* to = static_cast<float*>(p.sums) + (long long)outer * p.rows_inner + row + lane;
            *to = p.accumulate ? *to + sum[0] : sum[0];
          } else {
            static_cast<T*>(p.sums)[(long long)t.m_outer * p.rows_inner + row + lane] = static_cast<T>(sum[0]);
          }
        }
      }
      if (first_g >= groups) release(i);
      for (int g = first_g; g < groups; g += step_g) {
        const int n = t.n0 + g * 32;
        uint32_t aux[16];
        if constexpr (kAux) {
          if (has_aux) {
            ok = mbar_wait_warp(aux_bar, taken & 1, abort_flag);
            if (!ok) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint4 x = lds128(slabs + sw64_offset(lane, j));
              aux[4 * j] = x.x, aux[4 * j + 1] = x.y, aux[4 * j + 2] = x.z, aux[4 * j + 3] = x.w;
            }
            ++taken;
            __threadfence_block();  // the reads are complete before the next load may overwrite the slab
            __syncwarp();
            load_aux();
          }
        }
        // Accumulators are taken 16 columns at a time (kDense, kPlain: 32), to stay within the registers that 18 warps leave a thread.
        constexpr int kStep = kForm == kDense || kForm == kPlain ? 32 : 16;
        uint32_t y[16], yg[16];
        auto step = [&](auto first) {
          constexpr int kFirst = decltype(first)::value;
          float v[kStep], gate[kStep];
          uint32_t bv[kStep / 2];
          [[maybe_unused]] uint32_t bg[kStep / 2];
          if ((kForm == kDense || kForm == kGated) && bias != nullptr) {  // (the gradients' registers do not suffice)
            load_bias<T, kStep>(bv, bias, n + kFirst, p.columns);
            if constexpr (kTwo) load_bias<T, kStep>(bg, bias + p.columns, n + kFirst, p.columns);
          }
          tmem_load(acc + g * 32 + kFirst, v);
          if constexpr (kTwo) tmem_load(acc + units + g * 32 + kFirst, gate);
          tmem_ld_wait();
          if (kFirst + kStep == 32 && g + step_g >= groups) release(i);
          if constexpr (kForm == kPartial) {
            uint32_t x[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(v[j]);
            if (n + kFirst < p.columns) store(tm_out, x, n + kFirst, row, t.split * (p.tiles_m / p.tiles_m_inner) + t.m_outer);
          } else if constexpr (kForm == kPlain) {
#pragma unroll
            for (int j = 0; j < kStep / 2; ++j) y[kFirst / 2 + j] = pack2<T>(v[2 * j], v[2 * j + 1]);
          } else {
            if (bias != nullptr) {
              if constexpr (kGrad) load_bias<T, kStep>(bv, bias, n + kFirst, p.columns);
              add_bias<T>(v, bv);
              if constexpr (kGrad && kTwo) load_bias<T, kStep>(bg, bias + p.columns, n + kFirst, p.columns);
              if constexpr (kTwo) add_bias<T>(gate, bg);
            }
            if ((kForm == kDense || kForm == kGated) && p.has_saved) {
#pragma unroll
              for (int c = 0; c < kStep; c += 16) {
                if (n + kFirst + c >= p.columns) break;
                uint32_t x[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(v[c + j]);
                store(tm_saved, x, n + kFirst + c, row, 0);
                if constexpr (kTwo) {
#pragma unroll
                  for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(gate[c + j]);
                  store(tm_saved, x, n + kFirst + c, row, 1);
                }
              }
            }
            finish_any<T, kForm, kFirst, kStep>(p.activation, v, gate, has_aux, aux, y, yg);
          }
        };
        step(std::integral_constant<int, 0>());
        if constexpr (kStep == 16) step(std::integral_constant<int, 16>());
        if constexpr (kForm != kPartial) {
          store(tm_out, y, n, row, kForm == kPlain ? t.m_outer : 0);
          if (kForm == kGatedGrad) store(tm_out, yg, n, row, 1);
        }
      }
    }
    if (!ok && taken < loads) mbar_wait(aux_bar, taken & 1, abort_flag + 1);  // a load still in flight
    if (lane == 0) tma_store_wait_all();
    if (p.beside == kBesideSecond) pdl_wait();
  }

  __syncwarp();
  tc_fence_before();
  // a pair's blocks stay until the other no longer arrives on their barriers or reads their operands
  if constexpr (kPair) cluster_sync();
  else __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    if constexpr (kPair) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) *p.status = B200TA_ERR_DEVICE_WAIT;
}

}  // namespace matmul
#endif  // __CUDACC__

// An operand or result as the kernel sees it: rows x columns elements (x outer planes), the columns contiguous.
struct Plane {
  const void* base = nullptr;
  int64_t rows = 0, columns = 0, pitch = 0;  // elements
  int64_t outer = 1, outer_stride = 0;
};

// One product.  Operands lie as their forms say: kGated* take B as two planes (value and gate rows) and write two; a K-major
// A of two planes is contracted over both (with an MN-major B of two planes), an MN-major A of two planes gives the rows of
// two planes of the result.
struct Matmul {
  MatmulForm form = kDense;
  bool f16 = false, a_mn = false, b_mn = false;
  Plane a, b, out, aux, saved;  // aux / saved without a base: none
  const void* bias = nullptr;
  int activation = kActNone;
  int kblocks_split = 0;  // blocks of 64 of a part (kPartial); 0: all of them
  bool accumulate = false;
  int beside = kBesideNone;
  void* sums = nullptr;  // see MatmulParams
  const char* what = "matmul";
};
int run_matmul(const Matmul& m, void* stream);

// The three sets of kernels, each compiled by itself; a set returns B200TA_ERR_UNSUPPORTED for a product that is not its own.
struct MatmulMaps {
  CUtensorMap a, b, out, aux, saved;
};
int launch_matmul_forward(DeviceState* st, const Matmul& m, const MatmulMaps& maps, const MatmulParams& p, int grid, void* stream);
int launch_matmul_grad(DeviceState* st, const Matmul& m, const MatmulMaps& maps, const MatmulParams& p, int grid, void* stream);
int launch_matmul_product(DeviceState* st, const Matmul& m, const MatmulMaps& maps, const MatmulParams& p, int grid, void* stream);

#ifdef __CUDACC__
namespace matmul {
template <MatmulForm kForm, bool kAMn, bool kBMn>
int launch(DeviceState* st, int id, const Matmul& m, const MatmulMaps& maps, const MatmulParams& p, int grid, void* stream) {
  const KernelId kernel = KernelId(kKernelMatmul + 4 * id + (m.f16 ? 2 : 0) + (p.pair ? 1 : 0));
  auto* function = p.pair ? (m.f16 ? matmul_kernel<__half, kForm, kAMn, kBMn, true> : matmul_kernel<__nv_bfloat16, kForm, kAMn, kBMn, true>)
                          : (m.f16 ? matmul_kernel<__half, kForm, kAMn, kBMn, false> : matmul_kernel<__nv_bfloat16, kForm, kAMn, kBMn, false>);
  return launch_clusters(st, kernel, function, dim3(unsigned(grid)), p.pair ? 2 : 1, kThreads, kSmDynamic, stream, maps.a, maps.b,
                         maps.out, maps.aux, maps.saved, p);
}
}  // namespace matmul
#endif

}  // namespace b200ta

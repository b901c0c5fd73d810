// The tensor-core products of the trainable dense layers (sm_100a): D[m, n] = sum_k A[m, k] B[n, k], finished in one of
// five forms, for bf16 or fp16 operands with accumulators in 32 bits.
//
//   kDense      y = act(D + bias) + residual, and D + bias itself where the backward pass is to have it
//   kGated      value and gate columns in one tile: y = (value + b) act(gate + b')
//   kDenseGrad  dz = dy act'(D + bias)                                  D computed again from the layer's input
//   kGatedGrad  dz = [dy act(gate) | dy value act'(gate)]
//   kPartial    D in 32 bits, over one of several parts of k            weight gradients, joined by another kernel
//
// An operand lies with k contiguous (K-major) or with its rows contiguous (MN-major): x and W as they are make the forward
// product, dz and W that of dx, dz and x that of dW; nothing is transposed in memory.  Sizes are free (tiles past the edge
// are zero-filled by the loads and clipped by the stores); base addresses and row pitches are multiples of 16 bytes.
//
// A persistent block walks [128 x tile_n] tiles.  Warp roles (320 threads): warps 0-7 finish tiles (TMEM lane = row, two
// halves of the columns), warp 8 loads [128 x 64] and [tile_n x 64] operand blocks by TMA into a ring, warp 9 issues
// tcgen05.mma into two accumulators of 256 columns, one filled while the other is finished.  The finishing warps fetch what
// they read beside the accumulators (residual, dy) by TMA two groups of 32 columns ahead and store by TMA from a ring of
// slabs: a lane's own accesses to 32 rows occupy the load-store unit for some 56 clocks.
#pragma once

#include "activation.cuh"
#include "common.cuh"

namespace b200ta {

enum MatmulForm { kDense, kGated, kDenseGrad, kGatedGrad, kPartial };

struct MatmulParams {
  int tiles_m, tiles_n, splits, work;  // work = tiles_m * tiles_n * splits items
  int group_m;                         // row tiles that are walked together
  int tiles_m_inner;                   // row tiles of one outer index of A (MN-major A with two halves)
  int kblocks, kblocks_inner;          // blocks of 64 along k: in all, of one outer index
  int kblocks_split;                   // of one split
  int rows_inner;                      // valid rows of D for one outer index
  int columns;                         // valid result columns (kGated*: hidden units)
  int tile_n;                          // accumulator columns of a tile: 64, 128 or 256
  int stages;
  const void* bias;                    // [columns] (kGated*: value biases, then gate biases), or NULL
  int activation;
  int has_aux;                         // kDense: a residual
  int has_saved;                       // kDense, kGated: D + bias is stored as well
  int accumulate;                      // kPartial: add to what the parts hold
  int* status;
};

#ifdef __CUDACC__

namespace matmul {

constexpr int kThreads = 320;
constexpr int kBM = 128, kBK = 64;
constexpr int kABytes = kBM * kBK * 2;
constexpr int kRingBytes = 147456;     // operand stages
constexpr int kMaxStages = 6;
constexpr int kSmSlabs = kRingBytes;   // 8 warps x 8 KiB
constexpr int kWarpSlabs = 8192;
constexpr int kSmBars = kSmSlabs + 8 * kWarpSlabs;
enum Bar {
  FULL = 0, EMPTY = kMaxStages, ACC_FULL = 2 * kMaxStages, ACC_EMPTY = ACC_FULL + 2, AUX = ACC_EMPTY + 2, NUM_BARS = AUX + 16
};
constexpr int kSmTotal = kSmBars + NUM_BARS * 8 + 32;
constexpr int kSmDynamic = kSmTotal + 1024;
static_assert(kSmDynamic <= 232448, "shared memory of a block");

struct Item {
  int split, m_outer, m0, n0, kb0, kb1;
};
__device__ __forceinline__ Item decode(const MatmulParams& p, int t, int units) {
  Item r;
  const int tiles = p.tiles_m * p.tiles_n;
  r.split = t / tiles;
  t -= r.split * tiles;
  // groups of row tiles, all columns of a group before the next: what the blocks of a wave read stays in L2
  const int per_group = p.group_m * p.tiles_n, g = t / per_group, first = g * p.group_m;
  const int rows = p.tiles_m - first < p.group_m ? p.tiles_m - first : p.group_m;
  t -= g * per_group;
  const int nt = t / rows, mt = first + (t - nt * rows);
  r.m_outer = mt / p.tiles_m_inner;
  r.m0 = (mt - r.m_outer * p.tiles_m_inner) * kBM;
  r.n0 = nt * units;
  r.kb0 = r.split * p.kblocks_split;
  const int end = r.kb0 + p.kblocks_split;
  r.kb1 = end < p.kblocks ? end : p.kblocks;
  return r;
}

__host__ __device__ constexpr uint32_t idesc(bool f16, int m, int n, bool a_mn, bool b_mn) {
  return make_idesc_bf16(m, n, a_mn, b_mn) & ~(f16 ? (1u << 7 | 1u << 10) : 0u);
}

// y / dz of 32 columns of one row.  v: accumulators (kGated*: of the values), g: of the gates, aux: residual or dy.
// Results replace v (and g).
template <MatmulForm kForm, int kAct>
__device__ __forceinline__ void finish(float (&v)[32], float (&g)[32], const float (&aux)[32]) {
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    float a0, a1, s0, s1;
    if constexpr (kForm == kDense) {
      activate2<kAct, false>(v[j], v[j + 1], a0, a1, s0, s1);
      v[j] = a0 + aux[j], v[j + 1] = a1 + aux[j + 1];
    } else if constexpr (kForm == kGated) {
      activate2<kAct, false>(g[j], g[j + 1], a0, a1, s0, s1);
      v[j] *= a0, v[j + 1] *= a1;
    } else if constexpr (kForm == kDenseGrad) {
      activate2<kAct, true>(v[j], v[j + 1], a0, a1, s0, s1);
      v[j] = aux[j] * s0, v[j + 1] = aux[j + 1] * s1;
    } else {
      activate2<kAct, true>(g[j], g[j + 1], a0, a1, s0, s1);
      g[j] = aux[j] * v[j] * s0, g[j + 1] = aux[j + 1] * v[j + 1] * s1;
      v[j] = aux[j] * a0, v[j + 1] = aux[j + 1] * a1;
    }
  }
}
template <MatmulForm kForm>
__device__ __forceinline__ void finish_any(int activation, float (&v)[32], float (&g)[32], const float (&aux)[32]) {
  switch (activation) {
    case kActNone: return finish<kForm, kActNone>(v, g, aux);
    case kActRelu: return finish<kForm, kActRelu>(v, g, aux);
    case kActSilu: return finish<kForm, kActSilu>(v, g, aux);
    case kActGelu: return finish<kForm, kActGelu>(v, g, aux);
    case kActGeluTanh: return finish<kForm, kActGeluTanh>(v, g, aux);
    default: return finish<kForm, kActSigmoid>(v, g, aux);
  }
}

// Adds biases n .. n + 31 (those below `columns`) to v; every lane reads the same addresses.
template <typename T>
__device__ __forceinline__ void add_bias(float (&v)[32], const T* bias, int n, int columns) {
  const T* b = bias + n;
  if (n + 32 <= columns && (reinterpret_cast<uintptr_t>(b) & 15u) == 0) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(b) + c);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack2<T>(w[e]);
        v[c * 8 + 2 * e] += f.x, v[c * 8 + 2 * e + 1] += f.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (n + j < columns) v[j] += static_cast<float>(b[j]);
  }
}

__device__ __forceinline__ void tma_add_3d(const CUtensorMap* m, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(m), "r"(src),
               "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}

template <typename T, MatmulForm kForm, bool kAMn, bool kBMn>
__global__ void __launch_bounds__(kThreads, 1)
matmul_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
              const __grid_constant__ CUtensorMap tm_out, const __grid_constant__ CUtensorMap tm_aux,
              const __grid_constant__ CUtensorMap tm_saved, const MatmulParams p) {
  constexpr bool kTwo = kForm == kGated || kForm == kGatedGrad;  // value and gate columns in a tile
  constexpr bool kGrad = kForm == kDenseGrad || kForm == kGatedGrad;
  constexpr int kRing = kForm == kGated ? 4 : 2;                 // output slabs of a warp
  constexpr int kSlab = kForm == kPartial ? 4096 : 2048;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + kSmBars;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + kSmBars + NUM_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + kSmBars + NUM_BARS * 8 + 8);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    abort_flag[0] = 0, abort_flag[1] = 0;
    for (int i = 0; i < kMaxStages; ++i) {
      mbar_init(bars + (FULL + i) * 8, 1);
      mbar_init(bars + (EMPTY + i) * 8, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + (ACC_FULL + i) * 8, 1);
      mbar_init(bars + (ACC_EMPTY + i) * 8, 8);
    }
    for (int i = 0; i < 16; ++i) mbar_init(bars + (AUX + i) * 8, 1);
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    pdl_trigger();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int items = (p.work - 1 - int(blockIdx.x)) / int(gridDim.x) + 1;
  const int units = kTwo ? p.tile_n / 2 : p.tile_n;  // result columns of a tile
  const int stage_bytes = kABytes + p.tile_n * kBK * 2;

  if (warp == 8) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&tm_a);
      tma_prefetch_desc(&tm_b);
      pdl_wait();
      int stage = 0, issued = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int i = 0; ok && i < items; ++i) {
        const Item t = decode(p, blockIdx.x + i * gridDim.x, units);
        int ko = t.kb0 / p.kblocks_inner, ki = t.kb0 - ko * p.kblocks_inner;
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          ok = mbar_wait(bars + (EMPTY + stage) * 8, phase, abort_flag);
          if (!ok) break;
          const uint32_t full = bars + (FULL + stage) * 8;
          const uint32_t sa = base + stage * stage_bytes, sb = sa + kABytes;
          const int k0 = ki * kBK;
          mbar_expect_tx(full, stage_bytes);
          if constexpr (kAMn) {
            tma_load_3d(sa, &tm_a, full, t.m0, k0, t.m_outer);
            tma_load_3d(sa + kABytes / 2, &tm_a, full, t.m0 + 64, k0, t.m_outer);
          } else {
            tma_load_3d(sa, &tm_a, full, k0, t.m0, ko);
          }
          if constexpr (kBMn) {
            for (int n = 0; n < p.tile_n; n += 64) tma_load_3d(sb + n * kBK * 2, &tm_b, full, t.n0 + n, k0, ko);
          } else {
            tma_load_3d(sb, &tm_b, full, k0, t.n0, 0);  // kTwo: a box of value rows and a box of gate rows in one
          }
          ++issued;
          if (++stage == p.stages) stage = 0, phase ^= 1u;
          if (++ki == p.kblocks_inner) ki = 0, ++ko;
        }
      }
      // If the loop was abandoned, give copies still in flight a bounded chance to land.
      if (*abort_flag)
        for (int j = issued > p.stages ? issued - p.stages : 0; j < issued; ++j)
          mbar_wait(bars + (FULL + j % p.stages) * 8, (j / p.stages) & 1, abort_flag + 1);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------ MMA issuer (whole warp, one lane issues)
    const uint32_t id = idesc(__is_same(T, __half), kBM, p.tile_n, kAMn, kBMn);
    const uint32_t tb = __shfl_sync(0xffffffffu, tmem_base, 0);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; ok && i < items; ++i) {
      const Item t = decode(p, blockIdx.x + i * gridDim.x, units);
      const uint32_t acc = tb + (i & 1) * 256;
      ok = mbar_wait_warp(bars + (ACC_EMPTY + (i & 1)) * 8, ((i >> 1) & 1) ^ 1, abort_flag);
      for (int kb = t.kb0; ok && kb < t.kb1; ++kb) {
        ok = mbar_wait_warp(bars + (FULL + stage) * 8, phase, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sa = base + stage * stage_bytes;
        // K-major: rows of 128 bytes, groups of 8 rows 1 KiB apart, a step of 16 k is 32 bytes.  MN-major: rows (k) of 64
        // elements, blocks of 64 elements 8 KiB apart, a step of 16 k is 2 KiB.
        const uint64_t da = kAMn ? smem_desc<8192, 1024, kLayoutSw128>(sa) : smem_desc<16, 1024, kLayoutSw128>(sa);
        const uint64_t db = kBMn ? smem_desc<8192, 1024, kLayoutSw128>(sa + kABytes) : smem_desc<16, 1024, kLayoutSw128>(sa + kABytes);
#pragma unroll
        for (int k = 0; k < kBK / 16; ++k)
          umma_ss_warp(acc, da + k * (kAMn ? 128 : 2), db + k * (kBMn ? 128 : 2), id, (kb > t.kb0 || k > 0) ? 1u : 0u);
        umma_commit_warp(bars + (EMPTY + stage) * 8);
        if (++stage == p.stages) stage = 0, phase ^= 1u;
      }
      if (ok) umma_commit_warp(bars + (ACC_FULL + (i & 1)) * 8);
    }
  } else {
    // ------------------------------------------------------------------ finishing warps
    pdl_wait();
    const int half = warp >> 2, m = (warp & 3) * 32, c0 = half * (units / 2);
    const uint32_t lane_acc = tmem_base + (uint32_t(m) << 16);
    const uint32_t slabs = base + kSmSlabs + warp * kWarpSlabs;
    const uint32_t out_slabs = slabs + (kForm == kDense || kGrad ? 4096 : 0);
    const uint32_t aux_bar = bars + (AUX + warp * 2) * 8;
    const bool has_aux = kGrad || (kForm == kDense && p.has_aux);
    const T* bias = static_cast<const T*>(p.bias);
    // groups of 32 columns that this warp has in an item
    auto groups_of = [&](const Item& t) {
      if (t.m0 + m >= p.rows_inner) return 0;
      const int left = p.columns - t.n0 - c0, most = units / 2;
      return left <= 0 ? 0 : ((left < most ? left : most) + 31) / 32;
    };
    // residual or dy: the loads run two groups ahead
    int next_i = 0, next_g = 0, next_groups = -1;
    Item next{};
    uint32_t loads = 0, taken = 0;
    auto load_aux = [&]() {
      for (; next_i < items; ++next_i, next_g = 0, next_groups = -1) {
        if (next_groups < 0) next = decode(p, blockIdx.x + next_i * gridDim.x, units), next_groups = groups_of(next);
        if (next_g >= next_groups) continue;
        if (lane == 0) {
          const uint32_t bar = aux_bar + (loads & 1) * 8;
          mbar_expect_tx(bar, 2048);
          tma_load_3d(slabs + (loads & 1) * 2048, &tm_aux, bar, next.n0 + c0 + next_g * 32, next.m0 + m, 0);
        }
        ++loads, ++next_g;
        return;
      }
    };
    if (has_aux) load_aux(), load_aux();

    uint32_t stores = 0;
    auto store = [&](const CUtensorMap& map, const float (&x)[32], int column, int row, int outer) {
      const uint32_t slab = out_slabs + (stores & (kRing - 1)) * kSlab;
      if (lane == 0) tma_store_wait_read<kRing - 1>();  // the store that used this slab before has read it
      __syncwarp();
      if constexpr (kForm == kPartial) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          sts128(slab + sw128_offset(lane, j), make_uint4(__float_as_uint(x[4 * j]), __float_as_uint(x[4 * j + 1]),
                                                          __float_as_uint(x[4 * j + 2]), __float_as_uint(x[4 * j + 3])));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sts128(slab + sw64_offset(lane, j), make_uint4(pack2<T>(x[8 * j], x[8 * j + 1]), pack2<T>(x[8 * j + 2], x[8 * j + 3]),
                                                         pack2<T>(x[8 * j + 4], x[8 * j + 5]), pack2<T>(x[8 * j + 6], x[8 * j + 7])));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (kForm == kPartial && p.accumulate) tma_add_3d(&map, slab, column, row, outer);
        else tma_store_3d(&map, slab, column, row, outer);
        tma_store_commit();
      }
      ++stores;
    };

    bool ok = true;
    for (int i = 0; ok && i < items; ++i) {
      const Item t = decode(p, blockIdx.x + i * gridDim.x, units);
      const int groups = groups_of(t);
      ok = mbar_wait_warp(bars + (ACC_FULL + (i & 1)) * 8, (i >> 1) & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = lane_acc + (i & 1) * 256 + c0;
      for (int g = 0; g < groups; ++g) {
        uint32_t r[32], q[32];
        tmem_ld32(acc + g * 32, r);
        if constexpr (kTwo) tmem_ld32(acc + units + g * 32, q);
        const int n = t.n0 + c0 + g * 32, row = t.m0 + m;
        float aux[32];
        if constexpr (kGrad || kForm == kDense) {
          if (has_aux) {
            ok = mbar_wait_warp(aux_bar + (taken & 1) * 8, (taken >> 1) & 1, abort_flag);
            if (!ok) break;
            const uint32_t slab = slabs + (taken & 1) * 2048;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint4 x = lds128(slab + sw64_offset(lane, j));
              const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2<T>(w[e]);
                aux[j * 8 + 2 * e] = f.x, aux[j * 8 + 2 * e + 1] = f.y;
              }
            }
            ++taken;
            __threadfence_block();  // the reads are complete before the next load may overwrite the slab
            __syncwarp();
            load_aux();
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) aux[j] = 0.f;
          }
        }
        tmem_ld_wait();
        if (g == groups - 1) {  // the accumulator is in registers
          tc_fence_before();
          __syncwarp();
          mbar_arrive_warp(bars + (ACC_EMPTY + (i & 1)) * 8);
        }
        float v[32], gate[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]), gate[j] = kTwo ? __uint_as_float(q[j]) : 0.f;
        if constexpr (kForm == kPartial) {
          store(tm_out, v, n, row, t.split * (p.tiles_m / p.tiles_m_inner) + t.m_outer);
        } else {
          if (bias != nullptr) {
            add_bias(v, bias, n, p.columns);
            if (kTwo) add_bias(gate, bias + p.columns, n, p.columns);
          }
          if constexpr (kForm == kDense || kForm == kGated) {
            if (p.has_saved) {
              store(tm_saved, v, n, row, 0);
              if (kTwo) store(tm_saved, gate, n, row, 1);
            }
          }
          finish_any<kForm>(p.activation, v, gate, aux);
          store(tm_out, v, n, row, kForm == kDense ? t.m_outer : 0);
          if (kForm == kGatedGrad) store(tm_out, gate, n, row, 1);
        }
      }
      if (ok && groups == 0) {
        tc_fence_before();
        __syncwarp();
        mbar_arrive_warp(bars + (ACC_EMPTY + (i & 1)) * 8);
      }
    }
    if (!ok)  // loads of the residual or of dy still in flight
      for (uint32_t j = taken; j < loads; ++j) mbar_wait(aux_bar + (j & 1) * 8, (j >> 1) & 1, abort_flag + 1);
    if (lane == 0) tma_store_wait_all();
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
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
  const KernelId kernel = KernelId(kKernelMatmul + 2 * id + (m.f16 ? 1 : 0));
  return launch_kernel(st, kernel, m.f16 ? matmul_kernel<__half, kForm, kAMn, kBMn> : matmul_kernel<__nv_bfloat16, kForm, kAMn, kBMn>,
                       dim3(unsigned(grid)), kThreads, kSmDynamic, stream, maps.a, maps.b, maps.out, maps.aux, maps.saved, p);
}
}  // namespace matmul
#endif

}  // namespace b200ta

// dz and dx of a narrow dense layer (at most 128 inputs, many rows) in one kernel (sm_100a).
//
// dz is N or 2 N wide and the layer's input and its gradient K and N, so passing dz through memory (written once, read for dx
// and for dW) is most of the backward pass's traffic, and HBM bounds it.  Here a block takes 256 rows and walks the hidden units
// in chunks of 64: S = x Wc^T -> dz -> dx += dz Wc, the same tile of W as the operand of both products; dz goes to memory only
// if dW is wanted.  S and dx are accumulators in 32 bits, dz is rounded once, as the operand of its products.  (A second kernel
// of this kind for dW = dz^T x took 100 us for 147456 rows, 128 -> 512 gated, where reading dz takes 56: its operands' way
// through shared memory bounded it.)
//
// The finishing warps bound the kernel (activation, its slope and two products a unit: 250 instructions for 16 units of 32 rows, and
// one and a half special-function operations a unit).  Two row tiles of 128 share every tile of W and take turns: all sixteen
// warps finish one while the tensor cores work on the other, and what a step stores has until the tile's next step to leave.
// (Eight warps for each tile with one buffer for their stores: 147456 rows, 128 -> 512 gated, 135 us, now 125.  Chunks of 32 units
// with S twice: 147; its MMAs are too small.)  Shared memory: x 2 x 32 KiB, W in two stages of a chunk's value and gate rows (32
// KiB each), dy 16 x 2 KiB, results on their way out 16 x 4 KiB.  Tensor memory: S 2 x 128 columns, dz in their place as the left
// operand of the second product (from shared memory its tiles would be written and read again: that pipe bounded the kernel, dx
// alone 117 us where it now takes 88), dx 2 x 128.
//
// Warp roles (576 threads): warps 0-15 finish (TMEM lane = row, 16 units each), warp 16 loads by TMA, warp 17 issues tcgen05.mma.
#pragma once

#include "matmul.cuh"

namespace b200ta {

struct NarrowParams {
  int rows, K, N;      // N: hidden units
  int kblocks;         // blocks of 64 inputs, 1 or 2
  int chunks;          // of 64 units
  int store_dz;
  const void* bias;
  int activation;
  int* status;
};

struct Narrow {
  bool f16, gated;
  Plane x, dy, w, dx, dz;  // gated: w of two planes, dz of two planes; dz without a base: not stored
  const void* bias = nullptr;
  int activation = kActNone;
  const char* what = "narrow";
};
int run_narrow(const Narrow& n, void* stream);

#ifdef __CUDACC__
namespace narrow {

constexpr int kThreads = 576;
constexpr int kSlab = 2048;       // 32 rows of 64 bytes, or two of 32 rows of 32
constexpr int kHalf = kSlab / 2;

__device__ __forceinline__ void store_slab(uint32_t slab, int lane, const uint32_t (&x)[16]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) sts128(slab + sw64_offset(lane, j), make_uint4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]));
}
// 32 rows of 16 units; 16-byte vectors swapped in every second group of four rows (SWZ_32), so that lanes meet no bank twice.
__device__ __forceinline__ uint32_t half_offset(int lane, int j) { return lane * 32u + ((uint32_t(j) ^ ((uint32_t(lane) >> 2) & 1u)) << 4); }
__device__ __forceinline__ void store_half(uint32_t slab, int lane, const uint32_t (&x)[16]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) sts128(slab + half_offset(lane, j), make_uint4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]));
}
__device__ __forceinline__ void load_half(uint32_t slab, int lane, uint32_t (&aux)[16]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint4 x = lds128(slab + half_offset(lane, j));
    aux[4 * j] = x.x, aux[4 * j + 1] = x.y, aux[4 * j + 2] = x.z, aux[4 * j + 3] = x.w;
  }
}
// dz of 16 units (in the first halves of y, yg): accumulators of the values at `v` and of the gates at `g` (kDenseGrad: only `v`).
template <typename T, MatmulForm kForm>
__device__ __forceinline__ void units_dz(uint32_t v_addr, uint32_t g_addr, int n, const NarrowParams& p, const uint32_t (&aux)[16],
                                         uint32_t (&y)[16], uint32_t (&yg)[16]) {
  constexpr bool kTwo = kForm == kGatedGrad;
  const T* bias = static_cast<const T*>(p.bias);
  float v[16], gate[16];
  matmul::tmem_load(v_addr, v);
  if constexpr (kTwo) matmul::tmem_load(g_addr, gate);
  tmem_ld_wait();
  if (bias != nullptr) {
    uint32_t b[8];
    matmul::load_bias<T, 16>(b, bias, n, p.N);
    matmul::add_bias<T>(v, b);
    if constexpr (kTwo) {
      matmul::load_bias<T, 16>(b, bias + p.N, n, p.N);
      matmul::add_bias<T>(gate, b);
    }
  }
  matmul::finish_any<T, kForm, 0, 16>(p.activation, v, gate, true, aux, y, yg);
}

constexpr int kStages = 2;
constexpr int kSmX = 0, kSmW = 65536, kSmOut = kSmW + kStages * 32768, kSmSlabs = kSmOut + 32 * kSlab, kSmBars = kSmSlabs + 16 * kSlab;
enum Bar {
  X_FULL = 0, X_EMPTY = 2, S_FULL = 4, D_FULL = 6, DX_FULL = 8, DX_EMPTY = 10, W_FULL = 12, W_EMPTY = W_FULL + kStages,
  AUX = W_EMPTY + kStages, NUM_BARS = AUX + 32
};
constexpr int kSmTotal = kSmBars + NUM_BARS * 8 + 32, kSmDynamic = kSmTotal + 1024;
static_assert(kSmDynamic <= 232448, "shared memory of a block");

template <typename T, MatmulForm kForm>
__global__ void __launch_bounds__(kThreads, 1)
narrow_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
              const __grid_constant__ CUtensorMap tm_dy, const __grid_constant__ CUtensorMap tm_dx,
              const __grid_constant__ CUtensorMap tm_dz, const NarrowParams p) {
  constexpr bool kTwo = kForm == kGatedGrad;
  constexpr int kColumns = kTwo ? 128 : 64;     // accumulator columns of a chunk
  constexpr int kWBlock = kColumns * 128;       // bytes of a chunk's rows of W for 64 inputs

  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + kSmBars;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + kSmBars + NUM_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + kSmBars + NUM_BARS * 8 + 8);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    abort_flag[0] = 0, abort_flag[1] = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + (X_FULL + i) * 8, 1), mbar_init(bars + (X_EMPTY + i) * 8, 1);
      mbar_init(bars + (S_FULL + i) * 8, 1);
      mbar_init(bars + (D_FULL + i) * 8, 16);
      mbar_init(bars + (DX_FULL + i) * 8, 1), mbar_init(bars + (DX_EMPTY + i) * 8, 16);
    }
    for (int i = 0; i < kStages; ++i) mbar_init(bars + (W_FULL + i) * 8, 1), mbar_init(bars + (W_EMPTY + i) * 8, 1);
    for (int i = 0; i < 32; ++i) mbar_init(bars + (AUX + i) * 8, 1);
    fence_mbar_init();
  }
  if (warp == 17) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    pdl_trigger();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int items = (((p.rows + 255) / 256 - 1) - int(blockIdx.x)) / int(gridDim.x) + 1;

  if (warp == 16) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&tm_x);
      tma_prefetch_desc(&tm_w);
      pdl_wait();
      bool ok = true;
      int w_issued = 0, x_issued = 0;
      auto load_x = [&](int i, int t) {
        ok = mbar_wait(bars + (X_EMPTY + t) * 8, (i & 1) ^ 1, abort_flag);
        if (!ok) return;
        const uint32_t full = bars + (X_FULL + t) * 8;
        mbar_expect_tx(full, p.kblocks * 16384);
        for (int kb = 0; kb < p.kblocks; ++kb)
          tma_load_3d(base + kSmX + t * 32768 + kb * 16384, &tm_x, full, kb * 64, (blockIdx.x + i * gridDim.x) * 256 + t * 128, 0);
        if (t == 1) x_issued = i + 1;
      };
      for (int i = 0; ok && i < items; ++i) {
        for (int c = 0; ok && c < p.chunks; ++c) {
          // the first tile of W before the second x: the order in which they are used
          if (c == 0) load_x(i, 0);
          if (!ok) break;
          const int stage = w_issued % kStages;
          ok = mbar_wait(bars + (W_EMPTY + stage) * 8, ((w_issued / kStages) & 1) ^ 1, abort_flag);
          if (!ok) break;
          const uint32_t full = bars + (W_FULL + stage) * 8;
          mbar_expect_tx(full, p.kblocks * kWBlock);
          for (int kb = 0; kb < p.kblocks; ++kb)
            for (int g = 0; g < 2; ++g)  // kTwo: 32 value rows, then their gate rows
              tma_load_3d(base + kSmW + stage * 32768 + kb * kWBlock + g * (kWBlock / 2), &tm_w, full, kb * 64, c * 64 + g * 32, 0);
          ++w_issued;
          if (c == 0) load_x(i, 1);
        }
      }
      if (*abort_flag) {  // a bounded chance to land for copies in flight
        for (int j = w_issued > kStages ? w_issued - kStages : 0; j < w_issued; ++j)
          mbar_wait(bars + (W_FULL + j % kStages) * 8, (j / kStages) & 1, abort_flag + 1);
        for (int t = 0; t < 2 && x_issued > 0; ++t) mbar_wait(bars + (X_FULL + t) * 8, (x_issued - 1) & 1, abort_flag + 1);
      }
    }
  } else if (warp == 17) {
    // ------------------------------------------------------------------ MMA issuer (whole warp, one lane issues)
    constexpr bool kF16 = __is_same(T, __half);
    const uint32_t id_s = matmul::idesc(kF16, 128, kColumns, false, false);
    const uint32_t id_dx = matmul::idesc(kF16, 128, (p.K + 15) / 16 * 16, false, true);
    const uint32_t tb = __shfl_sync(0xffffffffu, tmem_base, 0);
    const int steps = items * p.chunks * 2;
    bool ok = true;
    // step s: row tile s & 1, chunk (s / 2) % chunks of item s / 2 / chunks
    auto issue_s = [&](int s) {
      const int t = s & 1, w = s >> 1, i = w / p.chunks, c = w - i * p.chunks, stage = w % kStages;
      if (c == 0) ok = mbar_wait_warp(bars + (X_FULL + t) * 8, i & 1, abort_flag);
      if (ok && t == 0) ok = mbar_wait_warp(bars + (W_FULL + stage) * 8, (w / kStages) & 1, abort_flag);
      if (!ok) return;
      tc_fence_after();
      for (int kb = 0; kb < p.kblocks; ++kb) {
        const uint64_t da = smem_desc<16, 1024, kLayoutSw128>(base + kSmX + t * 32768 + kb * 16384);
        const uint64_t db = smem_desc<16, 1024, kLayoutSw128>(base + kSmW + stage * 32768 + kb * kWBlock);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_ss_warp(tb + t * 128, da + k * 2, db + k * 2, id_s, (kb > 0 || k > 0) ? 1u : 0u);
      }
      umma_commit_warp(bars + (S_FULL + t) * 8);
      if (c == p.chunks - 1) umma_commit_warp(bars + (X_EMPTY + t) * 8);
    };
    if (ok) issue_s(0);
    if (ok) issue_s(1);
    for (int s = 0; ok && s < steps; ++s) {
      const int t = s & 1, w = s >> 1, i = w / p.chunks, c = w - i * p.chunks, stage = w % kStages;
      ok = mbar_wait_warp(bars + (D_FULL + t) * 8, w & 1, abort_flag);
      if (ok && c == 0) ok = mbar_wait_warp(bars + (DX_EMPTY + t) * 8, (i & 1) ^ 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      // dz of 16 units in the first 8 columns of their part of S; W: rows (hidden units) of 64 inputs, blocks of 64 inputs kWBlock apart
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint64_t db = smem_desc<kWBlock, 1024, kLayoutSw128>(base + kSmW + stage * 32768 + g * (kWBlock / 2));
#pragma unroll
        for (int k = 0; k < kColumns / 32; ++k)
          umma_ts_warp(tb + 256 + t * 128, tb + t * 128 + g * (kColumns / 2) + k * 16, db + k * 128, id_dx, (c > 0 || g > 0 || k > 0) ? 1u : 0u);
      }
      if (t == 1) umma_commit_warp(bars + (W_EMPTY + stage) * 8);
      if (c == p.chunks - 1) umma_commit_warp(bars + (DX_FULL + t) * 8);
      if (s + 2 < steps) issue_s(s + 2);  // behind the product that reads dz, whose columns it overwrites
    }
  } else {
    // ------------------------------------------------------------------ finishing warps: all of them on every step
    pdl_wait();
    const int quad = warp & 3, part = warp >> 2;  // 32 rows, 16 of the chunk's units
    const uint32_t lane_tmem = tmem_base + (uint32_t(quad * 32) << 16);
    const uint32_t slabs = base + kSmSlabs + warp * kSlab, aux_bars = bars + (AUX + warp * 2) * 8;  // one for each row tile
    const uint32_t outs = base + kSmOut + warp * 2 * kSlab;
    const uint32_t s_column = (part >> 1) * (kColumns / 2) + (part & 1) * 16;
    const int steps = items * p.chunks;
    auto row_of = [&](int i, int t) { return (int(blockIdx.x) + i * int(gridDim.x)) * 256 + t * 128 + quad * 32; };
    auto load_dy = [&](int i, int c, int t) {
      if (lane == 0) {
        mbar_expect_tx(aux_bars + t * 8, kHalf);
        tma_load_3d(slabs + t * kHalf, &tm_dy, aux_bars + t * 8, c * 64 + part * 16, row_of(i, t), 0);
      }
    };
    load_dy(0, 0, 0);
    load_dy(0, 0, 1);
    bool ok = true;
    int i = 0, c = 0;
    for (int w = 0; ok && w < steps; ++w) {
      const int unit = c * 64 + part * 16;
      const bool last = c + 1 == p.chunks;
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        uint32_t aux[16], y[16], yg[16];
        ok = mbar_wait2_warp(bars + (S_FULL + t) * 8, w & 1, aux_bars + t * 8, w & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        load_half(slabs + t * kHalf, lane, aux);
        const uint32_t s_addr = lane_tmem + t * 128 + s_column;
        units_dz<T, kForm>(s_addr, s_addr + 32, unit, p, aux, y, yg);
        // (dz takes the place of accumulators that have been read, by this warp alone)
        tmem_st8(s_addr, reinterpret_cast<const uint32_t(&)[8]>(y));
        if constexpr (kTwo) tmem_st8(s_addr + 32, reinterpret_cast<const uint32_t(&)[8]>(yg));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_warp(bars + (D_FULL + t) * 8);
        if (p.store_dz) {
          const uint32_t out = outs + t * kSlab;
          if (lane == 0) tma_store_wait_read<1>();  // the stores of this row tile's step before have read the slabs
          __syncwarp();
          store_half(out, lane, y);
          if constexpr (kTwo) store_half(out + kHalf, lane, yg);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (row_of(i, t) < p.rows && unit < p.N) {
              tma_store_3d(&tm_dz, out, unit, row_of(i, t), 0);
              if constexpr (kTwo) tma_store_3d(&tm_dz, out + kHalf, unit, row_of(i, t), 1);
            }
            tma_store_commit();  // (an empty group as well: they are counted)
          }
        }
        // what the slab held has been used
        if (!last) load_dy(i, c + 1, t);
        else if (i + 1 < items) load_dy(i + 1, 0, t);
      }
      if (!ok) break;
      if (++c < p.chunks) continue;
      // dx of the row tiles
#pragma unroll 1
      for (int t = 0; ok && t < 2; ++t) {
        ok = mbar_wait_warp(bars + (DX_FULL + t) * 8, i & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const int n = part * 32;
        if (n < p.K) {
          const uint32_t out = outs + t * kSlab;
          float v[32];
          uint32_t x[16];
          matmul::tmem_load(lane_tmem + 256 + t * 128 + n, v);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
          if (lane == 0) tma_store_wait_read<0>();
          __syncwarp();
          store_slab(out, lane, x);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (row_of(i, t) < p.rows) tma_store_3d(&tm_dx, out, n, row_of(i, t), 0);
            tma_store_commit();
          }
        }
        tc_fence_before();
        __syncwarp();
        mbar_arrive_warp(bars + (DX_EMPTY + t) * 8);
      }
      c = 0, ++i;
    }
    if (!ok && lane == 0)  // loads in flight land
      for (int t = 0; t < 2; ++t) mbar_wait(aux_bars + t * 8, 0, abort_flag + 1), mbar_wait(aux_bars + t * 8, 1, abort_flag + 1);
    if (lane == 0) tma_store_wait_all();
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) *p.status = B200TA_ERR_DEVICE_WAIT;
}

}  // namespace narrow
#endif  // __CUDACC__
}  // namespace b200ta

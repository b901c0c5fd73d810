// Layer norm over the last axis and its gradients (sm_100a), for bf16, fp16 or fp32 rows:
//
//   y  = (x - mean) rstd w + b                          rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd (g - mean(g) - xh mean(g xh))             g = dy w, xh = (x - mean) rstd
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Bound: HBM.  Forward reads x and writes y, backward reads x and dy and writes dx, each once: a row is held in the
// registers of the 2 to 512 threads that share it, and its mean and variance, or its two sums, are taken there in 32 bits,
// the variance from centred values.  Issue slots come next (a first version with 64-bit index arithmetic and unpacked sums
// needed 200 instructions for 16 values a lane and stayed at half the bandwidth), so addresses advance by constants, sums
// and products are made in packed pairs, and groups of lanes have a size known at compile time.  Blocks are persistent; a
// thread keeps its columns, and with them their parameters in registers (of up to 16 columns), and copies the next rows'
// vectors into its own slots of shared memory while it works on one (registers alone hold too few bytes in flight).
// Measured: 262144 rows of 128 in bf16 forward 23 us (5.8 TB/s), backward 38 us from a cold L2 (5.2 TB/s) and 4.4 for its join;
// 20000 rows of 1024 in fp32 28 and 46; 6001 of 8192 in fp16 45 and 87.
//
// Rows that are not 16-byte aligned (odd widths, odd pitches) take the same path: vectors lie on the 16-byte boundaries of the
// row that is written, and the at most 2 * 7 elements (fp32: 3) before the first and behind the last whole vector are taken by
// the row's first lanes, an element each.  Blocks step by a multiple of 8 (fp32: 4) rows, after which every pitch is back on
// the same boundary, so a thread keeps its columns.  A tensor whose rows lie otherwise is read by two aligned vectors that are
// shifted into place.  (A 16-byte vector with a byte of the row in it lies in the row's allocation.)  Vectors on the boundaries
// of x's columns instead, shifted on their way in and out, cost three times the instructions: 9000 rows of 1027 in bf16 took 39 us
// forward and 50 backward, now 16 and 28; 100000 of 127 took 29 and 36, now 18 and 28.
#pragma once

#include "activation.cuh"
#include "common.cuh"

namespace b200ta {

struct NormParams {
  const void *x, *dy, *w, *b;
  void *y, *dx;
  float2* stats;   // {rstd, -mean * rstd} per row: written by the forward pass (if not NULL), read by the backward pass
  float* partial;  // [blocks][2][width], or NULL where sums are not wanted or one block has them all
  void *dw, *db;   // of that block, each may be NULL
  long long xs, ys, dys, dxs, rows;
  int width;
  int lanes;           // threads that share a row, a power of two
  float eps;
};

struct NormShape {
  int lanes, items, threads;
  bool shifted;
};
constexpr int kNormThreads = 256;  // of a block, unless a row takes more
constexpr int kNormMaxWidth = 16384;
// Threads that share a row: a warp or less (from 2, shifted 8), or up to `most_lanes` of them, as long as 16 values a thread hold the row;
// up to 512 with 32 values for what is wider.
inline NormShape norm_shape(int width, int vec, int most_lanes, bool shifted) {
  NormShape s;
  s.shifted = shifted;
  const int n = width / vec, most = (n > most_lanes * 16 / vec ? 32 : 16) / vec;
  s.lanes = shifted ? 8 : 2;  // (with fewer a lane would take four or eight single elements)
  while (s.lanes < 32 && s.lanes < n) s.lanes *= 2;
  while (s.lanes * most < n) s.lanes *= 2;
  s.items = n > 0 ? (n + s.lanes - 1) / s.lanes : 1;
  // the kernels are made for 1, 2 and all items of 16 values, and for those of 32
  s.items = s.items <= 2 ? s.items : s.items * vec <= 16 ? 16 / vec : 32 / vec;
  s.threads = s.lanes > kNormThreads ? s.lanes : kNormThreads;
  return s;
}
// Blocks of a grid, at most `most`: those of shifted rows step by whole periods of their alignment.
inline int norm_blocks(int64_t rows, int64_t most, int per_block, int vec, bool shifted) {
  const int64_t need = (rows + per_block - 1) / per_block;
  if (need <= most) return int(need);
  return int(shifted && per_block < vec ? most - most % (vec / per_block) : most);
}
inline int norm_element_bytes(int dtype) { return dtype == B200TA_DTYPE_F32 ? 4 : 2; }
inline bool norm_aligned(const void* p, int64_t stride, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride * bytes % 16 == 0;
}

#ifdef __CUDACC__
namespace norm {

// kVec values of 16 bytes in packed pairs.
template <typename T>
struct Values {
  static constexpr int kVec = 16 / int(sizeof(T));
  F2 p[kVec / 2];
  __device__ __forceinline__ explicit Values(uint4 x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < kVec / 2; ++j) {
      if constexpr (sizeof(T) == 4) {
        p[j] = F2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
      } else {
        const float2 f = unpack2<T>(w[j]);
        p[j] = F2(f.x, f.y);
      }
    }
  }
};
template <typename T>
__device__ __forceinline__ uint4 bits_of(const F2* p) {
  float a[8];
  if constexpr (sizeof(T) == 4) {
    p[0].to(a[0], a[1]), p[1].to(a[2], a[3]);
    return make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j].to(a[2 * j], a[2 * j + 1]);
    return make_uint4(pack2<T>(a[0], a[1]), pack2<T>(a[2], a[3]), pack2<T>(a[4], a[5]), pack2<T>(a[6], a[7]));
  }
}

// Bytes `at` .. `at` + 15 of the 32 bytes of lo and hi (0 <= at < 16, a multiple of the element size).
template <typename T>
__device__ __forceinline__ uint4 window(uint4 lo, uint4 hi, uint32_t at) {
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  if (at & 8u) w[0] = w[2], w[1] = w[3], w[2] = w[4], w[3] = w[5], w[4] = w[6], w[5] = w[7];
  if (at & 4u) w[0] = w[1], w[1] = w[2], w[2] = w[3], w[3] = w[4], w[4] = w[5];
  if (sizeof(T) == 2 && (at & 2u)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The first `valid` elements of a vector, zeros behind them.
template <typename T>
__device__ __forceinline__ uint4 first(uint4 x, int valid) {
  constexpr int kPer = 4 / int(sizeof(T));
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int left = valid - j * kPer;
    w[j] = left >= kPer ? w[j] : left <= 0 ? 0u : w[j] & 0xFFFFu;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows that a group of threads works on at a time: two where a thread holds 16 values, so that a row's sums over the group
// (shuffles, and a barrier beyond a warp) cost half.
__host__ __device__ constexpr int rows_at_a_time(int values) { return values == 16 ? 2 : 1; }
// Slots of shared memory for rows of `vectors` vectors a thread, those that are worked on included.
__host__ __device__ constexpr int stages_of(int vectors, int threads, int blocks) {
  const int by_bytes = 196608 / blocks / (vectors * threads * 16);
  return by_bytes < 4 ? by_bytes : 4;
}
__device__ __forceinline__ void copy_ahead(uint32_t slot, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// 16 bytes, or zeros without an access: no branch, so that a thread's loads are on their way together.
__device__ __forceinline__ uint4 load_if(bool in, const void* p) {
  uint4 v;
  asm volatile(
      "{\n.reg .pred q;\nsetp.ne.u32 q, %5, 0;\nmov.u32 %0, 0;\nmov.u32 %1, 0;\nmov.u32 %2, 0;\nmov.u32 %3, 0;\n"
      "@q ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"(static_cast<uint32_t>(in)));
  return v;
}
// The vector at `p`, of any alignment, of a row of `width` elements from `row` on: from the two aligned vectors that hold it, as
// far as they touch the row.
template <typename T>
__device__ __forceinline__ uint4 load_anywhere(const T* p, const T* row, int width) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), at = a & 15u, lo = a - at, hi = lo + 16;
  const uintptr_t begin = reinterpret_cast<uintptr_t>(row), end = begin + width * sizeof(T);
  const uint4 x = load_if(hi > begin && lo < end, reinterpret_cast<const void*>(lo));
  const uint4 z = load_if(at != 0 && hi + 16 > begin && hi < end, reinterpret_cast<const void*>(hi));
  return window<T>(x, z, uint32_t(at));
}
template <typename T>
__device__ __forceinline__ float element_if(bool in, const T* p) {  // zero without an access
  if constexpr (sizeof(T) == 4) {
    float v;
    asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\nmov.f32 %0, 0f00000000;\n@q ld.global.nc.f32 %0, [%1];\n}"
                 : "=&f"(v) : "l"(p), "r"(static_cast<uint32_t>(in)));
    return v;
  } else {
    uint16_t v;
    asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %2, 0;\nmov.u16 %0, 0;\n@q ld.global.nc.u16 %0, [%1];\n}"
                 : "=&h"(v) : "l"(p), "r"(static_cast<uint32_t>(in)));
    return unpack2<T>(uint32_t(v)).x;
  }
}

// How a thread's part of a row lies: whole vectors from `column` on, one every lanes * kVec columns, and (kShifted) single
// elements before the first and behind the last vector of the row, kSingles of them at most.
template <typename T, bool kShifted, int kLanes>
struct Place {
  static constexpr int kVec = Values<T>::kVec;
  static constexpr int kSingles = !kShifted ? 0 : kLanes >= 2 * kVec ? 1 : 2 * kVec / kLanes, kSlots = kSingles ? kSingles : 1;
  int vectors;         // of the row, from this lane's first on
  int column;
  int single[kSlots];  // their columns, -1: none
  __device__ __forceinline__ Place(const T* row, int width, int lane, int lanes) {
    const int before = int((16u - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / int(sizeof(T));
    const int head = !kShifted ? 0 : before < width ? before : width, all = (width - head) / kVec, rest = head + all * kVec;
    vectors = all - lane, column = head + lane * kVec;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int e = lane + i * lanes, c = e < kVec ? e : rest + e - kVec;
      single[i] = kShifted && (e < kVec ? e < head : e < 2 * kVec && c < width) ? c : -1;
    }
  }
};

// The parameters of kVec columns from c on, or `none` where there are none.
template <typename T, typename W, bool kShifted>
__device__ __forceinline__ void load_param(const NormParams& p, const void* param, int c, float none, F2* v) {
  constexpr int kVec = Values<T>::kVec, kHalf = Values<W>::kVec;
  if (param == nullptr) {
#pragma unroll
    for (int j = 0; j < kVec / 2; ++j) v[j] = F2(none);
    return;
  }
  const W* q = static_cast<const W*>(param) + c;
#pragma unroll
  for (int h = 0; h < kVec; h += kHalf) {  // 16-bit rows with 32-bit parameters: two vectors
    uint4 raw;
    if constexpr (kShifted) raw = load_anywhere(q + h, static_cast<const W*>(param), p.width);
    else raw = __ldg(reinterpret_cast<const uint4*>(q + h));
    const Values<W> x(raw);
#pragma unroll
    for (int j = 0; j < kHalf / 2; ++j) v[h / 2 + j] = x.p[j];
  }
}
template <typename W>
__device__ __forceinline__ float single_param(const void* param, int c, float none) {
  return param == nullptr ? none : element_if(c >= 0, static_cast<const W*>(param) + c);
}

__device__ __forceinline__ float sum_of(F2 p) {
  float a, b;
  p.to(a, b);
  return a + b;
}

// The sums over the threads that share a row; every one of them gets the result.  Rows of more than a warp go through one of
// two halves of `scratch` in turn (32 warps each): all threads of the block call this equally often.
template <int kLanes, int kSums>
__device__ __forceinline__ void row_sums(float (&s)[kSums], int lanes, float* scratch, int& turn) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < kSums; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
  if (kLanes == 32 && lanes > 32) {
    const int warp = threadIdx.x >> 5, warps = lanes >> 5, first = warp / warps * warps;
    float* half = scratch + turn * 32 * kSums;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < kSums; ++i) half[warp * kSums + i] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSums; ++i) s[i] = 0.f;
    for (int w = first; w < first + warps; w += 2)  // two warps' in one access
#pragma unroll
      for (int i = 0; i < kSums; i += 2) {
        if constexpr (kSums == 1) {
          const float2 x = *reinterpret_cast<const float2*>(half + w);
          s[0] += x.x + x.y;
        } else {
          const float2 x = *reinterpret_cast<const float2*>(half + w * kSums + i);
          const float2 z = *reinterpret_cast<const float2*>(half + (w + 1) * kSums + i);
          s[i] += x.x + z.x, s[i + 1] += x.y + z.y;
        }
      }
  }
}

// Launches one kernel; its shared-memory limit is raised once on each device.
template <auto kKernel>
int launch_one(DeviceState* st, int blocks, int threads, int smem, void* stream, const NormParams& p) {
  static std::atomic<uint64_t> raised{0};
  const uint64_t bit = 1ull << st->device;
  if (smem > 40 * 1024 && !(raised.load(std::memory_order_relaxed) & bit)) {
    B200TA_CHECK_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    raised.fetch_or(bit, std::memory_order_relaxed);
  }
  return launch_kernel(st, kKernelNorm, kKernel, dim3(unsigned(blocks)), threads, smem, stream, p);
}

// The launch of a shape's kernel<T, W, kShifted, kItems, kLanes, kMost>: 2, 4, 8, 16 or (at least) 32 lanes, blocks of at most
// kMost threads.
#define B200TA_NORM_PICK(kernel, T, W, kShifted, s)                                  \
  (s.threads > 256 && s.items > int(sizeof(T))                                       \
       ? &norm::launch_one<kernel<T, W, kShifted, 2 * int(sizeof(T)), 32, 512>>      \
   : s.threads > 256     ? &norm::launch_one<kernel<T, W, kShifted, int(sizeof(T)), 32, 512>>         \
   : s.lanes == 2        ? &norm::launch_one<kernel<T, W, kShifted, 1, kShifted ? 8 : 2, 256>>                       \
   : s.lanes == 4        ? &norm::launch_one<kernel<T, W, kShifted, 1, kShifted ? 8 : 4, 256>>                       \
   : s.lanes == 8        ? &norm::launch_one<kernel<T, W, kShifted, 1, 8, 256>>                       \
   : s.lanes == 16       ? &norm::launch_one<kernel<T, W, kShifted, 1, 16, 256>>                      \
   : s.items == 1        ? &norm::launch_one<kernel<T, W, kShifted, 1, 32, 256>>                      \
   : s.items == 2        ? &norm::launch_one<kernel<T, W, kShifted, 2, 32, 256>>                      \
   : s.items <= sizeof(T) ? &norm::launch_one<kernel<T, W, kShifted, int(sizeof(T)), 32, 256>>        \
                         : &norm::launch_one<kernel<T, W, kShifted, 2 * int(sizeof(T)), 32, 256>>)

}  // namespace norm
#endif  // __CUDACC__
}  // namespace b200ta

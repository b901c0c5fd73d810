// The kernels of low-rank adapters beside the tensor-core products: low-rank values, their weights' gradients, small layouts.
#include <algorithm>
#include <type_traits>

#include "adapters.cuh"
#include "layer_norm.cuh"
#include "warp_matmul.cuh"

namespace b200ta {
namespace {

// Eight elements of a row of K from k on, zeros behind it.
template <typename T, bool kVec>
__device__ __forceinline__ uint4 load_eight_of(const T* row, int k, int K) {
  const uint4 v = kVec ? norm::load_if(k < K, row + k) : norm::load_anywhere(row + k, row, K);
  return K - k >= 8 ? v : norm::first<T>(v, K - k);
}

template <typename T>
__device__ __forceinline__ void store_low(const LowProduct& p, long long row, int r, float v) {
  T* low = static_cast<T*>(p.low) + row * low_pitch(p.rank) + low_place(p.rank, r);
  const T rounded = static_cast<T>(v);
  *low = rounded;
  low[low_unit(p.rank)] = static_cast<T>(second_term(v, static_cast<float>(rounded)));
}

// ---- low-rank values, a warp for each ------------------------------------------------------------------------------
//
// Few rows, or rows of many different adapters: a warp multiplies a row of x with one row of its adapter, 16 bytes a lane at a time.
// Bound by latency, then by the adapters' way from L2 (each row reads its own).
constexpr int kDotWarps = 8;
template <typename T, bool kVec>
__global__ void __launch_bounds__(kDotWarps * 32)
low_dot_kernel(const LowProduct p, int groups) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, r = int(blockIdx.x % unsigned(groups)) * kDotWarps + (threadIdx.x >> 5);
  const long long row = blockIdx.x / unsigned(groups);
  if (r >= low_pitch(p.rank) / 2) return;
  const int g = adapter_of(p.index, uint32_t(row));
  float sum = 0.f;
  if (g != kNoAdapter && r < p.rank) {
    for (int plane = 0; plane < p.planes; ++plane) {
      const T* x = static_cast<const T*>(p.x) + row * p.xs + plane * p.x_plane;
      const T* a = static_cast<const T*>(p.a) + ((long long)(g * p.planes + plane) * p.rank + r) * p.as;
      float2 s = make_float2(0.f, 0.f);
#pragma unroll 4
      for (int k = lane * 8; k < p.K; k += 256) {
        const uint4 u = load_eight_of<T, kVec>(x, k, p.K), v = load_eight_of<T, kVec>(a, k, p.K);
        const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 c = unpack2<T>(uw[j]), d = unpack2<T>(vw[j]);
          s.x = fmaf(c.x, d.x, s.x), s.y = fmaf(c.y, d.y, s.y);
        }
      }
      sum += s.x + s.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    sum *= p.scale != nullptr ? __ldg(p.scale + g) : p.scale_all;
  }
  if (lane == 0) store_low<T>(p, row, r, sum);
}

// ---- low-rank values by warp-wide products ---------------------------------------------------------------------------
//
// A warp takes 32 rows and kTiles * 8 ranks: products m16n8k16 with x as the left and the adapter's rows as the right operand, both read
// as they lie: a lane reads 16 bytes of each of its rows, eight neighbouring k, that serve as the pairs of two products (the order of
// k is the same in both operands and does not matter).  The warps of a block share the rows and take 32 of k in turn, or, where
// there are many rows and few k, take rows of their own.  Rows of other adapters than the first are taken in further
// passes; a pass stores the rows that are its own.  Bound by HBM (x once) or L2.
constexpr int kLowRows = 32;
__host__ __device__ constexpr int low_warps(int tiles) { return tiles == 8 ? 4 : 8; }
template <typename T, int kTiles, bool kVec, bool kExact>  // kExact: x in two terms
__global__ void __launch_bounds__(low_warps(kTiles) * 32)
low_product_kernel(const LowProduct p, int share) {
  constexpr int kWarps = low_warps(kTiles), kRanks = kTiles * 8;
  __shared__ float joined[kWarps][kLowRows][kRanks + 1];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = lane >> 2, t = lane & 3;
  const long long row0 = ((long long)blockIdx.x * (share ? 1 : kWarps) + (share ? 0 : warp)) * kLowRows;
  const int r0 = blockIdx.y * kRanks, first = share ? warp * 32 : 0, step = share ? kWarps * 32 : 32;
  if (row0 >= p.rows) return;  // (of a block whose warps share rows: all of them)
  TileAdapters<1> mine(p.index);
  mine.fetch(p.index, int(row0), int(p.rows));
  mine.arrived(p.index);
  auto store = [&](int row, int r, float v) {  // a value of this warp's rows
    if (r < low_pitch(p.rank) / 2) store_low<T>(p, row0 + row, r, r < p.rank ? v : 0.f);
  };
  const uint32_t in = p.rows - row0 < kLowRows ? (1u << (p.rows - row0)) - 1u : ~0u;  // rows that there are
  // rows without an adapter
  for (int row = share ? warp : 0; row < kLowRows && (in >> row & 1u); row += share ? kWarps : 1)
    if (__shfl_sync(0xffffffffu, mine.g[0], row) == kNoAdapter)
      for (int r = lane; r < kRanks; r += 32) store(row, r0 + r, 0.f);
  for (uint32_t taken[1]; mine.more();) {
    const int g = mine.take(taken);
    const uint32_t own = taken[0] & in;
    const float scale = p.scale != nullptr ? __ldg(p.scale + g) : p.scale_all;
    float acc[2][kTiles][4] = {};
    for (int plane = 0; plane < p.planes; ++plane) {
      const T *x[2][2], *a[kTiles];
      const long long second = kExact ? static_cast<const T*>(p.x2) - static_cast<const T*>(p.x) : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long row = row0 + i * 8 + q;
        x[i >> 1][i & 1] = static_cast<const T*>(p.x) + (row < p.rows ? row : p.rows - 1) * p.xs + plane * p.x_plane;
      }
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        const int r = r0 + j * 8 + q;
        a[j] = static_cast<const T*>(p.a) + ((long long)(g * p.planes + plane) * p.rank + (r < p.rank ? r : p.rank - 1)) * p.as;
      }
#pragma unroll 2
      for (int k = first + t * 8; k - t * 8 < p.K; k += step) {
        uint4 u[2][2], v[kTiles];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i >> 1][i & 1] = load_eight_of<T, kVec>(x[i >> 1][i & 1], k, p.K);
#pragma unroll
        for (int j = 0; j < kTiles; ++j) v[j] = load_eight_of<T, kVec>(a[j], k, p.K);
        auto multiply = [&]() {
#pragma unroll
          for (int j = 0; j < kTiles; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              mma16816<T>(acc[i][j], u[i][0].x, u[i][1].x, u[i][0].y, u[i][1].y, v[j].x, v[j].y);
              mma16816<T>(acc[i][j], u[i][0].z, u[i][1].z, u[i][0].w, u[i][1].w, v[j].z, v[j].w);
            }
        };
        if constexpr (kExact) {
          uint4 rest[2][2];
#pragma unroll
          for (int i = 0; i < 4; ++i) rest[i >> 1][i & 1] = load_eight_of<T, kVec>(x[i >> 1][i & 1] + second, k, p.K);
          multiply();
#pragma unroll
          for (int i = 0; i < 4; ++i) u[i >> 1][i & 1] = rest[i >> 1][i & 1];
        }
        multiply();
      }
    }
    if (share) {
      __syncthreads();  // (all warps have the same rows, and so the same passes)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) joined[warp][i * 16 + q + 8 * (e >> 1)][j * 8 + t * 2 + (e & 1)] = acc[i][j][e];
      __syncthreads();
      for (int i = threadIdx.x; i < kLowRows * kRanks; i += kWarps * 32) {
        const int row = i / kRanks, r = i % kRanks;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += joined[w][row][r];
        if (own >> row & 1u) store(row, r0 + r, sum * scale);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = i * 16 + q + 8 * h, r = r0 + j * 8 + t * 2;
            if (!(own >> row & 1u) || r >= low_pitch(p.rank) / 2) continue;
            const float v0 = r < p.rank ? acc[i][j][2 * h] * scale : 0.f, v1 = r + 1 < p.rank ? acc[i][j][2 * h + 1] * scale : 0.f;
            T* to = static_cast<T*>(p.low) + (row0 + row) * low_pitch(p.rank) + low_place(p.rank, r);
            const uint32_t rounded = pack2<T>(v0, v1);
            const float2 f = unpack2<T>(rounded);
            *reinterpret_cast<uint32_t*>(to) = rounded;
            *reinterpret_cast<uint32_t*>(to + low_unit(p.rank)) = pack2<T>(second_term(v0, f.x), second_term(v1, f.y));
          }
    }
  }
}

int dot_groups(int rank) { return (low_pitch(rank) / 2 + kDotWarps - 1) / kDotWarps; }
bool low_by_dots(const LowProduct& m, int num_sms) {
  return low_by_rows(m.rows, m.rank, m.K * m.planes, m.index, dot_groups(m.rank), num_sms);
}
// (Of dz with second terms by products alone: run_low_up() takes what low_by_rows() says, which comprises what low_by_dots() would.)
template <typename T, bool kVec>
int launch_low(DeviceState* st, const LowProduct& m, void* stream) {
  if (low_by_dots(m, st->num_sms)) {
    const int groups = dot_groups(m.rank);
    return launch_kernel(st, kKernelAdapter, low_dot_kernel<T, kVec>, dim3(unsigned(m.rows * groups)), kDotWarps * 32, 0, stream, m, groups);
  }
  const int64_t groups = (m.rows + kLowRows - 1) / kLowRows;
  // All ranks in a block, up to 64, or more blocks of fewer where these leave multiprocessors idle (158 rows of 1448, rank 76, two adapters
  // in turn: 10 us for 30; a gated training step of 300 rows of 2048, rank 64: 115 for 175).
  int tiles = m.rank <= 16 ? 2 : m.rank <= 32 ? 4 : 8;
  for (int i = 0; i < 2; ++i)
    if (tiles > 2 && groups * ((low_pitch(m.rank) / 2 + tiles * 8 - 1) / (tiles * 8)) * 2 <= st->num_sms) tiles /= 2;
  const int warps = low_warps(tiles);
  const int share = groups < int64_t(st->num_sms) * warps * 2 || m.K > 512;
  const dim3 grid{unsigned(share ? groups : (groups + warps - 1) / warps), unsigned((low_pitch(m.rank) / 2 + tiles * 8 - 1) / (tiles * 8))};
  auto pick = [&](auto exact) {
    constexpr bool kExact = decltype(exact)::value;
    return tiles == 2 ? low_product_kernel<T, 2, kVec, kExact> : tiles == 4 ? low_product_kernel<T, 4, kVec, kExact> : low_product_kernel<T, 8, kVec, kExact>;
  };
  // (dz with its second terms is aligned)
  auto* kernel = kVec && m.x2 != nullptr ? pick(std::integral_constant<bool, kVec>()) : pick(std::false_type());
  return launch_kernel(st, kKernelAdapter, kernel, grid, warps * 32, 0, stream, m, share);
}

// The same of dz and U as it lies, [columns][rank]: a block for a row, whose threads take eight ranks of every so many columns.
struct LowUpParams {
  const void *dz, *dz2, *up;
  void* low;
  const float* scale;
  float scale_all;
  long long zs, z_plane, us;
  int N, planes, rank;
  AdapterIndex index;
};
template <typename T>
__global__ void __launch_bounds__(256)
low_up_kernel(const LowUpParams p) {
  __shared__ float joined[256][9];
  pdl_wait();
  pdl_trigger();
  const long long row = blockIdx.x;
  const int vectors = low_pitch(p.rank) / 16, ways = 256 / vectors, v = threadIdx.x % vectors, way = threadIdx.x / vectors;
  const int g = adapter_of(p.index, uint32_t(row));
  float sum[8] = {};
  if (g != kNoAdapter && way < ways && v * 8 < p.rank) {
    for (int plane = 0; plane < p.planes; ++plane) {
      const T* dz = static_cast<const T*>(p.dz) + row * p.zs + plane * p.z_plane;
      const T* dz2 = p.dz2 == nullptr ? nullptr : static_cast<const T*>(p.dz2) + row * p.zs + plane * p.z_plane;
      const T* up = static_cast<const T*>(p.up) + (long long)(g * p.planes + plane) * p.N * p.us + v * 8;
#pragma unroll 8
      for (int n = way; n < p.N; n += ways) {
        const float d = dz2 == nullptr ? static_cast<float>(dz[n]) : static_cast<float>(dz[n]) + static_cast<float>(dz2[n]);
        const uint4 x = norm::first<T>(__ldg(reinterpret_cast<const uint4*>(up + n * p.us)), p.rank - v * 8);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack2<T>(w[j]);
          sum[2 * j] = fmaf(d, f.x, sum[2 * j]), sum[2 * j + 1] = fmaf(d, f.y, sum[2 * j + 1]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) joined[threadIdx.x][j] = sum[j];
  __syncthreads();
  const int r = threadIdx.x;
  if (r >= low_pitch(p.rank) / 2) return;
  float total = 0.f;
#pragma unroll 8
  for (int w = 0; w < ways; ++w) total += joined[w * vectors + r / 8][r % 8];
  if (r >= p.rank || g == kNoAdapter) total = 0.f;
  else total *= p.scale != nullptr ? __ldg(p.scale + g) : p.scale_all;
  T* low = static_cast<T*>(p.low) + row * low_pitch(p.rank) + low_place(p.rank, r);
  const T rounded = static_cast<T>(total);
  low[0] = rounded, low[low_unit(p.rank)] = static_cast<T>(second_term(total, static_cast<float>(rounded)));
}

// ---- up matrices with their columns contiguous -----------------------------------------------------------------------

struct TransposeParams {
  const uint16_t* up;
  uint16_t* out;
  long long up_pitch, out_pitch;
  int rank, N, planes;
};
__global__ void __launch_bounds__(256)
transpose_up_kernel(const TransposeParams p) {
  __shared__ uint16_t tile[32][34];
  pdl_trigger();
  pdl_wait();
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, n0 = blockIdx.x * 32, r0 = blockIdx.y * 32;
  const long long g = blockIdx.z / p.planes, plane = blockIdx.z % p.planes;
  const uint16_t* up = p.up + (g * p.planes + plane) * p.N * p.up_pitch;
  uint16_t* out = p.out + (g * p.planes + plane) * p.rank * p.out_pitch;
  for (int i = y; i < 32; i += 8)
    if (n0 + i < p.N && r0 + x < p.rank) tile[i][x] = up[(n0 + i) * p.up_pitch + r0 + x];
  __syncthreads();
  for (int i = y; i < 32; i += 8)
    if (r0 + i < p.rank && n0 + x < p.N) out[(long long)(r0 + i) * p.out_pitch + n0 + x] = tile[x][i];
}

// ---- gradients of the adapters' weights ---------------------------------------------------------------------------------
//
// dD_g = sum over the rows of g of dt^T x, dU_g likewise of t and dz: bound by HBM or L2 (x and dz once), with 64 ranks by the warp-wide
// products.  A block takes 128 columns, one adapter, up to 64 ranks and a part of the rows, 64 at a time through a ring of stages that a
// ninth warp fills by TMA.  Products m16n8k16 with ranks as rows and the tensor's rows along k: both operands lie with k across and
// are transposed on their way from shared memory.  Of several adapters a block first lists the groups of 64 rows that hold its own;
// in a group that others have a part of, their rows are cleared in the operands' registers, so that infinities and NaN in them stay
// out.  Parts are written in 32 bits, with a mark that they have been (a part of the rows may have none of an adapter's), and joined in
// a fixed order: results repeat bit by bit.  A single part is the result.  147456 rows of 128 and 1024 columns, rank 16: 57 us (359 MB at
// 6.3 TB/s; filled by cp.async from all threads 89); 8192 rows of 8192 columns, rank 64: 50 us (the products' pipe 0.73 full).
constexpr int kGradRows = 64, kGradColumns = 128, kGradChunks = 1024, kGradWarps = 8;
// (up to 16, 32 or 64 ranks with their two terms are rows of 64 or 128 bytes, or two blocks of the latter)
constexpr int kGradV = kGradRows * kGradColumns * 2;
__host__ __device__ constexpr int grad_stage(int tiles) { return kGradV + kGradRows * tiles * 64; }
__host__ __device__ constexpr int grad_stages(int tiles) { return tiles == 4 ? 3 : 4; }

struct GradParams {
  LowGrad job[2];
  AdapterIndex index;
  int rows, rank, rank_groups, slabs0, chunks_part, accumulate, direct;
  int terms;  // of the second job's tensor: logarithm
  uint8_t* marks;  // of each block
  int* status;
};
struct GradMaps {
  CUtensorMap t[2], v[2], v2;
};
__device__ __forceinline__ void ldmatrix4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Halves that stay of a pair of rows, whose bits are bits[0] and bits[1].
__device__ __forceinline__ uint32_t pair_mask(uint32_t bits) { return ((bits & 1u) ? 0xFFFFu : 0u) | ((bits & 2u) ? 0xFFFF0000u : 0u); }

template <typename T, int kTiles>  // tiles of 16 ranks
__global__ void __launch_bounds__((kGradWarps + 1) * 32, 2)
low_grad_kernel(const GradParams p, const __grid_constant__ GradMaps maps) {
  constexpr int kStages = grad_stages(kTiles), kStage = grad_stage(kTiles);
  extern __shared__ uint8_t raw[];
  __shared__ uint32_t masks[kGradChunks][2];
  __shared__ uint16_t list[kGradChunks];
  __shared__ __align__(8) uint64_t bars[2 * kStages];  // full, then empty
  __shared__ int listed, aborted[2];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u, bar0 = smem_u32(bars);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    aborted[0] = aborted[1] = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bar0 + i * 8, 1);
      mbar_init(bar0 + (kStages + i) * 8, kGradWarps);
    }
    fence_mbar_init();
  }
  pdl_trigger();
  pdl_wait();
  const int second = int(blockIdx.x) >= p.slabs0;
  const LowGrad& job = second ? p.job[1] : p.job[0];
  const int slab = int(blockIdx.x) - (second ? p.slabs0 : 0), slabs_plane = (job.columns + kGradColumns - 1) / kGradColumns;
  const int plane = slab / slabs_plane, c0 = (slab - plane * slabs_plane) * kGradColumns;
  const int g = blockIdx.z / p.rank_groups, r0 = int(blockIdx.z % unsigned(p.rank_groups)) * 64;
  const int first_row = int(blockIdx.y) * p.chunks_part * kGradRows;
  const int rows = min(p.rows - first_row, p.chunks_part * kGradRows), chunks = rows > 0 ? (rows + kGradRows - 1) / kGradRows : 0;

  // Bits of a group's rows that are g's.  (Rows behind the last one are zeros in shared memory and count where others do.)
  if (p.index.index == nullptr || p.index.rows_per_index >= 16) {  // a thread for a group, of a few entries
    for (int c = threadIdx.x; c < chunks; c += (kGradWarps + 1) * 32) {
      const int row0 = c * kGradRows, in = min(rows - row0, kGradRows);
      uint64_t own = 0;
      if (p.index.index == nullptr) {
        own = ~0ull;
      } else {
        for (int row = 0; row < in;) {
          const uint32_t at = p.index.first_row + uint32_t(first_row + row0 + row), next = (at / p.index.rows_per_index + 1) * p.index.rows_per_index;
          const int end = int(min(uint32_t(in), row + (next - at)));
          if (adapter_of(p.index, uint32_t(first_row + row0 + row)) == g) own |= (end - row >= 64 ? ~0ull : (1ull << (end - row)) - 1) << row;
          row = end;
        }
        if (own != 0 && in < 64) own |= ~0ull << in;
      }
      masks[c][0] = uint32_t(own), masks[c][1] = uint32_t(own >> 32);
    }
  } else {
    for (int c0 = warp; c0 < chunks; c0 += 4 * (kGradWarps + 1)) {
      int own[4][2];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = (c0 + u * (kGradWarps + 1)) * kGradRows + h * 32 + lane;
          own[u][h] = row < rows ? adapter_of(p.index, uint32_t(first_row + row)) : g;
        }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t bits = __ballot_sync(0xffffffffu, own[u][h] == g);
          const int c = c0 + u * (kGradWarps + 1);
          if (lane == 0 && c < chunks) masks[c][h] = bits;
        }
    }
  }
  __syncthreads();
  if (warp == 0) {
    int n = 0;
    for (int c = 0; c < chunks; c += 32) {
      const int at = c + lane < chunks ? c + lane : 0;
      const bool in = c + lane < chunks && (masks[at][0] | masks[at][1]) != 0;
      const uint32_t vote = __ballot_sync(0xffffffffu, in);
      if (in) list[n + __popc(vote & ((1u << lane) - 1u))] = uint16_t(c + lane);
      n += __popc(vote);
    }
    if (lane == 0) listed = n;
  }
  __syncthreads();
  const int terms = second ? p.terms : 0, count = listed << terms;
  volatile int* abort_flag = aborted;
  uint8_t* mark = p.direct ? nullptr : p.marks + ((long long)blockIdx.y * gridDim.z + blockIdx.z) * gridDim.x + blockIdx.x;
  if (count == 0 && !p.direct) {
    if (threadIdx.x == 0 && !p.accumulate) *mark = 0;
    return;
  }

  if (warp == kGradWarps) {
    if (lane == 0) {
      const CUtensorMap *tm_t = &maps.t[second], *tm_first = &maps.v[second];
      bool ok = true;
      int i = 0;
      for (; i < count; ++i) {
        const int s = i % kStages;
        ok = mbar_wait(bar0 + (kStages + s) * 8, (i / kStages & 1) ^ 1, abort_flag);
        if (!ok) break;
        const uint32_t stage = base + s * kStage, bar = bar0 + s * 8;
        const int row = first_row + list[i >> terms] * kGradRows;
        const CUtensorMap* tm_v = i & terms ? &maps.v2 : tm_first;
        mbar_expect_tx(bar, kStage);
        tma_load_3d(stage, tm_v, bar, c0, row, plane);
        tma_load_3d(stage + kGradV / 2, tm_v, bar, c0 + 64, row, plane);
#pragma unroll
        for (int b = 0; b < (kTiles == 4 ? 2 : 1); ++b) tma_load_3d(stage + kGradV + b * kGradRows * 128, tm_t, bar, 2 * r0 + b * 64, row, 0);
      }
      if (!ok)  // copies still in flight get a bounded chance to land
        for (int j = i > kStages ? i - kStages : 0; j < i; ++j) mbar_wait(bar0 + j % kStages * 8, j / kStages & 1, abort_flag + 1);
    }
  } else {
    // A warp has 16 columns and all ranks, or of 64 ranks half and 32 columns: fewer operands for as many products (each warp reads its
    // part of t from shared memory, which bounds it; 8192 rows of 8192 columns: 61 us with all ranks, now 50).
    constexpr int kWays = kTiles == 4 ? 2 : 1, kOwn = kTiles / kWays;
    const int way = kWays == 2 ? warp >> 2 : 0, columns0 = kWays == 2 ? (warp & 3) * 32 : warp * 16;
    float acc[kOwn][2 * kWays][4] = {};
    // rows of 128 bytes (t of 16 ranks: 64) whose 16-byte vectors are swizzled by the row
    const int vr = lane & 15, tr = (lane >> 4) * 8 + (lane & 7);
    uint32_t v_at[kWays];
#pragma unroll
    for (int j = 0; j < kWays; ++j) {
      const int vec = columns0 / 8 + j * 2 + (lane >> 4);
      v_at[j] = (vec >> 3) * (kGradV / 2) + vr * 128 + (((vec & 7) ^ (vr & 7)) << 4);
    }
    bool ok = true;
    for (int i = 0; i < count; ++i) {
      const int s = i % kStages;
      ok = mbar_wait_warp(bar0 + s * 8, i / kStages & 1, abort_flag);
      if (!ok) break;
      const uint32_t stage = base + s * kStage;
      const uint32_t bits0 = masks[list[i >> terms]][0], bits1 = masks[list[i >> terms]][1];
      auto walk = [&](auto&& mask) {
#pragma unroll
        for (int k = 0; k < kGradRows; k += 16) {
          uint32_t b[kWays][4];
#pragma unroll
          for (int j = 0; j < kWays; ++j) {
            ldmatrix4_t(stage + v_at[j] + k * 128, b[j]);
            mask(k, b[j][0], b[j][2], b[j][1], b[j][3]);
          }
#pragma unroll
          for (int m = 0; m < 2 * kOwn; ++m) {  // tiles of the block's first, then of its second terms
            const int row = k + tr;
            const uint32_t t_at = kTiles == 1 ? row * 64 + ((m * 2 + (lane >> 3 & 1)) ^ (row >> 1 & 3)) * 16
                                              : way * (kGradRows * 128) + row * 128 + ((m * 2 + (lane >> 3 & 1)) ^ (row & 7)) * 16;
            uint32_t a[4];
            ldmatrix4_t(stage + kGradV + t_at, a);
            mask(k, a[0], a[1], a[2], a[3]);
#pragma unroll
            for (int j = 0; j < kWays; ++j) {
              mma16816<T>(acc[m % kOwn][2 * j], a[0], a[1], a[2], a[3], b[j][0], b[j][1]);
              mma16816<T>(acc[m % kOwn][2 * j + 1], a[0], a[1], a[2], a[3], b[j][2], b[j][3]);
            }
          }
        }
      };
      if ((bits0 & bits1) == ~0u) {
        walk([](int, uint32_t&, uint32_t&, uint32_t&, uint32_t&) {});
      } else {
        walk([&](int k, uint32_t& x0, uint32_t& x1, uint32_t& y0, uint32_t& y1) {  // rows k + 2 t, + 1, and those eight further
          const uint32_t bits = (k < 32 ? bits0 : bits1) >> ((k & 31) + (lane & 3) * 2), lo = pair_mask(bits), hi = pair_mask(bits >> 8);
          x0 &= lo, x1 &= lo, y0 &= hi, y1 &= hi;
        });
      }
      mbar_arrive_warp_after_reads(bar0 + (kStages + s) * 8);
    }
    const int pitch = int(low_grad_columns(job.columns, job.planes)), plane_columns = pitch / job.planes, adapters = gridDim.z / p.rank_groups;
    const int all = job.columns * job.planes;
    const bool add = !p.direct && p.accumulate && *mark;
    float* part = job.part + ((long long)blockIdx.y * adapters + g) * p.rank * pitch + plane * plane_columns;
    T* out = static_cast<T*>(job.out) + (long long)g * p.rank * all;
#pragma unroll
    for (int m = 0; m < kOwn; ++m)
#pragma unroll
      for (int n = 0; n < 2 * kWays; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = r0 + (way * kOwn + m) * 16 + (lane >> 2) + 8 * (e >> 1), c = c0 + columns0 + n * 8 + (lane & 3) * 2 + (e & 1);
          if (r >= p.rank || c >= job.columns) continue;
          if (p.direct) {
            const long long column = (long long)plane * job.columns + c;
            out[job.transposed ? column * p.rank + r : (long long)r * all + column] = static_cast<T>(acc[m][n][e]);
          } else {
            float* to = part + (long long)r * pitch + c;
            *to = add ? *to + acc[m][n][e] : acc[m][n][e];
          }
        }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (!p.direct) *mark = 1;
    if (*abort_flag) *p.status = B200TA_ERR_DEVICE_WAIT;
  }
}

template <typename T, int kTiles>
int launch_grad(DeviceState* st, dim3 grid, void* stream, const GradParams& p, const GradMaps& maps) {
  constexpr int kIndex = (kTiles == 4 ? 2 : kTiles - 1) + (__is_same(T, __half) ? 3 : 0);
  return launch_kernel(st, KernelId(kKernelLowGrad + kIndex), low_grad_kernel<T, kTiles>, grid, (kGradWarps + 1) * 32,
                       grad_stages(kTiles) * grad_stage(kTiles) + 1024, stream, p, maps);
}

// Sums over the parts: a thread takes one value, or eight ranks of a column whose results lie together, of every kSlices-th part; the
// threads of an item are in different warps.
struct LowJoinParams {
  LowGrad job[2];
  int rank, parts, adapters;
  long long items0, items;  // of the first job, of both
  const uint8_t* marks;     // [part][adapter, group of 64 ranks][slab of 128 columns]: parts that were written
  int slabs, slabs0;
};
template <typename T, int kSlices, typename Int>  // Int: unsigned, wide enough for all items
__global__ void __launch_bounds__(256, 4)
low_join_kernel(const LowJoinParams p) {
  constexpr int kItems = 256 / kSlices;
  __shared__ float joined[kSlices > 1 ? kSlices - 1 : 1][8][kItems];
  pdl_trigger();
  pdl_wait();
  const int own = threadIdx.x % kItems, slice = threadIdx.x / kItems;
  const Int items = Int(p.items), items0 = Int(p.items0);
  for (Int first = Int(blockIdx.x) * kItems; first < items; first += Int(gridDim.x) * kItems) {
    const Int i = first + own;
    const bool second = i >= items0;
    const LowGrad& job = second ? p.job[1] : p.job[0];
    const Int at = second ? i - items0 : i;
    const uint32_t all = uint32_t(job.columns) * job.planes;
    const int plane_columns = (job.columns + 3) / 4 * 4, ranks = job.transposed ? 8 : 1;
    const long long pitch = (long long)plane_columns * job.planes, stride = (long long)p.adapters * p.rank * pitch;
    const Int row = at / all;
    const int column = int(at - row * all), plane = column >= job.columns;
    const uint32_t groups = uint32_t(p.rank + ranks - 1) / ranks;
    const long long g = row / groups;
    const int r0 = int(row - Int(g) * groups) * ranks;
    const float* part = job.part + (g * p.rank + r0) * pitch + plane * plane_columns + (column - plane * job.columns);
    const int rank_groups = (p.rank + 63) / 64, slabs_plane = (job.columns + kGradColumns - 1) / kGradColumns;
    const uint8_t* mark = p.marks + (g * rank_groups + r0 / 64) * p.slabs + (second ? p.slabs0 : 0) + plane * slabs_plane + (column - plane * job.columns) / kGradColumns;
    const long long mark_stride = (long long)p.adapters * rank_groups * p.slabs;
    float sum[8] = {};
    const int n = p.rank - r0 < ranks ? p.rank - r0 : ranks;
    if (i < items) {
      if (job.transposed) {
#pragma unroll 2
        for (int s = slice; s < p.parts; s += kSlices) {
          float x[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) x[r] = norm::element_if(r < n, part + s * stride + r * pitch);
          const bool written = __ldg(mark + s * mark_stride);
#pragma unroll
          for (int r = 0; r < 8; ++r) sum[r] += written ? x[r] : 0.f;
        }
      } else {
#pragma unroll 8
        for (int s = slice; s < p.parts; s += kSlices) {
          const float x = norm::element_if(true, part + s * stride);  // (loaded whether it was written or not: loads overlap)
          sum[0] += __ldg(mark + s * mark_stride) ? x : 0.f;
        }
      }
    }
    if constexpr (kSlices > 1) {
      if (slice > 0)
#pragma unroll
        for (int r = 0; r < 8; ++r) joined[slice - 1][r][own] = sum[r];
      __syncthreads();
      if (slice == 0)
#pragma unroll
        for (int s = 0; s < kSlices - 1; ++s)
#pragma unroll
          for (int r = 0; r < 8; ++r) sum[r] += joined[s][r][own];
      __syncthreads();
    }
    if (slice > 0 || i >= items) continue;
    if (!job.transposed) {
      static_cast<T*>(job.out)[(g * p.rank + r0) * all + column] = static_cast<T>(sum[0]);
      continue;
    }
    T* out = static_cast<T*>(job.out) + (g * all + column) * p.rank + r0;
    if (n == 8 && p.rank % 8 == 0 && (reinterpret_cast<uintptr_t>(job.out) & 15u) == 0) {
      *reinterpret_cast<uint4*>(out) = make_uint4(pack2<T>(sum[0], sum[1]), pack2<T>(sum[2], sum[3]), pack2<T>(sum[4], sum[5]), pack2<T>(sum[6], sum[7]));
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < n) out[r] = static_cast<T>(sum[r]);
    }
  }
}

}  // namespace

// Each row's own adapter read for it alone, from L2 at some 2 TB/s, rather than a pass over 32 rows' k for each adapter among them,
// whose loads and products follow one another: 0.4 us for 256 of k and 2 us besides.  (288 rows of 1336, rank 32, 8 rows a request: 30 us
// by passes, now 15.)  Blocks (`blocks_row` for each row) come in rounds of eight on each multiprocessor (1310 rows of 88, rank 20, 10
// rows a request: 16 us so, 8 by passes).
bool low_by_rows(int64_t rows, int rank, int K, const AdapterIndex& index, int blocks_row, int num_sms) {
  const double adapters = double(adapters_of_tile(index, rows, 32));
  const double each = 3 + double(rows) * rank * K * 2 / 2e6 + 2.5 * double(rows * blocks_row / (num_sms * 8)), passes = 4 + adapters * (2 + 0.4 * K / 256);
  return rows <= 8192 && each < passes;
}

int run_low(const LowProduct& m, void* stream) {
  DeviceState* st = nullptr;
  const int rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  // Tiles of 128 rows on the tensor cores, unless those of several requests are too few to fill the device, or few ranks of a few
  // thousand rows are done sooner by blocks of 32 (a layer of 4 x 768 rows, 1536 -> 384, rank 16: 18.0 us so and 20.5 by tiles; of 768
  // rows with rank 64: 18.6 and 15.5; 2048 rows of 4096, rank 64: 75 and 57).
  const int64_t tiles = (m.rows + 127) / 128;
  const bool mixed = m.index.index != nullptr && m.index.count > 1 && m.index.rows_per_index < 128;
  const bool small = m.rows <= 512 || (mixed && tiles < st->num_sms) || (m.rank <= 16 && m.rows <= 8192 && m.K * m.planes <= 2048);
  if (!small && !low_by_dots(m, st->num_sms)) return run_matmul_low(m, stream);
  if (m.f16) return m.aligned ? launch_low<__half, true>(st, m, stream) : launch_low<__half, false>(st, m, stream);
  return m.aligned ? launch_low<__nv_bfloat16, true>(st, m, stream) : launch_low<__nv_bfloat16, false>(st, m, stream);
}

int run_low_up(const LowProduct& m, const void* up, int64_t up_pitch, void* stream) {
  DeviceState* st = nullptr;
  const int rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  const LowUpParams p{m.x, m.x2, up, m.low, m.scale, m.scale_all, m.xs, m.x_plane, up_pitch, m.K, m.planes, m.rank, m.index};
  return launch_kernel(st, kKernelAdapter, m.f16 ? low_up_kernel<__half> : low_up_kernel<__nv_bfloat16>, dim3(unsigned(m.rows)), 256, 0, stream, p);
}

int run_transpose_up(const void* up, int64_t up_pitch, void* out, int64_t out_pitch, int count, int rank, int N, int planes, void* stream) {
  DeviceState* st = nullptr;
  const int rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  const TransposeParams p{static_cast<const uint16_t*>(up), static_cast<uint16_t*>(out), up_pitch, out_pitch, rank, N, planes};
  return launch_kernel(st, kKernelAdapter, transpose_up_kernel, dim3(unsigned((N + 31) / 32), unsigned((rank + 31) / 32), unsigned(count * planes)), 256,
                       0, stream, p);
}

// Parts of the rows: one wave of two blocks on each multiprocessor if all adapters have their share of the rows, and up to four (rows may
// be of few of them) as long as the parts stay below 16 MiB; blocks that have nothing to do end early.
LowGradShape low_grad_shape(int64_t rows, int K, int N, int planes, int count, int rank, int num_sms) {
  LowGradShape s{};
  const int64_t chunks = (rows + kGradRows - 1) / kGradRows, columns = int64_t(K) + int64_t(planes) * N;
  s.slabs = (K + kGradColumns - 1) / kGradColumns + planes * ((N + kGradColumns - 1) / kGradColumns);
  const int64_t blocks = s.slabs * ((rank + 63) / 64), wave = int64_t(num_sms) * 2;
  const int64_t wanted = std::max<int64_t>(wave / blocks, 1), shared = std::max<int64_t>(wave / (blocks * count), 1);
  const int64_t by_bytes = (int64_t(1) << 24) / (int64_t(count) * rank * columns * 4), most = 4 * wave / (blocks * count);
  const int64_t parts = std::max(std::min(std::max(shared, std::min(std::min(wanted, most), by_bytes)), (chunks + 3) / 4),
                                 (chunks + kGradChunks - 1) / kGradChunks);
  const int64_t per = (chunks + parts - 1) / parts;
  s.parts = int((chunks + per - 1) / per);
  s.marks = s.slabs * s.parts * count * ((rank + 63) / 64);
  return s;
}

int run_low_grads(const LowGrads& m, void* stream) {
  DeviceState* st = nullptr;
  const int rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  GradParams p{};
  GradMaps maps{};
  const int tiles = m.rank <= 16 ? 1 : m.rank <= 32 ? 2 : 4, t_row = tiles == 1 ? 32 : 64;
  for (int i = 0; i < 2; ++i) {
    const LowGrad& j = m.job[i];
    if (j.v == nullptr) continue;
    const uint64_t dims[3] = {uint64_t(j.columns), uint64_t(m.rows), uint64_t(j.planes)};
    const uint64_t strides[2] = {uint64_t(j.v_pitch) * 2, uint64_t(j.planes > 1 ? j.v_plane : j.v_pitch) * 2};
    const uint32_t box[3] = {64, kGradRows, 1};
    int rc = encode_tensor_map(&maps.v[i], j.v, 2, 3, dims, strides, box, SWZ_128, "adapters");
    if (rc != B200TA_OK) return rc;
    if (i == 1 && j.v2 != nullptr && (rc = encode_tensor_map(&maps.v2, j.v2, 2, 3, dims, strides, box, SWZ_128, "adapters")) != B200TA_OK) return rc;
    const uint64_t t_dims[3] = {uint64_t(low_pitch(m.rank)), uint64_t(m.rows), 1};
    const uint64_t t_strides[2] = {uint64_t(low_pitch(m.rank)) * 2, uint64_t(low_pitch(m.rank)) * 2};
    const uint32_t t_box[3] = {uint32_t(t_row), kGradRows, 1};
    rc = encode_tensor_map(&maps.t[i], j.t, 2, 3, t_dims, t_strides, t_box, tiles == 1 ? SWZ_64 : SWZ_128, "adapters");
    if (rc != B200TA_OK) return rc;
  }
  auto slabs_of = [](const LowGrad& j) { return j.v == nullptr ? 0 : j.planes * ((j.columns + kGradColumns - 1) / kGradColumns); };
  p.job[0] = m.job[0], p.job[1] = m.job[1], p.index = m.index, p.rows = int(m.rows), p.rank = m.rank, p.rank_groups = (m.rank + 63) / 64;
  p.slabs0 = slabs_of(m.job[0]), p.accumulate = m.accumulate, p.direct = m.direct, p.marks = m.marks, p.status = st->status_dev;
  p.terms = m.job[1].v2 != nullptr;
  const int64_t chunks = (m.rows + kGradRows - 1) / kGradRows;
  p.chunks_part = int((chunks + m.parts - 1) / m.parts);
  B200TA_REQUIRE(p.chunks_part <= kGradChunks, "adapters: too many rows for %d parts", m.parts);
  // (all columns of a part's rows at a time: memory is read in whole rows)
  const dim3 grid{unsigned(p.slabs0 + slabs_of(m.job[1])), unsigned(m.parts), unsigned(m.index.count * p.rank_groups)};
  int (*launch)(DeviceState*, dim3, void*, const GradParams&, const GradMaps&);
  if (m.f16) launch = tiles == 1 ? launch_grad<__half, 1> : tiles == 2 ? launch_grad<__half, 2> : launch_grad<__half, 4>;
  else launch = tiles == 1 ? launch_grad<__nv_bfloat16, 1> : tiles == 2 ? launch_grad<__nv_bfloat16, 2> : launch_grad<__nv_bfloat16, 4>;
  return launch(st, grid, stream, p, maps);
}

int run_low_join(const LowGrads& m, void* stream) {
  DeviceState* st = nullptr;
  const int rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  LowJoinParams p{};
  auto items_of = [&](const LowGrad& j) {
    return j.v == nullptr ? int64_t(0) : int64_t(m.index.count) * j.columns * j.planes * (j.transposed ? (m.rank + 7) / 8 : m.rank);
  };
  p.job[0] = m.job[0], p.job[1] = m.job[1], p.rank = m.rank, p.parts = m.parts, p.adapters = m.index.count;
  p.items0 = items_of(m.job[0]), p.items = p.items0 + items_of(m.job[1]);
  auto slabs_of = [](const LowGrad& j) { return j.v == nullptr ? 0 : j.planes * ((j.columns + kGradColumns - 1) / kGradColumns); };
  p.marks = m.marks, p.slabs0 = slabs_of(m.job[0]), p.slabs = p.slabs0 + slabs_of(m.job[1]);
  // several threads to an item where there are many parts of few values
  // (170000 values of 24 parts: 24 us sliced, 19 otherwise; 46000 of 29: 8 and 10)
  const bool sliced = m.parts >= 4 && p.items < int64_t(st->num_sms) * 28 * m.parts;
  const int64_t each = sliced ? 32 : 256, blocks = std::min<int64_t>((p.items + each - 1) / each, int64_t(st->num_sms) * 16);
  void (*kernel)(LowJoinParams);
  if (p.items < (int64_t(1) << 31))
    kernel = m.f16 ? (sliced ? low_join_kernel<__half, 8, uint32_t> : low_join_kernel<__half, 1, uint32_t>)
                   : (sliced ? low_join_kernel<__nv_bfloat16, 8, uint32_t> : low_join_kernel<__nv_bfloat16, 1, uint32_t>);
  else kernel = m.f16 ? low_join_kernel<__half, 1, uint64_t> : low_join_kernel<__nv_bfloat16, 1, uint64_t>;
  return launch_kernel(st, kKernelAdapter, kernel, dim3(unsigned(blocks)), 256, 0, stream, p);
}

}  // namespace b200ta

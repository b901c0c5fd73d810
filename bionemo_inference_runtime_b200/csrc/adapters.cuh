// Low-rank adapters beside the dense layers (sm_100a): z = x W^T + b + t U_g^T with t = s_g x D_g^T, g the adapter of a row's request.
//
// t and its gradient dt = s_g dz U_g are [rows, rank], formed in 32 bits and held as two numbers of the operands' type, the second what
// the rounding to the first left out: 16 bits of a value's mantissa in bf16, 22 in fp16, for twice the products with a rank's few
// columns.  One number would turn the slopes of relu where z is near zero (2047 rows of 515 -> 1283, rank 12: gradients 0.015 of
// their size off in bf16 and 0.005 in fp16, now 0.0024 and 0.0003) and make the adapters' gradients a quarter less exact (0.0030 and
// 0.0024).  Each product that t or dt joins (z, and dx = dz W + dt D_g) takes them as further blocks along k of its own tiles
// (matmul.cuh).  Rows whose index is no adapter's have t = 0 and take part in none.
#pragma once

#include "common.cuh"

namespace b200ta {

// Which adapter each row has: index[(first_row + row) / rows_per_index], of 4 or 8 bytes; without an index all rows have adapter 0.
struct AdapterIndex {
  const void* index;
  int bytes;
  uint32_t rows_per_index, first_row;
  int count;
};
constexpr int kNoAdapter = 0x7FFFFFFF;
constexpr int kMaxRank = 256;
__host__ __device__ constexpr int padded_rank(int rank) { return (rank + 7) / 8 * 8; }

// An adapter's part of a product: low [rows][2][pad8(rank)] in 16 bits; high [count][planes of columns][rank], or [count][rank][columns] for a
// product whose right operand has its rows along k.
struct LowRank {
  AdapterIndex index;
  int rank;
  const void* low;
  const void* high;
  int64_t high_pitch;
};

// low[row][0][0 .. pad8(rank)) = scale[g] * sum over planes and k of x[row][plane][k] a[g][r][plane][k], zeros where there is no adapter and
// behind the last rank; low[row][1] is what the rounding of low[row][0] left out.
struct LowProduct {
  const void *x, *a;
  void* low;
  const float* scale;  // per adapter on the device, or NULL:
  float scale_all;
  long long xs, x_plane, as, a_plane, rows;  // adapter g begins at row g * rank of a
  int K, planes, rank;
  bool f16, aligned;  // aligned: 16-byte rows
  AdapterIndex index;
};
int run_low(const LowProduct& m, void* stream);

// up [count][columns (two planes of N)][rank] as [count][rank][planes][pitch], for dz U.
int run_transpose_up(const void* up, int64_t up_pitch, void* out, int64_t out_pitch, int count, int rank, int N, int planes, void* stream);

// part[p][g][r][column] (+)= sum over the rows of part p that have adapter g of (t[row][0][r] + t[row][1][r]) v[row][column], for one or two such sums, in
// 32 bits; then the parts joined, in their order, to [count][rank][columns] or (transposed) [count][columns][rank] in 16 bits.
struct LowGrad {
  const void *t, *v;  // v NULL: not wanted
  float* part;
  void* out;
  long long v_pitch, v_plane;
  int columns, planes;  // of v
  int transposed;
};
struct LowGrads {
  LowGrad job[2];
  AdapterIndex index;
  long long rows;
  int rank, parts, accumulate;
  bool f16;
};
int low_grad_parts(int64_t rows, int64_t columns, int count, int rank, int num_sms);
__host__ __device__ inline int64_t low_grad_columns(int columns, int planes) { return int64_t(planes) * ((columns + 3) / 4 * 4); }
int run_low_grads(const LowGrads& m, void* stream);
int run_low_join(const LowGrads& m, void* stream);

#ifdef __CUDACC__
// (Past the first-level cache: a kernel that starts beside the one before it reads what was complete before both.)
__device__ __forceinline__ int adapter_of(const AdapterIndex& x, uint32_t row) {
  if (x.index == nullptr) return 0;
  const uint32_t i = (x.first_row + row) / x.rows_per_index;
  const long long g = x.bytes == 8 ? __ldcg(static_cast<const long long*>(x.index) + i) : (long long)__ldcg(static_cast<const int*>(x.index) + i);
  return g >= 0 && g < x.count ? int(g) : kNoAdapter;
}
// The adapters of 32 * kWords rows, which a warp walks in ascending order: lane l has those of rows 32 j + l.
template <int kWords>
struct TileAdapters {
  int g[kWords];
  __device__ __forceinline__ void load(const AdapterIndex& x, long long row0, long long rows) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      const long long row = row0 + j * 32 + lane;
      g[j] = row < rows ? adapter_of(x, uint32_t(row)) : kNoAdapter;
    }
  }
  // The first adapter behind `last` (-1: the first of all), kNoAdapter where there is none.
  __device__ __forceinline__ int next(int last) const {
    int least = kNoAdapter;
#pragma unroll
    for (int j = 0; j < kWords; ++j)
      if (g[j] > last && g[j] < least) least = g[j];
    return int(__reduce_min_sync(0xffffffffu, unsigned(least)));
  }
  // Bit l: row 32 j + l has adapter a.
  __device__ __forceinline__ uint32_t rows_of(int j, int a) const { return __ballot_sync(0xffffffffu, g[j] == a); }
};
#endif

}  // namespace b200ta

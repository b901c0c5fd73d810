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
  uint32_t factor, shift;  // n / rows_per_index = n * factor >> shift for all n below 2^31
  int count;
};
inline AdapterIndex adapter_index(const void* index, int bytes, int64_t rows_per_index, int count) {
  const uint64_t d = rows_per_index < 1 ? 1 : rows_per_index > (int64_t(1) << 31) ? uint64_t(1) << 31 : uint64_t(rows_per_index);
  uint32_t s = 0;
  while ((uint64_t(1) << s) < d) ++s;
  // 2^(31 + s) / d, rounded up: what is added to it, times n, stays below 2^(31 + s)
  return {index, bytes, uint32_t(d), 0, uint32_t(((uint64_t(1) << (31 + s)) + d - 1) / d), 31 + s, count};
}
// Adapters that a tile of `tile` of `rows` rows is expected to have: of the entries of its index, one each.
inline int64_t adapters_of_tile(const AdapterIndex& x, int64_t rows, int tile) {
  const int64_t entries = x.index == nullptr ? 1 : ((rows < tile ? rows : tile) - 1) / x.rows_per_index + 1;
  return entries < x.count ? entries : x.count;
}
constexpr int kNoAdapter = 0x7FFFFFFF;
constexpr int kMaxRank = 256;
// How low-rank values lie: a row has blocks of 16 or 32 ranks, of each its first and then its second terms (64 or 128 bytes: a tensor
// copy takes as long for a row of 32 bytes as for one of 128), zeros behind the last rank.
__host__ __device__ constexpr int low_unit(int rank) { return rank <= 16 ? 16 : 32; }
__host__ __device__ constexpr int low_blocks(int rank) { return (rank + low_unit(rank) - 1) / low_unit(rank); }
__host__ __device__ constexpr int low_pitch(int rank) { return 2 * low_unit(rank) * low_blocks(rank); }
__host__ __device__ constexpr int low_place(int rank, int r) { return r / low_unit(rank) * 2 * low_unit(rank) + r % low_unit(rank); }

// An adapter's part of a product: low [rows][low_pitch] in 16 bits; high [count][planes of columns][rank], or [count][rank][columns] for a
// product whose right operand has its rows along k.
struct LowRank {
  AdapterIndex index;
  int64_t rows;
  int rank;
  const void* low;
  const void* high;
  int64_t high_pitch;
};

// low[row][r] = scale[g] * sum over planes and k of x[row][plane][k] a[g][plane][r][k], in two terms; zeros where there is no adapter.
struct LowProduct {
  const void *x, *a;
  const void* x2;  // what the rounding of x left out, laid out alike (up to kExactRows rows), or NULL
  void* low;
  const float* scale;  // of each adapter, on the device, or NULL: scale_all
  float scale_all;
  long long xs, x_plane, as, rows;
  int K, planes, rank;
  bool f16, aligned;  // aligned: 16-byte rows
  AdapterIndex index;
};
constexpr int64_t kExactRows = 512;  // (run_low() takes as many without tensor cores)
int run_low(const LowProduct& m, void* stream);
int run_matmul_low(const LowProduct& m, void* stream);  // of it: on the tensor cores (dense.cu)
// dz U with U as it lies (for m.x = dz, its N columns as m.K; 16-byte rows), where low_by_rows() says so.
bool low_by_rows(int64_t rows, int rank, int K, const AdapterIndex& index, int blocks_row, int num_sms);
int run_low_up(const LowProduct& m, const void* up, int64_t up_pitch, void* stream);

// up [count][columns (two planes of N)][rank] as [count][planes][rank][pitch], for dz U.
int run_transpose_up(const void* up, int64_t up_pitch, void* out, int64_t out_pitch, int count, int rank, int N, int planes, void* stream);

// part[p][g][r][column] (+)= sum over the rows of part p that have adapter g of t[row][r] (both terms) v[row][column], for one or two such sums, in
// 32 bits; then the parts joined, in their order, to [count][rank][columns] or (transposed) [count][columns][rank] in 16 bits.
struct LowGrad {
  const void *t, *v;  // v NULL: not wanted
  const void* v2;     // second terms of v, laid out alike, or NULL
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
  int rank, parts, accumulate, direct;  // direct: one part of all rows, whose sums are the results (no join)
  uint8_t* marks;
  bool f16;
};
struct LowGradShape {
  int parts;
  int64_t slabs, marks;  // marks: bytes
};
LowGradShape low_grad_shape(int64_t rows, int K, int N, int planes, int count, int rank, int num_sms);
__host__ __device__ inline int64_t low_grad_columns(int columns, int planes) { return int64_t(planes) * ((columns + 3) / 4 * 4); }
int run_low_grads(const LowGrads& m, void* stream);
int run_low_join(const LowGrads& m, void* stream);

#ifdef __CUDACC__
// What the rounding of v to `rounded` left out; nothing of what has no number in 16 bits, so that infinities stay infinities.
__device__ __forceinline__ float second_term(float v, float rounded) {
  const float rest = v - rounded;
  return fabsf(rest) <= 3.402823466e38f ? rest : 0.f;
}
// (Past the first-level cache: a kernel that starts beside the one before it reads what was complete before both.)
__device__ __forceinline__ long long index_entry(const AdapterIndex& x, uint32_t row) {
  const uint32_t i = uint32_t(uint64_t(x.first_row + row) * x.factor >> x.shift);
  return x.bytes == 8 ? __ldcg(static_cast<const long long*>(x.index) + i) : (long long)__ldcg(static_cast<const int*>(x.index) + i);
}
__device__ __forceinline__ int adapter_of_entry(const AdapterIndex& x, long long entry) {
  return entry >= 0 && entry < x.count ? int(entry) : kNoAdapter;
}
__device__ __forceinline__ int adapter_of(const AdapterIndex& x, uint32_t row) {
  return x.index == nullptr ? 0 : adapter_of_entry(x, index_entry(x, row));
}
// The adapters of 32 * kWords rows, which a warp takes in the order of their first rows: of rows that share an entry the one, of others
// lane l has those of rows 32 j + l.  fetch() starts the loads, arrived() waits for them.  The usual case is short (rows of the same entry as
// before: two comparisons), since the warps that call this share their issue slots with sixteen others and an instruction takes them
// some ten clocks.
template <int kWords>
struct TileAdapters {
  long long entry[kWords];
  int g[kWords];
  uint32_t left[kWords];  // rows whose adapter has not been taken
  int count;              // rows that there are
  uint32_t begin, end;    // rows of the whole tensor that entry[0] is of
  bool same, next_same;
  __device__ __forceinline__ explicit TileAdapters(const AdapterIndex& x) : begin(0), end(x.index == nullptr ? ~0u : 0u) { entry[0] = 0; }
  __device__ __forceinline__ void fetch(const AdapterIndex& x, int row0, int rows) {
    const uint32_t first = x.first_row + uint32_t(row0), last = x.first_row + uint32_t(min(row0 + 32 * kWords, rows) - 1);
    next_same = first >= begin && last < end;
    if (next_same) return;
    const uint32_t i = uint32_t(uint64_t(first) * x.factor >> x.shift);
    begin = i * x.rows_per_index, end = begin + x.rows_per_index;
    next_same = last < end;
    if (next_same) {
      entry[0] = index_entry(x, uint32_t(row0));
      return;
    }
    end = begin;
    count = rows - row0;
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      const int row = j * 32 + int(threadIdx.x & 31);
      entry[j] = row < count ? index_entry(x, uint32_t(row0 + row)) : -1;
    }
  }
  __device__ __forceinline__ void arrived(const AdapterIndex& x) {
    same = next_same;
    if (same) {
      g[0] = adapter_of_entry(x, entry[0]);
      left[0] = g[0] != kNoAdapter;
      return;
    }
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      g[j] = adapter_of_entry(x, entry[j]);
      left[j] = __ballot_sync(0xffffffffu, g[j] != kNoAdapter);
    }
  }
  // Whether rows are left whose adapter has not been taken.
  __device__ __forceinline__ bool more() const {
    uint32_t any = left[0];
    if (!same)
#pragma unroll
      for (int j = 1; j < kWords; ++j) any |= left[j];
    return any != 0;
  }
  // Takes the adapter of the first row that is left; bit l of rows[j]: row 32 j + l has it.
  __device__ __forceinline__ int take(uint32_t (&rows)[kWords]) {
    if (same) {
      left[0] = 0;
#pragma unroll
      for (int j = 0; j < kWords; ++j) rows[j] = ~0u;
      return g[0];
    }
    int value = g[0];
    uint32_t bits = left[0];
#pragma unroll
    for (int j = 1; j < kWords; ++j)
      if (bits == 0) value = g[j], bits = left[j];
    const int a = __shfl_sync(0xffffffffu, value, __ffs(bits) - 1);
#pragma unroll
    for (int j = 0; j < kWords; ++j) rows[j] = __ballot_sync(0xffffffffu, g[j] == a), left[j] &= ~rows[j];
    return a;
  }
  // Whether these are all rows that there are.
  __device__ __forceinline__ bool all(const uint32_t (&rows)[kWords]) const {
    if (same) return true;
    bool every = true;
#pragma unroll
    for (int j = 0; j < kWords; ++j) every &= rows[j] == (count >= 32 * (j + 1) ? ~0u : count > 32 * j ? (1u << (count - 32 * j)) - 1u : 0u);
    return every;
  }
};
#endif

}  // namespace b200ta

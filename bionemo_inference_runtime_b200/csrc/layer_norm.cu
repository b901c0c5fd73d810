// Layer norm, forward; see layer_norm.cuh for the mathematics and what bounds it.
#include "layer_norm.cuh"

namespace b200ta {
namespace {

// Rows of more than 4096 are held by 256 threads of 32 values (blocks whose barriers fall apart) rather than 512 of 16: 6001 rows
// of 8192 in fp16 take 43 us and 53 us.  Their parameters are read again for every row, which with the rows' way through shared
// memory would fill the L1 pipe (51 us), so the next rows wait in registers; of 16 bits two rows at a time share the parameters
// (12000 rows of 5120: 76 us one by one, 69 in twos).  Shifted rows would pay for their parameters' shifting as well, and take
// up to 512 threads of 16 values (3000 rows of 5003: 41 us with 32 values, 31 so).
__host__ __device__ constexpr int rows_of(int values, int bytes) {
  return values == 16 || (values == 32 && bytes == 2) ? 2 : 1;
}
__host__ __device__ constexpr int blocks_of(int threads, int values, int bytes, bool shifted) {
  return threads > 256 ? 1 : values <= 8 ? (shifted ? 3 : 4) : rows_of(values, bytes) == 2 ? 2 : 3;
}

template <typename T, typename W, bool kShifted, int kItems, int kLanes, int kMost>
__global__ void __launch_bounds__(kMost, blocks_of(kMost, kItems * (16 / int(sizeof(T))), sizeof(T), kShifted))
norm_kernel(const NormParams p) {
  constexpr int kVec = norm::Values<T>::kVec, kPairs = kVec / 2;
  constexpr int kRows = rows_of(kItems * kVec, sizeof(T));
  constexpr int kStages = norm::stages_of(kItems, kMost, blocks_of(kMost, kItems * kVec, sizeof(T), kShifted));
  constexpr bool kHold = kItems * kVec <= 16, kAhead = !kHold;
  extern __shared__ uint4 slots[];  // [stage][item][thread]
  __shared__ __align__(8) float scratch[64 * kRows];
  pdl_trigger();
  pdl_wait();
  const int lanes = kLanes == 32 ? p.lanes : kLanes, lane = threadIdx.x & (lanes - 1);
  const int per_block = blockDim.x / lanes;
  const float inv = 1.f / float(p.width);
  const long long row0 = (long long)blockIdx.x * per_block + threadIdx.x / lanes, step = (long long)gridDim.x * per_block;
  T* y = static_cast<T*>(p.y) + row0 * p.ys;
  const norm::Place<T, kShifted, kLanes> place(y, p.width, lane, lanes);
  constexpr int kSingles = place.kSingles, kSlots = place.kSlots;
  auto has = [&](int i) { return place.vectors > i * lanes; };
  int turn = 0;
  const T* x = static_cast<const T*>(p.x) + row0 * p.xs;
  const T* x_row = x;  // of the single elements that are fetched next
  T* y_row = y;
  x += place.column, y += place.column;
  const bool same = !kShifted || (reinterpret_cast<uintptr_t>(x) & 15u) == 0;  // x lies as y does
  const long long x_step = step * p.xs, y_step = step * p.ys;
  long long left = p.rows - row0;                                     // rows from this one on
  long long block_left = p.rows - (long long)blockIdx.x * per_block;  // the same for the block's first row
  const uint32_t slot0 = smem_u32(slots) + threadIdx.x * 16, stage_bytes = kItems * blockDim.x * 16;
  long long ahead = left;  // the same for the row that is fetched next
  int fill = 0, take = 0;
  auto fetch = [&]() {
    if (ahead > 0)
#pragma unroll
      for (int i = 0; i < kItems; ++i)
        if (has(i)) {
          const uint32_t slot = slot0 + fill * stage_bytes + i * blockDim.x * 16;
          if (same) norm::copy_ahead(slot, x + i * lanes * kVec);
          else sts128(slot, norm::load_anywhere(x + i * lanes * kVec, x - place.column, p.width));
        }
    norm::copy_commit();
    x += x_step, ahead -= step;
    if (++fill == kStages) fill = 0;
  };
  uint4 next[kRows][kAhead ? kItems : 1];
  auto load_next = [&](long long from) {  // `from`: rows from the first of them on
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const bool in = from > r * step && has(i);
        uint4& to = next[r][kAhead ? i : 0];
        to = norm::load_if(in && same, x + i * lanes * kVec);
        if (kShifted && in && !same) to = norm::load_anywhere(x + i * lanes * kVec, x - place.column, p.width);
      }
      x += x_step;
    }
  };
  float single[kRows][kSlots], next_single[kRows][kSlots], single_w[kSlots], single_b[kSlots];
  auto load_singles = [&](long long from) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int i = 0; i < kSingles; ++i) next_single[r][i] = norm::element_if(from > r * step && place.single[i] >= 0, x_row + place.single[i]);
      x_row += x_step;
    }
  };
  if constexpr (kSingles > 0) load_singles(left);
  if constexpr (kHold)
    for (int i = 0; i < kStages - kRows; ++i) fetch();
  if constexpr (kAhead) load_next(left);
  F2 w[kHold ? kItems : 1][kPairs] = {}, b[kHold ? kItems : 1][kPairs] = {};
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    if (kHold && has(i)) {
      norm::load_param<T, W, kShifted>(p, p.w, place.column + i * lanes * kVec, 1.f, w[kHold ? i : 0]);
      norm::load_param<T, W, kShifted>(p, p.b, place.column + i * lanes * kVec, 0.f, b[kHold ? i : 0]);
    }
  }
#pragma unroll
  for (int i = 0; i < kSingles; ++i) {
    single_w[i] = norm::single_param<W>(p.w, place.single[i], 1.f);
    single_b[i] = norm::single_param<W>(p.b, place.single[i], 0.f);
  }
  long long row = row0;
  for (; block_left > 0; block_left -= kRows * step, left -= kRows * step, row += kRows * step) {
    F2 v[kRows][kItems][kPairs];
    if constexpr (kHold) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) fetch();
      norm::copy_wait<kStages - kRows>();
    }
    float s[kRows], mean[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      F2 sum(0.f);
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (kAhead) raw = next[r][i];
        else if (left > r * step && has(i)) raw = lds128(slot0 + take * stage_bytes + i * blockDim.x * 16);
        const norm::Values<T> values(raw);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) v[r][i][j] = values.p[j], sum = sum + values.p[j];  // zeros behind the row
      }
      s[r] = norm::sum_of(sum);
#pragma unroll
      for (int i = 0; i < kSingles; ++i) single[r][i] = next_single[r][i], s[r] += single[r][i];
      if (++take == kStages) take = 0;
    }
    if constexpr (kAhead) load_next(left - kRows * step);
    if constexpr (kSingles > 0) load_singles(left - kRows * step);
    norm::row_sums<kLanes>(s, lanes, scratch, turn);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      mean[r] = s[r] * inv;
      F2 sq(0.f);
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        if (has(i)) {
#pragma unroll
          for (int j = 0; j < kPairs; ++j) v[r][i][j] = v[r][i][j] + F2(-mean[r]), sq = fma2(v[r][i][j], v[r][i][j], sq);
        }
      }
      s[r] = norm::sum_of(sq);
#pragma unroll
      for (int i = 0; i < kSingles; ++i) {
        single[r][i] = place.single[i] >= 0 ? single[r][i] - mean[r] : 0.f;
        s[r] = fmaf(single[r][i], single[r][i], s[r]);
      }
    }
    norm::row_sums<kLanes>(s, lanes, scratch, turn);
    float rstd[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      rstd[r] = rsqrtf(s[r] * inv + p.eps);
      if (p.stats != nullptr && lane == 0 && left > r * step) p.stats[row + r * step] = make_float2(rstd[r], -mean[r] * rstd[r]);
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (!kHold && has(i)) {
        norm::load_param<T, W, kShifted>(p, p.w, place.column + i * lanes * kVec, 1.f, w[0]);
        norm::load_param<T, W, kShifted>(p, p.b, place.column + i * lanes * kVec, 0.f, b[0]);
      }
      const int k = kHold ? i : 0;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) v[r][i][j] = fma2(v[r][i][j] * F2(rstd[r]), w[k][j], b[k][j]);
        if (has(i) && left > r * step) *reinterpret_cast<uint4*>(y + r * y_step + i * lanes * kVec) = norm::bits_of<T>(v[r][i]);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int i = 0; i < kSingles; ++i)
        if (place.single[i] >= 0 && left > r * step)
          y_row[place.single[i]] = static_cast<T>(fmaf(single[r][i] * rstd[r], single_w[i], single_b[i]));
      y_row += y_step;
    }
    y += kRows * y_step;
  }
}

template <typename T, typename W>
auto pick(const NormShape& s) {
  return s.shifted ? B200TA_NORM_PICK(norm_kernel, T, W, true, s) : B200TA_NORM_PICK(norm_kernel, T, W, false, s);
}

}  // namespace
}  // namespace b200ta

extern "C" {

int b200ta_layer_norm(const void* x, int64_t xs, const void* weight, const void* bias, int param_dtype, void* y, int64_t ys,
                      void* stats, int dtype, int64_t rows, int width, float eps, void* stream) {
  using namespace b200ta;
  B200TA_REQUIRE(x && y, "layer_norm: NULL pointer");
  B200TA_REQUIRE(dtype >= 0 && dtype <= B200TA_DTYPE_F16, "layer_norm: unknown dtype %d", dtype);
  B200TA_REQUIRE((!weight && !bias) || param_dtype == dtype || param_dtype == B200TA_DTYPE_F32,
                 "layer_norm: parameters are in the dtype of x or in float32");
  B200TA_REQUIRE(rows > 0 && width > 0 && width <= kNormMaxWidth, "layer_norm: rows=%lld, width=%d (1 to %d)", (long long)rows, width,
                 kNormMaxWidth);
  DeviceState* st = nullptr;
  const int rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  NormParams p{};
  p.x = x, p.w = weight, p.b = bias, p.y = y, p.stats = static_cast<float2*>(stats);
  p.xs = xs, p.ys = ys, p.rows = rows, p.width = width, p.eps = eps;
  const int bytes = norm_element_bytes(dtype), vec = 16 / bytes;
  const bool whole = width % vec == 0 && norm_aligned(x, xs, bytes) && norm_aligned(y, ys, bytes) &&
                     norm_aligned(weight, 0, 4) && norm_aligned(bias, 0, 4);
  const NormShape s = norm_shape(width, vec, whole ? 256 : 512, !whole);
  p.lanes = s.lanes;
  const int resident = blocks_of(s.threads, s.items * vec, bytes, s.shifted);  // blocks that run at once on a multiprocessor
  const int blocks = norm_blocks(rows, int64_t(st->num_sms) * resident, s.threads / s.lanes, vec, s.shifted);
  const int smem = s.items * vec <= 16 ? norm::stages_of(s.items, s.threads, resident) * s.items * s.threads * 16 : 0;
  const bool f32 = param_dtype == B200TA_DTYPE_F32;
  int (*launch)(DeviceState*, int, int, int, void*, const NormParams&);
  if (dtype == B200TA_DTYPE_BF16) launch = f32 ? pick<__nv_bfloat16, float>(s) : pick<__nv_bfloat16, __nv_bfloat16>(s);
  else if (dtype == B200TA_DTYPE_F16) launch = f32 ? pick<__half, float>(s) : pick<__half, __half>(s);
  else launch = pick<float, float>(s);
  return launch(st, blocks, s.threads, smem, stream, p);
}

}  // extern "C"

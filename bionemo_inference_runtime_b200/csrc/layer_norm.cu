// Layer norm, forward; see layer_norm.cuh for the mathematics and what bounds it.
#include "layer_norm.cuh"

namespace b200ta {
namespace {

// Rows of more than 4096 are held by 256 threads of 32 values (three blocks, whose barriers fall apart) rather than 512 of 16:
// 6001 rows of 8192 in fp16 take 43 us and 53 us.  Their parameters are read again for every row, which with the rows' way
// through shared memory would fill the L1 pipe (51 us), so the next row waits in registers.
__host__ __device__ constexpr int rows_of(int values, int bytes, bool shifted) {
  return !shifted && (values == 16 || (values == 32 && bytes == 2)) ? 2 : 1;
}
__host__ __device__ constexpr int blocks_of(int threads, int values, int bytes, bool shifted) {
  return threads > 256 ? 1 : values <= 8 ? 4 : rows_of(values, bytes, shifted) == 2 ? 2 : 3;
}

template <typename T, typename W, bool kShifted, int kItems, int kLanes, int kMost>
__global__ void __launch_bounds__(kMost, blocks_of(kMost, kItems * (16 / int(sizeof(T))), sizeof(T), kShifted))
norm_kernel(const NormParams p) {
  constexpr int kVec = norm::Values<T>::kVec, kPairs = kVec / 2;
  constexpr int kRows = rows_of(kItems * kVec, sizeof(T), kShifted);
  constexpr int kStages = norm::stages_of(kItems, kMost, blocks_of(kMost, kItems * kVec, sizeof(T), kShifted));
  constexpr bool kHold = kItems * kVec <= 16, kCopies = !kShifted && kHold, kAhead = !kShifted && !kHold;
  extern __shared__ uint4 slots[];  // [stage][item][thread] (not for shifted rows)
  __shared__ __align__(8) float scratch[64 * kRows];
  pdl_trigger();
  pdl_wait();
  const int lanes = kLanes == 32 ? p.lanes : kLanes, lane = threadIdx.x & (lanes - 1);
  const int per_block = blockDim.x / lanes;
  const float inv = 1.f / float(p.width);
  int turn = 0, valid[kItems];  // elements of an item's vector that are in the row
#pragma unroll
  for (int i = 0; i < kItems; ++i) valid[i] = p.width - (i * lanes + lane) * kVec;
  const long long row0 = (long long)blockIdx.x * per_block + threadIdx.x / lanes, step = (long long)gridDim.x * per_block;
  const T* x = static_cast<const T*>(p.x) + row0 * p.xs + lane * kVec;
  T* y = static_cast<T*>(p.y) + row0 * p.ys + lane * kVec;
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
        if (valid[i] > 0) norm::copy_ahead(slot0 + fill * stage_bytes + i * blockDim.x * 16, x + i * lanes * kVec);
    norm::copy_commit();
    x += x_step, ahead -= step;
    if (++fill == kStages) fill = 0;
  };
  uint4 next[kRows][kAhead ? kItems : 1];
  auto load_next = [&](long long from) {  // `from`: rows from the first of them on
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) next[r][kAhead ? i : 0] = norm::load_if(from > r * step && valid[i] > 0, x + i * lanes * kVec);
      x += x_step;
    }
  };
  if constexpr (kCopies)
    for (int i = 0; i < kStages - kRows; ++i) fetch();
  if constexpr (kAhead) load_next(left);
  F2 w[kHold ? kItems : 1][kPairs] = {}, b[kHold ? kItems : 1][kPairs] = {};
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    if (kHold && valid[i] > 0) {
      norm::load_param<T, W, kShifted>(p, p.w, (i * lanes + lane) * kVec, valid[i], 1.f, w[kHold ? i : 0]);
      norm::load_param<T, W, kShifted>(p, p.b, (i * lanes + lane) * kVec, valid[i], 0.f, b[kHold ? i : 0]);
    }
  }
  long long row = row0;
  for (; block_left > 0; block_left -= kRows * step, left -= kRows * step, row += kRows * step) {
    F2 v[kRows][kItems][kPairs];
    if constexpr (kCopies) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) fetch();
      norm::copy_wait<kStages - kRows>();
    }
    float s[kRows], mean[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      F2 sum(0.f);
      norm::Pending pending[kShifted ? kItems : 1];
      if constexpr (kShifted) {
#pragma unroll
        for (int i = 0; i < kItems; ++i) pending[i] = norm::load<T, true>(x + i * lanes * kVec, left > 0 ? valid[i] : 0);
      }
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (kAhead) raw = next[r][i];
        else if constexpr (kShifted) raw = norm::arrived<T, true>(pending[i], x + i * lanes * kVec, left > 0 ? valid[i] : 0);
        else if (left > r * step && valid[i] > 0) raw = lds128(slot0 + take * stage_bytes + i * blockDim.x * 16);
        const norm::Values<T> values(raw);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) v[r][i][j] = values.p[j], sum = sum + values.p[j];  // zeros behind the row
      }
      s[r] = norm::sum_of(sum);
      if (++take == kStages) take = 0;
    }
    if (kShifted) x += x_step;
    if constexpr (kAhead) load_next(left - kRows * step);
    norm::row_sums<kLanes>(s, lanes, scratch, turn);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      mean[r] = s[r] * inv;
      F2 sq(0.f);
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        if (kShifted && valid[i] < kVec) {
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            float a, c;
            v[r][i][j].to(a, c);
            v[r][i][j] = F2(2 * j < valid[i] ? a - mean[r] : 0.f, 2 * j + 1 < valid[i] ? c - mean[r] : 0.f);
            sq = fma2(v[r][i][j], v[r][i][j], sq);
          }
        } else if (valid[i] > 0) {
#pragma unroll
          for (int j = 0; j < kPairs; ++j) v[r][i][j] = v[r][i][j] + F2(-mean[r]), sq = fma2(v[r][i][j], v[r][i][j], sq);
        }
      }
      s[r] = norm::sum_of(sq);
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
      if (!kHold && valid[i] > 0) {
        norm::load_param<T, W, kShifted>(p, p.w, (i * lanes + lane) * kVec, valid[i], 1.f, w[0]);
        norm::load_param<T, W, kShifted>(p, p.b, (i * lanes + lane) * kVec, valid[i], 0.f, b[0]);
      }
      const int k = kHold ? i : 0;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) v[r][i][j] = fma2(v[r][i][j] * F2(rstd[r]), w[k][j], b[k][j]);
        norm::store<T, kShifted>(y + r * y_step + i * lanes * kVec, norm::bits_of<T>(v[r][i]), left > r * step ? valid[i] : 0,
                                 lane & (kLanes - 1), kLanes);
      }
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
  p.params_aligned = norm_aligned(weight, 0, 4) && norm_aligned(bias, 0, 4);
  const int bytes = norm_element_bytes(dtype), vec = 16 / bytes;
  const bool whole = width % vec == 0 && norm_aligned(x, xs, bytes) && norm_aligned(y, ys, bytes) && p.params_aligned;
  const NormShape s = norm_shape(width, vec, 256, !whole);
  p.lanes = s.lanes;
  const int64_t per_block = s.threads / s.lanes, need = (rows + per_block - 1) / per_block;
  const int resident = blocks_of(s.threads, s.items * vec, bytes, s.shifted);  // blocks that run at once on a multiprocessor
  const int64_t most = int64_t(st->num_sms) * resident;
  const int smem = whole && s.items * vec <= 16 ? norm::stages_of(s.items, s.threads, resident) * s.items * s.threads * 16 : 0;
  const bool f32 = param_dtype == B200TA_DTYPE_F32;
  int (*launch)(DeviceState*, int, int, int, void*, const NormParams&);
  if (dtype == B200TA_DTYPE_BF16) launch = f32 ? pick<__nv_bfloat16, float>(s) : pick<__nv_bfloat16, __nv_bfloat16>(s);
  else if (dtype == B200TA_DTYPE_F16) launch = f32 ? pick<__half, float>(s) : pick<__half, __half>(s);
  else launch = pick<float, float>(s);
  return launch(st, int(need < most ? need : most), s.threads, smem, stream, p);
}

}  // extern "C"

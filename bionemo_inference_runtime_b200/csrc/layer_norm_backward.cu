// Gradients of the layer norm; see layer_norm.cuh for the mathematics and what bounds it.
//
// A thread keeps its columns, so dw and db add up in its registers over all of its rows, are joined over the block in shared
// memory, and one row of partial sums per block goes to the workspace, which a second kernel adds up.  The order is fixed:
// results repeat bit by bit.  Rows are walked from the last to the first: what came before (the forward pass, or the kernel that
// made dy) ended with the last ones, which L2 still holds (262144 rows of 128 in bf16, forward and backward: 72 us, so 68).
#include "layer_norm.cuh"

namespace b200ta {
namespace {

constexpr int64_t kOneBlock = 16384;  // elements of x

// Blocks of a multiprocessor: 8 values a thread leave room for three of 256 threads, more (or single elements beside
// them) for two.
__host__ __device__ constexpr int grad_blocks_of(int threads, int values, bool shifted) {
  return threads > 256 ? 1 : values <= 8 && !shifted ? 3 : 2;
}

template <typename T, typename W, bool kShifted, int kItems, int kLanes, int kMost>
__global__ void __launch_bounds__(kMost, grad_blocks_of(kMost, kItems * norm::Values<T>::kVec, kShifted))
norm_grad_kernel(const NormParams p) {
  constexpr int kVec = norm::Values<T>::kVec, kPairs = kVec / 2;
  constexpr int kRows = norm::rows_at_a_time(kItems * kVec);
  constexpr int kStages = norm::stages_of(2 * kItems, kMost, grad_blocks_of(kMost, kItems * kVec, kShifted));
  constexpr bool kHold = kItems * kVec <= 16;
  constexpr bool kKeep = kRows == 1 && kHold;  // xh and g stay in registers between the two passes over a row
  extern __shared__ uint4 slots[];    // [stage][x items, dy items][thread]; joined sums at the end
  float* joined = reinterpret_cast<float*>(slots);  // [groups / 2][2][width]
  __shared__ __align__(8) float scratch[128 * kRows];
  pdl_trigger();
  pdl_wait();
  const int lanes = kLanes == 32 ? p.lanes : kLanes, lane = threadIdx.x & (lanes - 1);
  const int per_block = blockDim.x / lanes, group = threadIdx.x / lanes;
  const float inv = 1.f / float(p.width);
  const long long row0 = (long long)blockIdx.x * per_block + group, step = (long long)gridDim.x * per_block;
  const long long first = p.rows - 1 - row0;  // row0, left and so on count from the last row
  const T* x = static_cast<const T*>(p.x) + first * p.xs;
  const T* dy = static_cast<const T*>(p.dy) + first * p.dys;
  T* dx = static_cast<T*>(p.dx) + first * p.dxs;
  const norm::Place<T, kShifted, kLanes> place(p.dx != nullptr ? dx : x, p.width, lane, lanes);
  constexpr int kSingles = place.kSingles, kSlots = place.kSlots;
  auto has = [&](int i) { return place.vectors > i * lanes; };
  int turn = 0;
  const T *x_row = x, *dy_row = dy;  // of the single elements that are fetched next
  T* dx_row = dx;
  x += place.column, dy += place.column, dx += place.column;
  const bool same_x = !kShifted || (reinterpret_cast<uintptr_t>(x) & 15u) == 0;  // lies as dx does
  const bool same_dy = !kShifted || (reinterpret_cast<uintptr_t>(dy) & 15u) == 0;
  const float2* stats = p.stats + first;
  long long left = p.rows - row0, block_left = p.rows - (long long)blockIdx.x * per_block;
  const uint32_t slot0 = smem_u32(slots) + threadIdx.x * 16, item_bytes = blockDim.x * 16, stage_bytes = 2 * kItems * item_bytes;
  long long ahead = left;
  int fill = 0, take = 0;
  auto fetch = [&]() {
    if (ahead > 0)
#pragma unroll
      for (int i = 0; i < kItems; ++i)
        if (has(i)) {
          const int c = i * lanes * kVec;
          const uint32_t to_x = slot0 + fill * stage_bytes + i * item_bytes, to_dy = to_x + kItems * item_bytes;
          if (same_x) norm::copy_ahead(to_x, x + c);
          else sts128(to_x, norm::load_anywhere(x + c, x - place.column, p.width));
          if (same_dy) norm::copy_ahead(to_dy, dy + c);
          else sts128(to_dy, norm::load_anywhere(dy + c, dy - place.column, p.width));
        }
    norm::copy_commit();
    x -= step * p.xs, dy -= step * p.dys, ahead -= step;
    if (++fill == kStages) fill = 0;
  };
  for (int i = 0; i < kStages - kRows; ++i) fetch();
  float2 next_single[kRows][kSlots];  // {x, dy}
  float single_w[kSlots], single_dw[kSlots] = {}, single_db[kSlots] = {};
  auto load_singles = [&](long long from) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int i = 0; i < kSingles; ++i) {
        const bool in = from > r * step && place.single[i] >= 0;
        next_single[r][i] = make_float2(norm::element_if(in, x_row + place.single[i]), norm::element_if(in, dy_row + place.single[i]));
      }
      x_row -= step * p.xs, dy_row -= step * p.dys;
    }
  };
  if constexpr (kSingles > 0) load_singles(left);
#pragma unroll
  for (int i = 0; i < kSingles; ++i) single_w[i] = norm::single_param<W>(p.w, place.single[i], 1.f);
  F2 dw[kItems][kPairs] = {}, db[kItems][kPairs] = {}, w[kHold ? kItems : 1][kPairs] = {};
#pragma unroll
  for (int i = 0; i < kItems; ++i)
    if (kHold && has(i)) norm::load_param<T, W, kShifted>(p, p.w, place.column + i * lanes * kVec, 1.f, w[kHold ? i : 0]);
  float2 next[kRows];
  auto fetch_stats = [&](long long rows_left) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) next[r] = rows_left > r * step ? __ldg(stats - r * step) : make_float2(0.f, 0.f);
    stats -= kRows * step;
  };
  fetch_stats(left);
  for (; block_left > 0; block_left -= kRows * step, left -= kRows * step) {
    F2 xh[kKeep ? kItems : 1][kPairs], g[kKeep ? kItems : 1][kPairs];
    float2 st[kRows];
    float s[2 * kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) st[r] = next[r];
    fetch_stats(left - kRows * step);
#pragma unroll
    for (int r = 0; r < kRows; ++r) fetch();
    norm::copy_wait<kStages - kRows>();
    // xh and g = dy w of item i of a row; with kSum also dw and db
    auto load = [&](int i, int r, int stage, auto sum) {
      uint4 raw_x = make_uint4(0u, 0u, 0u, 0u), raw_dy = raw_x;
      if (left > r * step && has(i)) {
        raw_x = lds128(slot0 + stage * stage_bytes + i * item_bytes);
        raw_dy = lds128(slot0 + stage * stage_bytes + (kItems + i) * item_bytes);
      }
      const norm::Values<T> vx(raw_x), vd(raw_dy);
      const int k = kKeep ? i : 0, kw = kHold ? i : 0;
      if (!kHold && has(i)) norm::load_param<T, W, kShifted>(p, p.w, place.column + i * lanes * kVec, 1.f, w[0]);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        // (behind the row dy is zero, and what xh is there does not count)
        xh[k][j] = fma2(vx.p[j], F2(st[r].x), F2(st[r].y));
        if constexpr (decltype(sum)::value) {
          dw[i][j] = fma2(vd.p[j], xh[k][j], dw[i][j]);
          db[i][j] = db[i][j] + vd.p[j];
        }
        g[k][j] = vd.p[j] * w[kw][j];
      }
    };
    float2 single[kRows][kSlots];  // {xh, g}
    int stage = take;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      F2 s0(0.f), s1(0.f);
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        load(i, r, stage, std::true_type());
#pragma unroll
        for (int j = 0; j < kPairs; ++j) s0 = s0 + g[kKeep ? i : 0][j], s1 = fma2(g[kKeep ? i : 0][j], xh[kKeep ? i : 0][j], s1);
      }
      s[2 * r] = norm::sum_of(s0), s[2 * r + 1] = norm::sum_of(s1);
#pragma unroll
      for (int i = 0; i < kSingles; ++i) {
        const float2 v = next_single[r][i];
        const float xh_i = fmaf(v.x, st[r].x, st[r].y), g_i = v.y * single_w[i];
        single_dw[i] = fmaf(v.y, xh_i, single_dw[i]), single_db[i] += v.y;
        s[2 * r] += g_i, s[2 * r + 1] = fmaf(g_i, xh_i, s[2 * r + 1]);
        single[r][i] = make_float2(xh_i, g_i);
      }
      if (++stage == kStages) stage = 0;
    }
    if constexpr (kSingles > 0) load_singles(left - kRows * step);
    if (p.dx != nullptr) {
      norm::row_sums<kLanes>(s, lanes, scratch, turn);
      stage = take;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const F2 a(st[r].x), b(-s[2 * r] * inv * st[r].x), c(-s[2 * r + 1] * inv * st[r].x);
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
          if constexpr (!kKeep) load(i, r, stage, std::false_type());
          F2 out[kPairs];
#pragma unroll
          for (int j = 0; j < kPairs; ++j) out[j] = fma2(xh[kKeep ? i : 0][j], c, fma2(g[kKeep ? i : 0][j], a, b));
          if (has(i) && left > r * step) *reinterpret_cast<uint4*>(dx + i * lanes * kVec) = norm::bits_of<T>(out);
        }
#pragma unroll
        for (int i = 0; i < kSingles; ++i) {
          const float out = -(single[r][i].x * s[2 * r + 1] + s[2 * r]) * inv * st[r].x + single[r][i].y * st[r].x;
          if (place.single[i] >= 0 && left > r * step) dx_row[place.single[i]] = static_cast<T>(out);
        }
        dx_row -= step * p.dxs;
        dx -= step * p.dxs;
        if (++stage == kStages) stage = 0;
      }
    }
    take = stage;
  }
  if (p.partial == nullptr && p.dw == nullptr && p.db == nullptr) return;
  norm::copy_wait<0>();
  __syncthreads();  // the slots are free
  // the groups' sums, joined in pairs: half of the groups that are left hand theirs to the other half
  auto each = [&](float* to, bool add) {
#pragma unroll
    for (int i = 0; i < kItems; ++i)
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const int c = place.column + i * lanes * kVec + 2 * j;
        float w0, w1, b0, b1;
        dw[i][j].to(w0, w1), db[i][j].to(b0, b1);
        if (!has(i)) continue;
        if (add) dw[i][j] = F2(w0 + to[c], w1 + to[c + 1]), db[i][j] = F2(b0 + to[p.width + c], b1 + to[p.width + c + 1]);
        else to[c] = w0, to[c + 1] = w1, to[p.width + c] = b0, to[p.width + c + 1] = b1;
      }
#pragma unroll
    for (int i = 0; i < kSingles; ++i) {
      const int c = place.single[i];
      if (c < 0) continue;
      if (add) single_dw[i] += to[c], single_db[i] += to[p.width + c];
      else to[c] = single_dw[i], to[p.width + c] = single_db[i];
    }
  };
  for (int left_groups = per_block; left_groups > 1; left_groups >>= 1) {
    const int half = left_groups >> 1;
    if (group >= half && group < left_groups) each(joined + (group - half) * 2 * p.width, false);
    __syncthreads();
    if (group < half) each(joined + group * 2 * p.width, true);
    __syncthreads();
  }
  if (group != 0) return;
  if (p.partial != nullptr) return each(p.partial + (long long)blockIdx.x * 2 * p.width, false);
  W *out_w = static_cast<W*>(p.dw), *out_b = static_cast<W*>(p.db);
  auto put = [&](int c, float w_c, float b_c) {
    if (out_w != nullptr) out_w[c] = static_cast<W>(w_c);
    if (out_b != nullptr) out_b[c] = static_cast<W>(b_c);
  };
#pragma unroll
  for (int i = 0; i < kItems; ++i)
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const int c = place.column + i * lanes * kVec + 2 * j;
      float w0, w1, b0, b1;
      dw[i][j].to(w0, w1), db[i][j].to(b0, b1);
      if (has(i)) put(c, w0, b0), put(c + 1, w1, b1);
    }
#pragma unroll
  for (int i = 0; i < kSingles; ++i)
    if (place.single[i] >= 0) put(place.single[i], single_dw[i], single_db[i]);
}

// dw and db: column sums of the blocks' partial sums.  A block takes kColumns of the 2 * width columns, 1024 / kColumns threads a
// column: 8 columns while that gives no more blocks than run at once, then 32 or 128 (backward of 2000 rows of 16384 in bf16:
// 124 us by eights alone, 103 so; of 8192 rows of 4096: 62 and 56).
template <typename T, int kColumns>
__global__ void __launch_bounds__(1024)
norm_join_kernel(const float* partial, int blocks, int width, T* dw, T* db) {
  constexpr int kThreads = 1024 / kColumns, kRows = kColumns < 32 ? 32 : kThreads;  // rows of `part`
  __shared__ float part[kRows][kColumns];
  pdl_trigger();
  pdl_wait();
  const int k = threadIdx.x / kColumns, c = blockIdx.x * kColumns + threadIdx.x % kColumns;
  float sum = 0.f;
  if (c < 2 * width)
#pragma unroll 4
    for (int b = k; b < blocks; b += kThreads) sum += __ldg(partial + (long long)b * 2 * width + c);
  if constexpr (kColumns < 32) {
#pragma unroll
    for (int o = kColumns; o < 32; o *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) < kColumns) part[threadIdx.x >> 5][threadIdx.x & 31] = sum;
  } else {
    part[k][threadIdx.x % kColumns] = sum;
  }
  __syncthreads();
  if (threadIdx.x < kColumns && c < 2 * width) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) sum += part[i][threadIdx.x];
    T* dst = c < width ? dw : db;
    if (dst != nullptr) dst[c < width ? c : c - width] = static_cast<T>(sum);
  }
}

template <typename T, typename W>
auto pick(const NormShape& s) {
  return s.shifted ? B200TA_NORM_PICK(norm_grad_kernel, T, W, true, s) : B200TA_NORM_PICK(norm_grad_kernel, T, W, false, s);
}

}  // namespace
}  // namespace b200ta

extern "C" {

size_t b200ta_layer_norm_workspace_bytes(int64_t rows, int width) {
  // a row of partial sums for each block; at most three blocks run on a multiprocessor
  using namespace b200ta;
  DeviceState* st = nullptr;
  if (rows <= 0 || width <= 0 || get_device_state(&st) != B200TA_OK) return 0;
  const int64_t most = int64_t(st->num_sms) * 3;
  return size_t(rows < most ? rows : most) * 2 * size_t(width) * sizeof(float);
}

int b200ta_layer_norm_backward(const void* dy, int64_t dys, const void* x, int64_t xs, const void* stats, const void* weight,
                               int param_dtype, void* dx, int64_t dxs, void* dweight, void* dbias, void* workspace,
                               size_t workspace_bytes, int dtype, int64_t rows, int width, void* stream) {
  using namespace b200ta;
  B200TA_REQUIRE(dy && x && stats, "layer_norm_backward: NULL pointer");
  B200TA_REQUIRE(dtype >= 0 && dtype <= B200TA_DTYPE_F16, "layer_norm_backward: unknown dtype %d", dtype);
  B200TA_REQUIRE(param_dtype == dtype || param_dtype == B200TA_DTYPE_F32,
                 "layer_norm_backward: parameters are in the dtype of x or in float32");
  B200TA_REQUIRE(rows > 0 && width > 0 && width <= kNormMaxWidth, "layer_norm_backward: rows=%lld, width=%d (1 to %d)",
                 (long long)rows, width, kNormMaxWidth);
  const bool sums = dweight != nullptr || dbias != nullptr;
  B200TA_REQUIRE(!sums || (workspace != nullptr && workspace_bytes >= b200ta_layer_norm_workspace_bytes(rows, width)),
                 "layer_norm_backward: the workspace is too small");
  if (!sums && dx == nullptr) return B200TA_OK;
  DeviceState* st = nullptr;
  int rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  NormParams p{};
  p.x = x, p.dy = dy, p.w = weight, p.dx = dx, p.stats = static_cast<float2*>(const_cast<void*>(stats));
  p.partial = sums ? static_cast<float*>(workspace) : nullptr;
  p.xs = xs, p.dys = dys, p.dxs = dxs, p.rows = rows, p.width = width;
  const int bytes = norm_element_bytes(dtype), vec = 16 / bytes;
  const bool whole = width % vec == 0 && norm_aligned(x, xs, bytes) && norm_aligned(dy, dys, bytes) &&
                     (!dx || norm_aligned(dx, dxs, bytes)) && norm_aligned(weight, 0, 4);
  const NormShape s = norm_shape(width, vec, 512, !whole);
  p.lanes = s.lanes;
  const int groups = s.threads / s.lanes, resident = grad_blocks_of(s.threads, s.items * vec, s.shifted);
  const int joined = sums && groups > 1 ? groups / 2 * 2 * width * int(sizeof(float)) : 0;
  const int ring = norm::stages_of(2 * s.items, s.threads, resident) * 2 * s.items * s.threads * 16;
  const int smem = joined > ring ? joined : ring;
  // Little work is for one block, whose sums are dw and db (4 rows of 317 in fp32: 8.9 us in two launches, 6.4 in one;
  // with twice the limit, 85 rows of 384 in bf16, 9.0 and 10.3), unless its step would not be a whole period of the rows' alignment.
  const bool one = sums && rows * width <= kOneBlock && (!s.shifted || groups % vec == 0 || rows <= groups);
  if (one) p.partial = nullptr, p.dw = dweight, p.db = dbias;
  const int blocks = one ? 1 : norm_blocks(rows, int64_t(st->num_sms) * resident, groups, vec, s.shifted);
  const bool f32 = param_dtype == B200TA_DTYPE_F32;
  int (*launch)(DeviceState*, int, int, int, void*, const NormParams&);
  if (dtype == B200TA_DTYPE_BF16) launch = f32 ? pick<__nv_bfloat16, float>(s) : pick<__nv_bfloat16, __nv_bfloat16>(s);
  else if (dtype == B200TA_DTYPE_F16) launch = f32 ? pick<__half, float>(s) : pick<__half, __half>(s);
  else launch = pick<float, float>(s);
  rc = launch(st, blocks, s.threads, smem, stream, p);
  if (rc != B200TA_OK || !sums || one) return rc;
  auto join = [&](auto* dw, auto* db) {
    using P = std::remove_pointer_t<decltype(dw)>;
    auto launch_join = [&](auto* kernel, int columns) {
      return launch_kernel(st, kKernelNorm, kernel, dim3(unsigned((2 * width + columns - 1) / columns)), 1024, 0, stream,
                           static_cast<const float*>(p.partial), blocks, width, dw, db);
    };
    if (2 * width <= st->num_sms * 2 * 8) return launch_join(&norm_join_kernel<P, 8>, 8);
    return 2 * width <= st->num_sms * 2 * 32 ? launch_join(&norm_join_kernel<P, 32>, 32) : launch_join(&norm_join_kernel<P, 128>, 128);
  };
  if (f32) return join(static_cast<float*>(dweight), static_cast<float*>(dbias));
  if (param_dtype == B200TA_DTYPE_F16) return join(static_cast<__half*>(dweight), static_cast<__half*>(dbias));
  return join(static_cast<__nv_bfloat16*>(dweight), static_cast<__nv_bfloat16*>(dbias));
}

}  // extern "C"

// Layer norm over the last axis and its gradients (sm_100a), for bf16, fp16 or fp32 rows:
//
//   y  = (x - mean) rstd w + b                          rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd (g - mean(g) - xh mean(g xh))             g = dy w, xh = (x - mean) rstd
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Bound: HBM.  Forward reads x and writes y, backward reads x and dy and writes dx, each once: a row is held in the
// registers of the 1 to 1024 threads that share it (at most 16 values each, in 32 bits), and its mean and variance, or its
// two sums, are taken there, the variance from centred values.  Blocks are persistent; a thread keeps its columns, so dw
// and db add up in its registers over all of its rows, are joined over the block in shared memory, and one row of partial
// sums per block goes to the workspace, which a second kernel adds up.  The order is fixed: results repeat bit by bit.
#include "activation.cuh"
#include "common.cuh"

namespace b200ta {
namespace {

constexpr int kThreads = 256;  // of a block, unless a row takes more
constexpr int kMaxWidth = 16384;

struct NormParams {
  const void *x, *dy, *w, *b;
  void *y, *dx;
  float2* stats;      // {rstd, -mean * rstd} per row: written by the forward pass (if not NULL), read by the backward pass
  float* partial;     // [blocks][2][width]
  long long xs, ys, dys, dxs, rows;
  int width, param_f32, lanes;  // lanes: threads that share a row, a power of two
  float eps;
};

template <typename T>
__device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }

// kVec consecutive elements, 16 bytes or one element.
template <typename T, int kVec>
__device__ __forceinline__ void load(const T* p, float* v) {
  if constexpr (kVec == 1) {
    v[0] = to_float(*p);
  } else {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 4) {
        v[e] = __uint_as_float(w[e]);
      } else {
        const float2 f = unpack2<T>(w[e]);
        v[2 * e] = f.x, v[2 * e + 1] = f.y;
      }
    }
  }
}
template <typename T, int kVec>
__device__ __forceinline__ void store(T* p, const float* v) {
  if constexpr (kVec == 1) {
    *p = static_cast<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  }
}
// Parameters are in the type of the rows or in fp32; their alignment is looked at once, by the host (kVec).
template <typename T, int kVec>
__device__ __forceinline__ void load_param(const void* p, int f32, int c, float* v) {
  if (f32) {
    const float* q = static_cast<const float*>(p) + c;
    if constexpr (kVec >= 4) {
#pragma unroll
      for (int e = 0; e < kVec; e += 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(q + e));
        v[e] = x.x, v[e + 1] = x.y, v[e + 2] = x.z, v[e + 3] = x.w;
      }
    } else {
      v[0] = __ldg(q);
    }
  } else {
    load<T, kVec>(static_cast<const T*>(p) + c, v);
  }
}

// The sums of `a` (and `b`) over the threads that share a row; every one of them gets the result.  Rows of more than a warp
// go through shared memory: all threads of the block call this equally often.
template <int kSums>
__device__ __forceinline__ void row_sums(float (&s)[kSums], int lanes, float* scratch) {
  const int in_warp = lanes < 32 ? lanes : 32;
  for (int o = in_warp >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < kSums; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
  if (lanes > 32) {
    const int warp = threadIdx.x >> 5, warps = lanes >> 5, first = warp / warps * warps;
    __syncthreads();  // the sums before these have been read
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < kSums; ++i) scratch[warp * kSums + i] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSums; ++i) s[i] = 0.f;
    for (int w = first; w < first + warps; ++w)
#pragma unroll
      for (int i = 0; i < kSums; ++i) s[i] += scratch[w * kSums + i];
  }
}

template <typename T, int kVec, int kItems, int kMost>
__global__ void __launch_bounds__(kMost, 1)
norm_kernel(const NormParams p) {
  __shared__ float scratch[32];
  pdl_trigger();
  pdl_wait();
  const int per_block = blockDim.x / p.lanes, group = threadIdx.x / p.lanes, lane = threadIdx.x % p.lanes;
  const float inv = 1.f / float(p.width);
  for (long long r0 = (long long)blockIdx.x * per_block; r0 < p.rows; r0 += (long long)gridDim.x * per_block) {
    const long long row = r0 + group;
    const bool valid = row < p.rows;
    float v[kItems * kVec];
    float sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int c = (i * p.lanes + lane) * kVec;
      if (valid && c < p.width) {
        load<T, kVec>(static_cast<const T*>(p.x) + row * p.xs + c, v + i * kVec);
#pragma unroll
        for (int e = 0; e < kVec; ++e) sum[0] += v[i * kVec + e];
      }
    }
    row_sums(sum, p.lanes, scratch);
    const float mean = sum[0] * inv;
    float sq[1] = {0.f};
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (valid && (i * p.lanes + lane) * kVec < p.width) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float d = v[i * kVec + e] - mean;
          v[i * kVec + e] = d;
          sq[0] = fmaf(d, d, sq[0]);
        }
      }
    }
    row_sums(sq, p.lanes, scratch);
    const float rstd = rsqrtf(sq[0] * inv + p.eps);
    if (!valid) continue;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int c = (i * p.lanes + lane) * kVec;
      if (c < p.width) {
        float w[kVec], b[kVec];
        if (p.w != nullptr) load_param<T, kVec>(p.w, p.param_f32, c, w);
        if (p.b != nullptr) load_param<T, kVec>(p.b, p.param_f32, c, b);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float n = v[i * kVec + e] * rstd;
          v[i * kVec + e] = fmaf(n, p.w != nullptr ? w[e] : 1.f, p.b != nullptr ? b[e] : 0.f);
        }
        store<T, kVec>(static_cast<T*>(p.y) + row * p.ys + c, v + i * kVec);
      }
    }
    if (p.stats != nullptr && lane == 0) p.stats[row] = make_float2(rstd, -mean * rstd);
  }
}

template <typename T, int kVec, int kItems, int kMost>
__global__ void __launch_bounds__(kMost, 1)
norm_grad_kernel(const NormParams p) {
  extern __shared__ float joined[];  // [groups - 1][2][width], if sums over rows are wanted
  __shared__ float scratch[64];
  pdl_trigger();
  pdl_wait();
  const int per_block = blockDim.x / p.lanes, group = threadIdx.x / p.lanes, lane = threadIdx.x % p.lanes;
  const float inv = 1.f / float(p.width);
  float dw[kItems * kVec], db[kItems * kVec];
#pragma unroll
  for (int j = 0; j < kItems * kVec; ++j) dw[j] = 0.f, db[j] = 0.f;
  for (long long r0 = (long long)blockIdx.x * per_block; r0 < p.rows; r0 += (long long)gridDim.x * per_block) {
    const long long row = r0 + group;
    const bool valid = row < p.rows;
    float xh[kItems * kVec], g[kItems * kVec];
    const float2 st = valid ? __ldg(p.stats + row) : make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int c = (i * p.lanes + lane) * kVec;
      if (valid && c < p.width) {
        load<T, kVec>(static_cast<const T*>(p.x) + row * p.xs + c, xh + i * kVec);
        load<T, kVec>(static_cast<const T*>(p.dy) + row * p.dys + c, g + i * kVec);
      }
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int c = (i * p.lanes + lane) * kVec;
      if (valid && c < p.width) {
        float w[kVec];
        if (p.w != nullptr) load_param<T, kVec>(p.w, p.param_f32, c, w);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const int j = i * kVec + e;
          xh[j] = fmaf(xh[j], st.x, st.y);
          dw[j] = fmaf(g[j], xh[j], dw[j]);
          db[j] += g[j];
          if (p.w != nullptr) g[j] *= w[e];
          s[0] += g[j];
          s[1] = fmaf(g[j], xh[j], s[1]);
        }
      }
    }
    if (p.dx == nullptr) continue;
    row_sums(s, p.lanes, scratch);
    const float m0 = s[0] * inv, m1 = s[1] * inv;
    if (!valid) continue;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int c = (i * p.lanes + lane) * kVec;
      if (c < p.width) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const int j = i * kVec + e;
          g[j] = st.x * (g[j] - m0 - xh[j] * m1);
        }
        store<T, kVec>(static_cast<T*>(p.dx) + row * p.dxs + c, g + i * kVec);
      }
    }
  }
  if (p.partial == nullptr) return;
  // the groups' sums, joined in pairs: half of the groups that are left hand theirs to the other half
  for (int left = per_block; left > 1; left >>= 1) {
    const int half = left >> 1;
    if (group >= half && group < left) {
      float* dst = joined + (long long)(group - half) * 2 * p.width;
#pragma unroll
      for (int i = 0; i < kItems; ++i)
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const int c = (i * p.lanes + lane) * kVec + e;
          if (c < p.width) dst[c] = dw[i * kVec + e], dst[p.width + c] = db[i * kVec + e];
        }
    }
    __syncthreads();
    if (group < half) {
      const float* src = joined + (long long)group * 2 * p.width;
#pragma unroll
      for (int i = 0; i < kItems; ++i)
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const int c = (i * p.lanes + lane) * kVec + e;
          if (c < p.width) dw[i * kVec + e] += src[c], db[i * kVec + e] += src[p.width + c];
        }
    }
    __syncthreads();
  }
  if (group == 0) {
    float* dst = p.partial + (long long)blockIdx.x * 2 * p.width;
#pragma unroll
    for (int i = 0; i < kItems; ++i)
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const int c = (i * p.lanes + lane) * kVec + e;
        if (c < p.width) dst[c] = dw[i * kVec + e], dst[p.width + c] = db[i * kVec + e];
      }
  }
}

// dw and db: column sums of the blocks' partial sums.  A block takes 32 of the 2 * width columns, eight threads a column.
template <typename T>
__global__ void __launch_bounds__(256)
norm_join_kernel(const float* partial, int blocks, int width, T* dw, T* db) {
  __shared__ float part[8][33];
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
  float sum = 0.f;
  if (c < 2 * width)
    for (int b = k; b < blocks; b += 8) sum += partial[(long long)b * 2 * width + c];
  part[k][threadIdx.x & 31] = sum;
  __syncthreads();
  if (k == 0 && c < 2 * width) {
    for (int i = 1; i < 8; ++i) sum += part[i][threadIdx.x];
    T* dst = c < width ? dw : db;
    if (dst != nullptr) dst[c < width ? c : c - width] = static_cast<T>(sum);
  }
}

struct Shape {
  int lanes, items, threads;
  bool vec;
};
// Threads that share a row: as few as hold it with at most 16 values each, a power of two.
Shape shape_of(int width, int vec, bool may_vec) {
  Shape s;
  s.vec = may_vec;
  const int v = may_vec ? vec : 1, most = may_vec ? 16 / vec : 16, n = (width + v - 1) / v;
  s.lanes = 1;
  while (s.lanes * most < n) s.lanes *= 2;
  // a warp's loads stay wide: up to 16 lanes of one vector before a lane takes a second one
  while (s.lanes < 16 && s.lanes < n) s.lanes *= 2;
  s.items = (n + s.lanes - 1) / s.lanes;
  s.threads = s.lanes > kThreads ? s.lanes : kThreads;
  return s;
}
int element_bytes(int dtype) { return dtype == B200TA_DTYPE_F32 ? 4 : 2; }
bool aligned(const void* p, int64_t stride, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride * bytes % 16 == 0;
}

// Blocks of the backward pass: as many as run at once with up to 80 registers a thread, so that there are few partial sums.
int grad_blocks(DeviceState* st, const Shape& s, int64_t rows) {
  const int64_t per_block = s.threads / s.lanes, need = (rows + per_block - 1) / per_block;
  const int64_t most = int64_t(st->num_sms) * (s.threads > 512 ? 1 : s.threads > 256 ? 1 : 3);
  return int(need < most ? need : most);
}

// Blocks of more than 256 threads hold rows that need all 16 values a thread.
template <typename T, int kVec, bool kGrad>
auto pick(const Shape& s) {
  constexpr int kMost = 16 / kVec, kFew = kVec == 1 ? 4 : 1, kSome = kVec == 1 ? 16 : 2;
  if constexpr (kGrad) {
    if (s.threads > 512) return &norm_grad_kernel<T, kVec, kMost, 1024>;
    if (s.threads > 256) return &norm_grad_kernel<T, kVec, kMost, 512>;
    if (s.items <= kFew) return &norm_grad_kernel<T, kVec, kFew, 256>;
    return s.items <= kSome ? &norm_grad_kernel<T, kVec, kSome, 256> : &norm_grad_kernel<T, kVec, kMost, 256>;
  } else {
    if (s.threads > 512) return &norm_kernel<T, kVec, kMost, 1024>;
    if (s.threads > 256) return &norm_kernel<T, kVec, kMost, 512>;
    if (s.items <= kFew) return &norm_kernel<T, kVec, kFew, 256>;
    return s.items <= kSome ? &norm_kernel<T, kVec, kSome, 256> : &norm_kernel<T, kVec, kMost, 256>;
  }
}
template <bool kGrad>
int launch_norm(DeviceState* st, int dtype, const Shape& s, const NormParams& p, int blocks, int smem, void* stream) {
  void (*kernel)(NormParams);
  if (dtype == B200TA_DTYPE_BF16) kernel = s.vec ? pick<__nv_bfloat16, 8, kGrad>(s) : pick<__nv_bfloat16, 1, kGrad>(s);
  else if (dtype == B200TA_DTYPE_F16) kernel = s.vec ? pick<__half, 8, kGrad>(s) : pick<__half, 1, kGrad>(s);
  else kernel = s.vec ? pick<float, 4, kGrad>(s) : pick<float, 1, kGrad>(s);
  return launch_kernel(st, kKernelNorm, kernel, dim3(unsigned(blocks)), s.threads, smem, stream, p);
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
  B200TA_REQUIRE(rows > 0 && width > 0 && width <= kMaxWidth, "layer_norm: rows=%lld, width=%d (1 to %d)", (long long)rows, width,
                 kMaxWidth);
  DeviceState* st = nullptr;
  const int rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  NormParams p{};
  p.x = x, p.w = weight, p.b = bias, p.y = y, p.stats = static_cast<float2*>(stats);
  p.xs = xs, p.ys = ys, p.rows = rows, p.width = width, p.eps = eps;
  p.param_f32 = param_dtype == B200TA_DTYPE_F32;
  const int bytes = element_bytes(dtype), vec = 16 / bytes;
  const bool wide = width % vec == 0 && aligned(x, xs, bytes) && aligned(y, ys, bytes) && aligned(weight, 0, 4) && aligned(bias, 0, 4);
  const Shape s = shape_of(width, vec, wide);
  p.lanes = s.lanes;
  const int64_t per_block = s.threads / s.lanes, need = (rows + per_block - 1) / per_block, most = int64_t(st->num_sms) * 16;
  const int blocks = int(need < most ? need : most);
  return launch_norm<false>(st, dtype, s, p, blocks, 0, stream);
}

size_t b200ta_layer_norm_workspace_bytes(int64_t rows, int width) {
  // a row of partial sums for each of at most 3 * 148 blocks (more on a device with more multiprocessors)
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
  B200TA_REQUIRE(rows > 0 && width > 0 && width <= kMaxWidth, "layer_norm_backward: rows=%lld, width=%d (1 to %d)",
                 (long long)rows, width, kMaxWidth);
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
  p.param_f32 = param_dtype == B200TA_DTYPE_F32;
  const int bytes = element_bytes(dtype), vec = 16 / bytes;
  const bool wide = width % vec == 0 && aligned(x, xs, bytes) && aligned(dy, dys, bytes) && (!dx || aligned(dx, dxs, bytes)) &&
                    aligned(weight, 0, 4);
  const Shape s = shape_of(width, vec, wide);
  p.lanes = s.lanes;
  const int blocks = grad_blocks(st, s, rows);
  const int groups = s.threads / s.lanes, smem = sums && groups > 1 ? groups / 2 * 2 * width * int(sizeof(float)) : 0;
  rc = launch_norm<true>(st, dtype, s, p, blocks, smem, stream);
  if (rc != B200TA_OK || !sums) return rc;
  const dim3 grid{unsigned((2 * width + 31) / 32)};
  if (param_dtype == B200TA_DTYPE_F32)
    return launch_kernel(st, kKernelNorm, norm_join_kernel<float>, grid, 256, 0, stream, p.partial, blocks, width,
                         static_cast<float*>(dweight), static_cast<float*>(dbias));
  if (param_dtype == B200TA_DTYPE_F16)
    return launch_kernel(st, kKernelNorm, norm_join_kernel<__half>, grid, 256, 0, stream, p.partial, blocks, width,
                         static_cast<__half*>(dweight), static_cast<__half*>(dbias));
  return launch_kernel(st, kKernelNorm, norm_join_kernel<__nv_bfloat16>, grid, 256, 0, stream, p.partial, blocks, width,
                       static_cast<__nv_bfloat16*>(dweight), static_cast<__nv_bfloat16*>(dbias));
}

}  // extern "C"

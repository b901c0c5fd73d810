// Dropout with a mask that is never stored (sm_100a), for bf16, fp16 or fp32:
//
//   y = residual + [u(m) >= d] x 2^16 / (2^16 - d)        d = round(p 2^16), m the element's number
//
// u(m) are the 16 bits of place m mod 8 in the 128 bits that Philox 4x32 with ten rounds (J. Salmon, M. Moraes, R. Dror, D. Shaw:
// Parallel random numbers: as easy as 1, 2, 3, 2011) makes of the counter (m / 8, sequence) under the key `seed`: a function of
// the element's number alone, so the backward pass is this kernel on dy, whatever the two launches look like.  With a shared axis
// its entries have one draw: x is [outer, axis, inner] and m numbers [outer, inner].  The probability is p to 2^-17, and the
// factor is that of the probability as it is, so that the mean stays.  A dropped element is left out, not multiplied by zero:
// infinities and NaN in it vanish.
//
// Bound: HBM (x and residual are read, y is written, once), or issue slots where the generator runs for every element of 16 bits: a
// block of it serves eight elements, 60 slots of the 32 bytes' 140.  A thread takes several vectors, whose loads are on their way while
// the generator runs; along a shared axis it makes one block of the generator for all of them.  Measured back to back: 262144 rows of
// 128 in bf16 with a residual and a shared axis 31 us (6.5 TB/s), 16384 rows of 2048 in fp16 without either 23 us (5.8 TB/s; 28 with a
// mask of bits between the generator and the elements), in fp32 41 us (6.6 TB/s).  Loads and stores mark their lines as used once, for
// the sake of what else is in L2: alone the kernel takes as long without.
#include <algorithm>

#include "activation.cuh"
#include "common.cuh"
#include "dropout_windows.h"

namespace b200ta {
namespace {

constexpr int kThreads = 256;

struct DropoutParams {
  const void *x, *residual;
  void* y;
  long long count;        // numbered elements: outer * inner
  long long axis, inner;  // (without a shared axis: 1, count)
  long long chunk;        // entries of the shared axis that a thread takes
  uint32_t dropped;       // of 65536
  float scale;
  uint64_t seed, sequence;
  const uint64_t* seed_at;  // read instead of seed, or NULL
};

__device__ __forceinline__ void philox_round(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
  const uint64_t a = uint64_t(c[0]) * 0xD2511F53u, b = uint64_t(c[2]) * 0xCD9E8D57u;
  const uint32_t c0 = uint32_t(b >> 32) ^ c[1] ^ k0, c2 = uint32_t(a >> 32) ^ c[3] ^ k1;
  c[0] = c0, c[1] = uint32_t(b), c[2] = c2, c[3] = uint32_t(a);
}
__device__ __forceinline__ void philox(uint32_t (&c)[4], uint64_t block, uint64_t sequence, uint64_t seed) {
  c[0] = uint32_t(block), c[1] = uint32_t(block >> 32), c[2] = uint32_t(sequence), c[3] = uint32_t(sequence >> 32);
  uint32_t k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    philox_round(c, k0, k1);
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
}
// Bit e of the result: element 8 * block + e stays.
__device__ __forceinline__ uint32_t keep_bits(uint64_t block, uint64_t sequence, uint64_t seed, uint32_t dropped) {
  uint32_t c[4];
  philox(c, block, sequence, seed);
  uint32_t bits = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    bits |= ((c[w] & 0xFFFFu) >= dropped ? 1u : 0u) << (2 * w);
    bits |= ((c[w] >> 16) >= dropped ? 1u : 0u) << (2 * w + 1);
  }
  return bits;
}
__device__ __forceinline__ uint64_t seed_of(const DropoutParams& p) { return p.seed_at != nullptr ? __ldg(p.seed_at) : p.seed; }

// Which of eight elements stay: by bits, or by the generator's words as they are (fewer instructions where they serve once).
struct KeepBits {
  uint32_t bits;
  __device__ __forceinline__ bool operator()(int e) const { return bits >> e & 1u; }
};
struct KeepWords {
  uint32_t c[4], dropped;  // dropped: below 65536
  __device__ __forceinline__ bool operator()(int e) const { return e & 1 ? c[e >> 1] >= dropped << 16 : (c[e >> 1] & 0xFFFFu) >= dropped; }
};
template <typename T>
struct Eight {  // elements, as they lie
  static constexpr int kVecs = int(sizeof(T)) / 2;
  uint4 v[kVecs];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, v[i]);
  }
};
// The 16 bytes of elements first, first + 1, ... of those that `keep` knows.
template <typename T, bool kResidual, typename Keep>
__device__ __forceinline__ uint4 drop_vec(uint4 x, uint4 residual, const Keep& keep, int first, float scale) {
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
  const uint32_t r[4] = {residual.x, residual.y, residual.z, residual.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) {
      const float r0 = kResidual ? __uint_as_float(r[j]) : 0.f;
      w[j] = __float_as_uint(keep(first + j) ? fmaf(__uint_as_float(w[j]), scale, r0) : r0);
    } else {
      const float2 f = unpack2<T>(w[j]), g = kResidual ? unpack2<T>(r[j]) : make_float2(0.f, 0.f);
      w[j] = pack2<T>(keep(first + 2 * j) ? fmaf(f.x, scale, g.x) : g.x, keep(first + 2 * j + 1) ? fmaf(f.y, scale, g.y) : g.y);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T, bool kResidual, typename Keep>
__device__ __forceinline__ void drop_eight(Eight<T>& x, const Eight<T>& residual, const Keep& keep, float scale) {
#pragma unroll
  for (int i = 0; i < Eight<T>::kVecs; ++i) x.v[i] = drop_vec<T, kResidual>(x.v[i], residual.v[i], keep, i * (16 / int(sizeof(T))), scale);
}
template <typename T, bool kResidual>
__device__ __forceinline__ void drop_one(const T* x, const T* residual, T* y, long long at, bool keep, float scale) {
  const float r = kResidual ? static_cast<float>(residual[at]) : 0.f;
  y[at] = static_cast<T>(keep ? fmaf(static_cast<float>(x[at]), scale, r) : r);
}

// Whole vectors of eight numbered elements: everything 16-byte aligned, and `inner` a multiple of eight where an axis is shared.
// A thread takes kUnroll of them at a time: blocks of the generator (kShared false) or entries of the shared axis.
template <typename T>
constexpr int kUnroll = sizeof(T) == 4 ? 2 : 4;
template <typename T, bool kShared, bool kResidual>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(const DropoutParams p) {
  constexpr int kN = kUnroll<T>;
  pdl_trigger();
  pdl_wait();
  const uint64_t seed = seed_of(p);
  const T *x = static_cast<const T*>(p.x), *residual = static_cast<const T*>(p.residual);
  T* y = static_cast<T*>(p.y);
  if constexpr (kShared) {
    const long long block = (long long)blockIdx.x * kThreads + threadIdx.x, m = block * 8;
    if (m >= p.count) return;
    const long long outer = m / p.inner, a0 = blockIdx.y * p.chunk, left = p.axis - a0 < p.chunk ? p.axis - a0 : p.chunk;
    long long at = (outer * p.axis + a0) * p.inner + (m - outer * p.inner);
    uint32_t keep = 0;
    for (long long a = 0; a < left; a += kN, at += kN * p.inner) {
      Eight<T> v[kN], r[kN];
#pragma unroll
      for (int u = 0; u < kN; ++u)
        if (a + u < left) {
          v[u].load(x + at + u * p.inner);
          if constexpr (kResidual) r[u].load(residual + at + u * p.inner);
        }
      if (a == 0) keep = keep_bits(block, p.sequence, seed, p.dropped);
#pragma unroll
      for (int u = 0; u < kN; ++u)
        if (a + u < left) {
          drop_eight<T, kResidual>(v[u], r[u], KeepBits{keep}, p.scale);
          v[u].store(y + at + u * p.inner);
        }
    }
  } else {
    const long long first = (long long)blockIdx.x * (kThreads * kN) + threadIdx.x;
    Eight<T> v[kN], r[kN];
#pragma unroll
    for (int u = 0; u < kN; ++u) {
      const long long m = (first + u * kThreads) * 8;
      if (m + 8 <= p.count) {
        v[u].load(x + m);
        if constexpr (kResidual) r[u].load(residual + m);
      }
    }
#pragma unroll
    for (int u = 0; u < kN; ++u) {
      const long long block = first + u * kThreads, m = block * 8;
      if (m >= p.count) break;
      KeepWords keep;
      philox(keep.c, block, p.sequence, seed);
      keep.dropped = p.dropped;
      if (m + 8 <= p.count) {
        drop_eight<T, kResidual>(v[u], r[u], keep, p.scale);
        v[u].store(y + m);
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (m + e < p.count) drop_one<T, kResidual>(x, residual, y, m + e, keep(e), p.scale);
      }
    }
  }
}

// An odd inner size beside a shared axis: rows of `inner` elements begin off the 16-byte boundaries, each on another.  A block makes the
// bits of 2048 numbered elements of one outer index; a row's whole vectors find their eight (fp32: four) bits at any place, and the
// elements before and behind them are taken one by one.  `lanes` threads share a row.
constexpr int kOdd = kThreads * 8;
static_assert(kOdd == kDropoutBits, "a byte of bits from each thread");
template <typename T, bool kResidual>
__global__ void __launch_bounds__(kThreads)
dropout_rows_kernel(const DropoutParams p, int windows, int lanes) {
  constexpr int kVec = 16 / int(sizeof(T)), kRows = 4;
  __shared__ uint32_t bits[kOdd / 32 + 2];  // (the numbered elements from the last multiple of eight before the window on)
  pdl_trigger();
  pdl_wait();
  const DropoutWindow window = dropout_window(blockIdx.x, unsigned(windows), p.inner);
  const int width = window.width;
  const long long m0 = window.outer * p.inner + window.first;
  reinterpret_cast<uint8_t*>(bits)[threadIdx.x] = uint8_t(keep_bits(m0 / 8 + threadIdx.x, p.sequence, seed_of(p), p.dropped));
  if (threadIdx.x < 2) bits[kOdd / 32 + threadIdx.x] = 0;
  __syncthreads();
  const int skew = int(m0 & 7), lane = threadIdx.x & (lanes - 1), step = kThreads / lanes;
  const T *x = static_cast<const T*>(p.x), *residual = static_cast<const T*>(p.residual);
  T* y = static_cast<T*>(p.y);
  auto keep_from = [&](int e) {  // bits of elements e, e + 1, ... of the window
    const int b = e + skew;
    return KeepBits{__funnelshift_r(bits[b >> 5], bits[(b >> 5) + 1], b & 31)};
  };
  const long long a1 = (blockIdx.y + 1) * p.chunk < p.axis ? (blockIdx.y + 1) * p.chunk : p.axis;
  for (long long a = blockIdx.y * p.chunk + threadIdx.x / lanes; a < a1; a += kRows * step) {
    long long row[kRows];  // the window's first element
    int head[kRows];       // elements before its first whole vector
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      row[r] = (window.outer * p.axis + a + r * step) * p.inner + window.first;
      head[r] = min(int(-row[r] & (kVec - 1)), width);
    }
    for (int v = lane; v * kVec < width; v += lanes) {
      uint4 from[kRows], add[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int e = head[r] + v * kVec;
        if (a + r * step < a1 && e + kVec <= width) {
          from[r] = __ldcs(reinterpret_cast<const uint4*>(x + row[r] + e));
          if constexpr (kResidual) add[r] = __ldcs(reinterpret_cast<const uint4*>(residual + row[r] + e));
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int e = head[r] + v * kVec;
        if (a + r * step < a1 && e + kVec <= width)
          __stcs(reinterpret_cast<uint4*>(y + row[r] + e), drop_vec<T, kResidual>(from[r], add[r], keep_from(e), 0, p.scale));
      }
    }
    // up to kVec - 1 elements on either side
    for (int k = lane; k < 2 * kVec; k += lanes) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (a + r * step >= a1) break;
        const int tail = head[r] + (width - head[r]) / kVec * kVec, e = k < kVec ? k : tail + k - kVec;
        if (k < kVec ? e < head[r] : e < width) drop_one<T, kResidual>(x, residual, y, row[r] + e, keep_from(e)(0), p.scale);
      }
    }
  }
}

// Everything else (addresses off the 16-byte boundaries, or p = 1, which the words' comparison cannot say): a block makes the bits of
// 2048 numbered elements, then its threads take neighbouring elements, eight of an entry of the shared axis at a time.
template <typename T, bool kResidual>
__global__ void __launch_bounds__(kThreads)
dropout_odd_kernel(const DropoutParams p) {
  __shared__ uint32_t bits[kOdd / 32];
  pdl_trigger();
  pdl_wait();
  const long long m0 = (long long)blockIdx.x * kOdd;
  reinterpret_cast<uint8_t*>(bits)[threadIdx.x] = uint8_t(keep_bits(m0 / 8 + threadIdx.x, p.sequence, seed_of(p), p.dropped));
  __syncthreads();
  const T *x = static_cast<const T*>(p.x), *residual = static_cast<const T*>(p.residual);
  T* y = static_cast<T*>(p.y);
  const long long a0 = blockIdx.y * p.chunk, a1 = a0 + p.chunk < p.axis ? a0 + p.chunk : p.axis;
  long long at[8];
  uint32_t keep = 0, in = 0;
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const int k = s * kThreads + threadIdx.x;
    const long long m = m0 + k, outer = m / p.inner;
    at[s] = (outer * p.axis + a0) * p.inner + (m - outer * p.inner);
    in |= (m < p.count ? 1u : 0u) << s;
    keep |= (bits[k >> 5] >> (k & 31) & 1u) << s;
  }
  for (long long a = a0; a < a1; ++a) {
    float v[8], r[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      v[s] = (in >> s & 1u) ? static_cast<float>(x[at[s]]) : 0.f;
      r[s] = kResidual && (in >> s & 1u) ? static_cast<float>(residual[at[s]]) : 0.f;
    }
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      if (in >> s & 1u) y[at[s]] = static_cast<T>((keep >> s & 1u) ? fmaf(v[s], p.scale, r[s]) : r[s]);
      at[s] += p.inner;
    }
  }
}

template <typename T>
int launch(DeviceState* st, DropoutParams p, void* stream) {
  auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
  const bool shared = p.axis > 1, based = aligned(p.x) && aligned(p.residual) && aligned(p.y);
  const bool whole = based && (shared ? p.inner % 8 == 0 : p.dropped < 65536), rows = based && shared && !whole && p.inner >= 16;
  const int64_t windows = dropout_windows(p.inner);
  const int64_t each = !whole ? kOdd : shared ? kThreads * 8 : kThreads * 8 * kUnroll<T>;
  const int64_t blocks = rows ? p.count / p.inner * windows : (p.count + each - 1) / each;
  B200TA_REQUIRE(blocks < (int64_t(1) << 31), "dropout: too many elements");
  int lanes = 4;  // as many threads as take a row's window at a time
  while (lanes < kThreads && lanes * (16 / int(sizeof(T))) < std::min<int64_t>(p.inner, kDropoutWindow)) lanes *= 2;
  // Two waves of eight blocks on each multiprocessor, as long as a thread has several entries of the axis.
  const int64_t wanted = std::max<int64_t>((int64_t(st->num_sms) * 16 + blocks - 1) / blocks, 1);
  p.chunk = std::max<int64_t>((p.axis + wanted - 1) / wanted, std::min<int64_t>(p.axis, rows ? 4 * (kThreads / lanes) : kUnroll<T>));
  p.chunk = std::max<int64_t>(p.chunk, (p.axis + 65534) / 65535);
  const dim3 grid{unsigned(blocks), unsigned((p.axis + p.chunk - 1) / p.chunk)};
  if (rows)
    return launch_kernel(st, kKernelDropout, p.residual ? &dropout_rows_kernel<T, true> : &dropout_rows_kernel<T, false>, grid, kThreads, 0, stream, p,
                         int(windows), lanes);
  void (*kernel)(DropoutParams);
  if (!whole) kernel = p.residual ? &dropout_odd_kernel<T, true> : &dropout_odd_kernel<T, false>;
  else if (shared) kernel = p.residual ? &dropout_kernel<T, true, true> : &dropout_kernel<T, true, false>;
  else kernel = p.residual ? &dropout_kernel<T, false, true> : &dropout_kernel<T, false, false>;
  return launch_kernel(st, kKernelDropout, kernel, grid, kThreads, 0, stream, p);
}

}  // namespace
}  // namespace b200ta

extern "C" int b200ta_dropout(const void* x, const void* residual, void* y, int dtype, int64_t outer, int64_t axis, int64_t inner, int dropped,
                              uint64_t seed, uint64_t sequence, const uint64_t* seed_at, void* stream) {
  using namespace b200ta;
  B200TA_REQUIRE(x && y, "dropout: NULL pointer");
  B200TA_REQUIRE(dtype >= 0 && dtype <= B200TA_DTYPE_F16, "dropout: unknown dtype %d", dtype);
  B200TA_REQUIRE(outer > 0 && axis > 0 && inner > 0, "dropout: bad sizes outer=%lld axis=%lld inner=%lld", (long long)outer, (long long)axis,
                 (long long)inner);
  B200TA_REQUIRE(dropped >= 0 && dropped <= 65536, "dropout: %d of 65536 dropped", dropped);
  const int size = dtype == B200TA_DTYPE_F32 ? 4 : 2;
  B200TA_REQUIRE((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(y)) % size == 0,
                 "dropout: an address is not a multiple of the element's size");
  DeviceState* st = nullptr;
  const int rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  DropoutParams p{};
  p.x = x, p.residual = residual, p.y = y;
  p.count = outer * inner, p.axis = axis, p.inner = axis == 1 ? p.count : inner;
  p.dropped = uint32_t(dropped), p.scale = dropped == 65536 ? 0.f : 65536.f / float(65536 - dropped);
  p.seed = seed, p.sequence = sequence, p.seed_at = seed_at;
  if (dtype == B200TA_DTYPE_BF16) return launch<__nv_bfloat16>(st, p, stream);
  if (dtype == B200TA_DTYPE_F16) return launch<__half>(st, p, stream);
  return launch<float>(st, p, stream);
}

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
// Bound: HBM (x and residual are read, y is written, once).  A generator's block serves eight elements, 60 issue slots for the 32
// or 48 bytes of a thread in 16 bits, half of what the memory pipe leaves; with 32 bits an element it would be the bound.  A thread
// takes several vectors, whose loads are on their way while the generator runs; along a shared axis it makes one block of the
// generator for all of them.
#include <algorithm>

#include "activation.cuh"
#include "common.cuh"

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
// Bit e of the result: element 8 * block + e stays.
__device__ __forceinline__ uint32_t keep_bits(uint64_t block, uint64_t sequence, uint64_t seed, uint32_t dropped) {
  uint32_t c[4] = {uint32_t(block), uint32_t(block >> 32), uint32_t(sequence), uint32_t(sequence >> 32)};
  uint32_t k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    philox_round(c, k0, k1);
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
  uint32_t bits = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    bits |= ((c[w] & 0xFFFFu) >= dropped ? 1u : 0u) << (2 * w);
    bits |= ((c[w] >> 16) >= dropped ? 1u : 0u) << (2 * w + 1);
  }
  return bits;
}
__device__ __forceinline__ uint64_t seed_of(const DropoutParams& p) { return p.seed_at != nullptr ? __ldg(p.seed_at) : p.seed; }

// Two neighbouring elements, of which bits `keep` say which stay.
__device__ __forceinline__ void drop2(float& a, float& b, float r0, float r1, uint32_t keep, float scale) {
  a = (keep & 1u) ? fmaf(a, scale, r0) : r0;
  b = (keep & 2u) ? fmaf(b, scale, r1) : r1;
}
template <typename T>
struct Eight {  // elements, as they lie
  static constexpr int kVecs = int(sizeof(T)) / 2;
  uint4 v[kVecs];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) reinterpret_cast<uint4*>(p)[i] = v[i];
  }
  template <bool kResidual>
  __device__ __forceinline__ void drop(const Eight& residual, uint32_t keep, float scale) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      const uint32_t r[4] = {residual.v[i].x, residual.v[i].y, residual.v[i].z, residual.v[i].w};
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          float a = __uint_as_float(w[j]), b = __uint_as_float(w[j + 1]);
          drop2(a, b, kResidual ? __uint_as_float(r[j]) : 0.f, kResidual ? __uint_as_float(r[j + 1]) : 0.f, keep >> (4 * i + j), scale);
          w[j] = __float_as_uint(a), w[j + 1] = __float_as_uint(b);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float2 f = unpack2<T>(w[j]);
          const float2 g = kResidual ? unpack2<T>(r[j]) : make_float2(0.f, 0.f);
          drop2(f.x, f.y, g.x, g.y, keep >> (2 * j), scale);
          w[j] = pack2<T>(f.x, f.y);
        }
      }
      v[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};
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
          v[u].template drop<kResidual>(r[u], keep, p.scale);
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
      const uint32_t keep = keep_bits(block, p.sequence, seed, p.dropped);
      if (m + 8 <= p.count) {
        v[u].template drop<kResidual>(r[u], keep, p.scale);
        v[u].store(y + m);
      } else {
        for (int e = 0; m + e < p.count; ++e) drop_one<T, kResidual>(x, residual, y, m + e, keep >> e & 1u, p.scale);
      }
    }
  }
}

// Everything else (odd inner sizes beside a shared axis, addresses off the 16-byte boundaries): a block makes the bits of 2048 numbered
// elements, then its threads take neighbouring elements, eight of an entry of the shared axis at a time.
constexpr int kOdd = kThreads * 8;
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
  const bool shared = p.axis > 1, whole = aligned(p.x) && aligned(p.residual) && aligned(p.y) && (!shared || p.inner % 8 == 0);
  const int64_t each = !whole ? kOdd : shared ? kThreads * 8 : kThreads * 8 * kUnroll<T>;
  const int64_t blocks = (p.count + each - 1) / each;
  B200TA_REQUIRE(blocks < (int64_t(1) << 31), "dropout: too many elements");
  // Two waves of eight blocks on each multiprocessor, as long as a thread has kUnroll entries of the axis.
  const int64_t wanted = std::max<int64_t>((int64_t(st->num_sms) * 16 + blocks - 1) / blocks, 1);
  p.chunk = std::max<int64_t>((p.axis + wanted - 1) / wanted, std::min<int64_t>(p.axis, kUnroll<T>));
  p.chunk = std::max<int64_t>(p.chunk, (p.axis + 65534) / 65535);
  const dim3 grid{unsigned(blocks), unsigned((p.axis + p.chunk - 1) / p.chunk)};
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

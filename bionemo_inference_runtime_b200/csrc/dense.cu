// The trainable dense layers around their products: argument checks, tensor maps and tiles of the products, and the small
// kernels beside them (few rows, dz from stored pre-activations, sums over rows, joining of parts, aligned copies).
#include <algorithm>

#include "layer_norm.cuh"
#include "matmul.cuh"
#include "narrow.cuh"

namespace b200ta {

namespace {

int map_of(CUtensorMap* map, const Plane& t, int bytes, uint32_t columns, uint32_t rows, uint32_t outer, SwizzleMode swz, const char* what) {
  const uint64_t dims[3] = {uint64_t(t.columns), uint64_t(t.rows), uint64_t(t.outer)};
  const uint64_t strides[2] = {uint64_t(t.pitch) * bytes, uint64_t(t.outer > 1 ? t.outer_stride : t.pitch) * bytes};
  const uint32_t box[3] = {columns, rows, outer};
  return encode_tensor_map(map, t.base, bytes, 3, dims, strides, box, swz, what);
}

// How the blocks share a product.  The costs are in clocks: a block of 64 along k costs its MMAs (4 * max(40, n * 0.54)) or its
// operands' way from L2 (46 bytes a clock and SM), a tile of 256 columns with its two stages waits for its loads besides, and
// a tile costs its finishing if that is more; all blocks take as many tiles as the busiest.  Pairs on 128 columns save loads of B
// (dW of 147456 rows, 128 -> 512 gated: 55 us, 58 by single blocks; 262144 rows of 512 -> 128: 71 and 73) and start later (768
// rows of 384 -> 1536 gated: 7.1 and 6.8).
struct Tiling {
  int tile_n, pair, resident;
  double clocks;
};
struct TilingOf {
  MatmulForm form;
  bool a_mn, sums;  // sums of A over k: tiles of up to 128 columns
  int64_t rows, outer, columns;
  int kblocks, splits;
};
Tiling choose_tiling(const TilingOf& m, int num_sms) {
  const bool two = m.form == kGated || m.form == kGatedGrad;
  const int64_t accumulated = two ? m.columns * 2 : m.columns;
  const double finish = m.form == kGatedGrad ? 12 : two ? 8 : 6.5;  // clocks for an accumulator column of 128 rows
  Tiling best{128, 0, 0, 1e300};
  auto consider = [&](int n, int pair, int resident, double waves, double main) {
    const double end = finish * n, cost = waves * std::max(main, end) + std::min(main, end) + (pair && n < 256 ? 3500 : 1500);
    if (cost < best.clocks * 0.98) best = {n, pair, resident, cost};
  };
  auto waves_of = [](int64_t items, int64_t blocks) { return double((items + blocks - 1) / blocks); };
  const int64_t tiles_m = (m.rows + 127) / 128 * m.outer;
  for (int n = m.sums ? 128 : 256; n >= 64; n /= 2) {
    if (n > 64 && n / 2 >= accumulated) continue;
    const int64_t tiles_n = (accumulated + n - 1) / n;
    const double mma = 4.0 * std::max(40.0, n * 0.54);
    if (!m.a_mn && m.splits == 1 && m.kblocks * n * matmul::kBK * 2 <= matmul::kResidentBytes && tiles_n <= num_sms) {
      const int64_t lanes = std::min(tiles_m, num_sms / tiles_n);
      consider(n, 0, int(lanes), waves_of(tiles_m, lanes), m.kblocks * std::max(mma, 356.0));
    } else {
      const double load = (n == 256 ? 1.2 : 1.0) * (16384 + n * 128) / 46;
      consider(n, 0, 0, waves_of(tiles_m * tiles_n * m.splits, num_sms), m.kblocks * std::max(mma, load));
    }
  }
  for (int n = 256; n >= 128 && m.rows > matmul::kBM && !m.sums; n /= 2) {
    if (n / 2 >= accumulated) continue;
    const int64_t tiles = (m.rows + 255) / 256 * m.outer * m.splits * ((accumulated + n - 1) / n);
    consider(n, 1, 0, waves_of(tiles, num_sms / 2), m.kblocks * std::max(4.0 * n * 0.54, (16384 + n * 64) / 46.0));
  }
  return best;
}

}  // namespace

int run_matmul(const Matmul& m, void* stream) {
  DeviceState* st = nullptr;
  int rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  const bool two = m.form == kGated || m.form == kGatedGrad;
  MatmulParams p{};
  const int64_t rows = m.a_mn ? m.a.columns : m.a.rows, columns = m.b_mn ? m.b.columns : m.b.rows;
  const int64_t k = m.a_mn ? m.a.rows : m.a.columns, m_outer = m.a_mn ? m.a.outer : 1, k_outer = m.a_mn ? 1 : m.a.outer;
  constexpr int64_t kMost = int64_t(1) << 31;
  B200TA_REQUIRE(rows < kMost - 512 && columns < kMost - 512 && k < kMost - 512, "%s: a size is past 2^31", m.what);
  p.kblocks_inner = int((k + matmul::kBK - 1) / matmul::kBK);
  p.kblocks = int(p.kblocks_inner * k_outer);
  p.kblocks_split = m.kblocks_split > 0 && m.kblocks_split < p.kblocks ? m.kblocks_split : p.kblocks;
  p.splits = (p.kblocks + p.kblocks_split - 1) / p.kblocks_split;
  p.rows_inner = int(rows), p.columns = int(columns);
  const Tiling tiling = choose_tiling({m.form, m.a_mn, m.sums != nullptr, rows, m_outer, columns, p.kblocks_split, p.splits}, st->num_sms);
  p.tile_n = tiling.tile_n, p.pair = tiling.pair, p.resident = tiling.resident;
  const int tile_m = p.pair ? 2 * matmul::kBM : matmul::kBM;
  p.tiles_m_inner = int((rows + tile_m - 1) / tile_m);
  p.tiles_m = int(p.tiles_m_inner * m_outer);
  const int units = two ? p.tile_n / 2 : p.tile_n;
  p.tiles_n = int((columns + units - 1) / units);
  const int64_t work = int64_t(p.tiles_m) * p.tiles_n * p.splits;
  B200TA_REQUIRE(work < kMost - 1024, "%s: too many tiles", m.what);
  p.work = int(work);
  p.group_m = p.pair ? 8 : 16;
  const int b_rows = p.pair ? p.tile_n / 2 : p.tile_n;
  p.stages = p.resident ? (matmul::kRingBytes - matmul::kResidentBytes) / matmul::kABytes
                        : matmul::kRingBytes / (matmul::kABytes + b_rows * matmul::kBK * 2);
  if (p.stages > matmul::kMaxStages) p.stages = matmul::kMaxStages;
  p.bias = m.bias;
  p.activation = m.activation;
  p.has_aux = m.aux.base != nullptr, p.has_saved = m.saved.base != nullptr, p.accumulate = m.accumulate, p.beside = m.beside, p.sums = m.sums;
  p.status = st->status_dev;

  MatmulMaps maps{};
  rc = m.a_mn ? map_of(&maps.a, m.a, 2, 64, 64, 1, SWZ_128, m.what) : map_of(&maps.a, m.a, 2, 64, matmul::kBM, 1, SWZ_128, m.what);
  if (rc != B200TA_OK) return rc;
  rc = m.b_mn ? map_of(&maps.b, m.b, 2, 64, 64, 1, SWZ_128, m.what)
              : map_of(&maps.b, m.b, 2, 64, uint32_t(p.pair || !two ? b_rows : units), two && !p.pair ? 2 : 1, SWZ_128, m.what);
  if (rc != B200TA_OK) return rc;
  const bool f32 = m.form == kPartial;
  const bool stored = f32 || ((reinterpret_cast<uintptr_t>(m.out.base) & 15u) == 0 && m.out.pitch % 8 == 0 &&
                              (m.out.outer == 1 || m.out.outer_stride % 8 == 0));
  if (!stored) {
    B200TA_REQUIRE(m.form == kDense || m.form == kGated || m.form == kPlain, "%s: the result must be aligned", m.what);
    p.direct = const_cast<void*>(m.out.base), p.direct_pitch = m.out.pitch, p.direct_outer = m.out.outer_stride;
  } else if ((rc = map_of(&maps.out, m.out, f32 ? 4 : 2, f32 ? 16 : 32, 32, 1, SWZ_64, m.what)) != B200TA_OK) {
    return rc;
  }
  if (p.has_aux && (rc = map_of(&maps.aux, m.aux, 2, 32, 32, 1, SWZ_64, m.what)) != B200TA_OK) return rc;
  if (p.has_saved && (rc = map_of(&maps.saved, m.saved, 4, 16, 32, 1, SWZ_64, m.what)) != B200TA_OK) return rc;
  const int blocks = p.resident ? p.resident * p.tiles_n : std::min(p.work, p.pair ? st->num_sms / 2 : st->num_sms);
  const int grid = p.pair ? 2 * blocks : blocks;
  // Sets of finishing warps are out of step, so that one computes while another loads and stores, and a warp's waits serve more
  // columns; with a single group of 32 result columns to a tile, two sets would leave half of the warps without work.  A block's
  // only tile is for all of them.  (Sums of A over k lie behind 128 accumulator columns.)
  const bool several = p.resident ? p.tiles_m > p.resident : p.work > blocks;
  p.buffers = p.tile_n <= 128 && p.sums == nullptr ? 2 : 1;
  p.sets = !several ? 0 : units <= 32 || p.columns <= 32 ? 2 : 1;
  // A set sees the phases of its own tiles alone, and a wait cannot tell a phase from the one after the next: every phase of an
  // accumulator has to be the same set's, so there are as many accumulators as sets at least.
  p.sets = std::min(p.sets, p.buffers);
  if (m.form == kDenseGrad || m.form == kGatedGrad) return launch_matmul_grad(st, m, maps, p, grid, stream);
  if (m.b_mn) return launch_matmul_product(st, m, maps, p, grid, stream);
  return launch_matmul_forward(st, m, maps, p, grid, stream);
}

namespace {

// ---- few rows ---------------------------------------------------------------------------------------------------
//
// Up to 16 rows: the weights are read once and that bounds the call, or its latency does.  A block takes 16 result columns (and
// their gates for kGated), whose rows of W are the left operand of warp-wide products m16n8k16, eight rows of x the right one; its
// warps take 32 of k in turn and add up in shared memory.  A lane reads 16 bytes of each of its rows, eight neighbouring k, which
// serve as pairs 2t, 2t + 8 of two products: the order of k is the same in both operands and does not matter.  128-row tiles of
// the tensor cores would leave all but N / 64 SMs idle and wait for tensor memory, and products by FMA want every row of x in
// registers for each column (13 rows, 960 -> 4648 gated: 45 us so, now 8; 16 rows, 4096 -> 4096: 130 and 18; one row the same).
// Rows that are not 16-byte aligned are shifted into place.
constexpr int kFewRows = 16;

struct FewParams {
  const void *x, *w, *bias, *residual;
  void *y, *saved;
  long long xs, ws, rs, ys, ss;
  int rows, K, N, activation;
};

template <typename T>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = unpack2<T>(w[e]);
    v[2 * e] = f.x, v[2 * e + 1] = f.y;
  }
}

__device__ __forceinline__ void activate_any(int activation, float z, float& a, float& s) {
  float a1, s1;
  switch (activation) {
    case kActNone: return activate2<kActNone, true>(z, z, a, a1, s, s1);
    case kActRelu: return activate2<kActRelu, true>(z, z, a, a1, s, s1);
    case kActSilu: return activate2<kActSilu, true>(z, z, a, a1, s, s1);
    case kActGelu: return activate2<kActGelu, true>(z, z, a, a1, s, s1);
    case kActGeluTanh: return activate2<kActGeluTanh, true>(z, z, a, a1, s, s1);
    default: return activate2<kActSigmoid, true>(z, z, a, a1, s, s1);
  }
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __half))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Eight elements of a row of K from k on, zeros behind it.
template <typename T, bool kVec>
__device__ __forceinline__ uint4 load_row(const T* row, int k, int K) {
  if constexpr (kVec) return norm::load_if(k < K, row + k);
  const uint4 v = norm::load_anywhere(row + k, row, K);
  return K - k >= 8 ? v : norm::first<T>(v, K - k);
}

constexpr int kFewWarps = 16, kFewColumns = 16;  // of a block, at most
template <typename T, bool kTwo, int kEights, bool kVec>
__global__ void __launch_bounds__(kFewWarps * 32, 1)
few_rows_kernel(const FewParams p) {
  __shared__ float joined[kFewWarps][kTwo ? 2 : 1][kEights * 8][kFewColumns + 1];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, n0 = blockIdx.x * kFewColumns, warps = blockDim.x >> 5;
  constexpr int kParts = kTwo ? 2 : 1;
  const T *w[kParts][2], *x[kEights];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int n = min(n0 + g + 8 * h, p.N - 1);  // (rows past the last are read again, their results not stored)
    w[0][h] = static_cast<const T*>(p.w) + n * p.ws;
    if constexpr (kTwo) w[1][h] = static_cast<const T*>(p.w) + (long long)(n + p.N) * p.ws;
  }
#pragma unroll
  for (int e = 0; e < kEights; ++e) x[e] = static_cast<const T*>(p.x) + min(g + 8 * e, p.rows - 1) * p.xs;
  float acc[kParts][kEights][4] = {};
#pragma unroll 4
  for (int k = warp * 32; k < p.K; k += warps * 32) {
    uint4 a[kParts][2], b[kEights];
#pragma unroll
    for (int i = 0; i < kParts; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) a[i][h] = load_row<T, kVec>(w[i][h], k + t * 8, p.K);
#pragma unroll
    for (int e = 0; e < kEights; ++e) b[e] = load_row<T, kVec>(x[e], k + t * 8, p.K);
#pragma unroll
    for (int i = 0; i < kParts; ++i)
#pragma unroll
      for (int e = 0; e < kEights; ++e) {
        mma16816<T>(acc[i][e], a[i][0].x, a[i][1].x, a[i][0].y, a[i][1].y, b[e].x, b[e].y);
        mma16816<T>(acc[i][e], a[i][0].z, a[i][1].z, a[i][0].w, a[i][1].w, b[e].z, b[e].w);
      }
  }
#pragma unroll
  for (int i = 0; i < kParts; ++i)
#pragma unroll
    for (int e = 0; e < kEights; ++e)
#pragma unroll
      for (int j = 0; j < 4; ++j) joined[warp][i][e * 8 + t * 2 + (j & 1)][g + 8 * (j >> 1)] = acc[i][e][j];
  __syncthreads();
  const int row = threadIdx.x / kFewColumns, c = threadIdx.x % kFewColumns, n = n0 + c;
  if (row >= p.rows || n >= p.N) return;
  float v = 0.f, gate = 0.f;
  for (int i = 0; i < warps; ++i) {
    v += joined[i][0][row][c];
    if constexpr (kTwo) gate += joined[i][1][row][c];
  }
  const T* bias = static_cast<const T*>(p.bias);
  if (bias != nullptr) {
    v += static_cast<float>(bias[n]);
    if (kTwo) gate += static_cast<float>(bias[n + p.N]);
  }
  if (p.saved != nullptr) {
    float* s = static_cast<float*>(p.saved) + row * p.ss + n;
    s[0] = v;
    if (kTwo) s[p.ss / 2] = gate;
  }
  float a, slope;
  activate_any(p.activation, kTwo ? gate : v, a, slope);
  if (kTwo) a *= v;
  if (p.residual != nullptr) a += static_cast<float>(static_cast<const T*>(p.residual)[row * p.rs + n]);
  static_cast<T*>(p.y)[row * p.ys + n] = static_cast<T>(a);
}

template <typename T, bool kTwo>
auto pick_few(int rows, bool vec) {
  if (rows <= 8) return vec ? &few_rows_kernel<T, kTwo, 1, true> : &few_rows_kernel<T, kTwo, 1, false>;
  return vec ? &few_rows_kernel<T, kTwo, 2, true> : &few_rows_kernel<T, kTwo, 2, false>;
}
template <typename T>
auto pick_few(int rows, bool vec, bool two) {
  return two ? pick_few<T, true>(rows, vec) : pick_few<T, false>(rows, vec);
}

// ---- dz from stored pre-activations ---------------------------------------------------------------------------------
//
// dz = dy act'(z), or [dy act(g) | dy v act'(g)], z kept in 32 bits: bound by HBM (8192 rows of 4096, bf16: 42 us, 268 MB at 6.4
// TB/s).  A block takes 256 columns of some rows, a thread eight columns of every eighth of them, whose sums (db) it has on the
// way: part[block.y][column] (+)= theirs, of the values before they are rounded.
struct SlopeParams {
  const void *dy, *saved;
  void* dz;
  float* part;  // or NULL
  long long dys, ss, zs, rows, part_pitch;
  int N, rows_block, accumulate;
};
__device__ __forceinline__ void load_eight(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
// The sums of the block's threads with the same columns, to the workspace.
__device__ __forceinline__ void store_sums(const float (&s)[8], float (&joined)[8][256 + 4], float* part, int columns, bool accumulate) {
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
#pragma unroll
  for (int j = 0; j < 8; ++j) joined[k][lane * 8 + j] = s[j];
  __syncthreads();
  if (int(threadIdx.x) < columns) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += joined[i][threadIdx.x];
    part[threadIdx.x] = accumulate ? part[threadIdx.x] + sum : sum;
  }
  __syncthreads();
}
template <typename T, int kAct, bool kTwo>
__global__ void __launch_bounds__(256, kTwo ? 3 : 4)
slope_kernel(const SlopeParams p) {
  __shared__ float joined[8][256 + 4];
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x * 256 + (threadIdx.x & 31) * 8;
  const long long r0 = (long long)blockIdx.y * p.rows_block, r1 = r0 + p.rows_block < p.rows ? r0 + p.rows_block : p.rows;
  float sv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sg[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (c < p.N) {
#pragma unroll 1
    for (long long row = r0 + (threadIdx.x >> 5); row < r1; row += 8) {
      const T* dy = static_cast<const T*>(p.dy) + row * p.dys + c;
      const float* z = static_cast<const float*>(p.saved) + row * p.ss + c;
      T* dz = static_cast<T*>(p.dz) + row * p.zs + c;
      float d[8], v[8], g[8];
      if (c + 8 <= p.N) {
        load_vec<T>(dy, d);
        load_eight(z, v);
        if constexpr (kTwo) load_eight(z + p.ss / 2, g);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = c + j < p.N;
          d[j] = in ? static_cast<float>(dy[j]) : 0.f, v[j] = in ? z[j] : 0.f;
          if constexpr (kTwo) g[j] = in ? z[p.ss / 2 + j] : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        float a0, a1, s0, s1;
        if constexpr (kTwo) {
          activate2<kAct, true>(g[j], g[j + 1], a0, a1, s0, s1);
          g[j] = d[j] * v[j] * s0, g[j + 1] = d[j + 1] * v[j + 1] * s1;
          v[j] = d[j] * a0, v[j + 1] = d[j + 1] * a1;
          sg[j] += g[j], sg[j + 1] += g[j + 1];
        } else {
          activate2<kAct, true>(v[j], v[j + 1], a0, a1, s0, s1);
          v[j] = d[j] * s0, v[j + 1] = d[j + 1] * s1;
        }
        sv[j] += v[j], sv[j + 1] += v[j + 1];
      }
      // (dz's rows are padded to eight columns: its last vector is stored whole)
      *reinterpret_cast<uint4*>(dz) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
      if constexpr (kTwo)
        *reinterpret_cast<uint4*>(dz + p.zs / 2) =
            make_uint4(pack2<T>(g[0], g[1]), pack2<T>(g[2], g[3]), pack2<T>(g[4], g[5]), pack2<T>(g[6], g[7]));
    }
  }
  if (p.part == nullptr) return;
  float* part = p.part + (long long)blockIdx.y * p.part_pitch + blockIdx.x * 256;
  const int columns = p.N - int(blockIdx.x) * 256;
  store_sums(sv, joined, part, columns, p.accumulate);
  if constexpr (kTwo) store_sums(sg, joined, part + p.zs / 2, columns, p.accumulate);
}
template <typename T, bool kTwo>
auto pick_slope(int activation) {
  switch (activation) {
    case kActNone: return &slope_kernel<T, kActNone, kTwo>;
    case kActRelu: return &slope_kernel<T, kActRelu, kTwo>;
    case kActSilu: return &slope_kernel<T, kActSilu, kTwo>;
    case kActGelu: return &slope_kernel<T, kActGelu, kTwo>;
    case kActGeluTanh: return &slope_kernel<T, kActGeluTanh, kTwo>;
    default: return &slope_kernel<T, kActSigmoid, kTwo>;
  }
}

// ---- sums over rows -------------------------------------------------------------------------------------------------
//
// part[block.y][n] (+)= sum over a block's rows of dz[., n], in 32 bits, of the values as they were rounded for dx and dW: the
// roundings of many rows add up to about that of the result.  32 lanes of eight columns, eight rows at a time, eight loads of a
// thread on their way: dz of 5003 rows and 6144 columns takes 14 us (61 MB).  (Blocks of half the rows with four loads: two waves
// of them, 19 us.)
template <typename T>
__global__ void __launch_bounds__(256, 4)
row_sum_kernel(const T* dz, long long pitch, long long rows, int N, long long part_pitch, int rows_block, int accumulate, float* part) {
  __shared__ float joined[8][256 + 4];
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x * 256 + (threadIdx.x & 31) * 8;
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const long long r0 = (long long)blockIdx.y * rows_block, r1 = r0 + rows_block < rows ? r0 + rows_block : rows;
  if (c < N) {
#pragma unroll 8
    for (long long r = r0 + (threadIdx.x >> 5); r < r1; r += 8) {
      float v[8];
      if (c + 8 <= N) {
        load_vec<T>(dz + r * pitch + c, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < N ? static_cast<float>(dz[r * pitch + c + j]) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
    }
  }
  store_sums(s, joined, part + (long long)blockIdx.y * part_pitch + blockIdx.x * 256, N - int(blockIdx.x) * 256, accumulate);
}

// out[r][c] = sum over the parts, in a fixed order; up to three such results (dW, db, dx) in one launch.
// A thread sums one value, four where they lie together, or eight threads sum one where there are many parts of few values (18 parts of
// 1024 x 128: 7.5 us, 9.4 MB mostly from L2; a launch and one round of loads bound it).
struct JoinParams {
  const float* part;
  void* out;  // rows of `columns`, dense
  long long part_stride, pitch, rows;
  int parts, columns, slices, blocks;  // slices: threads of a value, 1 or 8; 0: a thread takes four neighbouring values
};
template <typename T>
__device__ __forceinline__ void join_by_four(const JoinParams& p, long long first) {
  const int quads = p.columns / 4;
  for (long long i = first; i < p.rows * quads; i += p.blocks * 256LL) {
    const long long r = i / quads;
    const int c = int(i - r * quads) * 4;
    const float4* src = reinterpret_cast<const float4*>(p.part + r * p.pitch + c);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < p.parts; ++s) {
      const float4 x = __ldg(src + s * (p.part_stride / 4));
      sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
    }
    T* out = static_cast<T*>(p.out) + r * p.columns + c;  // 8-byte aligned: columns are a multiple of four
    *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(sum.x, sum.y), pack2<T>(sum.z, sum.w));
  }
}
template <typename T>
__global__ void __launch_bounds__(256)
join_kernel(const JoinParams a, const JoinParams b, const JoinParams c) {
  __shared__ float joined[8][33];
  pdl_trigger();
  pdl_wait();
  const int block = int(blockIdx.x);
  const JoinParams& p = block < a.blocks ? a : block < a.blocks + b.blocks ? b : c;
  const long long own = block - (block < a.blocks ? 0 : block < a.blocks + b.blocks ? a.blocks : a.blocks + b.blocks);
  if (p.slices == 0) return join_by_four<T>(p, own * 256 + threadIdx.x);
  const int values = 256 / p.slices, slice = p.slices == 1 ? 0 : threadIdx.x >> 5, lane = p.slices == 1 ? threadIdx.x : threadIdx.x & 31;
  const long long total = p.rows * p.columns;
  for (long long i0 = own * values; i0 < total; i0 += (long long)p.blocks * values) {
    const long long i = i0 + lane, r = i / p.columns;
    const float* src = p.part + r * p.pitch + (i - r * p.columns);
    float sum = 0.f;
    if (i < total)
#pragma unroll 8
      for (int s = slice; s < p.parts; s += p.slices) sum += __ldg(src + s * p.part_stride);
    if (p.slices > 1) {
      joined[slice][lane] = sum;
      __syncthreads();
      if (slice == 0)
#pragma unroll
        for (int s = 1; s < 8; ++s) sum += joined[s][lane];
      __syncthreads();
    }
    if (slice == 0 && i < total) static_cast<T*>(p.out)[i] = static_cast<T>(sum);
  }
}

// ---- aligned copies ---------------------------------------------------------------------------------------------------
//
// dst[r][c] = src[r * rs + c * cs] for 16-bit elements: tensors whose rows a TMA load cannot address (a pitch or base that is
// no multiple of 16 bytes, columns that are not contiguous) pass through a padded copy, up to four in one launch.  A thread
// makes a vector of eight columns, from two aligned loads shifted into place if they are contiguous, otherwise from eight
// loads with neighbouring threads in neighbouring rows.  (An aligned 16-byte vector with a byte of the source in it lies in
// the source's allocation.)  2047 rows of 515 and 1283 rows of 515 in one launch take 4.4 us, with 2047 of 1283 besides 6.2.
struct CopyParams {
  b200ta_copy job[B200TA_COPIES];
  long long end[B200TA_COPIES];  // vectors up to and with this job
  int jobs;
};
__global__ void __launch_bounds__(256)
copy_rows_kernel(const CopyParams p) {
  pdl_trigger();
  pdl_wait();
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < p.end[p.jobs - 1]; i += gridDim.x * 256LL) {
    int k = 0;
    while (i >= p.end[k]) ++k;
    const b200ta_copy& job = p.job[k];
    const long long v = i - (k == 0 ? 0 : p.end[k - 1]);
    const int vectors = (job.columns + 7) / 8;
    uint16_t* dst = static_cast<uint16_t*>(job.dst);
    const uint16_t* src = static_cast<const uint16_t*>(job.src);
    if (job.column_stride == 1) {
      const long long r = v / vectors;
      const int c = int(v - r * vectors) * 8, valid = job.columns - c;
      const __half* row = reinterpret_cast<const __half*>(src + r * job.row_stride);
      const uint4 x = norm::load_anywhere(row + c, row, job.columns);
      *reinterpret_cast<uint4*>(dst + r * job.dst_row_stride + c) = valid >= 8 ? x : norm::first<__half>(x, valid);
    } else {
      const long long c = v / job.rows * 8, r = v - v / job.rows * job.rows;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = c + 2 * j < job.columns ? src[r * job.row_stride + (c + 2 * j) * job.column_stride] : 0u;
        const uint32_t hi = c + 2 * j + 1 < job.columns ? src[r * job.row_stride + (c + 2 * j + 1) * job.column_stride] : 0u;
        w[j] = lo | hi << 16;
      }
      *reinterpret_cast<uint4*>(dst + r * job.dst_row_stride + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

bool rows_aligned(const void* p, int64_t pitch) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && pitch % 8 == 0; }
int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
int64_t pad4(int64_t n) { return (n + 3) / 4 * 4; }

int check_layer(const char* what, int dtype, int activation, int64_t rows, int K, int N) {
  B200TA_REQUIRE(dtype == B200TA_DTYPE_BF16 || dtype == B200TA_DTYPE_F16, "%s: activations and weights are bf16 or fp16 (dtype %d)", what, dtype);
  B200TA_REQUIRE(activation >= 0 && activation < kActCount, "%s: unknown activation %d", what, activation);
  B200TA_REQUIRE(rows > 0 && K > 0 && N > 0 && rows < (int64_t(1) << 31) - 512 && N < (1 << 30), "%s: rows=%lld, K=%d, N=%d", what,
                 (long long)rows, K, N);
  return B200TA_OK;
}

// How dW = dz^T x is cut along the rows, and whether db comes from the same product (sums of dz by MMAs with ones, which only
// tiles of up to 128 columns have room for) or from a pass over dz: its own, or the one that forms dz from kept values.  Parts are
// written and read once and sums read dz once more at some 2400 bytes a clock; a launch more costs some 4000 clocks.
struct Split {
  int kblocks, parts;  // of a part; in all
  bool sums;           // db from the product
};
Split split_rows(int64_t rows, int64_t n_rows, int64_t n_outer, int64_t columns, bool want_sums, bool kept, int num_sms) {
  const int64_t kblocks = (rows + matmul::kBK - 1) / matmul::kBK, values = n_rows * n_outer;
  Split best{int(kblocks), 1, false};
  double least = 1e300;
  for (int64_t tried = 1; tried <= 256 && tried <= kblocks; tried += tried < 8 ? 1 : tried < 24 ? 2 : tried < 64 ? 8 : 16) {
    const int64_t per = (kblocks + tried - 1) / tried, parts = (kblocks + per - 1) / per;
    for (int sums = 0; sums <= int(want_sums); ++sums) {
      const MatmulForm form = parts > 1 ? kPartial : kPlain;
      double cost = choose_tiling({form, true, sums != 0, n_rows, n_outer, columns, int(per), int(parts)}, num_sms).clocks;
      if (parts > 1) cost += 4000 + 8.0 * double(parts) * double(values) * double(columns) / 2400;
      if (want_sums && !sums) cost += (parts > 1 ? 0 : 4000) + (kept ? 0 : 4000 + 2.0 * double(values) * double(rows) / 2400);
      if (cost < least * 0.98) least = cost, best = {int(per), int(parts), sums != 0};
    }
  }
  return best;
}
// How dx = dz W is cut along the hidden units: in parts where few row tiles would walk many of them (1799 rows of 40, 5958 gated
// units: 66 us in one, 20 in parts with their join).  Many rows have tiles enough.
Split split_units(int64_t rows, int64_t units, int64_t outer, int64_t K, int num_sms) {
  const int64_t kblocks = (units + matmul::kBK - 1) / matmul::kBK * outer;
  Split best{int(kblocks), 1, false};
  double least = 1e300;
  for (int64_t tried = 1; tried <= 64 && tried <= kblocks && (tried == 1 || rows < int64_t(num_sms) * 64);
       tried += tried < 8 ? 1 : tried < 24 ? 2 : 8) {
    const int64_t per = (kblocks + tried - 1) / tried, parts = (kblocks + per - 1) / per;
    double cost = choose_tiling({parts > 1 ? kPartial : kPlain, false, false, rows, 1, K, int(per), int(parts)}, num_sms).clocks;
    if (parts > 1) cost += 8000 + 8.0 * double(parts) * double(rows) * double(K) / 2400;
    if (cost < least * 0.95) least = cost, best = {int(per), int(parts), false};
  }
  return best;
}
constexpr int kChunkRows = 256;  // chunks of the backward pass are multiples of this
// Rows of a partial sum of db: enough blocks of 256 columns to fill the device a few times, 32 to 1024 rows each; more where the
// second axis of a grid, on which the blocks of rows lie, has no room for so many blocks.
int sum_rows(int64_t rows, int64_t columns, int num_sms) {
  const int64_t blocks = std::max<int64_t>(4 * num_sms / ((columns + 255) / 256), 1), each = (rows + blocks - 1) / blocks;
  const int64_t wanted = std::min<int64_t>(std::max<int64_t>((each + 7) / 8 * 8, 32), 1024), least = (rows + 65534) / 65535;
  return int(std::max(wanted, (least + 7) / 8 * 8));
}

// The backward pass: how many rows at a time, and where its intermediates lie in the workspace.
struct BackwardPlan {
  int64_t chunk;      // rows of dz at a time
  int64_t dz_pitch;   // 0: dz is dy
  Split split;        // of a chunk's rows for dW
  bool direct;        // dW is written by its product
  Split dx_split;     // of the units for dx
  int rows_sum;       // rows of a partial sum of db
  int64_t dz, parts, sums, dx_parts, bytes;  // offsets, total
};
// Whether dz and dx come from one kernel (narrow.cuh).  Its blocks walk 64 units of 256 rows in some 6000 clocks (dense layers: 4800), one
// item of 256 rows after the other, where two products take some 9000 (5500) for 128 units of 128 rows, shared evenly, and 25000 for
// their launches and ends.  (Backward pass of a gated layer 128 -> 512: 9472 rows 46 us so and 44 otherwise, 16384 rows 48 and 57,
// 147456 rows 194 and 229; 128 -> 128, 9472 rows: 32 and 39; 104 -> 3160, 14196 rows: 265 and 208.)
bool narrow_pays(bool own_dz, bool kept, bool gated, int64_t rows, int K, int N, const void* dx, int64_t dxs, int num_sms) {
  if (!own_dz || kept || K > 128 || dx == nullptr || !rows_aligned(dx, dxs) || rows <= kChunkRows) return false;
  const double items = double((rows + 255) / 256), waves = double((int64_t(items) + num_sms - 1) / num_sms);
  const double one = waves * double((N + 63) / 64) * (gated ? 6000 : 4800) + 8000;
  return one < 25000 + (gated ? 9000 : 5500) * (double(rows) / 128) * (double(N) / 128) / num_sms;
}
BackwardPlan make_plan(bool gated, bool slope, bool kept, bool want_dbias, int64_t rows, int K, int N, int num_sms) {
  BackwardPlan p{};
  const int64_t outer = gated ? 2 : 1;
  p.dz_pitch = gated || slope ? outer * pad8(N) : 0;
  p.chunk = rows;
  if (p.dz_pitch != 0) {
    // At most half a gigabyte of dz, in whole waves of row tiles.  (Chunks that L2 keeps do not pay: a gated layer 128 -> 512
    // over 147456 rows took 347 us in chunks of 39 MB, 300 us of 116 MB and 241 us in one, which writes dz to HBM and reads
    // it twice; each launch's first loads and last stores cost more.)
    const int64_t wave = (int64_t(num_sms) * matmul::kBM + kChunkRows - 1) / kChunkRows * kChunkRows;
    p.chunk = std::min(rows, std::max<int64_t>((int64_t(1) << 29) / (p.dz_pitch * 2) / wave, 1) * wave);
  }
  p.split = split_rows(p.chunk, N, outer, K, want_dbias, kept, num_sms);
  p.direct = p.chunk >= rows && p.split.parts == 1;
  auto take = [&](int64_t bytes) {
    const int64_t at = p.bytes;
    p.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  p.dz = take(p.dz_pitch * (p.chunk < rows ? p.chunk : rows) * 2);
  p.parts = take(p.direct ? 0 : p.split.parts * outer * N * pad4(K) * int64_t(sizeof(float)));
  p.dx_split = p.chunk >= rows ? split_units(rows, N, outer, K, num_sms) : Split{0, 1, false};
  p.dx_parts = take(p.dx_split.parts == 1 ? 0 : p.dx_split.parts * rows * pad4(K) * int64_t(sizeof(float)));
  p.rows_sum = sum_rows(p.chunk, kept ? N : outer * N, num_sms);
  // Room for the sums of either way: db may be wanted without dW, whose product would have given them.
  const int64_t by_product = p.split.sums && !p.direct ? p.split.parts : 0, by_rows = (p.chunk + p.rows_sum - 1) / p.rows_sum;
  p.sums = take(want_dbias ? std::max(by_product, by_rows) * outer * pad8(N) * int64_t(sizeof(float)) : 0);
  return p;
}
// Whether kept pre-activations are read: a dense layer without an activation has dz = dy, whatever its caller kept.
bool reads_kept(bool given, bool gated, int activation) { return given && (gated || activation != kActNone); }
// The plan is a function of the sizes; the last few of a thread are kept, since making one takes longer than a launch.
const BackwardPlan& plan_backward(bool gated, bool slope, bool kept, bool want_dbias, int64_t rows, int K, int N, int num_sms) {
  struct Entry {
    int64_t rows = -1;
    int K, N, flags, num_sms;
    BackwardPlan plan;
  };
  thread_local Entry entries[16];
  const int flags = gated | slope << 1 | want_dbias << 2 | kept << 3;
  Entry& e = entries[(uint64_t(rows) * 31 + uint64_t(K) * 7 + uint64_t(N) * 3 + flags) % 16];
  if (e.rows != rows || e.K != K || e.N != N || e.flags != flags || e.num_sms != num_sms) {
    e.plan = make_plan(gated, slope, kept, want_dbias, rows, K, N, num_sms);
    e.rows = rows, e.K = K, e.N = N, e.flags = flags, e.num_sms = num_sms;
  }
  return e.plan;
}

}  // namespace
}  // namespace b200ta

extern "C" {

int b200ta_dense_few_rows(void) { return b200ta::kFewRows; }

int b200ta_dense(const void* x, int64_t xs, const void* w, int64_t ws, const void* bias, const void* residual, int64_t rs, void* y,
                 int64_t ys, void* saved, int64_t ss, int dtype, int activation, int gated, int64_t rows, int K, int N, void* stream) {
  using namespace b200ta;
  int rc = check_layer("dense", dtype, activation, rows, K, N);
  if (rc != B200TA_OK) return rc;
  B200TA_REQUIRE(x && w && y, "dense: NULL pointer");
  B200TA_REQUIRE(!gated || residual == nullptr, "dense: a gated layer has no residual");
  B200TA_REQUIRE(!gated || saved == nullptr || ss % 16 == 0, "dense: the pitch of a gated layer's saved values must be a multiple of 16");
  if (rows <= kFewRows) {
    DeviceState* st = nullptr;
    rc = get_device_state(&st);
    if (rc != B200TA_OK) return rc;
    const bool vec = K % 8 == 0 && rows_aligned(x, xs) && rows_aligned(w, ws), f16 = dtype == B200TA_DTYPE_F16;
    const FewParams p{x, w, bias, residual, y, saved, xs, ws, rs, ys, ss, int(rows), K, N, activation};
    // sixteen warps where blocks are few (three rows, 1536 -> 384: 9 us instead of 11), eight otherwise, of which more blocks fit
    const int blocks = (N + kFewColumns - 1) / kFewColumns, warps = blocks <= st->num_sms ? kFewWarps : kFewWarps / 2;
    return launch_kernel(st, kKernelDenseHelpers, f16 ? pick_few<__half>(int(rows), vec, gated) : pick_few<__nv_bfloat16>(int(rows), vec, gated),
                         dim3(unsigned(blocks)), warps * 32, 0, stream, p);
  }
  B200TA_REQUIRE(rows_aligned(x, xs) && rows_aligned(w, ws) && (!residual || rows_aligned(residual, rs)) &&
                     (!saved || rows_aligned(saved, ss)),
                 "dense: what is read must be 16-byte aligned with row strides that are multiples of 8 elements");
  Matmul m;
  m.form = gated ? kGated : kDense;
  m.f16 = dtype == B200TA_DTYPE_F16;
  m.a = {x, rows, K, xs};
  m.b = {w, N, K, ws, gated ? 2 : 1, int64_t(N) * ws};
  m.out = {y, rows, N, ys};
  if (residual) m.aux = {residual, rows, N, rs};
  if (saved) m.saved = {saved, rows, N, ss, gated ? 2 : 1, ss / 2};
  m.bias = bias, m.activation = activation, m.what = gated ? "gated dense" : "dense";
  return run_matmul(m, stream);
}

int b200ta_dense_keeps(int activation, int gated, int K) {
  // Kept values are written and read at 4 bytes each, computed ones cost 2 K operations each on the tensor cores: a training step
  // of a gated layer takes 399 us either way for 8192 rows, 1024 -> 4096, and 361 us kept, 406 us computed again for 4096 rows,
  // 2048 -> 4096.  (In 16 bits keeping would pay from 512 inputs on, but its rounding adds a third to the gradients' error.)
  return (gated || activation != b200ta::kActNone) && K >= 1536;
}

size_t b200ta_dense_backward_workspace_bytes(int activation, int gated, int kept, int want_dbias, int64_t rows, int K, int N) {
  using namespace b200ta;
  DeviceState* st = nullptr;
  if (rows <= 0 || K <= 0 || N <= 0 || get_device_state(&st) != B200TA_OK) return 0;
  return size_t(plan_backward(gated, activation != kActNone, reads_kept(kept != 0, gated != 0, activation), want_dbias != 0, rows, K, N,
                              st->num_sms)
                    .bytes);
}

int b200ta_dense_backward(const void* dy, int64_t dys, const void* x, int64_t xs, const void* w, int64_t ws, const void* bias,
                          const void* saved, int64_t ss, void* dx, int64_t dxs, void* dw, void* dbias, void* workspace,
                          size_t workspace_bytes, int dtype, int activation, int gated, int64_t rows, int K, int N, void* stream) {
  using namespace b200ta;
  int rc = check_layer("dense_backward", dtype, activation, rows, K, N);
  if (rc != B200TA_OK) return rc;
  B200TA_REQUIRE(dy && x && w, "dense_backward: NULL pointer");
  B200TA_REQUIRE(rows_aligned(dy, dys) && rows_aligned(x, xs) && rows_aligned(w, ws) &&
                     (!saved || (rows_aligned(saved, ss) && (!gated || ss % 16 == 0))),
                 "dense_backward: what is read must be 16-byte aligned with row strides that are multiples of 8 elements");
  DeviceState* st = nullptr;
  rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  const bool kept = reads_kept(saved != nullptr, gated != 0, activation);
  const BackwardPlan& plan = plan_backward(gated, activation != kActNone, kept, dbias != nullptr, rows, K, N, st->num_sms);
  B200TA_REQUIRE(plan.bytes == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0 &&
                                     workspace_bytes >= size_t(plan.bytes)),
                 "dense_backward: the workspace must be 256-byte aligned and of %lld bytes", (long long)plan.bytes);
  const bool f16 = dtype == B200TA_DTYPE_F16, own_dz = plan.dz_pitch != 0;
  const int64_t outer = gated ? 2 : 1;
  char* ws_base = static_cast<char*>(workspace);
  float* parts = reinterpret_cast<float*>(ws_base + plan.parts);
  float* sums = reinterpret_cast<float*>(ws_base + plan.sums);
  const int64_t sum_pitch = own_dz ? plan.dz_pitch : pad8(N);  // columns of dz that are summed, padding included
  const int sum_columns = int(own_dz ? plan.dz_pitch : N);
  const bool direct = plan.direct, product_sums = plan.split.sums && dw != nullptr && dbias != nullptr;

  auto join_of = [&](bool wanted, const float* part, int64_t count, int64_t stride, int64_t pitch, int64_t n_rows, int columns, void* out) {
    const bool four = columns % 4 == 0 && pitch % 4 == 0 && stride % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 7u) == 0;
    const int slices = n_rows * columns < 32768 && count > 8 ? 8 : four ? 0 : 1;
    const int64_t need = (slices == 0 ? n_rows * columns / 4 + 255 : n_rows * columns * slices + 255) / 256, most = int64_t(st->num_sms) * 16;
    return JoinParams{part, out, stride, pitch, n_rows, int(count), columns, slices, wanted ? int(std::min(need, most)) : 0};
  };
  auto join = [&](const JoinParams& a, const JoinParams& b, const JoinParams& c) {
    return launch_kernel(st, kKernelDenseHelpers, f16 ? join_kernel<__half> : join_kernel<__nv_bfloat16>,
                         dim3(unsigned(a.blocks + b.blocks + c.blocks)), 256, 0, stream, a, b, c);
  };
  const bool narrow = narrow_pays(own_dz, kept, gated != 0, rows, K, N, dx, dxs, st->num_sms);
  const bool dx_parts = dx != nullptr && !narrow && plan.dx_split.parts > 1 && dxs == K;  // (a join writes dense rows)

  for (int64_t r0 = 0; r0 < rows; r0 += plan.chunk) {
    const int64_t n = rows - r0 < plan.chunk ? rows - r0 : plan.chunk;
    const char* dy_c = static_cast<const char*>(dy) + r0 * dys * 2;
    const char* x_c = static_cast<const char*>(x) + r0 * xs * 2;
    const void* dz = dy_c;
    int64_t zs = dys;
    if (own_dz) {
      void* dst = ws_base + plan.dz;
      dz = dst, zs = plan.dz_pitch;
      if (narrow) {
        Narrow m;
        m.f16 = f16, m.gated = gated != 0;
        m.x = {x_c, n, K, xs};
        m.dy = {dy_c, n, N, dys};
        m.w = {w, N, K, ws, outer, int64_t(N) * ws};
        m.dx = {static_cast<char*>(dx) + r0 * dxs * 2, n, K, dxs};
        if (dw != nullptr || dbias != nullptr) m.dz = {dst, n, N, zs, outer, zs / 2};
        m.bias = bias, m.activation = activation, m.what = "dense_backward dx";
        rc = run_narrow(m, stream);
      } else if (kept) {
        const SlopeParams p{dy_c, static_cast<const float*>(saved) + r0 * ss, dst, dbias != nullptr && !product_sums ? sums : nullptr, dys, ss, zs, n,
                            sum_pitch, N, plan.rows_sum, r0 > 0};
        const dim3 grid{unsigned((N + 255) / 256), unsigned((n + plan.rows_sum - 1) / plan.rows_sum)};
        void (*kernel)(SlopeParams);
        if (f16) kernel = gated ? pick_slope<__half, true>(activation) : pick_slope<__half, false>(activation);
        else kernel = gated ? pick_slope<__nv_bfloat16, true>(activation) : pick_slope<__nv_bfloat16, false>(activation);
        rc = launch_kernel(st, kKernelDenseHelpers, kernel, grid, 256, 0, stream, p);
      } else {
        Matmul m;
        m.form = gated ? kGatedGrad : kDenseGrad, m.f16 = f16;
        m.a = {x_c, n, K, xs};
        m.b = {w, N, K, ws, outer, int64_t(N) * ws};
        m.out = {dst, n, N, zs, outer, zs / 2};
        m.aux = {dy_c, n, N, dys};
        m.bias = bias, m.activation = activation, m.what = "dense_backward dz";
        rc = run_matmul(m, stream);
      }
      if (rc != B200TA_OK) return rc;
    }
    if (dx != nullptr && !narrow) {
      Matmul m;
      m.form = dx_parts ? kPartial : kPlain, m.b_mn = true, m.f16 = f16;
      m.a = {dz, n, N, zs, outer, zs / 2};
      m.b = {w, N, K, ws, outer, int64_t(N) * ws};
      if (dx_parts) {
        m.out = {ws_base + plan.dx_parts, n, K, pad4(K), plan.dx_split.parts, n * pad4(K)};
        m.kblocks_split = plan.dx_split.kblocks;
      } else {
        m.out = {static_cast<char*>(dx) + r0 * dxs * 2, n, K, dxs};
      }
      if (dw != nullptr) m.beside = kBesideFirst;
      m.what = "dense_backward dx";
      if ((rc = run_matmul(m, stream)) != B200TA_OK) return rc;
    }
    if (dw != nullptr) {
      Matmul m;
      m.form = direct ? kPlain : kPartial, m.a_mn = m.b_mn = true, m.f16 = f16;
      m.a = {dz, n, N, zs, outer, zs / 2};
      m.b = {x_c, n, K, xs};
      if (direct) {
        m.out = {dw, N, K, K, outer, int64_t(N) * K};
      } else {
        m.out = {parts, N, K, pad4(K), plan.split.parts * outer, N * pad4(K)};
        m.kblocks_split = plan.split.kblocks;
        m.accumulate = r0 > 0;  // each part is added to by one block at a time, the chunks in their order
      }
      if (dx != nullptr && !narrow) m.beside = kBesideSecond;
      if (product_sums) m.sums = direct ? dbias : sums;
      m.what = "dense_backward dW";
      if ((rc = run_matmul(m, stream)) != B200TA_OK) return rc;
    }
    if (dbias != nullptr && !product_sums && !kept) {
      const dim3 grid{unsigned((sum_columns + 255) / 256), unsigned((n + plan.rows_sum - 1) / plan.rows_sum)};
      if (f16)
        rc = launch_kernel(st, kKernelDenseHelpers, row_sum_kernel<__half>, grid, 256, 0, stream, static_cast<const __half*>(dz), zs, n,
                           sum_columns, sum_pitch, plan.rows_sum, int(r0 > 0), sums);
      else
        rc = launch_kernel(st, kKernelDenseHelpers, row_sum_kernel<__nv_bfloat16>, grid, 256, 0, stream,
                           static_cast<const __nv_bfloat16*>(dz), zs, n, sum_columns, sum_pitch, plan.rows_sum, int(r0 > 0), sums);
      if (rc != B200TA_OK) return rc;
    }
  }
  const bool parts_left = dw != nullptr && !direct, sums_left = dbias != nullptr && !(product_sums && direct);
  if (!parts_left && !sums_left && !dx_parts) return B200TA_OK;
  const int64_t chunk = plan.chunk < rows ? plan.chunk : rows;
  const JoinParams a = join_of(parts_left, parts, plan.split.parts, outer * N * pad4(K), pad4(K), outer * N, K, dw);
  const JoinParams b = product_sums ? join_of(sums_left, sums, plan.split.parts, outer * N, N, outer, N, dbias)
                                    : join_of(sums_left, sums, (chunk + plan.rows_sum - 1) / plan.rows_sum, sum_pitch, sum_pitch / outer, outer, N, dbias);
  const JoinParams c = join_of(dx_parts, reinterpret_cast<const float*>(ws_base + plan.dx_parts), plan.dx_split.parts, rows * pad4(K), pad4(K), rows, K, dx);
  return join(a, b, c);
}

int b200ta_copy_rows(const b200ta_copy* jobs, int count, void* stream) {
  using namespace b200ta;
  B200TA_REQUIRE(jobs != nullptr && count > 0 && count <= B200TA_COPIES, "copy_rows: 1 to %d copies", B200TA_COPIES);
  CopyParams p{};
  p.jobs = count;
  for (int i = 0; i < count; ++i) {
    const b200ta_copy& job = p.job[i] = jobs[i];
    B200TA_REQUIRE(job.src && job.dst, "copy_rows: NULL pointer");
    B200TA_REQUIRE(job.rows > 0 && job.columns > 0, "copy_rows: rows=%lld, columns=%d", (long long)job.rows, job.columns);
    B200TA_REQUIRE(rows_aligned(job.dst, job.dst_row_stride) && job.dst_row_stride >= pad8(job.columns),
                   "copy_rows: dst must be 16-byte aligned with rows of at least %lld elements, a multiple of 8",
                   (long long)pad8(job.columns));
    p.end[i] = (i == 0 ? 0 : p.end[i - 1]) + job.rows * ((job.columns + 7) / 8);
  }
  DeviceState* st = nullptr;
  const int rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  const int64_t need = (p.end[count - 1] + 255) / 256, most = int64_t(st->num_sms) * 16;
  return launch_kernel(st, kKernelDenseHelpers, copy_rows_kernel, dim3(unsigned(need < most ? need : most)), 256, 0, stream, p);
}

}  // extern "C"

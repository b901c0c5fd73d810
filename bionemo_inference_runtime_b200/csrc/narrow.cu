// Launch of the narrow layers' backward kernel; see narrow.cuh.
#include <algorithm>

#include "narrow.cuh"

namespace b200ta {

namespace {
int map_of(CUtensorMap* map, const Plane& t, int bytes, uint32_t columns, uint32_t rows, uint32_t outer, SwizzleMode swz, const char* what) {
  const uint64_t dims[3] = {uint64_t(t.columns), uint64_t(t.rows), uint64_t(t.outer)};
  const uint64_t strides[2] = {uint64_t(t.pitch) * bytes, uint64_t(t.outer > 1 ? t.outer_stride : t.pitch) * bytes};
  const uint32_t box[3] = {columns, rows, outer};
  return encode_tensor_map(map, t.base, bytes, 3, dims, strides, box, swz, what);
}
}  // namespace

int run_narrow(const Narrow& n, void* stream) {
  DeviceState* st = nullptr;
  int rc = get_device_state(&st);
  if (rc != B200TA_OK) return rc;
  B200TA_REQUIRE(n.x.columns <= 128, "%s: at most 128 inputs", n.what);
  B200TA_REQUIRE(n.x.rows < (int64_t(1) << 31) - 512 && n.w.rows < (int64_t(1) << 30), "%s: a size is past its limit", n.what);
  NarrowParams p{};
  p.rows = int(n.x.rows), p.K = int(n.x.columns), p.N = int(n.w.rows);
  p.kblocks = (p.K + 63) / 64, p.chunks = (p.N + 63) / 64;
  p.store_dz = n.dz.base != nullptr;
  p.bias = n.bias, p.activation = n.activation, p.status = st->status_dev;
  CUtensorMap x, w, dy, dx, dz{};
  if ((rc = map_of(&x, n.x, 2, 64, 128, 1, SWZ_128, n.what)) != B200TA_OK ||
      (rc = map_of(&w, n.w, 2, 64, 32, n.gated ? 2 : 1, SWZ_128, n.what)) != B200TA_OK ||
      (rc = map_of(&dy, n.dy, 2, 16, 32, 1, SWZ_32, n.what)) != B200TA_OK || (rc = map_of(&dx, n.dx, 2, 32, 32, 1, SWZ_64, n.what)) != B200TA_OK ||
      (p.store_dz && (rc = map_of(&dz, n.dz, 2, 16, 32, 1, SWZ_32, n.what)) != B200TA_OK))
    return rc;
  const int grid = std::min((p.rows + 255) / 256, st->num_sms);
  auto* kernel = n.gated ? (n.f16 ? narrow::narrow_kernel<__half, kGatedGrad> : narrow::narrow_kernel<__nv_bfloat16, kGatedGrad>)
                         : (n.f16 ? narrow::narrow_kernel<__half, kDenseGrad> : narrow::narrow_kernel<__nv_bfloat16, kDenseGrad>);
  return launch_kernel(st, KernelId(kKernelNarrow + n.gated * 2 + n.f16), kernel, dim3(unsigned(grid)), narrow::kThreads, narrow::kSmDynamic,
                       stream, x, w, dy, dx, dz, p);
}

}  // namespace b200ta

// Low-rank values of many rows: x and the adapters' rows, both K-major.
#include "matmul.cuh"

namespace b200ta {
int launch_matmul_low(DeviceState* st, const Matmul& m, const MatmulMaps& maps, const MatmulParams& p, const MatmulAdapters& x, int grid, void* stream) {
  const KernelId kernel = KernelId(kKernelMatmulLow + (m.f16 ? 1 : 0));
  auto* function = m.f16 ? matmul::matmul_kernel<__half, kLow, false, false, false, MatmulAdapters>
                         : matmul::matmul_kernel<__nv_bfloat16, kLow, false, false, false, MatmulAdapters>;
  return launch_kernel(st, kernel, function, dim3(unsigned(grid)), matmul::kThreads, matmul::kSmDynamic, stream, maps.a, maps.b, maps.out, maps.aux,
                       maps.saved, p, x);
}
}  // namespace b200ta

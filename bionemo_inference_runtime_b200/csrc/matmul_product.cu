// The two products behind dz: dx = dz W (W with its rows along k) and dW = dz^T x (both with their rows along k), at
// once or in parts of k.
#include "matmul.cuh"

namespace b200ta {
int launch_matmul_product(DeviceState* st, const Matmul& m, const MatmulMaps& maps, const MatmulParams& p, int grid, void* stream) {
  if (m.form == kPlain && !m.a_mn) return matmul::launch<kPlain, false, true>(st, 4, m, maps, p, grid, stream);
  if (m.form == kPlain) return matmul::launch<kPlain, true, true>(st, 5, m, maps, p, grid, stream);
  if (m.form == kPartial && !m.a_mn) return matmul::launch<kPartial, false, true>(st, 7, m, maps, p, grid, stream);
  if (m.form == kPartial) return matmul::launch<kPartial, true, true>(st, 6, m, maps, p, grid, stream);
  return fail(B200TA_ERR_UNSUPPORTED, "%s: not a product of gradients", m.what);
}
}  // namespace b200ta

// Forward products of the trainable dense layers: y from x and W, both K-major.
#include "matmul.cuh"

namespace b200ta {
int launch_matmul_forward(DeviceState* st, const Matmul& m, const MatmulMaps& maps, const MatmulParams& p, int grid, void* stream) {
  if (m.form == kDense) return matmul::launch<kDense, false, false>(st, 0, m, maps, p, grid, stream);
  if (m.form == kGated) return matmul::launch<kGated, false, false>(st, 1, m, maps, p, grid, stream);
  return fail(B200TA_ERR_UNSUPPORTED, "%s: not a forward product", m.what);
}
}  // namespace b200ta

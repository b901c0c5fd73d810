// dz of the trainable dense layers from dy, with the pre-activations computed again from x and W.
#include "matmul.cuh"

namespace b200ta {
int launch_matmul_grad(DeviceState* st, const Matmul& m, const MatmulMaps& maps, const MatmulParams& p, const NoAdapters& x, int grid, void* stream) {
  if (m.form == kDenseGrad) return matmul::launch<kDenseGrad, false, false>(st, 2, m, maps, p, x, grid, stream);
  if (m.form == kGatedGrad) return matmul::launch<kGatedGrad, false, false>(st, 3, m, maps, p, x, grid, stream);
  return fail(B200TA_ERR_UNSUPPORTED, "%s: not a gradient of an activation", m.what);
}
}  // namespace b200ta

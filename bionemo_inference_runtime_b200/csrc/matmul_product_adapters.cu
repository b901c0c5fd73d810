// dx = dz W + dt D of the dense layers with adapters, at once or in parts of k.
#include "matmul.cuh"

namespace b200ta {
int launch_matmul_product(DeviceState* st, const Matmul& m, const MatmulMaps& maps, const MatmulParams& p, const MatmulAdapters& x, int grid, void* stream) {
  if (m.form == kPlain && !m.a_mn) return matmul::launch<kPlain, false, true>(st, 4, m, maps, p, x, grid, stream);
  if (m.form == kPartial && !m.a_mn) return matmul::launch<kPartial, false, true>(st, 7, m, maps, p, x, grid, stream);
  return fail(B200TA_ERR_UNSUPPORTED, "%s: not a product that adapters join", m.what);
}
}  // namespace b200ta

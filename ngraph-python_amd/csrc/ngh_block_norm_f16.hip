// The block norm kernels for f16 rows (a translation unit for each storage type: they build side by side).
#include "ngh_block_norm.h"

namespace ngh {
int launch_norm_f16(const NormShape& s, const NormArgs& a, NormPass pass, bool layer, unsigned grid, hipStream_t stream) {
    return launch_norm<f16_t>(s, a, pass, layer, grid, stream);
}
}  // namespace ngh

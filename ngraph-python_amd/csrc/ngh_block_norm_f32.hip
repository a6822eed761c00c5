// The block norm kernels for f32 rows (a translation unit for each storage type: they build side by side).
#include "ngh_block_norm.h"

namespace ngh {
int launch_norm_f32(const NormShape& s, const NormArgs& a, bool backward, bool bias, unsigned grid, hipStream_t stream) {
    return s.ragged ? launch_norm<float, true>(s, a, backward, bias, grid, stream) : launch_norm<float, false>(s, a, backward, bias, grid, stream);
}
}  // namespace ngh

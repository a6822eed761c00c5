// The block norm kernels for bf16 rows (a translation unit for each storage type: they build side by side).
#include "ngh_block_norm.h"

namespace ngh {
int launch_norm_bf16(const NormShape& s, const NormArgs& a, bool backward, bool bias, unsigned grid, hipStream_t stream) {
    return s.ragged ? launch_norm<bf16_t, true>(s, a, backward, bias, grid, stream) : launch_norm<bf16_t, false>(s, a, backward, bias, grid, stream);
}
}  // namespace ngh

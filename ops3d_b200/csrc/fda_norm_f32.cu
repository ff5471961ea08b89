// Layer norm kernels of fda_norm.cuh for f32 rows.
#include "fda_norm.cuh"

namespace fda_norm {
int norm_f32(bool backward, const NormArgs &p, const NormShape &s, int residual_dtype, cudaStream_t st) {
    return run_norm<float>(backward, p, s, residual_dtype, st);
}
}  // namespace fda_norm

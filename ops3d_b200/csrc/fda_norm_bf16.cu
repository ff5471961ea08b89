// Layer norm kernels of fda_norm.cuh for bf16 rows.
#include "fda_norm.cuh"

namespace fda_norm {
int norm_bf16(bool backward, const NormArgs &p, const NormShape &s, int residual_dtype, cudaStream_t st) {
    return run_norm<__nv_bfloat16>(backward, p, s, residual_dtype, st);
}
}  // namespace fda_norm

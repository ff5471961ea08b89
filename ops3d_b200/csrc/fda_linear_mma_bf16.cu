// The tensor-core kernels of the linear operators for bf16.
#include "fda_linear_mma_kernels.cuh"

namespace fda_linear {

int mma_rows_bf16(int mode, const MmaRows &p, cudaStream_t st) { return rows_of<__nv_bfloat16>(mode, p, st); }
int mma_weight_grad_bf16(const MmaWeightGrad &p, cudaStream_t st) { return weight_grad_of<__nv_bfloat16>(p, st); }
int mma_timeouts_bf16() { return timeouts(); }

}  // namespace fda_linear

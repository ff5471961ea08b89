// The tensor-core kernels of the linear operators for f16.
#include "fda_linear_mma_kernels.cuh"

namespace fda_linear {

int mma_pre_grad_unit(const MmaRows &p) { return pre_grad_unit(p); }
int mma_rows_f16(int mode, const MmaRows &p, cudaStream_t st) { return rows_of<__half>(mode, p, st); }
int mma_weight_grad_f16(const MmaWeightGrad &p, cudaStream_t st) { return weight_grad_of<__half>(p, st); }
int mma_timeouts_f16() { return timeouts(); }

}  // namespace fda_linear

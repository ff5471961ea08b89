// Layer norm: the sums of the parameters' gradients over blocks, rows too wide for registers, and the C entry points.
#include "fda_norm.cuh"

#include <algorithm>

namespace fda_norm {
namespace {

// grad_weight and grad_bias from the blocks' partial sums [count][2][width], added in a fixed order: 32 columns a block, its warps
// (as many as there are sums for, up to 32) taking turns over them.
__global__ void __launch_bounds__(1024) norm_sum_kernel(const float *partial, int count, int width, void *grad_weight, void *grad_bias, int dtype) {
    wait_for_previous_kernel();
    __shared__ float sums[32][32];
    const int lane = threadIdx.x % 32, part = threadIdx.x / 32, parts = blockDim.x / 32;
    const long long column = (long long)blockIdx.x * 32 + lane;
    // short chains of additions: eight sums side by side, then pairs of them
    float s[8] = {};
    if (column < 2ll * width) {
        for (int i = part; i < count; i += 8 * parts)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + k * parts < count) s[k] += partial[(size_t)(i + k * parts) * 2 * width + column];
    }
    sums[part][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    for (int half = 16; half > 0; half /= 2) {
        __syncthreads();
        if (part < half && part + half < parts) sums[part][lane] += sums[part + half][lane];
    }
    if (part != 0 || column >= 2ll * width) return;
    void *out = column < width ? grad_weight : grad_bias;
    if (out) store_from_f32(out, dtype, column < width ? column : column - width, sums[0][lane]);
}

// ---- rows that no block keeps in registers (beyond 8192 elements): a pass over the row for each step, from L2 after the first -----------------------------------------------
struct WideArgs {
    NormArgs n;
    int dtype, residual_dtype;
    float *statistics;  // [rows][2]: mean, 1 / deviation
    int rows_per_part;
};

__device__ __forceinline__ float wide_input(const WideArgs &p, size_t at) {
    const float v = load_as_f32(p.n.x, p.dtype, at);
    return p.n.residual ? v + load_as_f32(p.n.residual, p.residual_dtype, at) : v;
}
__device__ __forceinline__ float wide_weight(const WideArgs &p, int c) { return p.n.weight ? load_as_f32(p.n.weight, p.n.param_dtype, c) : 1.f; }

constexpr int kWideThreads = 512;
template <bool kBackward>
__global__ void __launch_bounds__(kWideThreads) norm_wide_kernel(const WideArgs p) {
    wait_for_previous_kernel();
    Team<0> team = block_team();
    const int width = p.n.width;
    const float inverse = 1.f / (float)width;
    for (long long row = blockIdx.x; row < p.n.rows; row += gridDim.x) {
        const size_t at = (size_t)row * width;
        float sum[1] = {0.f};
        for (int c = threadIdx.x; c < width; c += kWideThreads) sum[0] += wide_input(p, at + c);
        team.sum(sum);
        const float mean = sum[0] * inverse;
        float sums[3] = {0.f, 0.f, 0.f};
        for (int c = threadIdx.x; c < width; c += kWideThreads) {
            const float d = wide_input(p, at + c) - mean;
            sums[0] += d * d;
            if (kBackward) {
                const float g = load_as_f32(p.n.grad_y, p.dtype, at + c) * wide_weight(p, c);
                sums[1] += g * d;
                sums[2] += g;
            }
        }
        team.sum(sums);
        const float q = __frsqrt_rn(sums[0] * inverse + p.n.eps);
        if (kBackward && threadIdx.x == 0) {
            p.statistics[2 * row] = mean;
            p.statistics[2 * row + 1] = q;
        }
        const float along = q * q * sums[1] * inverse, level = sums[2] * inverse;
        for (int c = threadIdx.x; c < width; c += kWideThreads) {
            const float s = wide_input(p, at + c), d = s - mean;
            if (!kBackward) {
                if (p.n.sum) store_from_f32(p.n.sum, p.residual_dtype, at + c, s);
                const float bias = p.n.bias ? load_as_f32(p.n.bias, p.n.param_dtype, c) : 0.f;
                store_from_f32(p.n.y, p.dtype, at + c, d * q * wide_weight(p, c) + bias);
            } else {
                float ds = q * (load_as_f32(p.n.grad_y, p.dtype, at + c) * wide_weight(p, c) - level - d * along);
                if (p.n.grad_sum) ds += load_as_f32(p.n.grad_sum, p.residual_dtype, at + c);
                if (p.n.grad_x) store_from_f32(p.n.grad_x, p.dtype, at + c, ds);
                if (p.n.grad_residual) store_from_f32(p.n.grad_residual, p.residual_dtype, at + c, ds);
            }
        }
    }
}

// Partial sums of dweight and dbias over rows_per_part rows, a thread a column.
__global__ void __launch_bounds__(256) norm_wide_columns_kernel(const WideArgs p) {
    wait_for_previous_kernel();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.n.width) return;
    const long long first = (long long)blockIdx.y * p.rows_per_part, last = min(first + p.rows_per_part, p.n.rows);
    float weight = 0.f, bias = 0.f;
    for (long long row = first; row < last; ++row) {
        const size_t at = (size_t)row * p.n.width + c;
        const float dy = load_as_f32(p.n.grad_y, p.dtype, at);
        weight += dy * ((wide_input(p, at) - p.statistics[2 * row]) * p.statistics[2 * row + 1]);
        bias += dy;
    }
    float *out = p.n.partial + (size_t)blockIdx.y * 2 * p.n.width;
    out[c] = weight;
    out[p.n.width + c] = bias;
}

constexpr int kWideParts = 64;

struct Workspace {
    size_t partial, statistics, total;
};
Workspace workspace_of(long long rows, int width, int dtype) {
    const bool wide = is_wide(width, dtype);
    const size_t parts = wide ? (size_t)std::min<long long>(rows, kWideParts) : norm_backward_blocks(norm_shape(width, dtype, true), rows, dtype);
    Workspace w;
    w.partial = fda_linear::round256(parts * 2 * width * sizeof(float));
    w.statistics = wide ? fda_linear::round256((size_t)rows * 2 * sizeof(float)) : 0;
    w.total = w.partial + w.statistics;
    return w;
}

int run_fast(bool backward, const NormArgs &p, int dtype, int residual_dtype, cudaStream_t st) {
    const NormShape s = norm_shape(p.width, dtype, backward);
    if (dtype == FDA_DTYPE_F32) return norm_f32(backward, p, s, residual_dtype, st);
    if (dtype == FDA_DTYPE_F16) return norm_f16(backward, p, s, residual_dtype, st);
    return norm_bf16(backward, p, s, residual_dtype, st);
}

int check(long long rows, int width, int dtype, int param_dtype, int residual_dtype, bool residual) {
    if (!known_dtype(dtype)) return FDA_ERR_BAD_DTYPE;
    if (param_dtype != dtype && param_dtype != FDA_DTYPE_F32) return FDA_ERR_BAD_DTYPE;
    if (residual && residual_dtype != dtype && residual_dtype != FDA_DTYPE_F32) return FDA_ERR_BAD_DTYPE;
    if (rows < 0 || rows > INT32_MAX || width < 1 || width >= 1 << 26) return FDA_ERR_BAD_SHAPE;
    return FDA_OK;
}

}  // namespace
}  // namespace fda_norm

using namespace fda_norm;

extern "C" {

int fda_layer_norm_forward(const void *x, const void *weight, const void *bias, const void *residual, void *y, void *sum, long long rows,
                           int features, float eps, int dtype, int param_dtype, int residual_dtype, void *stream) {
    if (const int rc = check(rows, features, dtype, param_dtype, residual_dtype, residual)) return rc;
    if (sum && !residual) return FDA_ERR_NULL_POINTER;
    if (rows == 0) return FDA_OK;
    if (!x || !y) return FDA_ERR_NULL_POINTER;
    if (misaligned16(x) || misaligned16(residual) || misaligned16(y) || misaligned16(sum)) return FDA_ERR_MISALIGNED;
    NormArgs p{};
    p.x = x; p.residual = residual; p.weight = weight; p.bias = bias; p.y = y; p.sum = sum;
    p.rows = rows; p.width = features; p.param_dtype = param_dtype; p.eps = eps;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (is_wide(features, dtype)) {
        WideArgs w{p, dtype, residual_dtype, nullptr, 0};
        return launched(launch_early(norm_wide_kernel<false>, (unsigned)std::min<long long>(rows, 4 * kSms), kWideThreads, 0, st, 1, w));
    }
    return run_fast(false, p, dtype, residual_dtype, st);
}

size_t fda_layer_norm_backward_workspace_bytes(long long rows, int features, int dtype) {
    if (check(rows, features, dtype, dtype, dtype, false) != FDA_OK || rows == 0) return 0;
    return workspace_of(rows, features, dtype).total;
}

int fda_layer_norm_backward(const void *x, const void *weight, const void *residual, const void *grad_y, const void *grad_sum, void *grad_x,
                            void *grad_residual, void *grad_weight, void *grad_bias, void *workspace, size_t workspace_bytes, long long rows,
                            int features, float eps, int dtype, int param_dtype, int residual_dtype, void *stream) {
    if (const int rc = check(rows, features, dtype, param_dtype, residual_dtype, residual)) return rc;
    if ((grad_sum || grad_residual) && !residual) return FDA_ERR_NULL_POINTER;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {  // no row: the parameters' gradients are zero
        const size_t bytes = (size_t)features * type_size(param_dtype);
        cudaError_t e = cudaSuccess;
        if (grad_weight) e = cudaMemsetAsync(grad_weight, 0, bytes, st);
        if (grad_bias && e == cudaSuccess) e = cudaMemsetAsync(grad_bias, 0, bytes, st);
        return launched(e);
    }
    if (!x || !grad_y) return FDA_ERR_NULL_POINTER;
    const bool parameters = grad_weight || grad_bias, wide = is_wide(features, dtype);
    const Workspace need = workspace_of(rows, features, dtype);
    if (parameters || wide) {
        if (!workspace || workspace_bytes < need.total) return FDA_ERR_WORKSPACE;
        if ((uintptr_t)workspace % 256) return FDA_ERR_MISALIGNED;
    }
    if (misaligned16(x) || misaligned16(residual) || misaligned16(grad_y) || misaligned16(grad_sum) || misaligned16(grad_x) ||
        misaligned16(grad_residual))
        return FDA_ERR_MISALIGNED;
    NormArgs p{};
    p.x = x; p.residual = residual; p.weight = weight; p.grad_y = grad_y; p.grad_sum = grad_sum;
    p.grad_x = grad_x; p.grad_residual = grad_residual;
    p.partial = parameters ? static_cast<float *>(workspace) : nullptr;
    p.rows = rows; p.width = features; p.param_dtype = param_dtype; p.eps = eps;
    int parts;
    if (wide) {
        WideArgs w{p, dtype, residual_dtype, reinterpret_cast<float *>(static_cast<char *>(workspace) + need.partial), 0};
        parts = (int)std::min<long long>(rows, kWideParts);
        w.rows_per_part = (int)ceil_div(rows, parts);
        parts = (int)ceil_div(rows, w.rows_per_part);
        if (const int rc = launched(launch_early(norm_wide_kernel<true>, (unsigned)std::min<long long>(rows, 4 * kSms), kWideThreads, 0, st, 1, w)))
            return rc;
        if (!parameters) return FDA_OK;
        norm_wide_columns_kernel<<<dim3((unsigned)ceil_div(features, 256), parts), 256, 0, st>>>(w);
        if (const int rc = launched(cudaGetLastError())) return rc;
    } else {
        parts = (int)norm_backward_blocks(norm_shape(features, dtype, true), rows, dtype);
        if (const int rc = run_fast(true, p, dtype, residual_dtype, st)) return rc;
        if (!parameters) return FDA_OK;
    }
    const unsigned threads = 32 * (unsigned)std::min<long long>(32, ceil_div(parts, 4));
    return launched(launch_early(norm_sum_kernel, (unsigned)ceil_div(2ll * features, 32), threads, 0, st, 1, static_cast<const float *>(p.partial),
                                 parts, features, grad_weight, grad_bias, param_dtype));
}

}  // extern "C"

// Linear layers with bias, activation and residual in the product's epilogue, for one weight or one weight per ragged group of
// rows: C ABI, and the fp32 kernels.  16-bit products are in fda_linear_mma_kernels.cuh.
#include <algorithm>

#include "fda_config.h"
#include "fda_linear.cuh"

namespace {

using namespace fda_linear;

// ---------------------------------------------------------------------------------------------------------------------------
// Products on the fp32 pipes
// ---------------------------------------------------------------------------------------------------------------------------
// A block computes a 64 x 64 tile; its 256 threads own 4 x 4 sums each.  Operands pass through shared memory in slices of 16 along k,
// copied element by element (any size, any alignment; what does not exist arrives as zero) and three slices ahead: with one
// slice ahead, in registers, 3001 x 99 x 131 took 24 us, most of it waiting for memory slice by slice.
constexpr int kThreads = 256, kSlice = 16, kTile = 64, kOwn = 4, kAhead = 4, kPitch = kTile + 4;

struct Slices {
    float a[kAhead][kSlice][kPitch];
    float b[kAhead][kSlice][kPitch];
};

__device__ __forceinline__ void copy_element(float *dst, const float *src, bool exists) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(exists ? 4 : 0)
                 : "memory");
}

// Slice k0 .. k0 + 15 of A(i, k) = a[i * ai + k * ak], of which i < rows, k < depth exist; the stride that is 1 decides how
// threads cover it.
template <bool kContiguousK>
__device__ __forceinline__ void copy_slice(float (*dst)[kPitch], const float *a, long long ai, long long ak, int rows, int k0, int depth) {
#pragma unroll
    for (int j = 0; j < kTile * kSlice / kThreads; ++j) {
        const int i = kContiguousK ? (int)threadIdx.x / kSlice + j * (kThreads / kSlice) : (int)threadIdx.x % kTile;
        const int k = kContiguousK ? (int)threadIdx.x % kSlice : (int)threadIdx.x / kTile + j * (kThreads / kTile);
        const bool exists = i < rows && k0 + k < depth;
        copy_element(&dst[k][i], exists ? a + i * ai + (k0 + k) * ak : a, exists);
    }
}

// acc += A B over k in [0, depth); A is 64 x depth, B depth x 64.  A thread owns rows 4 ty .., columns 4 tx ..; with kSumA
// also sums = its rows of A added over k.  Every thread of the block takes part; the slices are free again at the end.
// Sums of 128 terms are made by themselves and then added: one chain over all of a long contraction is off by several times
// as much (a bias's gradient over 46567 rows by 1.5e-6 of its size).  Rows of A, which no product's rounding hides behind, are added
// slice by slice, 16 terms at a time, and the slices of a call by themselves.
constexpr int kChainSlices = 8;

template <bool kAK, bool kBK, bool kSumA>
__device__ __forceinline__ void tile_product(float (&acc)[kOwn][kOwn], float (&sums)[kOwn], Slices &s, const float *a, long long ai, long long ak,
                                             int rows, const float *b, long long bj, long long bk, int cols, int depth) {
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int slices = (depth + kSlice - 1) / kSlice;
    const auto copy = [&](int i) {
        if (i < slices) {
            copy_slice<kAK>(s.a[i % kAhead], a, ai, ak, rows, i * kSlice, depth);
            copy_slice<kBK>(s.b[i % kAhead], b, bj, bk, cols, i * kSlice, depth);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float part[kOwn][kOwn] = {}, slice_sums[kOwn] = {};
#pragma unroll
    for (int i = 0; i < kAhead - 1; ++i) copy(i);
    for (int i = 0; i < slices; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 2) : "memory");
        __syncthreads();  // slice i has arrived for every thread, and every thread is done with the one that is overwritten next
        copy(i + kAhead - 1);
        const float(*sa)[kPitch] = s.a[i % kAhead], (*sb)[kPitch] = s.b[i % kAhead];
        float slice_sum[kOwn] = {};
#pragma unroll
        for (int k = 0; k < kSlice; ++k) {
            const float4 qa = *reinterpret_cast<const float4 *>(&sa[k][kOwn * ty]), qb = *reinterpret_cast<const float4 *>(&sb[k][kOwn * tx]);
            const float ra[kOwn] = {qa.x, qa.y, qa.z, qa.w}, rb[kOwn] = {qb.x, qb.y, qb.z, qb.w};
#pragma unroll
            for (int r = 0; r < kOwn; ++r) {
                if (kSumA) slice_sum[r] += ra[r];
#pragma unroll
                for (int c = 0; c < kOwn; ++c) part[r][c] = fmaf(ra[r], rb[c], part[r][c]);
            }
        }
        if (kSumA)
#pragma unroll
            for (int r = 0; r < kOwn; ++r) slice_sums[r] += slice_sum[r];
        if (i % kChainSlices == kChainSlices - 1 || i + 1 == slices) {
#pragma unroll
            for (int r = 0; r < kOwn; ++r) {
#pragma unroll
                for (int c = 0; c < kOwn; ++c) {
                    acc[r][c] += part[r][c];
                    part[r][c] = 0.f;
                }
            }
        }
    }
    if (kSumA)
#pragma unroll
        for (int r = 0; r < kOwn; ++r) sums[r] += slice_sums[r];
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
}

template <typename T>
struct RowProduct {
    const T *a;      // x, or g for grad_x
    const T *w;
    const T *bias;   // forward and pre-gradient
    const T *extra;  // residual (forward), grad_output (pre-gradient)
    T *out;
    int depth, cols;  // contraction; columns of the result
    int in_features;  // row length of w
    int out_pitch;
    Groups g;
};

// kForward:  out = act(a W^T + bias) + extra    kPreGrad:  out = extra * act'(a W^T + bias)    kGradX:  out = a W
template <int kMode, int kAct>
__global__ void __launch_bounds__(kThreads) linear_rows_kernel(const RowProduct<float> p) {
    __shared__ RowTable table;
    __shared__ __align__(16) Slices slices;
    wait_for_previous_kernel();
    build_row_table(p.g, kTile, kMode != kPreGrad, table);
    __syncthreads();
    const int column_tiles = (p.cols + kTile - 1) / kTile;
    const long long tiles = (long long)table.unit_begin[p.g.groups + 2] * p.g.batch * column_tiles;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const RowUnit u = row_unit(p.g, table, kTile, (unsigned)(tile / column_tiles));
        const int col0 = (int)(tile % column_tiles) * kTile, cols = min(kTile, p.cols - col0);
        float acc[kOwn][kOwn] = {}, none[kOwn];
        if (u.group >= 0) {
            const float *w = p.w + (size_t)u.group * ((kMode == kGradX ? (size_t)p.depth : (size_t)p.cols) * p.in_features);
            const float *a = p.a + (size_t)u.row * p.depth;
            if (kMode == kGradX)
                tile_product<true, false, false>(acc, none, slices, a, p.depth, 1, u.count, w + col0, 1, p.in_features, cols, p.depth);
            else
                tile_product<true, true, false>(acc, none, slices, a, p.depth, 1, u.count, w + (size_t)col0 * p.in_features, p.in_features, 1,
                                                cols, p.depth);
        }
        float bias[kOwn] = {};
        if (kMode != kGradX && p.bias && u.group >= 0)
#pragma unroll
            for (int c = 0; c < kOwn; ++c)
                if (kOwn * tx + c < cols) bias[c] = p.bias[(size_t)u.group * p.cols + col0 + kOwn * tx + c];
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int r = kOwn * ty + i;
            if (r >= u.count) continue;
            float extra[kOwn] = {};
            if (kMode != kGradX && p.extra)
#pragma unroll
                for (int c = 0; c < kOwn; ++c)
                    if (kOwn * tx + c < cols) extra[c] = p.extra[(size_t)(u.row + r) * p.cols + col0 + kOwn * tx + c];
            float *out = p.out + (size_t)(u.row + r) * p.out_pitch + col0 + kOwn * tx;
#pragma unroll
            for (int c = 0; c < kOwn; ++c) {
                if (kOwn * tx + c >= cols) continue;
                float v = acc[i][c] + bias[c];
                if (kMode == kForward) v = (u.group >= 0 ? activate<kAct>(v) : v) + extra[c];
                else if (kMode == kPreGrad) v = activate_backward<kAct>(v, extra[c]);
                out[c] = v;
            }
        }
    }
}

// Few rows (one token, or a few per group): bound by latency and by reading the weight, which no tile of 128 rows helps.  A warp takes
// two outputs and up to eight rows, its lanes along the contraction, 16 bytes a load; lane 8 o + r finishes row r of output o.
// One token, 256 -> 1024: 5.3 us in the tile kernel, 2.9 here.
constexpr int kFewRows = 8, kFewOutputs = 2, kFewThreads = 128;

// 16 bytes of a row from element k on, or as many elements as exist.
template <typename T, bool kVector>
__device__ __forceinline__ void load_some(const T *row, int k, int depth, float (&v)[16 / sizeof(T)]) {
    constexpr int kCount = 16 / sizeof(T);
    if (kVector) {
        alignas(16) T raw[kCount];
        *reinterpret_cast<uint4 *>(raw) = __ldg(reinterpret_cast<const uint4 *>(row + k));
#pragma unroll
        for (int j = 0; j < kCount; ++j) v[j] = to_f32<T>(raw[j]);
    } else {
#pragma unroll
        for (int j = 0; j < kCount; ++j) v[j] = k + j < depth ? to_f32<T>(row[k + j]) : 0.f;
    }
}

// kForward and kPreGrad, whose results the backward of few rows keeps in fp32.
template <typename T, int kMode, bool kVector>
__global__ void __launch_bounds__(kFewThreads) linear_few_rows_kernel(const RowProduct<T> p, const int activation) {
    constexpr int kCount = 16 / sizeof(T);
    __shared__ RowTable table;
    wait_for_previous_kernel();
    build_row_table(p.g, kFewRows, kMode != kPreGrad, table);
    __syncthreads();
    const int lane = threadIdx.x % 32;
    const unsigned steps = (unsigned)((p.cols + kFewOutputs - 1) / kFewOutputs);
    const long long items = (long long)table.unit_begin[p.g.groups + 2] * p.g.batch * steps;
    const long long warps = (long long)gridDim.x * (kFewThreads / 32);
    for (long long item = (long long)blockIdx.x * (kFewThreads / 32) + threadIdx.x / 32; item < items; item += warps) {
        const RowUnit u = row_unit(p.g, table, kFewRows, (unsigned)(item / steps));
        const int col0 = (int)(item % steps) * kFewOutputs;
        float acc[kFewOutputs][kFewRows] = {};
        if (u.group >= 0) {
            const T *a = p.a + (size_t)u.row * p.depth;
            const T *w = p.w + ((size_t)u.group * p.cols + col0) * p.depth;
            const bool second = col0 + 1 < p.cols;
#pragma unroll 2
            for (int k = lane * kCount; k < p.depth; k += 32 * kCount) {
                float w0[kCount], w1[kCount];
                load_some<T, kVector>(w, k, p.depth, w0);
                load_some<T, kVector>(second ? w + p.depth : w, k, p.depth, w1);
#pragma unroll
                for (int r = 0; r < kFewRows; ++r)
                    if (r < u.count) {
                        float x[kCount];
                        load_some<T, kVector>(a + (size_t)r * p.depth, k, p.depth, x);
#pragma unroll
                        for (int j = 0; j < kCount; ++j) {
                            acc[0][r] = fmaf(x[j], w0[j], acc[0][r]);
                            acc[1][r] = fmaf(x[j], w1[j], acc[1][r]);
                        }
                    }
            }
        }
        float v = 0.f;
#pragma unroll
        for (int r = 0; r < kFewRows; ++r)
            if (r < u.count)
#pragma unroll
                for (int o = 0; o < kFewOutputs; ++o) {
                    float sum = acc[o][r];
#pragma unroll
                    for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                    if (lane == o * kFewRows + r) v = sum;
                }
        const int r = lane % kFewRows, c = col0 + lane / kFewRows;
        if (lane >= kFewOutputs * kFewRows || r >= u.count || c >= p.cols) continue;
        const size_t at = (size_t)(u.row + r) * p.cols + c;
        if (p.bias && u.group >= 0) v += to_f32<T>(p.bias[(size_t)u.group * p.cols + c]);
        if (kMode == kForward) {
            if (u.group >= 0) v = activate_any(activation, v);
            if (p.extra) v += to_f32<T>(p.extra[at]);
            p.out[at] = from_f32<T>(v);
        } else {
            reinterpret_cast<float *>(p.out)[at] = activate_backward_any(activation, v, to_f32<T>(p.extra[at]));
        }
    }
}

// The backward of few rows (64 in all), without a rounding between its products: g in fp32, or the output's gradient itself.
template <typename T, typename G>
struct FewGrad {
    const G *grad;  // [rows][out]
    const T *x, *w;
    T *grad_x, *grad_weight, *grad_bias;
    int in_features, out_features;
    Groups g;
};

// grad_x: 64 inputs of up to eight rows a block, two a lane; its warps share out the outputs and add their sums in order.
constexpr int kFewWarps = 8, kFewInputs = 64;

template <typename T, typename G>
__global__ void __launch_bounds__(32 * kFewWarps) linear_few_grad_x_kernel(const FewGrad<T, G> p) {
    __shared__ RowTable table;
    __shared__ float partial[kFewWarps][kFewRows][kFewInputs];
    wait_for_previous_kernel();
    build_row_table(p.g, kFewRows, true, table);
    __syncthreads();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const unsigned steps = (unsigned)((p.in_features + kFewInputs - 1) / kFewInputs);
    const long long items = (long long)table.unit_begin[p.g.groups + 2] * p.g.batch * steps;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const RowUnit u = row_unit(p.g, table, kFewRows, (unsigned)(item / steps));
        const int in0 = (int)(item % steps) * kFewInputs;
        const bool first = in0 + lane < p.in_features, second = in0 + 32 + lane < p.in_features;
        float acc[2][kFewRows] = {};
        if (u.group >= 0) {
            const T *w = p.w + (size_t)u.group * p.out_features * p.in_features + in0 + lane;
            const G *grad = p.grad + (size_t)u.row * p.out_features;
#pragma unroll 4
            for (int n = warp; n < p.out_features; n += kFewWarps) {
                const T *line = w + (size_t)n * p.in_features;
                const float w0 = first ? to_f32<T>(line[0]) : 0.f, w1 = second ? to_f32<T>(line[32]) : 0.f;
#pragma unroll
                for (int r = 0; r < kFewRows; ++r)
                    if (r < u.count) {
                        const float v = to_f32<G>(grad[(size_t)r * p.out_features + n]);
                        acc[0][r] = fmaf(v, w0, acc[0][r]);
                        acc[1][r] = fmaf(v, w1, acc[1][r]);
                    }
            }
        }
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
            partial[warp][r][lane] = acc[0][r];
            partial[warp][r][32 + lane] = acc[1][r];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < u.count * kFewInputs; i += 32 * kFewWarps) {
            const int r = i / kFewInputs, c = i % kFewInputs;
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < kFewWarps; ++k) sum += partial[k][r][c];
            if (in0 + c < p.in_features) p.grad_x[(size_t)(u.row + r) * p.in_features + in0 + c] = from_f32<T>(sum);
        }
        __syncthreads();
    }
}

// grad_weight and grad_bias: a warp an output and 256 inputs of it, eight a lane; the group's rows one after the other.
template <typename T, typename G>
__global__ void __launch_bounds__(kThreads) linear_few_weight_grad_kernel(const FewGrad<T, G> p) {
    constexpr int kEach = 8, kLine = 32 * kEach;
    __shared__ int start[kMaxGroups + 2];
    wait_for_previous_kernel();
    if (threadIdx.x < 32) scan_starts(p.g, start);
    __syncthreads();
    const int lane = threadIdx.x % 32, lines = (p.in_features + kLine - 1) / kLine;
    const long long items = (long long)p.g.groups * p.out_features * lines;
    const long long warps = (long long)gridDim.x * (kThreads / 32);
    for (long long item = (long long)blockIdx.x * (kThreads / 32) + threadIdx.x / 32; item < items; item += warps) {
        const int line = (int)(item % lines);
        const long long output = item / lines;  // counted over the groups
        const int e = (int)(output / p.out_features), n = (int)(output - (long long)e * p.out_features);
        float acc[kEach] = {}, bias = 0.f;
        for (int b = 0; b < p.g.batch; ++b)
            for (int m = start[e]; m < start[e + 1]; ++m) {
                const size_t row = (size_t)b * p.g.rows + m;
                const float v = to_f32<G>(p.grad[row * p.out_features + n]);
                const T *x = p.x + row * p.in_features + line * kLine + lane;
                bias += v;
#pragma unroll
                for (int j = 0; j < kEach; ++j)
                    if (line * kLine + 32 * j + lane < p.in_features) acc[j] = fmaf(v, to_f32<T>(x[32 * j]), acc[j]);
            }
        if (p.grad_weight)
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int k = line * kLine + 32 * j + lane;
                if (k < p.in_features) p.grad_weight[(size_t)output * p.in_features + k] = from_f32<T>(acc[j]);
            }
        if (p.grad_bias && line == 0 && lane == 0) p.grad_bias[output] = from_f32<T>(bias);
    }
}

// The bias's gradient from the sums over 32 rows that the pre-activation's gradient left behind (MmaRows::sums): a block takes 32 outputs
// of a group, its warps every 32nd of an element's sums, or of the elements where there are more, and adds the warps' in order.
constexpr int kBiasWarps = 32;

template <typename T>
__global__ void __launch_bounds__(32 * kBiasWarps) linear_bias_sum_kernel(const Groups g, const float *__restrict__ sums, int unit, int cols,
                                                                          T *__restrict__ grad_bias) {
    __shared__ RowTable table;
    __shared__ float partial[kBiasWarps][32];
    wait_for_previous_kernel();
    build_row_table(g, unit, false, table);
    __syncthreads();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, steps = (cols + 31) / 32, subs = unit / kSumRows;
    for (long long item = blockIdx.x; item < (long long)g.groups * steps; item += gridDim.x) {
        const int e = (int)(item / steps), c = (int)(item % steps) * 32 + lane;
        const int each = (int)(((long long)(table.start[e + 1] - table.start[e]) + kSumRows - 1) / kSumRows);  // sums of one batch element
        const size_t apart = (size_t)table.unit_begin[g.groups + 2] * subs;                                    // of two elements' sums
        const float *const first = sums + (size_t)table.unit_begin[e + 1] * subs * cols + c;
        float sum = 0.f;
        if (c < cols) {
            if (each >= kBiasWarps || each >= g.batch) {
                for (int b = 0; b < g.batch; ++b)
#pragma unroll 8
                    for (int k = warp; k < each; k += kBiasWarps) sum += first[(b * apart + k) * cols];
            } else {  // (one element after the other leaves most warps idle: 512 elements of 3 groups 300 us more)
#pragma unroll 1
                for (int b = warp; b < g.batch; b += kBiasWarps)
                    for (int k = 0; k < each; ++k) sum += first[(b * apart + k) * cols];
            }
        }
        partial[warp][lane] = sum;
        __syncthreads();
        if (warp == 0 && c < cols) {
            float total = 0.f;
#pragma unroll
            for (int w = 0; w < kBiasWarps; ++w) total += partial[w][lane];
            grad_bias[(size_t)e * cols + c] = from_f32<T>(total);
        }
        __syncthreads();
    }
}

template <typename T>
struct WeightGrad {
    const T *grad;  // g [rows][out]
    const T *x;     // [rows][in]
    T *grad_weight, *grad_bias;
    float *slots, *bias_slots;  // partial sums: [slot][out][in], [slot][out]
    int in_features, out_features;
    int block, piece;
    Groups g;
};

// A 64 x 64 tile of grad_weight (outputs x inputs) over one piece of a group's rows.
__global__ void __launch_bounds__(kThreads) linear_weight_grad_kernel(const WeightGrad<float> p) {
    __shared__ PieceTable table;
    __shared__ __align__(16) Slices slices;
    wait_for_previous_kernel();
    build_piece_table(p.g, p.block, p.piece, table);
    __syncthreads();
    const int out_tiles = (p.out_features + kTile - 1) / kTile, in_tiles = (p.in_features + kTile - 1) / kTile;
    const int per_piece = out_tiles * in_tiles;
    const long long items = (long long)table.piece_begin[p.g.groups] * per_piece;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const int piece = (int)(item / per_piece), t = (int)(item % per_piece);
        const int e = find_section(table.piece_begin, p.g.groups, piece), s = piece - table.piece_begin[e];
        const int out0 = (t / in_tiles) * kTile, in0 = (t % in_tiles) * kTile;
        const int outs = min(kTile, p.out_features - out0), ins = min(kTile, p.in_features - in0);
        const int blocks = group_blocks(p.g, table.start, e, p.block);
        const bool with_bias = in0 == 0 && p.grad_bias;
        float acc[kOwn][kOwn] = {}, bias[kOwn] = {};
        for (int j = s * p.piece; j < min(blocks, (s + 1) * p.piece); ++j) {
            long long row;
            int count;
            block_rows(p.g, table.start, e, p.block, j, row, count);
            const float *grad = p.grad + (size_t)row * p.out_features + out0, *x = p.x + (size_t)row * p.in_features + in0;
            if (with_bias)
                tile_product<false, false, true>(acc, bias, slices, grad, 1, p.out_features, outs, x, 1, p.in_features, ins, count);
            else
                tile_product<false, false, false>(acc, bias, slices, grad, 1, p.out_features, outs, x, 1, p.in_features, ins, count);
        }
        const bool whole = table.slot_begin[e + 1] == table.slot_begin[e];
        const size_t slot = whole ? (size_t)e : (size_t)table.slot_begin[e] + s;
        float *const weight = whole ? p.grad_weight : p.slots, *const biases = whole ? p.grad_bias : p.bias_slots;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int r = kOwn * ty + i;
            if (r >= outs) continue;
            if (p.grad_weight)
#pragma unroll
                for (int c = 0; c < kOwn; ++c)
                    if (kOwn * tx + c < ins) weight[(slot * p.out_features + out0 + r) * p.in_features + in0 + kOwn * tx + c] = acc[i][c];
            if (with_bias && tx == 0) biases[slot * p.out_features + out0 + r] = bias[i];
        }
    }
}

// Adds the slots of the groups that were computed in pieces, in order.  A block takes 1024 elements of a group's slots, or with
// kSplit 128, whose slots its eight warps share and whose eight sums are added in order: for many slots, where a thread's
// chain of loads would be the time (74 slots of 256 x 256 for each of 3 groups: 28 us in one chain, 13 in eight; 18 slots of 1024 x
// 256 8 us against 15).
constexpr int kSumWarps = 8, kLaneElements = 4;

template <typename T, bool kSplit>
__global__ void __launch_bounds__(32 * kSumWarps) linear_weight_grad_sum_kernel(const WeightGrad<T> p) {
    __shared__ PieceTable table;
    __shared__ float partial[kSplit ? kSumWarps : 1][32 * kLaneElements];
    wait_for_previous_kernel();
    build_piece_table(p.g, p.block, p.piece, table);
    __syncthreads();
    const size_t size = (size_t)p.out_features * p.in_features, both = size + p.out_features;
    constexpr int kEach = 32 * kLaneElements * (kSplit ? 1 : kSumWarps);
    const long long blocks = (long long)((both + kEach - 1) / kEach);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (long long item = blockIdx.x; item < blocks * p.g.groups; item += gridDim.x) {
        const int e = (int)(item / blocks);
        const int first = table.slot_begin[e], count = table.slot_begin[e + 1] - first;
        if (count == 0) continue;
        const size_t base = (size_t)(item % blocks) * kEach + (kSplit ? 0 : warp * 32 * kLaneElements) + lane;
        float sum[kLaneElements] = {};
        // weights: element i of slot s at slots[s * size + i]; biases behind them, in slots of their own
        const float *src[kLaneElements];
        size_t step[kLaneElements];
#pragma unroll
        for (int j = 0; j < kLaneElements; ++j) {
            const size_t i = base + 32 * j;
            const bool weight = i < size;
            step[j] = weight ? size : (size_t)p.out_features;
            src[j] = weight ? p.slots + first * size + i : p.bias_slots + (size_t)first * p.out_features + (i - size);
            if (i >= both || !(weight ? p.grad_weight : p.grad_bias)) src[j] = nullptr;
        }
        // eight slots on their way at a time, the last round's missing ones left out (not in a loop of single slots)
        constexpr int kRound = 8, kStep = kSplit ? kSumWarps : 1;
        for (int s = kSplit ? warp : 0; s < count; s += kRound * kStep) {
            float v[kRound][kLaneElements];
#pragma unroll
            for (int r = 0; r < kRound; ++r)
#pragma unroll
                for (int j = 0; j < kLaneElements; ++j)
                    v[r][j] = src[j] && s + r * kStep < count ? src[j][(size_t)(s + r * kStep) * step[j]] : 0.f;
#pragma unroll
            for (int r = 0; r < kRound; ++r)
#pragma unroll
                for (int j = 0; j < kLaneElements; ++j) sum[j] += v[r][j];
        }
        const auto put = [&](size_t i, float total) {
            if (i < size) {
                if (p.grad_weight) p.grad_weight[e * size + i] = from_f32<T>(total);
            } else if (i < both && p.grad_bias) {
                p.grad_bias[(size_t)e * p.out_features + (i - size)] = from_f32<T>(total);
            }
        };
        if constexpr (!kSplit) {
#pragma unroll
            for (int j = 0; j < kLaneElements; ++j) put(base + 32 * j, sum[j]);
        } else {
#pragma unroll
            for (int j = 0; j < kLaneElements; ++j) partial[warp][32 * j + lane] = sum[j];
            __syncthreads();
            if (warp < kLaneElements) {
                float total = 0.f;
#pragma unroll
                for (int w = 0; w < kSumWarps; ++w) total += partial[w][32 * warp + lane];
                put(base + 32 * warp, total);
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------------------------------------
inline size_t type_size(int dtype) { return dtype == FDA_DTYPE_F32 ? 4 : 2; }

// Upper bound of a piece table's slots, whatever the start indices are.  A group has slots when it has more than `piece` blocks, so more
// than floor(piece / batch) in each batch element, and all of these but the last are whole: that takes `least` rows of the element.  With k
// such groups of r rows an element (r >= k in all) there are at most r - k over `block` and one block a group more, times the
// batch; b blocks of a group are at most (b + piece - 1) / piece pieces.  The bound grows with k and with r.
long long most_slots(int batch, int rows, int groups, int block, int piece) {
    if (batch == 0) return 0;
    const long long least = (long long)block * (piece / batch) + 1, k = std::min<long long>(groups, rows / least);
    return k == 0 ? 0 : (batch * ((rows - k) / block + k) + k * (piece - 1)) / piece;
}

// As many pieces as `workers` take at once over `tiles` tiles of the weight, none shorter than `least_piece` blocks.
Cut cut_rows(int batch, int rows, int groups, long long tiles, int block, int least_piece, int workers) {
    Cut c;
    c.block = block;
    const long long blocks = std::max<long long>(1, most_units(batch, rows, groups, block, false));
    // One piece more than the SMs take would be a round of its own, and every further group can add one that is not full.  Where there
    // are many groups for the SMs, only those twice the mean are cut: each piece has its start and its sums to write and add
    // (16 uneven groups, 256 -> 1024: pieces of 8 blocks 42 + 14 us, of 34 28 + 7).
    const long long wanted = std::max<long long>(1, workers / tiles);
    const long long length = wanted >= 2 * groups ? ceil_div(blocks, wanted - (groups - 1)) : 2 * ceil_div(blocks, groups);
    c.piece = (int)std::max<long long>(least_piece, length);
    if (blocks <= 2 * least_piece) c.piece = (int)blocks;  // the second launch would cost more than it spreads
    c.pieces = ceil_div(blocks, c.piece) + groups;
    c.slots = most_slots(batch, rows, groups, block, c.piece);
    return c;
}

struct Shape {
    int batch, rows, groups, in_features, out_features, dtype;
};

int check_shape(const Shape &s) {
    if (s.dtype < 0 || s.dtype > 2) return FDA_ERR_BAD_DTYPE;
    if (s.batch < 0 || s.rows < 0 || s.groups < 1 || s.in_features < 1 || s.out_features < 1) return FDA_ERR_BAD_SHAPE;
    if ((long long)s.batch * s.rows >= (1ll << 31)) return FDA_ERR_BAD_SHAPE;
    if (s.in_features >= (1 << 26) || s.out_features >= (1 << 26)) return FDA_ERR_BAD_SHAPE;
    if (s.groups > FDA_LINEAR_MAX_GROUPS) return FDA_ERR_TOO_LARGE_STATIC;
    return FDA_OK;
}

int check_groups(const Shape &s, const int64_t *starts, int num_starts) {
    if (!starts) return s.groups == 1 ? FDA_OK : FDA_ERR_NULL_POINTER;
    return (num_starts == s.groups || num_starts == s.groups + 1) ? FDA_OK : FDA_ERR_BAD_SHAPE;
}

int launched(cudaError_t e) {
    if (e == cudaSuccess) return FDA_OK;
    fda::record_cuda_error((int)e);
    return FDA_ERR_CUDA;
}

constexpr int kPlainBlock = 256, kPlainLeastPiece = 1;

template <int kMode, int kAct>
int run_rows(const RowProduct<float> &p, cudaStream_t st) {
    const long long tiles = most_units(p.g.batch, p.g.rows, p.g.groups, kTile, kMode != kPreGrad) * ceil_div(p.cols, kTile);
    return launched(launch_early(linear_rows_kernel<kMode, kAct>, (unsigned)std::min<long long>(tiles, 8 * kSms), kThreads, 0, st, 1, p));
}

template <int kMode>
int run_rows(const RowProduct<float> &p, int activation, cudaStream_t st) {
    switch (activation) {
        case FDA_ACT_NONE: return run_rows<kMode, FDA_ACT_NONE>(p, st);
        case FDA_ACT_RELU: return run_rows<kMode, FDA_ACT_RELU>(p, st);
        case FDA_ACT_GELU: return run_rows<kMode, FDA_ACT_GELU>(p, st);
        case FDA_ACT_GELU_TANH: return run_rows<kMode, FDA_ACT_GELU_TANH>(p, st);
        default: return run_rows<kMode, FDA_ACT_SILU>(p, st);
    }
}

// 16-bit operands whose rows do not start on 16-byte boundaries are copied to rows that do, up to three of them in one launch.  A
// thread writes 16 bytes; what lies behind a row's elements is never read as anything.
struct Padding {
    const unsigned short *src[3];
    uint4 *dst[3];
    unsigned long long units[3];
    int line[3], count;
};

__global__ void __launch_bounds__(kThreads) linear_pad_kernel(const Padding p) {
    wait_for_previous_kernel();
    const unsigned long long step = (unsigned long long)gridDim.x * kThreads, first = (unsigned long long)blockIdx.x * kThreads + threadIdx.x;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        if (i >= p.count) break;
        const int line = p.line[i];
        const unsigned units = (unsigned)(line + 7) / 8;
        for (unsigned long long u = first; u < p.units[i]; u += step) {
            const unsigned long long row = u >> 32 ? u / units : (unsigned)u / units;
            const int c = (int)(u - row * units) * 8;
            const unsigned short *s = p.src[i] + row * line + c;
            unsigned v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = (c + 2 * j < line ? (unsigned)s[2 * j] : 0u) | (c + 2 * j + 1 < line ? (unsigned)s[2 * j + 1] << 16 : 0u);
            p.dst[i][u] = make_uint4(v[0], v[1], v[2], v[3]);
        }
    }
}

inline int padded(int line) { return (line + 7) & ~7; }

// Where rows of `line` elements are aligned src stays itself, else it becomes `place`, and the copy is noted.
void align_rows(Padding &p, const void *&src, char *place, size_t rows, int line) {
    if (line % 8 == 0) return;
    p.src[p.count] = static_cast<const unsigned short *>(src);
    p.dst[p.count] = reinterpret_cast<uint4 *>(place);
    p.units[p.count] = rows * (padded(line) / 8);
    p.line[p.count++] = line;
    src = place;
}

int pad(const Padding &p, cudaStream_t st) {
    if (p.count == 0) return FDA_OK;
    const unsigned long long most = *std::max_element(p.units, p.units + p.count);
    const unsigned blocks = (unsigned)std::min<unsigned long long>((most + kThreads - 1) / kThreads, 16 * kSms);
    return launched(launch_early(linear_pad_kernel, blocks, kThreads, 0, st, 1, p));
}

// What the workspaces hold, one behind the other.
struct Layout {
    size_t x = 0, w = 0, g = 0, slots = 0, bias_slots = 0, sums = 0, total = 0;
    size_t take(size_t bytes) {
        const size_t at = total;
        total += round256(bytes);
        return at;
    }
};

int mma_rows(int mode, const MmaRows &p, cudaStream_t st) {
    return p.dtype == FDA_DTYPE_F16 ? mma_rows_f16(mode, p, st) : mma_rows_bf16(mode, p, st);
}
int mma_weight_grad(const MmaWeightGrad &p, cudaStream_t st) {
    return p.dtype == FDA_DTYPE_F16 ? mma_weight_grad_f16(p, st) : mma_weight_grad_bf16(p, st);
}

size_t total_rows(const Shape &s) { return (size_t)s.batch * s.rows; }

void add_padded_operands(Layout &l, const Shape &s) {
    if (s.dtype == FDA_DTYPE_F32 || s.in_features % 8 == 0) return;
    l.x = l.take(total_rows(s) * padded(s.in_features) * 2);
    l.w = l.take((size_t)s.groups * s.out_features * padded(s.in_features) * 2);
}

// The 16-bit weight gradient's accumulators: 256 x 256 by pairs of blocks where that leaves every pair a piece of 16 blocks, else 128
// outputs and as many inputs as leave every SM a piece of 8.
struct WeightTile {
    int outputs, inputs;
    bool pair;
};

WeightTile mma_weight_tile(const Shape &s) {
    const long long blocks = most_units(s.batch, s.rows, s.groups, kMmaSlice, false);
    if (s.out_features > 128 && s.in_features > 128 &&
        ceil_div(s.out_features, 256) * ceil_div(s.in_features, 256) * ceil_div(blocks, 16) >= kSms / 2)
        return {256, 256, true};
    for (int tile = 256; tile > 64; tile /= 2)
        if (s.in_features > tile / 2 && ceil_div(s.out_features, kMmaTileRows) * ceil_div(s.in_features, tile) * ceil_div(blocks, 8) >= kSms)
            return {kMmaTileRows, tile, false};
    return {kMmaTileRows, 64, false};
}

Cut weight_cut(const Shape &s) {
    if (s.dtype != FDA_DTYPE_F32) {
        const WeightTile t = mma_weight_tile(s);
        return cut_rows(s.batch, s.rows, s.groups, ceil_div(s.out_features, t.outputs) * ceil_div(s.in_features, t.inputs), kMmaSlice, 8,
                        t.pair ? kSms / 2 : kSms);
    }
    return cut_rows(s.batch, s.rows, s.groups, ceil_div(s.out_features, kTile) * ceil_div(s.in_features, kTile), kPlainBlock,
                    kPlainLeastPiece, kSms);
}

bool few_rows(const Shape &s);

Layout forward_layout(const Shape &s) {
    Layout l;
    if (!few_rows(s)) add_padded_operands(l, s);
    return l;
}

bool few_rows_backward(const Shape &s) { return total_rows(s) <= 64; }

// A 16-bit bias's gradient behind an activation comes from g as it is (MmaRows::sums), not from g rounded by the weight gradient's product
// with ones: that would have the rounding's error twice, 1.4 times one rounding in the mean over many outputs and up to twice over few.  The
// sums cost the pre-activation's gradient 15 % (73728 x 256 x 1024: 119 instead of 103 us, 149504 x 256 x 256: 68 instead of 58),
// and some us to add them.
bool bias_from_sums(const Shape &s, int activation) { return s.dtype != FDA_DTYPE_F32 && activation != FDA_ACT_NONE; }

// g: the pre-activation's gradient, or a padded copy of grad_output.
Layout backward_layout(const Shape &s, int activation) {
    Layout l;
    if (few_rows_backward(s)) {
        if (activation != FDA_ACT_NONE) l.g = l.take(total_rows(s) * s.out_features * sizeof(float));
        return l;
    }
    add_padded_operands(l, s);
    const bool narrow = s.dtype != FDA_DTYPE_F32;
    if (activation != FDA_ACT_NONE || (narrow && s.out_features % 8))
        l.g = l.take(total_rows(s) * (narrow ? padded(s.out_features) : s.out_features) * type_size(s.dtype));
    if (bias_from_sums(s, activation)) l.sums = l.take(most_sum_rows(s.batch, s.rows, s.groups) * s.out_features * sizeof(float));
    const Cut c = weight_cut(s);
    l.slots = l.take((size_t)c.slots * s.out_features * s.in_features * sizeof(float));
    l.bias_slots = l.take((size_t)c.slots * s.out_features * sizeof(float));
    return l;
}

// Few rows in all (with groups: few enough that most groups have hardly any).
bool few_rows(const Shape &s) { return total_rows(s) <= (s.groups > 1 ? 64 : 8); }

template <typename T, int kMode>
int run_few_rows(const RowProduct<T> &p, int activation, cudaStream_t st) {
    const long long steps = ceil_div(p.cols, kFewOutputs);
    const long long warps = most_units(p.g.batch, p.g.rows, p.g.groups, kFewRows, kMode != kPreGrad && p.g.starts) * steps;
    const unsigned blocks = (unsigned)std::min<long long>(ceil_div(warps, kFewThreads / 32), 16 * kSms);
    const bool vector = p.depth % (16 / sizeof(T)) == 0 && ((uintptr_t)p.a | (uintptr_t)p.w) % 16 == 0;
    return launched(launch_early(vector ? linear_few_rows_kernel<T, kMode, true> : linear_few_rows_kernel<T, kMode, false>, blocks, kFewThreads, 0,
                                 st, 1, p, activation));
}

// out = act(x W^T + bias) + extra, or extra * act'(x W^T + bias)
template <typename T>
RowProduct<T> row_product(const Shape &s, const Groups &g, const void *x, const void *weight, const void *bias, const void *extra, void *out,
                          int out_pitch) {
    RowProduct<T> p;
    p.a = static_cast<const T *>(x);
    p.w = static_cast<const T *>(weight);
    p.bias = static_cast<const T *>(bias);
    p.extra = static_cast<const T *>(extra);
    p.out = static_cast<T *>(out);
    p.depth = p.in_features = s.in_features;
    p.cols = s.out_features;
    p.out_pitch = out_pitch;
    p.g = g;
    return p;
}

template <int kMode>
int run_few_rows(const Shape &s, const Groups &g, const void *x, const void *weight, const void *bias, const void *extra, void *out,
                 int out_pitch, int activation, cudaStream_t st) {
    if (s.dtype == FDA_DTYPE_F32)
        return run_few_rows<float, kMode>(row_product<float>(s, g, x, weight, bias, extra, out, out_pitch), activation, st);
    if (s.dtype == FDA_DTYPE_F16)
        return run_few_rows<__half, kMode>(row_product<__half>(s, g, x, weight, bias, extra, out, out_pitch), activation, st);
    return run_few_rows<__nv_bfloat16, kMode>(row_product<__nv_bfloat16>(s, g, x, weight, bias, extra, out, out_pitch), activation, st);
}

int forward(const Shape &s, const Groups &g, const void *x, const void *weight, const void *bias, const void *residual, void *y, char *ws,
            int activation, cudaStream_t st) {
    if (few_rows(s)) return run_few_rows<kForward>(s, g, x, weight, bias, residual, y, s.out_features, activation, st);
    if (s.dtype == FDA_DTYPE_F32)
        return run_rows<kForward>(row_product<float>(s, g, x, weight, bias, residual, y, s.out_features), activation, st);
    const Layout l = forward_layout(s);
    Padding pads{};
    align_rows(pads, x, ws + l.x, total_rows(s), s.in_features);
    align_rows(pads, weight, ws + l.w, (size_t)s.groups * s.out_features, s.in_features);
    if (const int rc = pad(pads, st)) return rc;
    const long long in = padded(s.in_features);
    const MmaRows p{x, weight, bias, residual, y, nullptr, in, in, s.out_features, s.out_features, s.in_features, s.out_features, s.dtype, activation, g};
    return mma_rows(kForward, p, st);
}

struct Gradients {
    void *x, *weight, *bias;
};

template <typename T>
int sum_slots(const WeightGrad<T> &q, const Shape &s, const Cut &c, cudaStream_t st) {
    if (c.slots == 0) return FDA_OK;
    const bool split = c.pieces > 32 + s.groups && c.pieces > 8ll * s.groups;
    const long long items = ceil_div(((long long)s.in_features + 1) * s.out_features, 32 * kLaneElements * (split ? 1 : kSumWarps)) * s.groups;
    const unsigned blocks = (unsigned)std::min<long long>(items, 4 * kSms);
    return launched(launch_early(split ? linear_weight_grad_sum_kernel<T, true> : linear_weight_grad_sum_kernel<T, false>, blocks,
                                 32 * kSumWarps, 0, st, 1, q));
}

template <typename T>
WeightGrad<T> weight_grad_args(const Shape &s, const Groups &g, const Cut &c, const void *grad, const void *x, const Gradients &out,
                               char *ws, const Layout &l) {
    WeightGrad<T> q;
    q.grad = static_cast<const T *>(grad);
    q.x = static_cast<const T *>(x);
    q.grad_weight = static_cast<T *>(out.weight);
    q.grad_bias = static_cast<T *>(out.bias);
    q.slots = reinterpret_cast<float *>(ws + l.slots);
    q.bias_slots = reinterpret_cast<float *>(ws + l.bias_slots);
    q.in_features = s.in_features;
    q.out_features = s.out_features;
    q.block = c.block;
    q.piece = c.piece;
    q.g = g;
    return q;
}

int sum_bias(const Shape &s, const Groups &g, const float *sums, int unit, void *grad_bias, cudaStream_t st) {
    const unsigned blocks = (unsigned)std::min<long long>(ceil_div(s.out_features, 32) * s.groups, 4 * kSms);
    if (s.dtype == FDA_DTYPE_F16)
        return launched(launch_early(linear_bias_sum_kernel<__half>, blocks, 32 * kBiasWarps, 0, st, 1, g, sums, unit, s.out_features,
                                     static_cast<__half *>(grad_bias)));
    return launched(launch_early(linear_bias_sum_kernel<__nv_bfloat16>, blocks, 32 * kBiasWarps, 0, st, 1, g, sums, unit, s.out_features,
                                 static_cast<__nv_bfloat16 *>(grad_bias)));
}

template <typename T, typename G>
int few_gradients(const Shape &s, const Groups &g, const void *grad, const void *x, const void *weight, const Gradients &out, cudaStream_t st) {
    FewGrad<T, G> p;
    p.grad = static_cast<const G *>(grad);
    p.x = static_cast<const T *>(x);
    p.w = static_cast<const T *>(weight);
    p.grad_x = static_cast<T *>(out.x);
    p.grad_weight = static_cast<T *>(out.weight);
    p.grad_bias = static_cast<T *>(out.bias);
    p.in_features = s.in_features;
    p.out_features = s.out_features;
    p.g = g;
    if (out.x) {
        const long long items = most_units(s.batch, s.rows, s.groups, kFewRows, true) * ceil_div(s.in_features, kFewInputs);
        const int rc = launched(launch_early(linear_few_grad_x_kernel<T, G>, (unsigned)std::min<long long>(items, 8 * kSms), 32 * kFewWarps, 0, st, 1, p));
        if (rc) return rc;
    }
    if (!out.weight && !out.bias) return FDA_OK;
    const long long items = (long long)s.groups * s.out_features * ceil_div(s.in_features, 256);
    return launched(launch_early(linear_few_weight_grad_kernel<T, G>, (unsigned)std::min<long long>(ceil_div(items, kThreads / 32), 16 * kSms),
                                 kThreads, 0, st, 1, p));
}

template <typename T>
int backward_few(const Shape &s, const Groups &g, const void *x, const void *weight, const void *bias, const void *grad_output,
                 const Gradients &out, char *ws, int activation, cudaStream_t st) {
    if (activation == FDA_ACT_NONE) return few_gradients<T, T>(s, g, grad_output, x, weight, out, st);
    const Layout l = backward_layout(s, activation);
    if (const int rc = run_few_rows<T, kPreGrad>(row_product<T>(s, g, x, weight, bias, grad_output, ws + l.g, s.out_features), activation, st))
        return rc;
    return few_gradients<T, float>(s, g, ws + l.g, x, weight, out, st);
}

int backward_f32(const Shape &s, const Groups &g, const void *x, const void *weight, const void *bias, const void *grad_output,
                 const Gradients &out, char *ws, int activation, cudaStream_t st) {
    const Layout l = backward_layout(s, activation);
    const void *grad = grad_output;
    if (activation != FDA_ACT_NONE) {
        grad = ws + l.g;
        const RowProduct<float> p = row_product<float>(s, g, x, weight, bias, grad_output, ws + l.g, s.out_features);
        if (const int rc = run_rows<kPreGrad>(p, activation, st)) return rc;
    }
    if (out.x) {
        RowProduct<float> p = row_product<float>(s, g, grad, weight, nullptr, nullptr, out.x, s.in_features);
        p.depth = s.out_features;
        p.cols = s.in_features;
        if (const int rc = run_rows<kGradX, FDA_ACT_NONE>(p, st)) return rc;
    }
    if (!out.weight && !out.bias) return FDA_OK;
    const Cut c = weight_cut(s);
    const WeightGrad<float> q = weight_grad_args<float>(s, g, c, grad, x, out, ws, l);
    const long long items = c.pieces * ceil_div(s.out_features, kTile) * ceil_div(s.in_features, kTile);
    if (const int rc = launched(launch_early(linear_weight_grad_kernel, (unsigned)std::min<long long>(items, 8 * kSms), kThreads, 0, st, 1, q)))
        return rc;
    return sum_slots(q, s, c, st);
}

int backward_narrow(const Shape &s, const Groups &g, const void *x, const void *weight, const void *bias, const void *grad_output,
                    Gradients out, char *ws, int activation, cudaStream_t st) {
    const Layout l = backward_layout(s, activation);
    bool weights = out.weight || out.bias;
    const long long in = padded(s.in_features), outs = padded(s.out_features);
    const void *grad = activation != FDA_ACT_NONE ? ws + l.g : grad_output;
    Padding pads{};
    if (activation != FDA_ACT_NONE || weights) align_rows(pads, x, ws + l.x, total_rows(s), s.in_features);
    if (activation != FDA_ACT_NONE || out.x) align_rows(pads, weight, ws + l.w, (size_t)s.groups * s.out_features, s.in_features);
    if (activation == FDA_ACT_NONE) align_rows(pads, grad, ws + l.g, total_rows(s), s.out_features);
    if (const int rc = pad(pads, st)) return rc;
    if (activation != FDA_ACT_NONE) {
        float *const sums = out.bias && bias_from_sums(s, activation) ? reinterpret_cast<float *>(ws + l.sums) : nullptr;
        const MmaRows p{x, weight, bias, grad_output, ws + l.g, sums, in, in, s.out_features, outs, s.in_features, s.out_features, s.dtype,
                        activation, g};
        if (const int rc = mma_rows(kPreGrad, p, st)) return rc;
        if (sums) {
            if (const int rc = sum_bias(s, g, sums, mma_pre_grad_unit(p), out.bias, st)) return rc;
            out.bias = nullptr;
            weights = out.weight;
        }
    }
    if (out.x) {
        const MmaRows p{grad, weight, nullptr, nullptr, out.x, nullptr, outs, in, 0, s.in_features, s.in_features, s.out_features, s.dtype,
                        FDA_ACT_NONE, g};
        if (const int rc = mma_rows(kGradX, p, st)) return rc;
    }
    if (!weights) return FDA_OK;
    const Cut c = weight_cut(s);
    const MmaWeightGrad q{grad, x, outs, in, out.weight, out.bias, reinterpret_cast<float *>(ws + l.slots),
                          reinterpret_cast<float *>(ws + l.bias_slots), s.in_features, s.out_features, s.dtype, mma_weight_tile(s).inputs, mma_weight_tile(s).pair, c, g};
    if (const int rc = mma_weight_grad(q, st)) return rc;
    if (s.dtype == FDA_DTYPE_F16) return sum_slots(weight_grad_args<__half>(s, g, c, nullptr, nullptr, out, ws, l), s, c, st);
    return sum_slots(weight_grad_args<__nv_bfloat16>(s, g, c, nullptr, nullptr, out, ws, l), s, c, st);
}

bool misaligned16(const void *p) { return (uintptr_t)p % 16 != 0; }

}  // namespace

extern "C" {

size_t fda_linear_forward_workspace_bytes(int batch, int rows, int groups, int in_features, int out_features, int dtype) {
    const Shape s{batch, rows, groups, in_features, out_features, dtype};
    return check_shape(s) == FDA_OK ? forward_layout(s).total : 0;
}

int fda_linear_forward(const void *x, const void *weight, const void *bias, const void *residual, const int64_t *group_start_index,
                       int num_starts, void *y, void *workspace, size_t workspace_bytes, int batch, int rows, int groups, int in_features,
                       int out_features, int activation, int dtype, void *stream) {
    const Shape s{batch, rows, groups, in_features, out_features, dtype};
    if (const int rc = check_shape(s)) return rc;
    if (activation < FDA_ACT_NONE || activation > FDA_ACT_SILU) return FDA_ERR_BAD_ACTIVATION;
    if (const int rc = check_groups(s, group_start_index, num_starts)) return rc;
    if (batch == 0 || rows == 0) return FDA_OK;
    if (!x || !weight || !y) return FDA_ERR_NULL_POINTER;
    const size_t need = forward_layout(s).total;
    if (need > 0 && (!workspace || workspace_bytes < need)) return FDA_ERR_WORKSPACE;
    if (need > 0 && (uintptr_t)workspace % 256) return FDA_ERR_MISALIGNED;
    const Groups g{group_start_index, num_starts, groups, batch, rows};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype != FDA_DTYPE_F32 && (misaligned16(x) || misaligned16(weight))) return FDA_ERR_MISALIGNED;
    return forward(s, g, x, weight, bias, residual, y, static_cast<char *>(workspace), activation, st);
}

size_t fda_linear_backward_workspace_bytes(int batch, int rows, int groups, int in_features, int out_features, int activation, int dtype) {
    const Shape s{batch, rows, groups, in_features, out_features, dtype};
    return check_shape(s) == FDA_OK ? backward_layout(s, activation).total : 0;
}

int fda_linear_backward(const void *x, const void *weight, const void *bias, const void *grad_output, const int64_t *group_start_index,
                        int num_starts, void *grad_x, void *grad_weight, void *grad_bias, void *workspace, size_t workspace_bytes,
                        int batch, int rows, int groups, int in_features, int out_features, int activation, int dtype, void *stream) {
    const Shape s{batch, rows, groups, in_features, out_features, dtype};
    if (const int rc = check_shape(s)) return rc;
    if (activation < FDA_ACT_NONE || activation > FDA_ACT_SILU) return FDA_ERR_BAD_ACTIVATION;
    if (const int rc = check_groups(s, group_start_index, num_starts)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (batch == 0 || rows == 0) {  // no row: the parameters' gradients are zero
        const size_t bytes = (size_t)groups * out_features * type_size(dtype);
        cudaError_t e = cudaSuccess;
        if (grad_weight) e = cudaMemsetAsync(grad_weight, 0, bytes * in_features, st);
        if (grad_bias && e == cudaSuccess) e = cudaMemsetAsync(grad_bias, 0, bytes, st);
        if (e != cudaSuccess) fda::record_cuda_error((int)e);
        return e == cudaSuccess ? FDA_OK : FDA_ERR_CUDA;
    }
    if (!x || !weight || !grad_output) return FDA_ERR_NULL_POINTER;
    const size_t need = backward_layout(s, activation).total;
    if (need > 0 && (!workspace || workspace_bytes < need)) return FDA_ERR_WORKSPACE;
    if (need > 0 && (uintptr_t)workspace % 256) return FDA_ERR_MISALIGNED;
    const Groups g{group_start_index, num_starts, groups, batch, rows};
    const Gradients out{grad_x, grad_weight, grad_bias};
    char *ws = static_cast<char *>(workspace);
    if (dtype != FDA_DTYPE_F32 && (misaligned16(x) || misaligned16(weight) || misaligned16(grad_output))) return FDA_ERR_MISALIGNED;
    if (few_rows_backward(s)) {
        if (dtype == FDA_DTYPE_F32) return backward_few<float>(s, g, x, weight, bias, grad_output, out, ws, activation, st);
        if (dtype == FDA_DTYPE_F16) return backward_few<__half>(s, g, x, weight, bias, grad_output, out, ws, activation, st);
        return backward_few<__nv_bfloat16>(s, g, x, weight, bias, grad_output, out, ws, activation, st);
    }
    if (dtype == FDA_DTYPE_F32) return backward_f32(s, g, x, weight, bias, grad_output, out, ws, activation, st);
    return backward_narrow(s, g, x, weight, bias, grad_output, out, ws, activation, st);
}

int fda_linear_timeouts(void) {
    // reading the counts would wait for streams only that wait for the default one
    if (launched(cudaDeviceSynchronize()) != FDA_OK) return -1;
    const int a = mma_timeouts_f16(), b = mma_timeouts_bf16();
    return a < 0 || b < 0 ? -1 : a + b;
}

}  // extern "C"

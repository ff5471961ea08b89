// What the kernels of the linear operators share: activations, the row groups, and how a grid walks them.
//
//     pre = x W^T + b,   y = act(pre) + residual            x [batch][rows][in], W [groups][out][in], y [batch][rows][out]
//     g = dy * act'(pre),   dx = g W,   dW = g^T x,   db = sum of g's rows
//
// Row m of every batch element belongs to group e for start(e) <= m < start(e + 1); start(e) is the largest of the given
// start indices up to e, each brought into 0 .. rows, so that no list of indices can lead out of a tensor or make two groups
// share a row.  With as many start indices as groups the last group ends with the rows, with one more it ends there; rows in
// front of the first group and behind the last belong to none: their product is nothing (y = residual or 0, dx = 0).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <stdint.h>

#include "../../include/fda_b200.h"

namespace fda_linear {

constexpr int kMaxGroups = FDA_LINEAR_MAX_GROUPS;

// A kernel may be set up while the one before it in the stream still runs: everything in front of this call touches no memory
// but its own block's, and nothing behind it comes before the earlier kernel has ended and its results are visible.
__device__ __forceinline__ void wait_for_previous_kernel() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr float kSqrtHalf = 0.70710678118654752f, kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kTanhScale = 0.79788456080286536f, kTanhCubic = 0.044715f;  // sqrt(2/pi)

// 1 / (1 + e^-v); where e^-v overflows the quotient is 0.
__device__ __forceinline__ float sigmoid(float v) { return 1.f / (1.f + expf(-v)); }

// act(pre).  A NaN stays one (a maximum would turn it into 0).
template <int kAct>
__device__ __forceinline__ float activate(float v) {
    if (kAct == FDA_ACT_RELU) return v < 0.f ? 0.f : v;
    if (kAct == FDA_ACT_GELU) {
        const float c = 1.f + erff(v * kSqrtHalf);
        return c == 0.f ? 0.f : 0.5f * v * c;  // 0 at minus infinity too, as in the paired form
    }
    if (kAct == FDA_ACT_GELU_TANH) return 0.5f * v * (1.f + tanhf(kTanhScale * (v + kTanhCubic * v * v * v)));
    if (kAct == FDA_ACT_SILU) return v * sigmoid(v);
    return v;
}

// dy * act'(pre); relu's derivative at 0 is 0.
template <int kAct>
__device__ __forceinline__ float activate_backward(float v, float dy) {
    if (kAct == FDA_ACT_RELU) return v <= 0.f ? 0.f : dy;
    if (kAct == FDA_ACT_GELU) return dy * (0.5f * (1.f + erff(v * kSqrtHalf)) + v * kInvSqrt2Pi * expf(-0.5f * v * v));
    if (kAct == FDA_ACT_GELU_TANH) {
        const float t = tanhf(kTanhScale * (v + kTanhCubic * v * v * v));
        // beyond 12 t is 1 or -1 to the last bit, and the slope's polynomial would overflow for very large v
        const float c = fminf(fmaxf(v, -12.f), 12.f);
        return dy * (0.5f * (1.f + t) + 0.5f * c * (1.f - t * t) * kTanhScale * (1.f + 3.f * kTanhCubic * c * c));
    }
    if (kAct == FDA_ACT_SILU) {
        const float s = sigmoid(v);
        return dy * (s * (1.f + v * (1.f - s)));
    }
    return dy;
}

// The same with the activation as an argument, where few elements pass.
__device__ __forceinline__ float activate_any(int act, float v) {
    switch (act) {
        case FDA_ACT_RELU: return activate<FDA_ACT_RELU>(v);
        case FDA_ACT_GELU: return activate<FDA_ACT_GELU>(v);
        case FDA_ACT_GELU_TANH: return activate<FDA_ACT_GELU_TANH>(v);
        case FDA_ACT_SILU: return activate<FDA_ACT_SILU>(v);
        default: return v;
    }
}
__device__ __forceinline__ float activate_backward_any(int act, float v, float dy) {
    switch (act) {
        case FDA_ACT_RELU: return activate_backward<FDA_ACT_RELU>(v, dy);
        case FDA_ACT_GELU: return activate_backward<FDA_ACT_GELU>(v, dy);
        case FDA_ACT_GELU_TANH: return activate_backward<FDA_ACT_GELU_TANH>(v, dy);
        case FDA_ACT_SILU: return activate_backward<FDA_ACT_SILU>(v, dy);
        default: return dy;
    }
}

struct Groups {
    const int64_t *starts;  // nullptr: one group of all rows
    int num_starts;         // groups or groups + 1
    int groups;
    int batch;
    int rows;  // of one batch element
};

// The groups of one batch element as a block sees them, in shared memory.  A product over rows walks units of `unit` rows:
// section 0 holds the rows in front of the first group, section e + 1 those of group e, the last section the rows behind.
struct RowTable {
    int start[kMaxGroups + 2];       // first row of group e; [groups] is where the last ends
    int unit_begin[kMaxGroups + 3];  // first unit of section s; the last entry is the number of units
};

// Running maximum / sum over 32 lanes.
__device__ __forceinline__ int warp_scan_max(int v) {
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, v, d);
        if ((threadIdx.x & 31) >= d) v = max(v, o);
    }
    return v;
}
__device__ __forceinline__ int warp_scan_sum(int v) {
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, v, d);
        if ((threadIdx.x & 31) >= d) v += o;
    }
    return v;
}

// start[0 .. groups] by one warp.
__device__ __forceinline__ void scan_starts(const Groups &g, int *start) {
    const int lane = threadIdx.x & 31;
    if (!g.starts) {
        if (lane == 0) { start[0] = 0; start[1] = g.rows; }
        __syncwarp();
        return;
    }
    int carry = 0;
    for (int base = 0; base <= g.groups; base += 32) {
        const int i = base + lane;
        int v = 0;
        if (i <= g.groups) {
            if (i < g.num_starts) {
                const int64_t s = g.starts[i];
                v = s < 0 ? 0 : s > g.rows ? g.rows : (int)s;
            } else {
                v = g.rows;
            }
        }
        v = max(warp_scan_max(v), carry);
        if (i <= g.groups) start[i] = v;
        carry = __shfl_sync(0xffffffffu, v, 31);
    }
    __syncwarp();
}

// The whole table by the first warp of a block; the caller synchronises.  `rest`: the rows of no group get units too.
__device__ __forceinline__ void build_row_table(const Groups &g, int unit, bool rest, RowTable &t) {
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    scan_starts(g, t.start);
    int carry = 0;
    for (int base = 0; base < g.groups + 2; base += 32) {
        const int s = base + lane;
        int n = 0;
        if (s < g.groups + 2) {
            const int lo = s == 0 ? 0 : t.start[s - 1];
            const int hi = s == g.groups + 1 ? g.rows : t.start[s];
            const bool counts = rest || (s > 0 && s <= g.groups);
            n = counts ? (int)(((long long)(hi - lo) + unit - 1) / unit) : 0;
        }
        const int sum = warp_scan_sum(n) + carry;
        if (s < g.groups + 2) t.unit_begin[s] = sum - n;
        if (s == g.groups + 1) t.unit_begin[s + 1] = sum;
        carry = __shfl_sync(0xffffffffu, sum, 31);
    }
}

struct RowUnit {
    long long row;  // first row, counted over all batch elements
    int count;      // rows of it
    int group;      // -1: of no group
};

// Which section of a table holds unit u: the last with begin[s] <= u.
__device__ __forceinline__ int find_section(const int *begin, int sections, int u) {
    int lo = 0, hi = sections;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (begin[mid] <= u) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ RowUnit row_unit(const Groups &g, const RowTable &t, int unit, unsigned u) {
    const unsigned per_batch = (unsigned)t.unit_begin[g.groups + 2];
    const unsigned b = u / per_batch;
    const int i = (int)(u - b * per_batch);
    const int s = find_section(t.unit_begin, g.groups + 2, i);
    const int lo = s == 0 ? 0 : t.start[s - 1];
    const int hi = s == g.groups + 1 ? g.rows : t.start[s];
    const int first = lo + (i - t.unit_begin[s]) * unit;
    RowUnit r;
    r.row = (long long)b * g.rows + first;
    r.count = min(unit, hi - first);
    r.group = (s > 0 && s <= g.groups) ? s - 1 : -1;
    return r;
}

// How a product over the rows themselves (the weight's gradient) is cut: the rows of a group, over all batch elements, are
// blocks of `block` rows that no batch element shares, and pieces of at most `piece` such blocks.  A group of one piece is
// finished where it is computed; the pieces of the others go to slots of partial sums that a second kernel adds in order.
struct PieceTable {
    int start[kMaxGroups + 2];
    int piece_begin[kMaxGroups + 1];  // a group without rows has one piece (of no blocks): its gradient is zero
    int slot_begin[kMaxGroups + 1];
};

__device__ __forceinline__ int group_blocks(const Groups &g, const int *start, int e, int block) {
    return g.batch * (int)(((long long)(start[e + 1] - start[e]) + block - 1) / block);
}

__device__ __forceinline__ void build_piece_table(const Groups &g, int block, int piece, PieceTable &t) {
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    scan_starts(g, t.start);
    int pieces = 0, slots = 0;
    for (int base = 0; base <= g.groups; base += 32) {
        const int e = base + lane;
        int n = 0;
        if (e < g.groups) {
            n = (group_blocks(g, t.start, e, block) + piece - 1) / piece;
            if (n == 0) n = 1;
        }
        const int slot = n > 1 ? n : 0;
        const int sum = warp_scan_sum(n) + pieces, slot_sum = warp_scan_sum(slot) + slots;
        if (e <= g.groups) {
            t.piece_begin[e] = sum - n;
            t.slot_begin[e] = slot_sum - slot;
        }
        pieces = __shfl_sync(0xffffffffu, sum, 31);
        slots = __shfl_sync(0xffffffffu, slot_sum, 31);
    }
}

// Block j of group e: its first row over all batch elements, and how many rows it has.
__device__ __forceinline__ void block_rows(const Groups &g, const int *start, int e, int block, int j, long long &row, int &count) {
    const int per = (int)(((long long)(start[e + 1] - start[e]) + block - 1) / block);
    const int b = j / per, i = j - b * per;
    const int first = start[e] + i * block;
    row = (long long)b * g.rows + first;
    count = min(block, start[e + 1] - first);
}

// ---- host -------------------------------------------------------------------------------------------------------------------
inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
inline size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

constexpr int kSms = 148;

// Launch of a kernel that calls wait_for_previous_kernel, by clusters of `cluster` blocks.
template <typename... Parameters, typename... Arguments>
cudaError_t launch_early(void (*kernel)(Parameters...), unsigned grid, unsigned threads, int shared, cudaStream_t st, int cluster,
                         const Arguments &...arguments) {
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t launch{};
    launch.gridDim = dim3(grid);
    launch.blockDim = dim3(threads);
    launch.dynamicSmemBytes = shared;
    launch.stream = st;
    launch.attrs = attributes;
    launch.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&launch, kernel, Parameters(arguments)...);
}

// Upper bound of a row table's units, whatever the start indices are: every section adds at most one incomplete unit per batch
// element.
inline long long most_units(int batch, int rows, int groups, int unit, bool rest) {
    const long long sections = groups + (rest ? 2 : 0);
    return (long long)batch * (rows < rows / unit + sections ? rows : rows / unit + sections);
}

// How the rows of the weight's gradient are cut (PieceTable).
struct Cut {
    int block, piece;
    long long pieces, slots;  // at most
};

// What a product over row units does with its sums (run_rows, mma_rows).
enum Mode {
    kForward,  // out = act(a W^T + bias) + extra
    kPreGrad,  // out = extra * act'(a W^T + bias)
    kGradX     // out = a W
};

// 16-bit products on the tensor cores (fda_linear_mma_kernels.cuh).  Rows of a and of w start on 16-byte boundaries: their pitches (in
// elements) are multiples of 8.
struct MmaRows {
    const void *a, *w, *bias, *extra;
    void *out;
    float *sums;  // kPreGrad: the results' sums over 32 rows each, before rounding; may be nullptr
    long long a_pitch, w_pitch, extra_pitch, out_pitch;
    int in_features, out_features, dtype, activation;
    Groups g;
};
// Row k of `sums` [..][out_features] for the k-th 32 rows of a unit of `unit` rows, unit / 32 of them for every unit of a row table
// without rest.  The launch says which unit it took.
constexpr int kSumRows = 32;
inline size_t most_sum_rows(int batch, int rows, int groups) {
    const long long a = most_units(batch, rows, groups, 128, false) * (128 / kSumRows);
    const long long b = most_units(batch, rows, groups, 256, false) * (256 / kSumRows);
    return (size_t)(a > b ? a : b);
}
int mma_pre_grad_unit(const MmaRows &p);
int mma_rows_f16(int mode, const MmaRows &p, cudaStream_t st);
int mma_rows_bf16(int mode, const MmaRows &p, cudaStream_t st);

struct MmaWeightGrad {
    const void *grad, *x;
    long long grad_pitch, x_pitch;
    void *grad_weight, *grad_bias;  // either may be nullptr
    float *slots, *bias_slots;
    int in_features, out_features, dtype;
    int tile;  // inputs of an accumulator: 64, 128 or 256
    bool pair; // two blocks to 256 outputs x 256 inputs
    Cut cut;
    Groups g;
};
constexpr int kMmaTileRows = 128, kMmaSlice = 64;  // accumulator rows; contraction indices of a slice (and rows of a PieceTable's block)
int mma_weight_grad_f16(const MmaWeightGrad &p, cudaStream_t st);  // without the sum over slots
int mma_weight_grad_bf16(const MmaWeightGrad &p, cudaStream_t st);
int mma_timeouts_f16();  // -1 where the device cannot be asked
int mma_timeouts_bf16();

}  // namespace fda_linear

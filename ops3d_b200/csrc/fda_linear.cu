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
// A block computes a BM x BN tile; its 256 threads own TM x TN sums each (rows ty + 16 i, columns tx + 16 j: neighbouring
// threads read neighbouring words of a k-slice from shared memory and write neighbouring outputs).  Operands pass through
// shared memory in slices of 16 along k, the next slice travelling in registers meanwhile.
constexpr int kThreads = 256, kSlice = 16;

// A(i, k) = a[i * ai + k * ak], of which i < rows, k < depth exist; the stride that is 1 decides how threads cover a slice.
template <typename T, int kTile, bool kContiguousK>
struct SliceLoader {
    static constexpr int kEach = kTile * kSlice / kThreads;
    float reg[kEach];
    __device__ __forceinline__ static int index(int j) {  // along the tile
        return kContiguousK ? (int)threadIdx.x / kSlice + j * (kThreads / kSlice) : ((int)threadIdx.x + j * kThreads) % kTile;
    }
    __device__ __forceinline__ static int depth(int j) {
        return kContiguousK ? (int)threadIdx.x % kSlice : ((int)threadIdx.x + j * kThreads) / kTile;
    }
    __device__ __forceinline__ void load(const T *a, long long ai, long long ak, int rows, int k0, int k_end) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = index(j), k = k0 + depth(j);
            reg[j] = (i < rows && k < k_end) ? to_f32<T>(a[i * ai + k * ak]) : 0.f;
        }
    }
    __device__ __forceinline__ void store(float (*s)[kTile + 1]) const {
#pragma unroll
        for (int j = 0; j < kEach; ++j) s[depth(j)][index(j)] = reg[j];
    }
};

template <int BM, int BN>
struct Slices {
    float a[kSlice][BM + 1];
    float b[kSlice][BN + 1];
};

// acc += A B over k in [0, depth); A is BM x depth, B depth x BN.
template <typename T, int BM, int BN, bool kAK, bool kBK>
__device__ __forceinline__ void tile_product(float (&acc)[BM / 16][BN / 16], Slices<BM, BN> &s, const T *a, long long ai, long long ak,
                                             int rows, const T *b, long long bj, long long bk, int cols, int depth) {
    constexpr int TM = BM / 16, TN = BN / 16;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    SliceLoader<T, BM, kAK> la;
    SliceLoader<T, BN, kBK> lb;
    la.load(a, ai, ak, rows, 0, depth);
    lb.load(b, bj, bk, cols, 0, depth);
    for (int k0 = 0; k0 < depth; k0 += kSlice) {
        __syncthreads();
        la.store(s.a);
        lb.store(s.b);
        __syncthreads();
        if (k0 + kSlice < depth) {
            la.load(a, ai, ak, rows, k0 + kSlice, depth);
            lb.load(b, bj, bk, cols, k0 + kSlice, depth);
        }
#pragma unroll
        for (int k = 0; k < kSlice; ++k) {
            float ra[TM], rb[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) ra[i] = s.a[k][ty + 16 * i];
#pragma unroll
            for (int j = 0; j < TN; ++j) rb[j] = s.b[k][tx + 16 * j];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = fmaf(ra[i], rb[j], acc[i][j]);
        }
    }
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
    Groups g;
};

// kForward:  out = act(a W^T + bias) + extra    kPreGrad:  out = extra * act'(a W^T + bias)    kGradX:  out = a W
template <typename T, int kMode, int kAct, int BM, int BN>
__global__ void __launch_bounds__(kThreads) linear_rows_kernel(const RowProduct<T> p) {
    __shared__ RowTable table;
    __shared__ Slices<BM, BN> slices;
    build_row_table(p.g, BM, kMode != kPreGrad, table);
    __syncthreads();
    const int column_tiles = (p.cols + BN - 1) / BN;
    const long long tiles = (long long)table.unit_begin[p.g.groups + 2] * p.g.batch * column_tiles;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const RowUnit u = row_unit(p.g, table, BM, (unsigned)(tile / column_tiles));
        const int col0 = (int)(tile % column_tiles) * BN, cols = min(BN, p.cols - col0);
        float acc[BM / 16][BN / 16] = {};
        if (u.group >= 0) {
            const T *w = p.w + (size_t)u.group * ((kMode == kGradX ? (size_t)p.depth : (size_t)p.cols) * p.in_features);
            const T *a = p.a + (size_t)u.row * p.depth;
            if (kMode == kGradX)
                tile_product<T, BM, BN, true, false>(acc, slices, a, p.depth, 1, u.count, w + col0, 1, p.in_features, cols, p.depth);
            else
                tile_product<T, BM, BN, true, true>(acc, slices, a, p.depth, 1, u.count, w + (size_t)col0 * p.in_features, p.in_features, 1,
                                                    cols, p.depth);
        }
#pragma unroll
        for (int j = 0; j < BN / 16; ++j) {
            const int c = tx + 16 * j;
            if (c >= cols) continue;
            const float bias = (kMode != kGradX && p.bias && u.group >= 0) ? to_f32<T>(p.bias[(size_t)u.group * p.cols + col0 + c]) : 0.f;
#pragma unroll
            for (int i = 0; i < BM / 16; ++i) {
                const int r = ty + 16 * i;
                if (r >= u.count) continue;
                const size_t at = (size_t)(u.row + r) * p.cols + col0 + c;
                float v = acc[i][j] + bias;
                if (kMode == kForward) {
                    if (u.group >= 0) v = activate<kAct>(v);
                    if (p.extra) v += to_f32<T>(p.extra[at]);
                } else if (kMode == kPreGrad) {
                    v = activate_backward<kAct>(v, to_f32<T>(p.extra[at]));
                }
                p.out[at] = from_f32<T>(v);
            }
        }
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

// grad_weight tile BM (outputs) x BN (inputs) over one piece of a group's rows.
template <typename T, int BM, int BN>
__global__ void __launch_bounds__(kThreads) linear_weight_grad_kernel(const WeightGrad<T> p) {
    __shared__ PieceTable table;
    __shared__ Slices<BM, BN> slices;
    build_piece_table(p.g, p.block, p.piece, table);
    __syncthreads();
    const int out_tiles = (p.out_features + BM - 1) / BM, in_tiles = (p.in_features + BN - 1) / BN;
    const int per_piece = out_tiles * in_tiles;
    const long long items = (long long)table.piece_begin[p.g.groups] * per_piece;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const int piece = (int)(item / per_piece), t = (int)(item % per_piece);
        const int e = find_section(table.piece_begin, p.g.groups, piece), s = piece - table.piece_begin[e];
        const int out0 = (t / in_tiles) * BM, in0 = (t % in_tiles) * BN;
        const int outs = min(BM, p.out_features - out0), ins = min(BN, p.in_features - in0);
        const int blocks = group_blocks(p.g, table.start, e, p.block);
        float acc[BM / 16][BN / 16] = {};
        float bias = 0.f;
        for (int j = s * p.piece; j < min(blocks, (s + 1) * p.piece); ++j) {
            long long row;
            int count;
            block_rows(p.g, table.start, e, p.block, j, row, count);
            const T *grad = p.grad + (size_t)row * p.out_features + out0;
            tile_product<T, BM, BN, false, false>(acc, slices, grad, 1, p.out_features, outs,
                                                  p.x + (size_t)row * p.in_features + in0, 1, p.in_features, ins, count);
            if (in0 == 0 && p.grad_bias && (int)threadIdx.x < outs)
                for (int r = 0; r < count; ++r) bias += to_f32<T>(grad[(size_t)r * p.out_features + threadIdx.x]);
        }
        const bool whole = table.slot_begin[e + 1] == table.slot_begin[e];
        const size_t slot = (size_t)table.slot_begin[e] + s;
        if (p.grad_weight)
#pragma unroll
            for (int i = 0; i < BM / 16; ++i)
#pragma unroll
                for (int j = 0; j < BN / 16; ++j) {
                    const int r = ty + 16 * i, c = tx + 16 * j;
                    if (r >= outs || c >= ins) continue;
                    const size_t at = (size_t)(out0 + r) * p.in_features + in0 + c, size = (size_t)p.out_features * p.in_features;
                    if (whole) p.grad_weight[e * size + at] = from_f32<T>(acc[i][j]);
                    else p.slots[slot * size + at] = acc[i][j];
                }
        if (in0 == 0 && p.grad_bias && (int)threadIdx.x < outs) {
            const size_t at = out0 + threadIdx.x;
            if (whole) p.grad_bias[(size_t)e * p.out_features + at] = from_f32<T>(bias);
            else p.bias_slots[slot * p.out_features + at] = bias;
        }
    }
}

// Adds the slots of the groups that were computed in pieces, in order.  A block takes 1024 elements of a group's slots, or with
// kSplit 128, whose slots its eight warps share and whose eight sums are added in order: for many slots, where a thread's
// chain of loads would be the time (148 slots of 256 x 256: 28 us in one chain, 11 in eight; 40 slots of 16 groups 27 us against 84).
constexpr int kSumWarps = 8, kLaneElements = 4;

template <typename T, bool kSplit>
__global__ void __launch_bounds__(32 * kSumWarps) linear_weight_grad_sum_kernel(const WeightGrad<T> p) {
    __shared__ PieceTable table;
    __shared__ float partial[kSplit ? kSumWarps : 1][32 * kLaneElements];
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
#pragma unroll 4
        for (int s = kSplit ? warp : 0; s < count; s += kSplit ? kSumWarps : 1)
#pragma unroll
            for (int j = 0; j < kLaneElements; ++j)
                if (src[j]) sum[j] += src[j][s * step[j]];
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

}  // namespace

namespace fda_linear {

Cut cut_rows(int batch, int rows, int groups, long long tiles, int block, int least_piece) {
    Cut c;
    c.block = block;
    const long long blocks = std::max<long long>(1, most_units(batch, rows, groups, block, false));
    // As many pieces as the SMs take at once: one more would be a round of its own.  Every further group can add a piece that is
    // not full; where there are too many groups for that, pieces half as long, so that the last round is short.
    const long long wanted = std::max<long long>(1, kSms / tiles);
    const long long full = wanted >= 2 * groups ? wanted - (groups - 1) : 2 * wanted;
    c.piece = (int)std::max<long long>(least_piece, ceil_div(blocks, full));
    c.pieces = ceil_div(blocks, c.piece) + groups;
    // a group of n > 1 pieces has more than (n - 1) * piece blocks, so at least n / 2 * piece
    c.slots = blocks <= c.piece ? 0 : std::min(c.pieces, 2 * (blocks / c.piece) + 1);
    return c;
}

}  // namespace fda_linear

namespace {

struct Shape {
    int batch, rows, groups, in_features, out_features, dtype;
};

int check_shape(const Shape &s) {
    if (s.dtype < 0 || s.dtype > 2) return FDA_ERR_BAD_DTYPE;
    if (s.batch < 0 || s.rows < 0 || s.groups < 1 || s.in_features < 1 || s.out_features < 1) return FDA_ERR_BAD_SHAPE;
    if ((long long)s.batch * s.rows >= (1ll << 31)) return FDA_ERR_BAD_SHAPE;
    if (s.groups > FDA_LINEAR_MAX_GROUPS) return FDA_ERR_TOO_LARGE_STATIC;
    return FDA_OK;
}

int check_groups(const Shape &s, const int64_t *starts, int num_starts) {
    if (!starts) return s.groups == 1 ? FDA_OK : FDA_ERR_NULL_POINTER;
    return (num_starts == s.groups || num_starts == s.groups + 1) ? FDA_OK : FDA_ERR_BAD_SHAPE;
}

int launched() {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return FDA_OK;
    fda::record_cuda_error((int)e);
    return FDA_ERR_CUDA;
}

constexpr int kTileSize = 64;
constexpr int kPlainBlock = 64, kPlainLeastPiece = 4;

template <typename T, int kMode, int kAct>
int run_rows_plain(const RowProduct<T> &p, cudaStream_t st) {
    const long long tiles = most_units(p.g.batch, p.g.rows, p.g.groups, kTileSize, kMode != kPreGrad) * ceil_div(p.cols, kTileSize);
    linear_rows_kernel<T, kMode, kAct, kTileSize, kTileSize><<<(unsigned)std::min<long long>(tiles, 8 * kSms), kThreads, 0, st>>>(p);
    return launched();
}

template <typename T, int kMode>
int run_rows(const RowProduct<T> &p, int activation, cudaStream_t st) {
    switch (kMode == kGradX ? FDA_ACT_NONE : activation) {
        case FDA_ACT_NONE: return run_rows_plain<T, kMode, FDA_ACT_NONE>(p, st);
        case FDA_ACT_RELU: return run_rows_plain<T, kMode, FDA_ACT_RELU>(p, st);
        case FDA_ACT_GELU: return run_rows_plain<T, kMode, FDA_ACT_GELU>(p, st);
        case FDA_ACT_GELU_TANH: return run_rows_plain<T, kMode, FDA_ACT_GELU_TANH>(p, st);
        default: return run_rows_plain<T, kMode, FDA_ACT_SILU>(p, st);
    }
}

// 16-bit operands whose rows do not start on 16-byte boundaries are copied to rows that do.
__global__ void __launch_bounds__(kThreads) linear_pad_kernel(const unsigned short *__restrict__ src, unsigned short *__restrict__ dst,
                                                              unsigned long long elements, int line, int pitch) {
    const unsigned long long step = (unsigned long long)gridDim.x * kThreads;
    for (unsigned long long i = (unsigned long long)blockIdx.x * kThreads + threadIdx.x; i < elements; i += step)
        dst[i / (unsigned)line * (unsigned)pitch + i % (unsigned)line] = src[i];
}

inline int padded(int line) { return (line + 7) & ~7; }

// src itself where its rows are aligned, else a padded copy in `place`; launches the copy.
int aligned_rows(const void *&src, char *place, size_t rows, int line, cudaStream_t st) {
    if (line % 8 == 0) return FDA_OK;
    const unsigned long long elements = (unsigned long long)rows * line;
    const unsigned blocks = (unsigned)std::min<unsigned long long>((elements + kThreads - 1) / kThreads, 16 * kSms);
    linear_pad_kernel<<<blocks, kThreads, 0, st>>>(static_cast<const unsigned short *>(src), reinterpret_cast<unsigned short *>(place),
                                                   elements, line, padded(line));
    src = place;
    return launched();
}

// What the workspaces hold, one behind the other.
struct Layout {
    size_t x = 0, w = 0, g = 0, slots = 0, bias_slots = 0, total = 0;
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

Cut weight_cut(const Shape &s) {
    if (s.dtype != FDA_DTYPE_F32) {
        const long long tiles = ceil_div(s.out_features, kMmaTileRows) * ceil_div(s.in_features, mma_weight_tile(s.in_features));
        return cut_rows(s.batch, s.rows, s.groups, tiles, kMmaSlice, 8);
    }
    return cut_rows(s.batch, s.rows, s.groups, ceil_div(s.out_features, kTileSize) * ceil_div(s.in_features, kTileSize), kPlainBlock,
                    kPlainLeastPiece);
}

Layout forward_layout(const Shape &s) {
    Layout l;
    add_padded_operands(l, s);
    return l;
}

// g: the pre-activation's gradient, or a padded copy of grad_output.
Layout backward_layout(const Shape &s, int activation) {
    Layout l;
    add_padded_operands(l, s);
    const bool narrow = s.dtype != FDA_DTYPE_F32;
    if (activation != FDA_ACT_NONE || (narrow && s.out_features % 8))
        l.g = l.take(total_rows(s) * (narrow ? padded(s.out_features) : s.out_features) * type_size(s.dtype));
    const Cut c = weight_cut(s);
    l.slots = l.take((size_t)c.slots * s.out_features * s.in_features * sizeof(float));
    l.bias_slots = l.take((size_t)c.slots * s.out_features * sizeof(float));
    return l;
}

int forward_f32(const Shape &s, const Groups &g, const void *x, const void *weight, const void *bias, const void *residual, void *y,
                int activation, cudaStream_t st) {
    RowProduct<float> p;
    p.a = static_cast<const float *>(x);
    p.w = static_cast<const float *>(weight);
    p.bias = static_cast<const float *>(bias);
    p.extra = static_cast<const float *>(residual);
    p.out = static_cast<float *>(y);
    p.depth = p.in_features = s.in_features;
    p.cols = s.out_features;
    p.g = g;
    return run_rows<float, kForward>(p, activation, st);
}

int forward_narrow(const Shape &s, const Groups &g, const void *x, const void *weight, const void *bias, const void *residual, void *y,
                   char *ws, int activation, cudaStream_t st) {
    const Layout l = forward_layout(s);
    if (const int rc = aligned_rows(x, ws + l.x, total_rows(s), s.in_features, st)) return rc;
    if (const int rc = aligned_rows(weight, ws + l.w, (size_t)s.groups * s.out_features, s.in_features, st)) return rc;
    const long long in = padded(s.in_features);
    const MmaRows p{x, weight, bias, residual, y, in, in, s.out_features, s.out_features, s.in_features, s.out_features, s.dtype, activation, g};
    return mma_rows(kForward, p, st);
}

struct Gradients {
    void *x, *weight, *bias;
};

template <typename T>
int sum_slots(const WeightGrad<T> &q, const Shape &s, const Cut &c, cudaStream_t st) {
    if (c.slots == 0) return FDA_OK;
    const bool split = c.pieces > 16ll * s.groups;
    const long long items = ceil_div(((long long)s.in_features + 1) * s.out_features, 32 * kLaneElements * (split ? 1 : kSumWarps)) * s.groups;
    const unsigned blocks = (unsigned)std::min<long long>(items, 4 * kSms);
    if (split) linear_weight_grad_sum_kernel<T, true><<<blocks, 32 * kSumWarps, 0, st>>>(q);
    else linear_weight_grad_sum_kernel<T, false><<<blocks, 32 * kSumWarps, 0, st>>>(q);
    return launched();
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

int backward_f32(const Shape &s, const Groups &g, const void *x, const void *weight, const void *bias, const void *grad_output,
                 const Gradients &out, char *ws, int activation, cudaStream_t st) {
    const Layout l = backward_layout(s, activation);
    RowProduct<float> p;
    p.w = static_cast<const float *>(weight);
    p.bias = static_cast<const float *>(bias);
    p.in_features = s.in_features;
    p.g = g;
    const float *grad = static_cast<const float *>(grad_output);
    if (activation != FDA_ACT_NONE) {
        p.a = static_cast<const float *>(x);
        p.extra = grad;
        p.out = reinterpret_cast<float *>(ws + l.g);
        p.depth = s.in_features;
        p.cols = s.out_features;
        if (const int rc = run_rows<float, kPreGrad>(p, activation, st)) return rc;
        grad = p.out;
    }
    if (out.x) {
        p.a = grad;
        p.bias = p.extra = nullptr;
        p.out = static_cast<float *>(out.x);
        p.depth = s.out_features;
        p.cols = s.in_features;
        if (const int rc = run_rows<float, kGradX>(p, FDA_ACT_NONE, st)) return rc;
    }
    if (!out.weight && !out.bias) return FDA_OK;
    const Cut c = weight_cut(s);
    const WeightGrad<float> q = weight_grad_args<float>(s, g, c, grad, x, out, ws, l);
    const long long items = c.pieces * ceil_div(s.out_features, kTileSize) * ceil_div(s.in_features, kTileSize);
    linear_weight_grad_kernel<float, kTileSize, kTileSize><<<(unsigned)std::min<long long>(items, 8 * kSms), kThreads, 0, st>>>(q);
    if (const int rc = launched()) return rc;
    return sum_slots(q, s, c, st);
}

int backward_narrow(const Shape &s, const Groups &g, const void *x, const void *weight, const void *bias, const void *grad_output,
                    const Gradients &out, char *ws, int activation, cudaStream_t st) {
    const Layout l = backward_layout(s, activation);
    const bool weights = out.weight || out.bias;
    const long long in = padded(s.in_features), outs = padded(s.out_features);
    if (activation != FDA_ACT_NONE || weights)
        if (const int rc = aligned_rows(x, ws + l.x, total_rows(s), s.in_features, st)) return rc;
    if (activation != FDA_ACT_NONE || out.x)
        if (const int rc = aligned_rows(weight, ws + l.w, (size_t)s.groups * s.out_features, s.in_features, st)) return rc;
    const void *grad = grad_output;
    if (activation != FDA_ACT_NONE) {
        const MmaRows p{x, weight, bias, grad_output, ws + l.g, in, in, s.out_features, outs, s.in_features, s.out_features, s.dtype,
                        activation, g};
        if (const int rc = mma_rows(kPreGrad, p, st)) return rc;
        grad = ws + l.g;
    } else if (const int rc = aligned_rows(grad, ws + l.g, total_rows(s), s.out_features, st)) {
        return rc;
    }
    if (out.x) {
        const MmaRows p{grad, weight, nullptr, nullptr, out.x, outs, in, 0, s.in_features, s.in_features, s.out_features, s.dtype,
                        FDA_ACT_NONE, g};
        if (const int rc = mma_rows(kGradX, p, st)) return rc;
    }
    if (!weights) return FDA_OK;
    const Cut c = weight_cut(s);
    const MmaWeightGrad q{grad, x, outs, in, out.weight, out.bias, reinterpret_cast<float *>(ws + l.slots),
                          reinterpret_cast<float *>(ws + l.bias_slots), s.in_features, s.out_features, s.dtype, c, g};
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
    if ((uintptr_t)workspace % 256) return FDA_ERR_MISALIGNED;
    const Groups g{group_start_index, num_starts, groups, batch, rows};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == FDA_DTYPE_F32) return forward_f32(s, g, x, weight, bias, residual, y, activation, st);
    if (misaligned16(x) || misaligned16(weight)) return FDA_ERR_MISALIGNED;
    return forward_narrow(s, g, x, weight, bias, residual, y, static_cast<char *>(workspace), activation, st);
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
    if ((uintptr_t)workspace % 256) return FDA_ERR_MISALIGNED;
    const Groups g{group_start_index, num_starts, groups, batch, rows};
    const Gradients out{grad_x, grad_weight, grad_bias};
    char *ws = static_cast<char *>(workspace);
    if (dtype == FDA_DTYPE_F32) return backward_f32(s, g, x, weight, bias, grad_output, out, ws, activation, st);
    if (misaligned16(x) || misaligned16(weight) || misaligned16(grad_output)) return FDA_ERR_MISALIGNED;
    return backward_narrow(s, g, x, weight, bias, grad_output, out, ws, activation, st);
}

int fda_linear_timeouts(void) {
    const int a = mma_timeouts_f16(), b = mma_timeouts_bf16();
    return a < 0 || b < 0 ? -1 : a + b;
}

}  // extern "C"

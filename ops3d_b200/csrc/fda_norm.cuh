// Layer norm of a residual sum, forward and backward.
//
//     s = x + residual,   mu = mean(s),   d = s - mu,   q = 1 / sqrt(mean(d d) + eps),   y = d q weight + bias          per row
//     g = dy weight,   ds = q (g - mean(g) - d q^2 mean(g d)) + dsum,   dweight = sum over rows of dy d q,   dbias = sum of dy
//
// One pass over memory in each direction: a row stays in the registers of the threads that share it (8 or 32 lanes of a warp, or a
// block), while its mean and then the sums of the deviations are taken, so the variance has no cancellation.  Nothing is kept for
// the backward but x and residual: the statistics come from the row again, which is there anyway.  Bound by DRAM traffic.
//
// Rows of any width are read in aligned 16-byte vectors.  Row r starts r * width elements into the tensor, that is at element
// (r * width) mod kWidth of a vector; rows a multiple of kWidth apart start at the same one.  A team takes such rows only, so its lanes
// keep their columns: parameters and the partial sums of dweight and dbias stay in registers.  Elements of the neighbouring rows in
// a row's first and last vector are masked out.
#pragma once

#include "fda_rows.cuh"

namespace fda_norm {

using namespace fda_rows;

struct NormArgs {
    const void *x, *residual, *weight, *bias;  // all but x may be nullptr
    const void *grad_y, *grad_sum;             // grad_sum may be nullptr
    void *y, *sum;                             // sum may be nullptr
    void *grad_x, *grad_residual;              // each may be nullptr
    float *partial;                            // [blocks][2][width], nullptr where the parameters have no gradient
    long long rows;
    int width, param_dtype;
    float eps;
};

constexpr int kTeamThreads = 256;   // of a block whose teams are lanes of a warp
constexpr int kBlockThreads = 512;  // most threads of a block that is a team

template <typename T> constexpr int kWidthOf = 16 / (int)sizeof(T);

// Vectors of one row that belong to a lane: columns, and whether they are all inside.
template <int kWidth, int kVectors, int kLanes, bool kRagged>
struct Columns {
    int first[kVectors];  // may be negative where kRagged
    int width;
    __device__ __forceinline__ Columns(int width, long long row, int lane, int size) : width(width) {
        const int shift = kRagged ? (int)((row * width) % kWidth) : 0;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) first[i] = (i * size + lane) * kWidth - shift;
    }
    __device__ __forceinline__ bool any(int i) const { return first[i] < width; }
    __device__ __forceinline__ bool whole(int i) const { return !kRagged || (first[i] >= 0 && first[i] + kWidth <= width); }
    __device__ __forceinline__ bool has(int i, int j) const { return kRagged ? first[i] + j >= 0 && first[i] + j < width : first[i] < width; }
};

template <typename T, int kWidth, bool kRagged>
__device__ __forceinline__ void load_vector(Raw<T, kWidth> &raw, const T *tensor, long long at, long long total) {
    if (kRagged && at + kWidth > total) {  // the tensor ends inside the vector
        alignas(16) T v[kWidth];
        for (int j = 0; j < kWidth; ++j) v[j] = at + j < total ? tensor[at + j] : from_f32<T>(0.f);
        raw.load(v);
        return;
    }
    raw.load(tensor + at);
}

template <typename T, int kWidth, int kVectors, int kLanes, bool kRagged>
__device__ __forceinline__ void load_row(Raw<T, kWidth> (&raw)[kVectors], const void *tensor, const Columns<kWidth, kVectors, kLanes, kRagged> &c,
                                         long long row, long long rows) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        if (row < rows && c.any(i)) load_vector<T, kWidth, kRagged>(raw[i], static_cast<const T *>(tensor), row * c.width + c.first[i], rows * c.width);
        else raw[i].clear();
    }
}

template <typename T, int kWidth, int kVectors, int kLanes, bool kRagged>
__device__ __forceinline__ void store_vector(void *tensor, const float *v, const Columns<kWidth, kVectors, kLanes, kRagged> &c, int i, long long row) {
    T *at = static_cast<T *>(tensor) + row * c.width + c.first[i];
    if (c.whole(i)) {
        Raw<T, kWidth> raw;
        raw.set(v);
        raw.store(at);
        return;
    }
#pragma unroll
    for (int j = 0; j < kWidth; ++j)
        if (c.has(i, j)) at[j] = from_f32<T>(v[j]);
}

// Which rows a team takes: the first one, and how far apart they are (a multiple of kWidth, because a grid's blocks are where a block
// is a team, and a block's teams are otherwise).
template <int kLanes>
__device__ __forceinline__ void team_rows(long long &first, long long &step) {
    if (kLanes == 0) {
        first = blockIdx.x;
        step = gridDim.x;
    } else {
        constexpr int kTeams = kTeamThreads / (kLanes ? kLanes : 1);
        first = (long long)blockIdx.x * kTeams + threadIdx.x / (kLanes ? kLanes : 1);
        step = (long long)gridDim.x * kTeams;
    }
}

// Shared memory of the sums over a block.
template <int kLanes>
__device__ __forceinline__ Team<kLanes> make_team() {
    Team<kLanes> team;
    if constexpr (kLanes == 0) {
        __shared__ float sums[2][Team<0>::kMost][Team<0>::kWarps];
        team.shared = sums;
    }
    return team;
}

// R: the residual's type; kResidual false: there is none.
template <typename T, typename R, bool kResidual, int kVectors, int kLanes, bool kRagged>
__global__ void __launch_bounds__(kLanes ? kTeamThreads : kBlockThreads) norm_forward_kernel(const NormArgs p) {
    constexpr int W = kWidthOf<T>;
    wait_for_previous_kernel();
    Team<kLanes> team = make_team<kLanes>();
    long long row, step;
    team_rows<kLanes>(row, step);
    const Columns<W, kVectors, kLanes, kRagged> c(p.width, row, team.lane(), team.size());
    Raw<T, W> x[kVectors];
    Raw<R, W> r[kVectors];
    load_row<T>(x, p.x, c, row, p.rows);
    if (kResidual) load_row<R>(r, p.residual, c, row, p.rows);
    float weight[kVectors][W], bias[kVectors][W];
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) {
            weight[i][j] = p.weight && c.has(i, j) ? load_as_f32(p.weight, p.param_dtype, c.first[i] + j) : 1.f;
            bias[i][j] = p.bias && c.has(i, j) ? load_as_f32(p.bias, p.param_dtype, c.first[i] + j) : 0.f;
        }
    const float inverse = 1.f / (float)p.width;
    // every lane of a warp stays to the end: they exchange sums
    const long long lanes_first = kLanes ? row - threadIdx.x % 32 / (kLanes ? kLanes : 1) : row;
    for (long long base = lanes_first; base < p.rows; base += step, row += step) {
        float s[kVectors][W], sums[1] = {0.f};
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            x[i].get(s[i]);
            if (kResidual) {
                float extra[W];
                r[i].get(extra);
#pragma unroll
                for (int j = 0; j < W; ++j) s[i][j] += extra[j];
            }
#pragma unroll
            for (int j = 0; j < W; ++j) sums[0] += c.has(i, j) ? s[i][j] : 0.f;
        }
        load_row<T>(x, p.x, c, row + step, p.rows);
        if (kResidual) load_row<R>(r, p.residual, c, row + step, p.rows);
        if (kResidual && p.sum && row < p.rows) {
#pragma unroll
            for (int i = 0; i < kVectors; ++i)
                if (c.any(i)) store_vector<R>(p.sum, s[i], c, i, row);
        }
        team.sum(sums);
        const float mean = sums[0] * inverse;
        sums[0] = 0.f;
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                s[i][j] = c.has(i, j) ? s[i][j] - mean : 0.f;
                sums[0] += s[i][j] * s[i][j];
            }
        team.sum(sums);
        const float q = __frsqrt_rn(sums[0] * inverse + p.eps);
        if (row >= p.rows) continue;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            if (!c.any(i)) continue;
#pragma unroll
            for (int j = 0; j < W; ++j) s[i][j] = s[i][j] * q * weight[i][j] + bias[i][j];
            store_vector<T>(p.y, s[i], c, i, row);
        }
    }
}

template <typename T, typename R, bool kResidual, int kVectors, int kLanes, bool kRagged>
__global__ void __launch_bounds__(kLanes ? kTeamThreads : kBlockThreads) norm_backward_kernel(const NormArgs p) {
    constexpr int W = kWidthOf<T>;
    wait_for_previous_kernel();
    Team<kLanes> team = make_team<kLanes>();
    long long row, step;
    team_rows<kLanes>(row, step);
    const Columns<W, kVectors, kLanes, kRagged> c(p.width, row, team.lane(), team.size());
    Raw<T, W> x[kVectors], dy[kVectors];
    Raw<R, W> r[kVectors];
    load_row<T>(x, p.x, c, row, p.rows);
    load_row<T>(dy, p.grad_y, c, row, p.rows);
    if (kResidual) load_row<R>(r, p.residual, c, row, p.rows);
    float weight[kVectors][W], grad_weight[kVectors][W], grad_bias[kVectors][W];
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) {
            weight[i][j] = p.weight && c.has(i, j) ? load_as_f32(p.weight, p.param_dtype, c.first[i] + j) : 1.f;
            grad_weight[i][j] = grad_bias[i][j] = 0.f;
        }
    const float inverse = 1.f / (float)p.width;
    const long long lanes_first = kLanes ? row - threadIdx.x % 32 / (kLanes ? kLanes : 1) : row;
    for (long long base = lanes_first; base < p.rows; base += step, row += step) {
        float d[kVectors][W], g[kVectors][W], mean[1] = {0.f};
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            x[i].get(d[i]);
            dy[i].get(g[i]);
            if (kResidual) {
                float extra[W];
                r[i].get(extra);
#pragma unroll
                for (int j = 0; j < W; ++j) d[i][j] += extra[j];
            }
#pragma unroll
            for (int j = 0; j < W; ++j) mean[0] += c.has(i, j) ? d[i][j] : 0.f;
        }
        load_row<T>(x, p.x, c, row + step, p.rows);
        load_row<T>(dy, p.grad_y, c, row + step, p.rows);
        if (kResidual) load_row<R>(r, p.residual, c, row + step, p.rows);
        team.sum(mean);
        mean[0] *= inverse;
        float sums[3] = {0.f, 0.f, 0.f};  // of d d, g d, g
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                d[i][j] = c.has(i, j) ? d[i][j] - mean[0] : 0.f;
                const float gw = c.has(i, j) ? g[i][j] * weight[i][j] : 0.f;
                sums[0] += d[i][j] * d[i][j];
                sums[1] += gw * d[i][j];
                sums[2] += gw;
            }
        team.sum(sums);
        const float q = __frsqrt_rn(sums[0] * inverse + p.eps);
        const float along = q * q * sums[1] * inverse, level = sums[2] * inverse;
        if (row >= p.rows) continue;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            if (!c.any(i)) continue;
            float ds[W];
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float dyv = c.has(i, j) ? g[i][j] : 0.f;
                ds[j] = q * (dyv * weight[i][j] - level - d[i][j] * along);
                grad_weight[i][j] += dyv * (d[i][j] * q);
                grad_bias[i][j] += dyv;
            }
            if (kResidual && p.grad_sum) {
                Raw<R, W> raw;
                load_vector<R, W, kRagged>(raw, static_cast<const R *>(p.grad_sum), row * p.width + c.first[i], p.rows * p.width);
                float extra[W];
                raw.get(extra);
#pragma unroll
                for (int j = 0; j < W; ++j) ds[j] += extra[j];
            }
            if (p.grad_x) store_vector<T>(p.grad_x, ds, c, i, row);
            if (kResidual && p.grad_residual) store_vector<R>(p.grad_residual, ds, c, i, row);
        }
    }
    if (!p.partial) return;
    // the block's sums, column by column; with several teams in a fixed order
    float *out = p.partial + (size_t)blockIdx.x * 2 * p.width;
    if constexpr (kLanes == 0) {
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (c.has(i, j)) {
                    out[c.first[i] + j] = grad_weight[i][j];
                    out[p.width + c.first[i] + j] = grad_bias[i][j];
                }
    } else {
        extern __shared__ float columns[];  // [2][width]
        for (int i = threadIdx.x; i < 2 * p.width; i += kTeamThreads) columns[i] = 0.f;
        for (int t = 0; t < kTeamThreads / (kLanes ? kLanes : 1); ++t) {
            __syncthreads();
            if ((int)threadIdx.x / (kLanes ? kLanes : 1) != t) continue;
#pragma unroll
            for (int i = 0; i < kVectors; ++i)
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (c.has(i, j)) {
                        columns[c.first[i] + j] += grad_weight[i][j];
                        columns[p.width + c.first[i] + j] += grad_bias[i][j];
                    }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * p.width; i += kTeamThreads) out[i] = columns[i];
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------
// Threads that share a row, and vectors of each.
struct NormShape {
    int lanes, vectors, threads;
    bool ragged;
};
// Up to 16 values of a row in a lane: twice as many spill in the backward (its sums take as many registers again).
constexpr int kMostValues = 16;
inline int most_fast_width(int) { return kBlockThreads * kMostValues - 16; }

inline NormShape norm_shape(int width, int dtype) {
    const int W = dtype == FDA_DTYPE_F32 ? 4 : 8;
    NormShape s;
    s.ragged = width % W != 0;
    const int vectors = (width + (s.ragged ? W - 1 : 0) + W - 1) / W;
    s.lanes = vectors <= 8 ? 8 : 32;
    s.threads = kTeamThreads;
    s.vectors = 1;
    while (s.vectors * W < kMostValues && s.lanes * s.vectors < vectors) s.vectors *= 2;
    if (s.lanes * s.vectors < vectors) {
        s.lanes = 0;
        s.threads = (int)ceil_div(ceil_div(vectors, s.vectors), 32) * 32;
    }
    return s;
}

// Blocks: as many as rows need, at most what fills the device; a multiple of 8 where a block is a team (rows 8 apart).
inline unsigned norm_blocks(const NormShape &s, long long rows, int most_per_sm) {
    const long long per_block = s.lanes ? s.threads / s.lanes : 1;
    const long long needed = ceil_div(rows, per_block);
    const long long room = (long long)kSms * most_per_sm;
    long long blocks = needed < room ? needed : room;
    if (!s.lanes) blocks = ceil_div(blocks, 8) * 8;
    return (unsigned)blocks;
}

// The kernels of one type (fda_norm_f32.cu and so on).
int norm_f32(bool backward, const NormArgs &p, const NormShape &s, int residual_dtype, unsigned blocks, cudaStream_t st);
int norm_f16(bool backward, const NormArgs &p, const NormShape &s, int residual_dtype, unsigned blocks, cudaStream_t st);
int norm_bf16(bool backward, const NormArgs &p, const NormShape &s, int residual_dtype, unsigned blocks, cudaStream_t st);

template <typename T, typename R, bool kResidual, int kVectors, int kLanes>
int run_norm(bool backward, const NormArgs &p, const NormShape &s, unsigned blocks, cudaStream_t st) {
    if (backward) {
        const int shared = kLanes && p.partial ? 2 * p.width * (int)sizeof(float) : 0;
        return launched(launch_early(s.ragged ? norm_backward_kernel<T, R, kResidual, kVectors, kLanes, true>
                                              : norm_backward_kernel<T, R, kResidual, kVectors, kLanes, false>,
                                     blocks, s.threads, shared, st, 1, p));
    }
    return launched(launch_early(s.ragged ? norm_forward_kernel<T, R, kResidual, kVectors, kLanes, true>
                                          : norm_forward_kernel<T, R, kResidual, kVectors, kLanes, false>,
                                 blocks, s.threads, 0, st, 1, p));
}

template <typename T, typename R, bool kResidual>
int run_norm(bool backward, const NormArgs &p, const NormShape &s, unsigned blocks, cudaStream_t st) {
    constexpr int kMost = kMostValues / kWidthOf<T>;
    if (s.lanes == 8) return run_norm<T, R, kResidual, 1, 8>(backward, p, s, blocks, st);
    if (s.lanes == 32) {
        if (s.vectors == 1) return run_norm<T, R, kResidual, 1, 32>(backward, p, s, blocks, st);
        if (s.vectors == 2) return run_norm<T, R, kResidual, 2, 32>(backward, p, s, blocks, st);
        return run_norm<T, R, kResidual, kMost, 32>(backward, p, s, blocks, st);
    }
    return run_norm<T, R, kResidual, kMost, 0>(backward, p, s, blocks, st);
}

template <typename T>
int run_norm(bool backward, const NormArgs &p, const NormShape &s, int residual_dtype, unsigned blocks, cudaStream_t st) {
    if (!p.residual) return run_norm<T, T, false>(backward, p, s, blocks, st);
    if (sizeof(T) == 2 && residual_dtype == FDA_DTYPE_F32) return run_norm<T, float, true>(backward, p, s, blocks, st);
    return run_norm<T, T, true>(backward, p, s, blocks, st);
}

}  // namespace fda_norm

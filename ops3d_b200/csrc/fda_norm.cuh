// Layer norm of a residual sum, forward and backward.
//
//     s = x + residual,   mu = mean(s),   d = s - mu,   q = 1 / sqrt(mean(d d) + eps),   y = d q weight + bias          per row
//     g = dy weight,   ds = q (g - mean(g) - d q^2 mean(g d)) + dsum,   dweight = sum over rows of dy d q,   dbias = sum of dy
//
// One pass over memory in each direction: a row stays in the registers of the threads that share it (4 to 32 lanes of a warp, or
// a block), while its mean and then the sums of the deviations are taken, so the variance has no cancellation.  Nothing is kept for
// the backward but x and residual: the statistics come from the row again, which is there anyway.  Bound by DRAM traffic.
//
// Rows of any width are read in aligned 16-byte vectors.  Row r starts r * width elements into the tensor, that is at element
// (r * width) mod kWidth of a vector; rows a multiple of kWidth apart start at the same one.  A team takes such rows only, so its lanes
// keep their columns: parameters and the partial sums of dweight and dbias stay in registers.  Elements of the neighbouring rows in
// a row's first and last vector are masked out.
#pragma once

#include "fda_norm_copy.h"
#include "fda_rows.cuh"

#include <algorithm>

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

constexpr int kTeamThreads = 256;    // of a block whose teams are lanes of a warp
constexpr int kBlockThreads = 1024;  // most threads of a block that is a team

template <typename T> constexpr int kWidthOf = 16 / (int)sizeof(T);

// Vectors of a row that belong to a lane.
template <int kWidth, int kVectors, bool kRagged>
struct Columns {
    int width;
    int first[kVectors];                // column of the first element; may be negative where kRagged
    int count[kVectors];                // elements from the first to the row's end, at most kWidth; 0 where the row has none
    unsigned bits[kVectors];            // bit j: element j is one of the row's
    Pair valid[kVectors][kRagged ? kWidth / 2 : 1];  // the same as factors
    unsigned keep[kVectors][kRagged ? 4 : 1];        // and as a mask of the vector's words
    __device__ __forceinline__ Columns(int width, long long row, int lane, int size) : width(width) {
        const int shift = kRagged ? (int)((row * width) % kWidth) : 0;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            first[i] = (i * size + lane) * kWidth - shift;
            count[i] = max(0, min(kWidth, width - first[i]));
            bits[i] = (1u << count[i]) - 1;
            if constexpr (kRagged) {
                if (first[i] < 0) bits[i] &= ~((1u << -first[i]) - 1);
#pragma unroll
                for (int k = 0; k < 4; ++k) keep[i][k] = 0;
#pragma unroll
                for (int j = 0; j < kWidth / 2; ++j) valid[i][j] = Pair(has(i, 2 * j) ? 1.f : 0.f, has(i, 2 * j + 1) ? 1.f : 0.f);
#pragma unroll
                for (int j = 0; j < kWidth; ++j) {
                    if (has(i, j)) keep[i][j * 4 / kWidth] |= kWidth == 4 ? 0xffffffffu : 0xffffu << (j % 2 * 16);
                }
            } else {
                valid[i][0] = Pair(count[i] ? 1.f : 0.f);
            }
        }
    }
    __device__ __forceinline__ bool any(int i) const { return count[i] != 0; }
    __device__ __forceinline__ bool whole(int i) const { return !kRagged || bits[i] == (1u << kWidth) - 1; }
    __device__ __forceinline__ bool has(int i, int j) const { return bits[i] >> j & 1; }
    __device__ __forceinline__ Pair ones(int i, int j) const { return valid[i][kRagged ? j : 0]; }  // of elements 2 j and 2 j + 1
};

// Rows on their way: every lane copies vectors into its own places of a ring in shared memory, kStages - 1 rows ahead of the one that it
// works on.  They are its own vectors, so that nothing has to wait for another lane; where a vector has 32 bytes (an fp32 residual beside 16-bit
// rows) lanes of a warp share them, so that their copies still cover whole lines (598016 x 256 forward 271 us without, 181 with).
__device__ __forceinline__ void copy16(unsigned to, const void *from, int bytes) {  // the rest of the 16 becomes 0
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// at: where the row's first vector of the lane starts in the tensor; left: rows from this one on.  kLanes: neighbouring lanes that share
// the row.
template <typename E, int kLanes, int kWidth, int kVectors, bool kRagged>
__device__ __forceinline__ void copy_row(unsigned slot, unsigned pitch, const void *tensor, const Columns<kWidth, kVectors, kRagged> &c,
                                         long long at, long long left) {
    constexpr int kUnits = kWidth * (int)sizeof(E) / 16, kEach = 16 / (int)sizeof(E);
    const int lane = threadIdx.x % kLanes, room = kRagged ? room_of(left, c.width, kEach) : 0;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            // elements from the lane's own vector to what it copies
            const int ahead = kUnits == 1 ? 0 : (u * kLanes + lane) * kEach - lane * kWidth;
            const int rest = kUnits == 1 ? c.count[i] : c.width - (c.first[i] + ahead);
            const int bytes = kRagged ? copied_elements(c.first[i] + ahead, c.width, kEach, room) * (int)sizeof(E) : rest <= 0 || left <= 0 ? 0 : 16;
            const E *from = static_cast<const E *>(tensor) + at + (c.first[i] - c.first[0]) + ahead;
            copy16(slot + (i * kUnits + u) * pitch, bytes ? from : tensor, bytes);
        }
    }
}

// A lane's vector i from its place, elements of neighbouring rows as 0.
template <typename E, int kLanes, int kWidth, int kVectors, bool kRagged>
__device__ __forceinline__ void read_vector(const char *slot, unsigned pitch, const Columns<kWidth, kVectors, kRagged> &c, int i, Pair *v) {
    constexpr int kUnits = kWidth * (int)sizeof(E) / 16;
    Raw<E, kWidth> raw;
    if constexpr (kUnits == 1) {
        raw.u[0] = *reinterpret_cast<const uint4 *>(slot + i * pitch);
        if constexpr (kRagged) {
            raw.u[0].x &= c.keep[i][0];
            raw.u[0].y &= c.keep[i][1];
            raw.u[0].z &= c.keep[i][2];
            raw.u[0].w &= c.keep[i][3];
        }
        raw.get(v);
    } else {
        const int lane = threadIdx.x % kLanes;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int chunk = lane * kUnits + u;
            raw.u[u] = *reinterpret_cast<const uint4 *>(slot + (i * kUnits + chunk / kLanes) * pitch + (chunk % kLanes - lane) * 16);
        }
        float f[kWidth];
        raw.get(f);
        if (kRagged) {
#pragma unroll
            for (int j = 0; j < kWidth; ++j) f[j] = c.has(i, j) ? f[j] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < kWidth / 2; ++j) v[j] = Pair(f[2 * j], f[2 * j + 1]);
    }
}

// at: as above, of the row that is stored.
template <typename E, int kWidth, int kVectors, bool kRagged>
__device__ __forceinline__ void store_vector(void *tensor, const Pair *v, const Columns<kWidth, kVectors, kRagged> &c, int i, long long at) {
    E *to = static_cast<E *>(tensor) + at + (c.first[i] - c.first[0]);
    Raw<E, kWidth> raw;
    raw.set(v);
    if (c.whole(i)) {
        raw.store(to);
        return;
    }
#pragma unroll
    for (int j = 0; j < kWidth; ++j)
        if (c.has(i, j)) to[j] = raw.element(j);
}

// ds += the gradient that reaches the sum from elsewhere.
template <typename E, int kWidth, int kVectors, bool kRagged>
__device__ __forceinline__ void add_sum_gradient(const void *tensor, Pair *ds, const Columns<kWidth, kVectors, kRagged> &c, int i, long long at) {
    const E *from = static_cast<const E *>(tensor) + at + (c.first[i] - c.first[0]);
    float v[kWidth];
    if (c.whole(i)) {
        Raw<E, kWidth> raw;
        raw.load(from);
        raw.get(v);
    } else {
#pragma unroll
        for (int j = 0; j < kWidth; ++j) v[j] = c.has(i, j) ? to_f32(from[j]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kWidth / 2; ++j) ds[j] = ds[j] + Pair(v[2 * j], v[2 * j + 1]);
}

// A parameter's numbers for a lane's columns, `otherwise` where there is none.
template <typename E, int kWidth, int kVectors, bool kRagged>
__device__ __forceinline__ void load_parameter(const E *tensor, const Columns<kWidth, kVectors, kRagged> &c, float (&v)[kVectors][kWidth]) {
    const bool vector = !kRagged && (uintptr_t)tensor % 16 == 0;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        if (vector && c.any(i)) {
            Raw<E, kWidth> raw;
            raw.load(tensor + c.first[i]);
            raw.get(v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < kWidth; ++j)
                if (c.has(i, j)) v[i][j] = to_f32(tensor[c.first[i] + j]);
        }
    }
}
template <typename T, int kWidth, int kVectors, bool kRagged>
__device__ __forceinline__ void load_parameter(const void *tensor, int dtype, float otherwise, const Columns<kWidth, kVectors, kRagged> &c,
                                               Pair (&pairs)[kVectors][kWidth / 2]) {
    float v[kVectors][kWidth];
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < kWidth; ++j) v[i][j] = otherwise;
    if (tensor) {
        if (dtype == FDA_DTYPE_F32) load_parameter(static_cast<const float *>(tensor), c, v);
        else load_parameter(static_cast<const T *>(tensor), c, v);
    }
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < kWidth / 2; ++j) pairs[i][j] = Pair(v[i][2 * j], v[i][2 * j + 1]);
}

// Which rows a team of lanes takes: the first one, and how far apart they are (a multiple of kWidth, because a block's teams are).
template <int kLanes>
__device__ __forceinline__ void team_rows(long long &first, long long &step) {
    constexpr int kTeams = kTeamThreads / kLanes;
    first = (long long)blockIdx.x * kTeams + threadIdx.x / kLanes;
    step = (long long)gridDim.x * kTeams;
}

// The block as a team, with shared memory for its sums.
__device__ __forceinline__ Team<0> block_team() {
    __shared__ alignas(16) float sums[2][Team<0>::kMost][Team<0>::kWarps];
    for (int i = threadIdx.x; i < 2 * Team<0>::kMost * Team<0>::kWarps; i += blockDim.x) (&sums[0][0][0])[i] = 0.f;
    __syncthreads();
    Team<0> team;
    team.shared = sums;
    return team;
}

// 16-byte places of a lane for one row, rows of the ring, and (where teams are lanes) blocks to an SM.  They are so many that 48 KB or so are
// on their way to an SM: that covers DRAM's latency, and more makes it slower (598016 x 256 bf16 forward with a residual: 32 KB 144 us, 48 KB
// 138, 72 KB 185).
template <typename T, typename R, bool kResidual, int kVectors, bool kBackward>
constexpr int kUnitsOf = kVectors * ((kBackward ? 2 : 1) + (kResidual ? (int)(sizeof(R) / sizeof(T)) : 0));
template <int kUnits, int kLanes, bool kBackward>
constexpr int kStagesOf = kLanes == 0  ? (kUnits == 1 ? 4 : kUnits == 2 && !kBackward ? 3 : 2)
                          : kBackward ? (kUnits == 2 ? 4 : kUnits == 3 ? 3 : 2)
                                      : (kUnits <= 2 ? 4 : kUnits == 3 ? 3 : 2);
template <int kUnits>
constexpr int kForwardBlocks = kUnits == 1 ? 4 : kUnits == 4 ? 3 : 2;

// R: the residual's type; kResidual false: there is none.  598016 x 256 bf16: 103 us (5.9 TB/s), with a residual 139 (6.6 TB/s, the speed of a
// copy); rows that start anywhere cost instructions and, a vector beyond a power of two, half of the lanes: 100000 x 259 with a residual 53 us
// (2.9 TB/s).
template <typename T, typename R, bool kResidual, int kVectors, int kLanes, bool kRagged>
__global__ void __launch_bounds__(kTeamThreads) norm_forward_kernel(const NormArgs p) {
    constexpr int W = kWidthOf<T>, kUnits = kUnitsOf<T, R, kResidual, kVectors, false>, kStages = kStagesOf<kUnits, kLanes, false>;
    extern __shared__ uint4 ring[];
    wait_for_previous_kernel();
    Team<kLanes> team;
    long long row, step;
    team_rows<kLanes>(row, step);
    const Columns<W, kVectors, kRagged> c(p.width, row, team.lane(), team.size());
    const unsigned pitch = blockDim.x * 16, stage = pitch * kUnits;
    const char *const mine = reinterpret_cast<const char *>(ring + threadIdx.x);
    const unsigned slots = (unsigned)__cvta_generic_to_shared(mine);
    long long at = row * p.width + c.first[0], left = p.rows - row;  // of the next row to be copied, then of the one that is worked on
    const long long stride = step * p.width;
    const auto issue = [&](int s) {
        copy_row<T, kLanes>(slots + s * stage, pitch, p.x, c, at, left);
        if (kResidual) copy_row<R, kLanes>(slots + s * stage + kVectors * pitch, pitch, p.residual, c, at, left);
        copies_issued();
        at += stride;
        left -= step;
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s);
    constexpr int H = W / 2;
    Pair weight[kVectors][H], bias[kVectors][H];
    load_parameter<T>(p.weight, p.param_dtype, 1.f, c, weight);
    load_parameter<T>(p.bias, p.param_dtype, 0.f, c, bias);
    const float inverse = 1.f / (float)p.width;
    // every lane of a warp stays to the end: they exchange sums
    int s = 0;
    for (long long base = row - threadIdx.x % 32 / kLanes; base < p.rows; base += step, row += step) {
        Pair d[kVectors][H], add(0.f);
        float sums[1];
        wait_copies<kStages - 2>();
        if (kResidual && sizeof(R) > sizeof(T)) __syncwarp();  // other lanes' copies are there too, and the places of the row before are free
        const char *const slot = mine + s * stage;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            read_vector<T, kLanes>(slot, pitch, c, i, d[i]);
            if (kResidual) {
                Pair extra[H];
                read_vector<R, kLanes>(slot + kVectors * pitch, pitch, c, i, extra);
#pragma unroll
                for (int j = 0; j < H; ++j) d[i][j] = d[i][j] + extra[j];
            }
#pragma unroll
            for (int j = 0; j < H; ++j) add = add + d[i][j];
        }
        issue(s == 0 ? kStages - 1 : s - 1);
        const long long here = at - kStages * stride;
        s = s == kStages - 1 ? 0 : s + 1;
        if (kResidual && p.sum && row < p.rows) {
#pragma unroll
            for (int i = 0; i < kVectors; ++i)
                if (c.any(i)) store_vector<R>(p.sum, d[i], c, i, here);
        }
        sums[0] = add.sum();
        team.sum(sums);
        const Pair minus_mean(-sums[0] * inverse);
        Pair square(0.f);
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
#pragma unroll
            for (int j = 0; j < H; ++j) {
                d[i][j] = fma2(minus_mean, c.ones(i, j), d[i][j]);
                square = fma2(d[i][j], d[i][j], square);
            }
        sums[0] = square.sum();
        team.sum(sums);
        const Pair q(__frsqrt_rn(sums[0] * inverse + p.eps));
        if (row >= p.rows) continue;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            if (!c.any(i)) continue;
#pragma unroll
            for (int j = 0; j < H; ++j) d[i][j] = fma2(d[i][j] * q, weight[i][j], bias[i][j]);
            store_vector<T>(p.y, d[i], c, i, here);
        }
    }
    wait_copies<0>();
}

// 598016 x 256 bf16: 157 us (5.8 TB/s), with a residual 185 (6.6); 300000 x 64 with one 30 (5.1).  Two rounds of sums over the lanes, the second of
// three numbers; issue slots are 73 % busy.
template <typename T, typename R, bool kResidual, int kVectors, int kLanes, bool kRagged>
__global__ void __launch_bounds__(kTeamThreads) norm_backward_kernel(const NormArgs p) {
    constexpr int W = kWidthOf<T>, kUnits = kUnitsOf<T, R, kResidual, kVectors, true>, kStages = kStagesOf<kUnits, kLanes, true>;
    extern __shared__ uint4 ring[];
    wait_for_previous_kernel();
    Team<kLanes> team;
    long long row, step;
    team_rows<kLanes>(row, step);
    const Columns<W, kVectors, kRagged> c(p.width, row, team.lane(), team.size());
    const unsigned pitch = blockDim.x * 16, stage = pitch * kUnits;
    const char *const mine = reinterpret_cast<const char *>(ring + threadIdx.x);
    const unsigned slots = (unsigned)__cvta_generic_to_shared(mine);
    long long at = row * p.width + c.first[0], left = p.rows - row;
    const long long stride = step * p.width;
    const auto issue = [&](int s) {
        copy_row<T, kLanes>(slots + s * stage, pitch, p.x, c, at, left);
        copy_row<T, kLanes>(slots + s * stage + kVectors * pitch, pitch, p.grad_y, c, at, left);
        if (kResidual) copy_row<R, kLanes>(slots + s * stage + 2 * kVectors * pitch, pitch, p.residual, c, at, left);
        copies_issued();
        at += stride;
        left -= step;
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s);
    constexpr int H = W / 2;
    Pair weight[kVectors][H], weight_sum[kVectors][H], bias_sum[kVectors][H];
    load_parameter<T>(p.weight, p.param_dtype, 1.f, c, weight);
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < H; ++j) weight_sum[i][j] = bias_sum[i][j] = Pair(0.f);
    const float inverse = 1.f / (float)p.width;
    int s = 0;
    for (long long base = row - threadIdx.x % 32 / kLanes; base < p.rows; base += step, row += step) {
        Pair d[kVectors][H], dy[kVectors][H], add(0.f);
        wait_copies<kStages - 2>();
        if (kResidual && sizeof(R) > sizeof(T)) __syncwarp();  // other lanes' copies are there too, and the places of the row before are free
        const char *const slot = mine + s * stage;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            read_vector<T, kLanes>(slot, pitch, c, i, d[i]);
            read_vector<T, kLanes>(slot + kVectors * pitch, pitch, c, i, dy[i]);
            if (kResidual) {
                Pair extra[H];
                read_vector<R, kLanes>(slot + 2 * kVectors * pitch, pitch, c, i, extra);
#pragma unroll
                for (int j = 0; j < H; ++j) d[i][j] = d[i][j] + extra[j];
            }
#pragma unroll
            for (int j = 0; j < H; ++j) add = add + d[i][j];
        }
        issue(s == 0 ? kStages - 1 : s - 1);
        const long long here = at - kStages * stride;
        s = s == kStages - 1 ? 0 : s + 1;
        float mean[1] = {add.sum()};
        team.sum(mean);
        const Pair minus_mean(-mean[0] * inverse);
        Pair dd(0.f), gd(0.f), gg(0.f);
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
#pragma unroll
            for (int j = 0; j < H; ++j) {
                d[i][j] = fma2(minus_mean, c.ones(i, j), d[i][j]);
                const Pair g = dy[i][j] * weight[i][j];
                dd = fma2(d[i][j], d[i][j], dd);
                gd = fma2(g, d[i][j], gd);
                gg = gg + g;
            }
        float sums[3] = {dd.sum(), gd.sum(), gg.sum()};
        team.sum(sums);
        const float scale = __frsqrt_rn(sums[0] * inverse + p.eps);
        if (row >= p.rows) continue;
        const Pair q(scale), level(-scale * (sums[2] * inverse)), along(-scale * (scale * scale * (sums[1] * inverse)));
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            if (!c.any(i)) continue;
            Pair ds[H];
#pragma unroll
            for (int j = 0; j < H; ++j) {
                ds[j] = fma2(dy[i][j] * weight[i][j], q, fma2(d[i][j], along, level));
                weight_sum[i][j] = fma2(dy[i][j], d[i][j] * q, weight_sum[i][j]);
                bias_sum[i][j] = bias_sum[i][j] + dy[i][j];
            }
            if (kResidual && p.grad_sum) add_sum_gradient<R>(p.grad_sum, ds, c, i, here);
            if (p.grad_x) store_vector<T>(p.grad_x, ds, c, i, here);
            if (kResidual && p.grad_residual) store_vector<R>(p.grad_residual, ds, c, i, here);
        }
    }
    wait_copies<0>();
    if (!p.partial) return;
    // the block's sums, column by column; with several teams in a fixed order
    float grad_weight[kVectors][W], grad_bias[kVectors][W];
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < H; ++j) {
            weight_sum[i][j].get(grad_weight[i][2 * j], grad_weight[i][2 * j + 1]);
            bias_sum[i][j].get(grad_bias[i][2 * j], grad_bias[i][2 * j + 1]);
        }
    float *out = p.partial + (size_t)blockIdx.x * 2 * p.width;
    // teams of a warp have the same columns unless rows are ragged
    constexpr int kTeams = kRagged ? kTeamThreads / kLanes : kTeamThreads / 32;
    if (!kRagged) {
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j)
                for (int o = kLanes; o < 32; o *= 2) {
                    grad_weight[i][j] += __shfl_xor_sync(0xffffffffu, grad_weight[i][j], o);
                    grad_bias[i][j] += __shfl_xor_sync(0xffffffffu, grad_bias[i][j], o);
                }
    }
    __syncthreads();
    float *columns = reinterpret_cast<float *>(ring);  // [kTeams][2][width]
    const int t = kRagged ? (int)threadIdx.x / kLanes : (int)threadIdx.x / 32;
    if (kRagged || threadIdx.x % 32 < kLanes) {
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (c.has(i, j)) {
                    columns[t * 2 * p.width + c.first[i] + j] = grad_weight[i][j];
                    columns[(t * 2 + 1) * p.width + c.first[i] + j] = grad_bias[i][j];
                }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.width; i += kTeamThreads) {
        float sum = 0.f;
#pragma unroll 8
        for (int k = 0; k < kTeams; ++k) sum += columns[k * 2 * p.width + i];
        out[i] = sum;
    }
}

// ---- a block to a row ----------------------------------------------------------------------------------------------------------
// As above, for rows that a warp has no registers for.  A row's mean is taken together with the sums of the row before it, so that the block
// meets once for a row: a row's time is that of the barrier and the exchange around it (100000 x 640 bf16 forward: two meetings 76 us, one 58).
template <typename T, typename R, bool kResidual, int kVectors, bool kRagged>
__global__ void __launch_bounds__(kBlockThreads) norm_forward_block_kernel(const NormArgs p) {
    constexpr int W = kWidthOf<T>, H = W / 2, kUnits = kUnitsOf<T, R, kResidual, kVectors, false>, kStages = kStagesOf<kUnits, 0, false>;
    extern __shared__ uint4 ring[];
    wait_for_previous_kernel();
    Team<0> team = block_team();
    const Columns<W, kVectors, kRagged> c(p.width, blockIdx.x, team.lane(), team.size());
    const unsigned pitch = blockDim.x * 16, stage = pitch * kUnits;
    const char *const mine = reinterpret_cast<const char *>(ring + threadIdx.x);
    const unsigned slots = (unsigned)__cvta_generic_to_shared(mine);
    long long at = (long long)blockIdx.x * p.width + c.first[0], left = p.rows - blockIdx.x;  // of the next row to be copied
    const long long stride = (long long)gridDim.x * p.width;
    const auto issue = [&](int s) {
        copy_row<T, 32>(slots + s * stage, pitch, p.x, c, at, left);
        if (kResidual) copy_row<R, 32>(slots + s * stage + kVectors * pitch, pitch, p.residual, c, at, left);
        copies_issued();
        at += stride;
        left -= gridDim.x;
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s);
    Pair weight[kVectors][H], bias[kVectors][H];
    load_parameter<T>(p.weight, p.param_dtype, 1.f, c, weight);
    load_parameter<T>(p.bias, p.param_dtype, 0.f, c, bias);
    const float inverse = 1.f / (float)p.width;
    int s = 0;
    // the row of place s, whose sum is returned; the place of the row before it is filled again
    const auto read_row = [&](Pair (&d)[kVectors][H], bool there) {
        wait_copies<kStages - 2>();
        if (kResidual && sizeof(R) > sizeof(T)) __syncwarp();
        const char *const slot = mine + s * stage;
        Pair add(0.f);
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            read_vector<T, 32>(slot, pitch, c, i, d[i]);
            if (kResidual) {
                Pair extra[H];
                read_vector<R, 32>(slot + kVectors * pitch, pitch, c, i, extra);
#pragma unroll
                for (int j = 0; j < H; ++j) d[i][j] = d[i][j] + extra[j];
            }
#pragma unroll
            for (int j = 0; j < H; ++j) add = add + d[i][j];
        }
        issue(s == 0 ? kStages - 1 : s - 1);
        s = s == kStages - 1 ? 0 : s + 1;
        if (kResidual && p.sum && there) {
#pragma unroll
            for (int i = 0; i < kVectors; ++i)
                if (c.any(i)) store_vector<R>(p.sum, d[i], c, i, at - kStages * stride);
        }
        return add.sum();
    };
    Pair d[kVectors][H], ahead[kVectors][H];
    float sums[2] = {0.f, read_row(d, blockIdx.x < p.rows)};
    team.sum(sums);
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const Pair minus_mean(-sums[1] * inverse);
        Pair square(0.f);
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
#pragma unroll
            for (int j = 0; j < H; ++j) {
                d[i][j] = fma2(minus_mean, c.ones(i, j), d[i][j]);
                square = fma2(d[i][j], d[i][j], square);
            }
        sums[1] = read_row(ahead, row + gridDim.x < p.rows);
        sums[0] = square.sum();
        team.sum(sums);
        const Pair q(__frsqrt_rn(sums[0] * inverse + p.eps));
        const long long here = at - (kStages + 1) * stride;
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            if (c.any(i)) {
#pragma unroll
                for (int j = 0; j < H; ++j) d[i][j] = fma2(d[i][j] * q, weight[i][j], bias[i][j]);
                store_vector<T>(p.y, d[i], c, i, here);
            }
#pragma unroll
            for (int j = 0; j < H; ++j) d[i][j] = ahead[i][j];
        }
    }
    wait_copies<0>();
}

// The backward has no registers for a second row: its block meets twice (73728 x 1024 f16 103 us; before its sums took fewer exchanges 108, and then 120 with the next row's mean ahead).
template <typename T, typename R, bool kResidual, int kVectors, bool kRagged>
__global__ void __launch_bounds__(kBlockThreads) norm_backward_block_kernel(const NormArgs p) {
    constexpr int W = kWidthOf<T>, H = W / 2, kUnits = kUnitsOf<T, R, kResidual, kVectors, true>, kStages = kStagesOf<kUnits, 0, true>;
    extern __shared__ uint4 ring[];
    wait_for_previous_kernel();
    Team<0> team = block_team();
    const Columns<W, kVectors, kRagged> c(p.width, blockIdx.x, team.lane(), team.size());
    const unsigned pitch = blockDim.x * 16, stage = pitch * kUnits;
    const char *const mine = reinterpret_cast<const char *>(ring + threadIdx.x);
    const unsigned slots = (unsigned)__cvta_generic_to_shared(mine);
    long long at = (long long)blockIdx.x * p.width + c.first[0], left = p.rows - blockIdx.x;
    const long long stride = (long long)gridDim.x * p.width;
    const auto issue = [&](int s) {
        copy_row<T, 32>(slots + s * stage, pitch, p.x, c, at, left);
        copy_row<T, 32>(slots + s * stage + kVectors * pitch, pitch, p.grad_y, c, at, left);
        if (kResidual) copy_row<R, 32>(slots + s * stage + 2 * kVectors * pitch, pitch, p.residual, c, at, left);
        copies_issued();
        at += stride;
        left -= gridDim.x;
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s);
    Pair weight[kVectors][H], weight_sum[kVectors][H], bias_sum[kVectors][H];
    load_parameter<T>(p.weight, p.param_dtype, 1.f, c, weight);
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < H; ++j) weight_sum[i][j] = bias_sum[i][j] = Pair(0.f);
    const float inverse = 1.f / (float)p.width;
    int s = 0;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        wait_copies<kStages - 2>();
        if (kResidual && sizeof(R) > sizeof(T)) __syncwarp();
        const char *const slot = mine + s * stage;
        Pair d[kVectors][H], dy[kVectors][H], add(0.f);
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            read_vector<T, 32>(slot, pitch, c, i, d[i]);
            read_vector<T, 32>(slot + kVectors * pitch, pitch, c, i, dy[i]);
            if (kResidual) {
                Pair extra[H];
                read_vector<R, 32>(slot + 2 * kVectors * pitch, pitch, c, i, extra);
#pragma unroll
                for (int j = 0; j < H; ++j) d[i][j] = d[i][j] + extra[j];
            }
#pragma unroll
            for (int j = 0; j < H; ++j) add = add + d[i][j];
        }
        issue(s == 0 ? kStages - 1 : s - 1);
        const long long here = at - kStages * stride;
        s = s == kStages - 1 ? 0 : s + 1;
        float mean[1] = {add.sum()};
        team.sum(mean);
        const Pair minus_mean(-mean[0] * inverse);
        Pair dd(0.f), gd(0.f), gg(0.f);
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
#pragma unroll
            for (int j = 0; j < H; ++j) {
                d[i][j] = fma2(minus_mean, c.ones(i, j), d[i][j]);
                const Pair g = dy[i][j] * weight[i][j];
                dd = fma2(d[i][j], d[i][j], dd);
                gd = fma2(g, d[i][j], gd);
                gg = gg + g;
            }
        float sums[3] = {dd.sum(), gd.sum(), gg.sum()};
        team.sum(sums);
        const float scale = __frsqrt_rn(sums[0] * inverse + p.eps);
        const Pair q(scale), level(-scale * (sums[2] * inverse)), along(-scale * (scale * scale * (sums[1] * inverse)));
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            Pair ds[H];
#pragma unroll
            for (int j = 0; j < H; ++j) {
                ds[j] = fma2(dy[i][j] * weight[i][j], q, fma2(d[i][j], along, level));
                weight_sum[i][j] = fma2(dy[i][j], d[i][j] * q, weight_sum[i][j]);
                bias_sum[i][j] = bias_sum[i][j] + dy[i][j];
            }
            if (!c.any(i)) continue;
            if (kResidual && p.grad_sum) add_sum_gradient<R>(p.grad_sum, ds, c, i, here);
            if (p.grad_x) store_vector<T>(p.grad_x, ds, c, i, here);
            if (kResidual && p.grad_residual) store_vector<R>(p.grad_residual, ds, c, i, here);
        }
    }
    wait_copies<0>();
    if (!p.partial) return;
    float *out = p.partial + (size_t)blockIdx.x * 2 * p.width;
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < H; ++j) {
            float w[2], b[2];
            weight_sum[i][j].get(w[0], w[1]);
            bias_sum[i][j].get(b[0], b[1]);
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (c.has(i, 2 * j + k)) {
                    out[c.first[i] + 2 * j + k] = w[k];
                    out[p.width + c.first[i] + 2 * j + k] = b[k];
                }
        }
}

// ---- host -------------------------------------------------------------------------------------------------------------------
// Threads that share a row, and 16-byte vectors of each.
struct NormShape {
    int lanes, vectors, threads;
    bool ragged;
};
// 8 values of a row to a lane; 16 where that still lets a warp take the row, which saves the barriers of a block (149504 x 512 70 + 98 us).  Not in the backward of
// ragged rows: masks and sums beside 16 values leave one block to an SM (100000 x 259 bf16: 130 us, by 64 threads 117; forward 49 and 58).
constexpr int kMostValues = 8;

inline NormShape norm_shape(int width, int dtype, bool backward) {
    const int W = dtype == FDA_DTYPE_F32 ? 4 : 8;
    NormShape s;
    s.ragged = width % W != 0;
    const int vectors = (width + (s.ragged ? W - 1 : 0) + W - 1) / W;
    s.vectors = kMostValues / W;
    s.threads = kTeamThreads;
    for (s.lanes = 4; s.lanes <= 32; s.lanes *= 2)
        if (s.lanes * s.vectors >= vectors) return s;
    s.lanes = 32;
    s.vectors *= 2;
    if (!(s.ragged && backward) && s.lanes * s.vectors >= vectors) return s;
    s.vectors /= 2;
    s.lanes = 0;
    s.threads = (int)ceil_div(ceil_div(vectors, s.vectors), 32) * 32;
    return s;
}
inline bool is_wide(int width, int dtype) { return norm_shape(width, dtype, true).threads > kBlockThreads; }  // for a block's registers

// Blocks: as many as rows need, at most what is on the device at once (blocks that are teams have 64 registers a thread); a multiple of 8
// where a block is a team (rows 8 apart).
inline unsigned norm_blocks(const NormShape &s, long long rows, int per_sm) {
    const long long needed = ceil_div(rows, s.lanes ? s.threads / s.lanes : 1);
    if (s.lanes) return (unsigned)std::min<long long>(needed, kSms * per_sm);
    const long long room = (long long)kSms * (kBlockThreads / s.threads) / 8 * 8;
    return (unsigned)std::min(ceil_div(needed, 8) * 8, room);
}
// Of the backward, whose blocks leave sums each.
inline unsigned norm_backward_blocks(const NormShape &s, long long rows, int dtype) {
    return norm_blocks(s, rows, s.vectors * (dtype == FDA_DTYPE_F32 ? 4 : 8) > kMostValues ? 2 : 3);
}

// The kernels of one type (fda_norm_f32.cu and so on).
int norm_f32(bool backward, const NormArgs &p, const NormShape &s, int residual_dtype, cudaStream_t st);
int norm_f16(bool backward, const NormArgs &p, const NormShape &s, int residual_dtype, cudaStream_t st);
int norm_bf16(bool backward, const NormArgs &p, const NormShape &s, int residual_dtype, cudaStream_t st);

template <typename T, typename R, bool kResidual, int kVectors, int kLanes>
int run_norm(bool backward, const NormArgs &p, const NormShape &s, cudaStream_t st) {
    constexpr int kForward = kUnitsOf<T, R, kResidual, kVectors, false>, kBackward = kUnitsOf<T, R, kResidual, kVectors, true>;
    const int units = backward ? kBackward * kStagesOf<kBackward, kLanes, true> : kForward * kStagesOf<kForward, kLanes, false>;
    const int shared = units * s.threads * 16;
    void (*kernel)(NormArgs);
    if constexpr (kLanes == 0)
        kernel = backward ? (s.ragged ? norm_backward_block_kernel<T, R, kResidual, kVectors, true>
                                      : norm_backward_block_kernel<T, R, kResidual, kVectors, false>)
                          : (s.ragged ? norm_forward_block_kernel<T, R, kResidual, kVectors, true>
                                      : norm_forward_block_kernel<T, R, kResidual, kVectors, false>);
    else
        kernel = backward ? (s.ragged ? norm_backward_kernel<T, R, kResidual, kVectors, kLanes, true>
                                      : norm_backward_kernel<T, R, kResidual, kVectors, kLanes, false>)
                          : (s.ragged ? norm_forward_kernel<T, R, kResidual, kVectors, kLanes, true>
                                      : norm_forward_kernel<T, R, kResidual, kVectors, kLanes, false>);
    if (shared > 40 * 1024)  // with the static part beyond what every launch may have; the attribute belongs to the current device
        if (const int rc = launched(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared))) return rc;
    const unsigned blocks = backward ? norm_backward_blocks(s, p.rows, sizeof(T) == 4 ? FDA_DTYPE_F32 : FDA_DTYPE_F16)
                                     : norm_blocks(s, p.rows, kForwardBlocks<kForward>);
    return launched(launch_early(kernel, blocks, s.threads, shared, st, 1, p));
}

template <typename T, typename R, bool kResidual>
int run_norm(bool backward, const NormArgs &p, const NormShape &s, cudaStream_t st) {
    constexpr int kEach = kMostValues / kWidthOf<T>;
    if (s.lanes == 4) return run_norm<T, R, kResidual, kEach, 4>(backward, p, s, st);
    if (s.lanes == 8) return run_norm<T, R, kResidual, kEach, 8>(backward, p, s, st);
    if (s.lanes == 16) return run_norm<T, R, kResidual, kEach, 16>(backward, p, s, st);
    if (s.lanes == 0) return run_norm<T, R, kResidual, kEach, 0>(backward, p, s, st);
    if (s.vectors == kEach) return run_norm<T, R, kResidual, kEach, 32>(backward, p, s, st);
    return run_norm<T, R, kResidual, 2 * kEach, 32>(backward, p, s, st);
}

template <typename T>
int run_norm(bool backward, const NormArgs &p, const NormShape &s, int residual_dtype, cudaStream_t st) {
    if (!p.residual) return run_norm<T, T, false>(backward, p, s, st);
    if (sizeof(T) == 2 && residual_dtype == FDA_DTYPE_F32) return run_norm<T, float, true>(backward, p, s, st);
    return run_norm<T, T, true>(backward, p, s, st);
}

}  // namespace fda_norm

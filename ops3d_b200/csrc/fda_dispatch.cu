// Rows sorted by expert, and back.
//
//     entry i = token * top_k + choice;  an entry whose expert is outside 0 .. n_experts - 1 belongs to none
//     position[i] = entries of lower experts + entries of its own expert before it, -1 for none;  start[e] = entries of lower experts
//     dispatch   rows[position[i]] = x[token]                                 rows behind the last expert's are 0
//     combine    y[token] = sum over choices of weight * rows[position] + residual
//     its gradients   drows[position] = weight * dy[token],   dweight = <rows[position], dy[token]>,   dresidual = dy
//     dispatch's      dx[token] = sum over choices of drows[position]  (a combine without weights)
//
// A counting sort: how many entries of each expert come before a block's own, then each entry's place among those.  The order is that
// of the entries, whatever the blocks do.  Few entries are counted by every block for itself, in the launch that moves the rows; many
// in a launch before it, block by block.  Moving the rows is bound by DRAM: dispatch reads a row of x once and writes it top_k times, its
// opposite the other way round, both without atomics.
//
// Rows of any width move in aligned 16-byte vectors of the side that is written.  The other side's row starts elsewhere in a vector; a
// lane loads the aligned vector that its own begins in, takes the next one from its neighbour and shifts the two.
#include "fda_rows.cuh"

#include <algorithm>

namespace {

using namespace fda_rows;

constexpr unsigned kAll = 0xffffffffu;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMostExperts = 1024, kMostChoices = 32;

// ---- rows --------------------------------------------------------------------------------------------------------------------
struct MoveArgs {
    const void *rows, *x, *weights, *residual, *grad;
    const int64_t *position, *end;  // end: where the last expert's rows end
    void *out, *grad_weights;
    long long tokens;
    int top_k, width, weight_dtype;
    int slots, passes;  // vectors that a row can touch, and how often a team of lanes takes some of them
};

template <typename T> constexpr int kWidthOf = 16 / (int)sizeof(T);

// Vector number `at` of a tensor of `total` elements; 0 outside.
template <typename T, bool kRagged>
__device__ __forceinline__ uint4 load_vector(const T *tensor, long long at, long long total) {
    constexpr int W = kWidthOf<T>;
    if (kRagged && (at < 0 || at * W + W > total)) {
        alignas(16) T v[W];
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = at >= 0 && at * W + j < total ? tensor[at * W + j] : from_f32<T>(0.f);
        return *reinterpret_cast<const uint4 *>(v);
    }
    return reinterpret_cast<const uint4 *>(tensor)[at];
}

// Elements by, by + 1, ... of the vectors a and b, one behind the other.
template <typename T>
__device__ __forceinline__ uint4 shifted(uint4 a, uint4 b, int by) {
    const int words = by * (int)sizeof(T) / 4;
    unsigned w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 7; ++i) w[i] = words & 1 ? w[i + 1] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = words & 2 ? w[i + 2] : w[i];
    if (sizeof(T) == 2) {
        const int bits = by % 2 * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint4 next_lane(uint4 v) {
    return make_uint4(__shfl_down_sync(kAll, v.x, 1), __shfl_down_sync(kAll, v.y, 1), __shfl_down_sync(kAll, v.z, 1), __shfl_down_sync(kAll, v.w, 1));
}

// A row that vectors of one tensor are aligned to: slot i holds its elements first, first + 1, ...
template <typename T, bool kRagged>
struct Slot {
    long long vector;  // in the tensor
    int first, width;
    __device__ __forceinline__ Slot(long long row, int width, int i) : width(width) {
        constexpr int W = kWidthOf<T>;
        const long long start = row * width;
        const int lead = kRagged ? (int)(start % W) : 0;
        vector = start / W + i;
        first = i * W - lead;
    }
    __device__ __forceinline__ bool any() const { return first < width; }
    __device__ __forceinline__ bool whole() const { return !kRagged || (first >= 0 && first + kWidthOf<T> <= width); }
    __device__ __forceinline__ bool has(int j) const { return !kRagged || (first + j >= 0 && first + j < width); }
    __device__ __forceinline__ void store(T *tensor, uint4 v) const {
        if (!any()) return;
        if (whole()) {
            reinterpret_cast<uint4 *>(tensor)[vector] = v;
            return;
        }
        Raw<T, kWidthOf<T>> raw;
        raw.u[0] = v;
#pragma unroll
        for (int j = 0; j < kWidthOf<T>; ++j)
            if (has(j)) tensor[vector * kWidthOf<T> + j] = raw.element(j);
    }
    // The same elements of the row `row` of a tensor of rows as wide; with elements of its neighbours where has(j) is false.  Every
    // lane of the warp takes part; `there` false: 0.
    __device__ __forceinline__ uint4 fetch(const T *tensor, long long row, long long rows, bool there) const {
        constexpr int W = kWidthOf<T>;
        there = there && any();
        if (!kRagged) return there ? reinterpret_cast<const uint4 *>(tensor)[row * (width / W) + first / W] : make_uint4(0, 0, 0, 0);
        const long long from = row * width + first;
        const long long at = from >= 0 ? from / W : -1;  // above -W
        const uint4 a = row >= 0 && first - W < width ? load_vector<T, true>(tensor, at, rows * width) : make_uint4(0, 0, 0, 0);
        const uint4 v = shifted<T>(a, next_lane(a), (int)(from - at * W));
        return there ? v : make_uint4(0, 0, 0, 0);
    }
};

// A position that leads nowhere counts as none.
__device__ __forceinline__ long long row_of(const MoveArgs &p, long long entry) {
    const int64_t at = p.position[entry];
    return at >= 0 && at < p.tokens * p.top_k ? at : -1;
}

// Rows first .. last - 1 are 0.
template <typename T, bool kRagged>
__device__ __forceinline__ void clear_rows(const MoveArgs &p, T *rows, long long first, long long last, long long thread, long long threads) {
    constexpr int W = kWidthOf<T>;
    const long long begin = first * p.width, end = last * p.width;
    for (long long v = begin / W + thread; v * W < end; v += threads) {
        if (!kRagged || (v * W >= begin && v * W + W <= end)) {
            reinterpret_cast<uint4 *>(rows)[v] = make_uint4(0, 0, 0, 0);
        } else {
            for (long long i = max(begin, v * W); i < min(end, v * W + W); ++i) rows[i] = from_f32<T>(0.f);
        }
    }
}

// Slots that a team of kLanes lanes (0: the block) takes in a pass: a ragged row's last lane only has the vector that the one before needs.
template <int kLanes, bool kRagged>
__device__ __forceinline__ int slot_of(int pass, int lane) {
    constexpr int kTake = kRagged ? 31 : 32;
    if (kLanes != 0) return pass * (kRagged ? kLanes - 1 : kLanes) + lane;
    return (pass * kWarps + (int)threadIdx.x / 32) * kTake + lane;  // warp by warp
}
template <int kLanes, bool kRagged>
__device__ __forceinline__ bool takes(int lane) {
    return !kRagged || lane + 1 < (kLanes ? kLanes : 32);
}

// kLanes lanes take a token's slots of one pass.
template <typename T, int kLanes, bool kRagged>
__global__ void __launch_bounds__(kThreads) combine_kernel(const MoveArgs p) {
    constexpr int W = kWidthOf<T>, H = W / 2, kTeams = kThreads / kLanes, kAtOnce = 4;
    wait_for_previous_kernel();
    const int lane = threadIdx.x % kLanes;
    const T *rows = static_cast<const T *>(p.rows);
    const long long units = p.tokens * p.passes, all = p.tokens * p.top_k;
    const long long own = (long long)blockIdx.x * kTeams + threadIdx.x / kLanes;
    for (long long unit = own; unit - own % (32 / kLanes) < units; unit += (long long)gridDim.x * kTeams) {
        const bool active = unit < units;
        const long long token = !active ? 0 : p.passes == 1 ? unit : unit / p.passes;
        const Slot<T, kRagged> slot(token, p.width, slot_of<kLanes, kRagged>((int)(unit - token * p.passes), lane));
        Pair sum[H];
#pragma unroll
        for (int i = 0; i < H; ++i) sum[i] = Pair(0.f);
        uint4 extra = make_uint4(0, 0, 0, 0);
        const bool mine = active && slot.any() && takes<kLanes, kRagged>(lane);
        if (p.residual && mine) extra = load_vector<T, kRagged>(static_cast<const T *>(p.residual), slot.vector, p.tokens * p.width);
        for (int j = 0; j < p.top_k; j += kAtOnce) {
            long long at[kAtOnce];
            float weight[kAtOnce];
            uint4 v[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                const long long entry = token * p.top_k + j + i;
                const bool there = active && j + i < p.top_k;
                at[i] = there ? row_of(p, entry) : -1;
                weight[i] = there && p.weights ? load_as_f32(p.weights, p.weight_dtype, entry) : 1.f;
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) v[i] = slot.fetch(rows, at[i], all, at[i] >= 0);
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                if (at[i] < 0) continue;  // the weight of no row may be anything
                Raw<T, W> raw;
                Pair e[H];
                raw.u[0] = v[i];
                raw.get(e);
#pragma unroll
                for (int h = 0; h < H; ++h) sum[h] = fma2(e[h], Pair(weight[i]), sum[h]);
            }
        }
        if (!mine) continue;
        Raw<T, W> raw;
        if (p.residual) {
            Pair e[H];
            raw.u[0] = extra;
            raw.get(e);
#pragma unroll
            for (int h = 0; h < H; ++h) sum[h] = sum[h] + e[h];
        }
        raw.set(sum);
        slot.store(static_cast<T *>(p.out), raw.u[0]);
    }
}

// kLanes lanes, or (0) a block, take a token.
template <typename T, int kLanes, bool kRagged>
__global__ void __launch_bounds__(kThreads) combine_backward_kernel(const MoveArgs p) {
    constexpr int W = kWidthOf<T>, H = W / 2, kLine = kLanes ? kLanes : 32, kTeams = kLanes ? kThreads / kLine : 1, kAtOnce = 4;
    __shared__ float dots[kWarps][kAtOnce];
    wait_for_previous_kernel();
    const int lane = threadIdx.x % kLine;
    const T *rows = static_cast<const T *>(p.rows), *grad = static_cast<const T *>(p.grad);
    T *out = static_cast<T *>(p.out);
    const long long all = p.tokens * p.top_k;
    const long long own = (long long)blockIdx.x * kTeams + (kLanes ? threadIdx.x / kLine : 0), step = (long long)gridDim.x * kTeams;
    for (long long unit = own; unit - (kLanes ? own % (32 / kLine) : 0) < p.tokens; unit += step) {
        const bool active = unit < p.tokens;
        const long long token = active ? unit : 0;
        for (int j = 0; j < p.top_k; j += kAtOnce) {
            long long at[kAtOnce];
            float weight[kAtOnce];
            Pair dot[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                const long long entry = token * p.top_k + j + i;
                const bool there = active && j + i < p.top_k;
                at[i] = there ? row_of(p, entry) : -1;
                weight[i] = there && p.weights ? load_as_f32(p.weights, p.weight_dtype, entry) : 1.f;
                dot[i] = Pair(0.f);
            }
            for (int pass = 0; pass < p.passes; ++pass) {
                const int number = slot_of<kLanes, kRagged>(pass, lane);
                uint4 dy[kAtOnce], v[kAtOnce];
                if (!kRagged) {
                    const Slot<T, kRagged> slot(token, p.width, number);
                    dy[0] = slot.fetch(grad, token, p.tokens, active);
                }
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    const Slot<T, kRagged> slot(max(at[i], 0ll), p.width, number);
                    if (kRagged) dy[i] = slot.fetch(grad, token, p.tokens, at[i] >= 0);
                    else dy[i] = dy[0];
                    v[i] = make_uint4(0, 0, 0, 0);
                    if (p.grad_weights && at[i] >= 0 && slot.any() && takes<kLanes, kRagged>(lane))
                        v[i] = load_vector<T, kRagged>(rows, slot.vector, all * p.width);
                }
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    if (at[i] < 0 || !takes<kLanes, kRagged>(lane)) continue;
                    const Slot<T, kRagged> slot(at[i], p.width, number);
                    Raw<T, W> raw;
                    Pair g[H], e[H];
                    raw.u[0] = dy[i];
                    raw.get(g);
                    if (p.grad_weights) {
                        raw.u[0] = v[i];
                        raw.get(e);
                        if (slot.whole()) {  // beyond the row's end both are 0
#pragma unroll
                            for (int h = 0; h < H; ++h) dot[i] = fma2(g[h], e[h], dot[i]);
                        } else {
#pragma unroll
                            for (int h = 0; h < H; ++h) {
                                float a, b, c, d;
                                g[h].get(a, b);
                                e[h].get(c, d);
                                const float first = slot.has(2 * h) ? a * c : 0.f, second = slot.has(2 * h + 1) ? b * d : 0.f;
                                dot[i] = dot[i] + Pair(first, second);
                            }
                        }
                    }
                    if (out) {
#pragma unroll
                        for (int h = 0; h < H; ++h) g[h] = g[h] * Pair(weight[i]);
                        raw.set(g);
                        slot.store(out, raw.u[0]);
                    }
                }
            }
            if (!p.grad_weights) continue;
            float sums[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) sums[i] = lanes_sum<kLine>(dot[i].sum());
            if constexpr (kLanes == 0) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i)
                    if (lane == 0) dots[threadIdx.x / 32][i] = sums[i];
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    sums[i] = dots[0][i];
                    for (int w = 1; w < kWarps; ++w) sums[i] += dots[w][i];
                }
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (active && j + i < p.top_k && (kLanes ? lane : (int)threadIdx.x) == 0)
                    store_from_f32(p.grad_weights, p.weight_dtype, token * p.top_k + j + i, at[i] < 0 ? 0.f : sums[i]);
        }
    }
    if (out) clear_rows<T, kRagged>(p, out, min(max((long long)*p.end, 0ll), all), all, (long long)blockIdx.x * kThreads + threadIdx.x,
                                    (long long)gridDim.x * kThreads);
}

// ---- sorting, and the rows with it -------------------------------------------------------------------------------------------
struct SortArgs {
    const int64_t *experts;
    int64_t *start, *position;
    int *counts;  // [blocks][n_experts]: of a block's entries; after the scan, of those before it
    int *total;   // [n_experts], where there is a scan
    long long entries;
    int n_experts, chunk, chunks;  // entries of a block, a multiple of top_k; blocks along the entries
};

__device__ __forceinline__ int expert_of(const SortArgs &p, long long i, long long last) {
    if (i >= last) return -1;
    const int64_t e = p.experts[i];
    return e >= 0 && e < p.n_experts ? (int)e : -1;
}

__global__ void __launch_bounds__(kThreads) sort_count_kernel(const SortArgs p) {
    __shared__ int count[kMostExperts];
    wait_for_previous_kernel();
    for (int e = threadIdx.x; e < p.n_experts; e += kThreads) count[e] = 0;
    __syncthreads();
    const long long first = (long long)blockIdx.x * p.chunk, last = min(first + p.chunk, p.entries);
#pragma unroll 4
    for (long long i = first + threadIdx.x; i < last; i += kThreads) {
        const int e = expert_of(p, i, last);
        if (e >= 0) atomicAdd(&count[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.n_experts; e += kThreads) p.counts[(size_t)blockIdx.x * p.n_experts + e] = count[e];
}

// Over the blocks, 32 experts at a time: 32 runs of blocks side by side.
__global__ void __launch_bounds__(1024) sort_scan_kernel(const SortArgs p) {
    __shared__ int sums[32][33];
    wait_for_previous_kernel();
    const int lane = threadIdx.x % 32, run = threadIdx.x / 32, e = blockIdx.x * 32 + lane;
    const int length = (p.chunks + 31) / 32, first = min(run * length, p.chunks), last = min(first + length, p.chunks);
    int s = 0;
    if (e < p.n_experts)
        for (int c = first; c < last; ++c) s += p.counts[(size_t)c * p.n_experts + e];
    sums[run][lane] = s;
    __syncthreads();
    int before = 0, all = 0;
    for (int k = 0; k < 32; ++k) {
        if (k == run) before = all;
        all += sums[k][lane];
    }
    if (e >= p.n_experts) return;
    for (int c = first; c < last; ++c) {
        const size_t at = (size_t)c * p.n_experts + e;
        const int n = p.counts[at];
        p.counts[at] = before;
        before += n;
    }
    if (run == 0) p.total[e] = all;
}

// How a block of the moving kernel learns how many entries of each expert there are, and how many before its own.
enum Counted {
    kByItself,  // it counts all entries
    kPerBlock,  // counts of each block: it adds them up
    kScanned    // added up by sort_scan_kernel
};

constexpr int kPart = 2048;  // entries of a block that are placed at a time
constexpr int kMoveThreads = 512, kMoveWarps = kMoveThreads / 32;

// Dynamic shared memory: next[kMoveWarps][n_experts], then total[n_experts], then start[n_experts + 1], then place[kPart].
inline int move_shared(int n_experts) { return ((kMoveWarps + 2) * n_experts + 1 + kPart) * (int)sizeof(int); }

// A block takes a chunk of entries (tokens), and of their rows the columns of one of gridDim.y slices.
template <typename T, int kLanes, bool kRagged, int kCounted>
__global__ void __launch_bounds__(kMoveThreads, 2) dispatch_kernel(const SortArgs p, const MoveArgs m) {
    extern __shared__ int shared[];
    __shared__ int carry[kMoveWarps];
    wait_for_previous_kernel();
    const int E = p.n_experts, warp = threadIdx.x / 32;
    int *next = shared, *total = shared + kMoveWarps * E, *start = total + E, *place = start + E + 1;
    const long long first = (long long)blockIdx.x * p.chunk, last = min(first + p.chunk, p.entries);
    // next[0][e]: entries of expert e before the block's; total[e]: all
    for (int i = threadIdx.x; i < (kMoveWarps + 1) * E; i += kMoveThreads) next[i] = 0;
    __syncthreads();
    if (kCounted == kByItself) {
#pragma unroll 4
        for (long long i = threadIdx.x; i < p.entries; i += kMoveThreads) {
            const int e = expert_of(p, i, p.entries);
            if (e >= 0) {
                atomicAdd(&total[e], 1);
                if (i < first) atomicAdd(&next[e], 1);
            }
        }
    } else if (kCounted == kPerBlock) {
        // threads side by side take neighbouring experts of one block
        const int rows = max(1, kMoveThreads / E);
        for (int base = 0; base < E; base += kMoveThreads) {
            const int e = E >= kMoveThreads ? base + threadIdx.x : threadIdx.x % E, row = E >= kMoveThreads ? 0 : threadIdx.x / E;
            int all = 0, before = 0;
            if (e < E && row < rows) {
#pragma unroll 4
                for (int c = row; c < p.chunks; c += rows) {
                    const int n = p.counts[(size_t)c * E + e];
                    all += n;
                    if (c < (int)blockIdx.x) before += n;
                }
                atomicAdd(&total[e], all);
                atomicAdd(&next[e], before);
            }
        }
    } else {
        for (int e = threadIdx.x; e < E; e += kMoveThreads) {
            total[e] = p.total[e];
            next[e] = p.counts[(size_t)blockIdx.x * E + e];
        }
    }
    __syncthreads();
    // start[0 .. E]: sums of the totals
    {
        constexpr int kEach = kMostExperts / kMoveThreads;
        int sum = 0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int e = threadIdx.x * kEach + k;
            if (e < E) sum += total[e];
        }
        const int upto = fda_linear::warp_scan_sum(sum);
        if (threadIdx.x % 32 == 31) carry[warp] = upto;
        __syncthreads();
        int at = upto - sum;
        for (int w = 0; w < warp; ++w) at += carry[w];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int e = threadIdx.x * kEach + k;
            if (e < E) {
                start[e] = at;
                at += total[e];
                if (e == E - 1) start[E] = at;
            }
        }
    }
    __syncthreads();
    const bool writes_order = blockIdx.y == 0;
    if (blockIdx.x == 0 && writes_order)
        for (int e = threadIdx.x; e <= E; e += kMoveThreads) p.start[e] = start[e];
    for (int e = threadIdx.x; e < E; e += kMoveThreads) total[e] = start[e] + next[e];  // where the block's first entry of e goes
    __syncthreads();

    T *rows = static_cast<T *>(m.out);
    const T *x = static_cast<const T *>(m.x);
    const int part_size = kPart / m.top_k * m.top_k;
    for (long long part = first; part < last; part += part_size) {
        const long long end = min(part + part_size, last);
        // a warp takes a run of the part; first its counts
        constexpr int kRun = kPart / kMoveWarps, kSteps = kRun / 32;
        for (int i = threadIdx.x; i < kMoveWarps * E; i += kMoveThreads) next[i] = 0;
        __syncthreads();
        const int lane = threadIdx.x % 32;
        int expert[kSteps];
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            expert[k] = expert_of(p, part + warp * kRun + k * 32 + lane, end);
            if (expert[k] >= 0) atomicAdd(&next[warp * E + expert[k]], 1);
        }
        __syncthreads();
        for (int e = threadIdx.x; e < E; e += kMoveThreads) {
            int at = total[e];
            for (int w = 0; w < kMoveWarps; ++w) {
                const int n = next[w * E + e];
                next[w * E + e] = at;
                at += n;
            }
            total[e] = at;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int i = warp * kRun + k * 32 + lane;
            if (part + warp * kRun + k * 32 >= end) break;
            const unsigned same = __match_any_sync(kAll, expert[k]);
            const int before = __popc(same & ((1u << lane) - 1));
            int at = -1;
            if (expert[k] >= 0) at = next[warp * E + expert[k]] + before;
            __syncwarp();
            if (expert[k] >= 0 && before == 0) next[warp * E + expert[k]] += __popc(same);
            __syncwarp();
            if (part + i < end) {
                place[i] = at;
                if (writes_order) p.position[part + i] = at;
            }
        }
        __syncthreads();
        // the rows of the part's tokens: kLanes lanes to a token and pass
        constexpr int kTeams = kMoveThreads / kLanes, kAtOnce = 4;
        const long long token0 = part / m.top_k;
        const int tokens = (int)((end - part) / m.top_k), tl = threadIdx.x % kLanes, team = threadIdx.x / kLanes;
        for (int pass = blockIdx.y; pass < m.passes; pass += gridDim.y) {
            const int number = slot_of<kLanes, kRagged>(pass, tl);
            for (int base = 0; base < tokens; base += kTeams * kAtOnce) {
                if (!kRagged) {
                    uint4 v[kAtOnce];
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        const int t = base + i * kTeams + team;
                        const Slot<T, kRagged> slot(token0 + t, m.width, number);
                        v[i] = slot.fetch(x, token0 + t, m.tokens, t < tokens);
                    }
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        const int t = base + i * kTeams + team;
                        if (t >= tokens) continue;
                        for (int j = 0; j < m.top_k; ++j) {
                            const int at = place[t * m.top_k + j];
                            if (at >= 0) Slot<T, kRagged>(at, m.width, number).store(rows, v[i]);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        const int t = base + i * kTeams + team;
                        for (int j = 0; j < m.top_k; ++j) {
                            const int at = t < tokens ? place[t * m.top_k + j] : -1;
                            const Slot<T, kRagged> slot(max(at, 0), m.width, number);
                            const uint4 v = slot.fetch(x, token0 + t, m.tokens, at >= 0);
                            if (at >= 0 && takes<kLanes, kRagged>(tl)) slot.store(rows, v);
                        }
                    }
                }
            }
        }
        __syncthreads();
    }
    clear_rows<T, kRagged>(m, rows, start[E], p.entries, ((long long)blockIdx.y * gridDim.x + blockIdx.x) * kMoveThreads + threadIdx.x,
                           (long long)gridDim.x * gridDim.y * kMoveThreads);
}

// ---- host --------------------------------------------------------------------------------------------------------------------
// Lanes that take a token, and passes over its vectors.
template <typename T>
void set_slots(MoveArgs &p, int &lanes, bool &ragged) {
    constexpr int W = kWidthOf<T>;
    ragged = p.width % W != 0;
    p.slots = ragged ? (p.width + 2 * W - 2) / W : p.width / W;
    const int extra = ragged ? 1 : 0;
    lanes = 32;
    while (lanes > 4 && lanes / 2 - extra >= p.slots) lanes /= 2;
    p.passes = (int)ceil_div(p.slots, lanes - extra);
}

template <typename T, int kLanes, bool kRagged>
int run_combine(const MoveArgs &p, cudaStream_t st) {
    const long long blocks = ceil_div(p.tokens * p.passes, kThreads / kLanes);
    return launched(launch_early(combine_kernel<T, kLanes, kRagged>, (unsigned)std::min<long long>(blocks, 32 * kSms), kThreads, 0, st, 1, p));
}
template <typename T, int kLanes, bool kRagged>
int run_combine_backward(const MoveArgs &p, cudaStream_t st) {
    const long long blocks = kLanes ? ceil_div(p.tokens, kThreads / (kLanes ? kLanes : 1)) : p.tokens;
    return launched(launch_early(combine_backward_kernel<T, kLanes, kRagged>, (unsigned)std::min<long long>(blocks, 32 * kSms), kThreads, 0, st, 1, p));
}

template <typename T, bool kRagged>
int run_combine(const MoveArgs &p, int lanes, bool backward, cudaStream_t st) {
    // wide rows of few tokens: a block to a token
    if (backward && p.passes > 1 && p.tokens < 8 * kSms * kWarps) {
        MoveArgs q = p;
        q.passes = (int)ceil_div(p.slots, kWarps * (kRagged ? 31 : 32));
        return run_combine_backward<T, 0, kRagged>(q, st);
    }
    if (lanes == 4) return backward ? run_combine_backward<T, 4, kRagged>(p, st) : run_combine<T, 4, kRagged>(p, st);
    if (lanes == 8) return backward ? run_combine_backward<T, 8, kRagged>(p, st) : run_combine<T, 8, kRagged>(p, st);
    if (lanes == 16) return backward ? run_combine_backward<T, 16, kRagged>(p, st) : run_combine<T, 16, kRagged>(p, st);
    return backward ? run_combine_backward<T, 32, kRagged>(p, st) : run_combine<T, 32, kRagged>(p, st);
}

template <typename T>
int run_combine(MoveArgs p, bool backward, cudaStream_t st) {
    int lanes;
    bool ragged;
    set_slots<T>(p, lanes, ragged);
    return ragged ? run_combine<T, true>(p, lanes, backward, st) : run_combine<T, false>(p, lanes, backward, st);
}

int run_combine(const MoveArgs &p, int dtype, bool backward, cudaStream_t st) {
    if (dtype == FDA_DTYPE_F32) return run_combine<float>(p, backward, st);
    if (dtype == FDA_DTYPE_F16) return run_combine<__half>(p, backward, st);
    return run_combine<__nv_bfloat16>(p, backward, st);
}

constexpr long long kFewEntries = 4096;  // that every block counts by itself

// Entries of a block, and blocks along them.
void set_chunks(SortArgs &s, int top_k, int passes, unsigned &slices) {
    const long long tokens = s.entries / top_k;
    const bool few = s.entries <= kFewEntries;
    // few: a token to a warp and pass, and slices of columns until every SM has a block; many: two blocks to an SM
    long long per = few ? std::max<long long>(1, kMoveWarps / passes) : ceil_div(tokens, 2 * kSms);
    s.chunk = (int)(per * top_k);
    s.chunks = (int)ceil_div(tokens, per);
    slices = few ? (unsigned)std::min<long long>(passes, std::max<long long>(1, kSms / s.chunks)) : 1;
}
Counted counted(const SortArgs &s) {
    if (s.entries <= kFewEntries) return kByItself;
    return s.n_experts <= 64 ? kPerBlock : kScanned;
}

template <typename T, int kLanes, bool kRagged>
int run_dispatch(const SortArgs &s, const MoveArgs &p, unsigned slices, cudaStream_t st) {
    const Counted c = counted(s);
    const int shared = move_shared(s.n_experts);
    const auto kernel = c == kByItself ? dispatch_kernel<T, kLanes, kRagged, kByItself>
                        : c == kPerBlock ? dispatch_kernel<T, kLanes, kRagged, kPerBlock> : dispatch_kernel<T, kLanes, kRagged, kScanned>;
    if (shared > 40 * 1024)  // the attribute belongs to the current device
        if (const int rc = launched(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared))) return rc;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t launch{};
    launch.gridDim = dim3(s.chunks, slices);
    launch.blockDim = dim3(kMoveThreads);
    launch.dynamicSmemBytes = shared;
    launch.stream = st;
    launch.attrs = &attribute;
    launch.numAttrs = 1;
    return launched(cudaLaunchKernelEx(&launch, kernel, s, p));
}

template <typename T, bool kRagged>
int run_dispatch(const SortArgs &s, const MoveArgs &p, int lanes, unsigned slices, cudaStream_t st) {
    if (lanes == 4) return run_dispatch<T, 4, kRagged>(s, p, slices, st);
    if (lanes == 8) return run_dispatch<T, 8, kRagged>(s, p, slices, st);
    if (lanes == 16) return run_dispatch<T, 16, kRagged>(s, p, slices, st);
    return run_dispatch<T, 32, kRagged>(s, p, slices, st);
}

template <typename T>
int run_dispatch(SortArgs s, MoveArgs p, cudaStream_t st) {
    int lanes;
    bool ragged;
    unsigned slices;
    set_slots<T>(p, lanes, ragged);
    set_chunks(s, p.top_k, p.passes, slices);
    const Counted c = counted(s);
    if (c != kByItself)
        if (const int rc = launched(launch_early(sort_count_kernel, s.chunks, kThreads, 0, st, 1, s))) return rc;
    if (c == kScanned)
        if (const int rc = launched(launch_early(sort_scan_kernel, (unsigned)ceil_div(s.n_experts, 32), 1024, 0, st, 1, s))) return rc;
    return ragged ? run_dispatch<T, true>(s, p, lanes, slices, st) : run_dispatch<T, false>(s, p, lanes, slices, st);
}

int check_rows(long long tokens, int top_k, int width, int dtype) {
    if (!known_dtype(dtype)) return FDA_ERR_BAD_DTYPE;
    if (tokens < 0 || top_k < 1 || width < 1 || width >= 1 << 26) return FDA_ERR_BAD_SHAPE;
    if (top_k > kMostChoices) return FDA_ERR_TOO_LARGE_STATIC;
    if (tokens > INT32_MAX / top_k) return FDA_ERR_BAD_SHAPE;
    return FDA_OK;
}

// Counts of the blocks; there are at most two to an SM.
size_t counts_bytes(int n_experts) { return fda_linear::round256((size_t)2 * kSms * n_experts * sizeof(int)); }

}  // namespace

extern "C" {

size_t fda_dispatch_workspace_bytes(long long tokens, int top_k, int n_experts) {
    if (tokens <= 0 || top_k < 1 || top_k > kMostChoices || tokens > INT32_MAX / top_k || n_experts < 1 || n_experts > kMostExperts) return 0;
    if (tokens * top_k <= kFewEntries) return 0;
    return counts_bytes(n_experts) + fda_linear::round256((size_t)n_experts * sizeof(int));
}

int fda_dispatch_rows(const void *x, const int64_t *experts, void *rows, int64_t *group_start_index, int64_t *position, void *workspace,
                      size_t workspace_bytes, long long tokens, int top_k, int n_experts, int features, int dtype, void *stream) {
    if (const int rc = check_rows(tokens, top_k, features, dtype)) return rc;
    if (n_experts < 1) return FDA_ERR_BAD_SHAPE;
    if (n_experts > kMostExperts) return FDA_ERR_TOO_LARGE_STATIC;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!group_start_index) return FDA_ERR_NULL_POINTER;
    if (tokens == 0) return launched(cudaMemsetAsync(group_start_index, 0, (size_t)(n_experts + 1) * sizeof(int64_t), st));
    if (!x || !experts || !rows || !position) return FDA_ERR_NULL_POINTER;
    const size_t need = fda_dispatch_workspace_bytes(tokens, top_k, n_experts);
    if (need > 0 && (!workspace || workspace_bytes < need)) return FDA_ERR_WORKSPACE;
    if ((need > 0 && (uintptr_t)workspace % 256) || misaligned16(x) || misaligned16(rows)) return FDA_ERR_MISALIGNED;
    SortArgs s{};
    s.experts = experts; s.start = group_start_index; s.position = position; s.entries = tokens * top_k; s.n_experts = n_experts;
    if (need > 0) {
        s.counts = static_cast<int *>(workspace);
        s.total = reinterpret_cast<int *>(static_cast<char *>(workspace) + counts_bytes(n_experts));
    }
    MoveArgs p{};
    p.x = x; p.out = rows; p.tokens = tokens; p.top_k = top_k; p.width = features;
    if (dtype == FDA_DTYPE_F32) return run_dispatch<float>(s, p, st);
    if (dtype == FDA_DTYPE_F16) return run_dispatch<__half>(s, p, st);
    return run_dispatch<__nv_bfloat16>(s, p, st);
}

int fda_combine_rows(const void *rows, const int64_t *position, const void *weights, const void *residual, void *y, long long tokens, int top_k,
                     int features, int dtype, int weight_dtype, void *stream) {
    if (const int rc = check_rows(tokens, top_k, features, dtype)) return rc;
    if (weights && !known_dtype(weight_dtype)) return FDA_ERR_BAD_DTYPE;
    if (tokens == 0) return FDA_OK;
    if (!rows || !position || !y) return FDA_ERR_NULL_POINTER;
    if (misaligned16(rows) || misaligned16(residual) || misaligned16(y)) return FDA_ERR_MISALIGNED;
    MoveArgs p{};
    p.rows = rows; p.position = position; p.weights = weights; p.residual = residual; p.out = y; p.tokens = tokens; p.top_k = top_k;
    p.width = features; p.weight_dtype = weight_dtype;
    return run_combine(p, dtype, false, static_cast<cudaStream_t>(stream));
}

int fda_combine_rows_backward(const void *rows, const int64_t *position, const int64_t *rows_end, const void *weights, const void *grad_y,
                              void *grad_rows, void *grad_weights, long long tokens, int top_k, int features, int dtype, int weight_dtype,
                              void *stream) {
    if (const int rc = check_rows(tokens, top_k, features, dtype)) return rc;
    if ((weights || grad_weights) && !known_dtype(weight_dtype)) return FDA_ERR_BAD_DTYPE;
    if (tokens == 0 || (!grad_rows && !grad_weights)) return FDA_OK;
    if (!position || !rows_end || !grad_y || (grad_weights && !rows)) return FDA_ERR_NULL_POINTER;
    if (misaligned16(rows) || misaligned16(grad_y) || misaligned16(grad_rows)) return FDA_ERR_MISALIGNED;
    MoveArgs p{};
    p.rows = rows; p.position = position; p.end = rows_end; p.weights = weights; p.grad = grad_y; p.out = grad_rows; p.grad_weights = grad_weights;
    p.tokens = tokens; p.top_k = top_k; p.width = features; p.weight_dtype = weight_dtype;
    return run_combine(p, dtype, true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

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
constexpr int kMostChunks = 2 * kSms;  // blocks along the entries where they are many

// ---- rows --------------------------------------------------------------------------------------------------------------------
struct MoveArgs {
    const void *rows, *x, *weights, *residual, *grad;
    const int64_t *position;
    void *out, *grad_weights;
    int *entry;  // [entries]: of each row the entry that wrote its gradient; anything where none did
    long long tokens, entries;
    int top_k, width, passes;  // passes: how often a team of lanes takes vectors of a row
    bool wide_weights;         // fp32, else in the rows' type
};

template <typename T> constexpr int kWidthOf = 16 / (int)sizeof(T);

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

// A tensor of rows.  Row numbers and offsets inside a row have 31 bits, their products 64.
template <typename T>
struct Rows {
    static constexpr int W = kWidthOf<T>;
    T *base;
    const T *end;
    unsigned width;
    __device__ __forceinline__ Rows(const void *tensor, long long rows, int width)
        : base(const_cast<T *>(static_cast<const T *>(tensor))), end(base + rows * width), width(width) {}
    // Where a row starts in its first vector.
    __device__ __forceinline__ int lead(int row) const { return (int)((unsigned)row * width % W); }
    __device__ __forceinline__ T *at(int row, int column) const { return base + ((unsigned long long)(unsigned)row * width + (long long)column); }
    // The vector that starts on a boundary; outside the tensor 0.  kOnce: it is not read again, and leaves the caches first.
    template <bool kRagged, bool kOnce = false>
    __device__ __forceinline__ uint4 load(const T *from) const {
        if (kRagged && (from < base || from + W > end)) {
            alignas(16) T v[W];
#pragma unroll
            for (int j = 0; j < W; ++j) v[j] = from + j >= base && from + j < end ? from[j] : from_f32<T>(0.f);
            return *reinterpret_cast<const uint4 *>(v);
        }
        return kOnce ? __ldcs(reinterpret_cast<const uint4 *>(from)) : *reinterpret_cast<const uint4 *>(from);
    }
    // Elements column .. column + W - 1 of a row, -W < column; what is not in the row may be anything.  Where rows are ragged every lane
    // of the warp takes part, and a lane needs the next one to have the next W columns.  `there` false: 0, nothing is read.
    template <bool kRagged, bool kOnce = false>
    __device__ __forceinline__ uint4 fetch(int row, int column, bool there) const {
        const uint4 none = make_uint4(0, 0, 0, 0);
        if (!kRagged) return there && column < (int)width ? load<false, kOnce>(at(row, column)) : none;
        const T *from = at(row, column);
        const int by = (int)((uintptr_t)from % 16) / (int)sizeof(T);
        const uint4 a = there && column < (int)width + W ? load<true, kOnce>(from - by) : none;
        return shifted<T>(a, next_lane(a), by);
    }
    // Columns column .. of a row at a vector's boundary; those outside the row stay as they are.
    template <bool kRagged>
    __device__ __forceinline__ void store(int row, int column, uint4 v) const {
        if (column >= (int)width) return;
        T *to = at(row, column);
        if (!kRagged || (column >= 0 && column + W <= (int)width)) {
            *reinterpret_cast<uint4 *>(to) = v;
            return;
        }
        Raw<T, W> raw;
        raw.u[0] = v;
        const unsigned bits = ((1u << min(W, (int)width - column)) - 1) & ~((1u << max(0, -column)) - 1);
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (bits >> j & 1) to[j] = raw.element(j);
    }
};

// A vector of a row that starts at `column`: elements outside the row as 0.
template <typename T>
__device__ __forceinline__ uint4 inside(uint4 v, int column, int width) {
    constexpr int kBits = (int)sizeof(T) * 8;
    const int low = max(0, -column) * kBits, high = max(0, min(kWidthOf<T>, width - column)) * kBits;
    unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int from = min(max(low - 32 * i, 0), 32), to = min(max(high - 32 * i, 0), 32);
        w[i] &= (unsigned)((0xffffffffull << from) & (0xffffffffull >> (32 - to)));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Positions and weights of kAtOnce choices of a token, as they are read; a choice beyond the last has none.
template <int kAtOnce>
struct Choices {
    int64_t position[kAtOnce];
    float weight[kAtOnce];
    template <typename T>
    __device__ __forceinline__ void load(const MoveArgs &p, long long token, int j, bool there) {
        const long long entry = token * p.top_k + j;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const bool one = there && j + i < p.top_k;
            position[i] = one ? p.position[entry + i] : -1;
            weight[i] = 1.f;
        }
        if (!p.weights) return;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const bool one = there && j + i < p.top_k;
            if (one) weight[i] = p.wide_weights ? static_cast<const float *>(p.weights)[entry + i] : to_f32(static_cast<const T *>(p.weights)[entry + i]);
        }
    }
    // The row; -1 for a position that leads nowhere.
    __device__ __forceinline__ int row(const MoveArgs &p, int i) const {
        return (unsigned long long)position[i] < (unsigned long long)p.entries ? (int)position[i] : -1;
    }
};

// Rows first .. last - 1 are 0.
template <typename T, bool kRagged>
__device__ __forceinline__ void clear_rows(T *rows, int width, long long first, long long last, long long thread, long long threads) {
    constexpr int W = kWidthOf<T>;
    const long long begin = first * width, end = last * width;
    for (long long v = begin / W + thread; v * W < end; v += threads) {
        if (!kRagged || (v * W >= begin && v * W + W <= end)) {
            reinterpret_cast<uint4 *>(rows)[v] = make_uint4(0, 0, 0, 0);
        } else {
            for (long long i = max(begin, v * W); i < min(end, v * W + W); ++i) rows[i] = from_f32<T>(0.f);
        }
    }
}

// Vectors that a team of kLanes lanes (0: the block, warp by warp) takes in a pass: a ragged row's last lane only has the vector that the
// one before needs.
template <int kLanes, bool kRagged>
__device__ __forceinline__ int slot_of(int pass, int lane) {
    if (kLanes != 0) return pass * (kRagged ? kLanes - 1 : kLanes) + lane;
    return (pass * kWarps + (int)threadIdx.x / 32) * (kRagged ? 31 : 32) + lane;
}
template <int kLanes, bool kRagged>
__device__ __forceinline__ bool takes(int lane) {
    return !kRagged || lane + 1 < (kLanes ? kLanes : 32);
}

// kLanes lanes take a token's vectors of one pass.  Positions and weights of the next choices are on their way while rows are added up.  Bound
// by DRAM (149504 x 4 x 256 bf16 77 us, 6.0 TB/s); read as data that is not used again rows come faster (73728 x 2 x 256: 27 -> 22 us).
constexpr int kCombineBlocks = 4;  // to an SM, all there at once
template <typename T, int kLanes, bool kRagged, int kAtOnce>
__global__ void __launch_bounds__(kThreads, kCombineBlocks) combine_kernel(const MoveArgs p) {
    constexpr int W = kWidthOf<T>, H = W / 2, kTeams = kThreads / kLanes;
    wait_for_previous_kernel();
    const int lane = threadIdx.x % kLanes;
    const Rows<T> rows(p.rows, p.entries, p.width), out(p.out, p.tokens, p.width), residual(p.residual, p.tokens, p.width);
    const long long units = p.tokens * p.passes, step = (long long)gridDim.x * kTeams;
    long long unit = (long long)blockIdx.x * kTeams + threadIdx.x / kLanes;
    const long long warp = threadIdx.x % 32 / kLanes;  // the warp's first team decides when it ends
    const auto token_of = [&](long long u) { return p.passes == 1 ? u : u / p.passes; };
    int j = 0;
    Pair sum[H];
#pragma unroll
    for (int h = 0; h < H; ++h) sum[h] = Pair(0.f);
    Choices<kAtOnce> next;
    next.template load<T>(p, token_of(unit), 0, unit < units);
    while (unit - warp < units) {
        const bool active = unit < units, last = j + kAtOnce >= p.top_k;
        const int token = active ? (int)token_of(unit) : 0, pass = active ? (int)(unit - (long long)token * p.passes) : 0;
        const int column = slot_of<kLanes, kRagged>(pass, lane) * W - (kRagged ? out.lead(token) : 0);
        const bool mine = active && column < p.width && takes<kLanes, kRagged>(lane);
        uint4 v[kAtOnce], extra = make_uint4(0, 0, 0, 0);
        float weight[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int row = next.row(p, i);
            v[i] = rows.template fetch<kRagged, true>(max(row, 0), column, row >= 0);
            weight[i] = row >= 0 ? next.weight[i] : 0.f;  // that of no row may be anything
        }
        if (p.residual && last && mine) extra = residual.template load<kRagged, true>(residual.at(token, column));
        j = last ? 0 : j + kAtOnce;
        if (last) unit += step;
        next.template load<T>(p, token_of(unit), j, unit < units);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            Raw<T, W> raw;
            Pair e[H];
            raw.u[0] = v[i];
            raw.get(e);
#pragma unroll
            for (int h = 0; h < H; ++h) sum[h] = fma2(e[h], Pair(weight[i]), sum[h]);
        }
        if (!last) continue;
        Raw<T, W> raw;
        if (p.residual) {
            Pair e[H];
            raw.u[0] = extra;
            raw.get(e);
#pragma unroll
            for (int h = 0; h < H; ++h) sum[h] = sum[h] + e[h];
        }
        raw.set(sum);
        if (mine) out.template store<kRagged>(token, column, raw.u[0]);
#pragma unroll
        for (int h = 0; h < H; ++h) sum[h] = Pair(0.f);
    }
}

// kLanes lanes, or (0) a block, take a token.  Bound by DRAM: 149504 x 4 x 256 bf16 124 us, 5.6 TB/s.
// Blocks that registers leave room for on an SM: where rows are aligned as many as are launched (149504 x 4: 132 us with more blocks than fit,
// 124 so), shifted rows need twice the registers.
template <bool kRagged, int kAtOnce>
constexpr int kCombineBackwardBlocks = kAtOnce == 2 ? (kRagged ? 3 : 4) : kRagged ? 2 : 3;
template <typename T, int kLanes, bool kRagged, int kAtOnce>
__global__ void __launch_bounds__(kThreads, kCombineBackwardBlocks<kRagged, kAtOnce>) combine_backward_kernel(const MoveArgs p) {
    constexpr int W = kWidthOf<T>, H = W / 2, kLine = kLanes ? kLanes : 32, kTeams = kLanes ? kThreads / kLine : 1;
    __shared__ float dots[kWarps][kAtOnce];
    wait_for_previous_kernel();
    const int lane = threadIdx.x % kLine;
    const Rows<T> rows(p.rows, p.entries, p.width), grad(p.grad, p.tokens, p.width), out(p.out, p.entries, p.width);
    const long long step = (long long)gridDim.x * kTeams, warp = kLanes ? threadIdx.x % 32 / kLine : 0;
    long long unit = (long long)blockIdx.x * kTeams + (kLanes ? threadIdx.x / kLine : 0);
    int j = 0;
    Choices<kAtOnce> next;
    next.template load<T>(p, unit, 0, unit < p.tokens);
    while (unit - warp < p.tokens) {
        const bool active = unit < p.tokens;
        const int token = active ? (int)unit : 0, first = j;
        int row[kAtOnce];
        Pair weight[kAtOnce], dot[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            row[i] = next.row(p, i);
            weight[i] = Pair(next.weight[i]);
            dot[i] = Pair(0.f);
        }
        const bool last = j + kAtOnce >= p.top_k;
        j = last ? 0 : j + kAtOnce;
        if (p.out && (kLanes ? lane : (int)threadIdx.x) == 0) {
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (row[i] >= 0) p.entry[row[i]] = token * p.top_k + first + i;
        }
        if (last) unit += step;
        next.template load<T>(p, unit, j, unit < p.tokens);
        for (int pass = 0; pass < p.passes; ++pass) {
            const int start = slot_of<kLanes, kRagged>(pass, lane) * W;
            uint4 dy[kRagged ? kAtOnce : 1], v[kAtOnce];
            int column[kAtOnce];
            if constexpr (!kRagged) dy[0] = grad.template fetch<false>(token, start, active);
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                column[i] = start - (kRagged ? rows.lead(max(row[i], 0)) : 0);
                if constexpr (kRagged) dy[i] = grad.template fetch<true>(token, column[i], row[i] >= 0);
                v[i] = make_uint4(0, 0, 0, 0);
                if (p.grad_weights && row[i] >= 0 && column[i] < p.width) v[i] = rows.template load<kRagged>(rows.at(row[i], column[i]));
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                if (row[i] < 0 || !takes<kLanes, kRagged>(lane)) continue;
                Raw<T, W> raw;
                Pair g[H], e[H];
                raw.u[0] = kRagged ? inside<T>(dy[kRagged ? i : 0], column[i], p.width) : dy[0];
                raw.get(g);
                if (p.grad_weights) {
                    raw.u[0] = kRagged ? inside<T>(v[i], column[i], p.width) : v[i];
                    raw.get(e);
#pragma unroll
                    for (int h = 0; h < H; ++h) dot[i] = fma2(g[h], e[h], dot[i]);
                }
                if (p.out) {
#pragma unroll
                    for (int h = 0; h < H; ++h) g[h] = g[h] * weight[i];
                    raw.set(g);
                    out.template store<kRagged>(row[i], column[i], raw.u[0]);
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
        if (!active || (kLanes ? lane : (int)threadIdx.x) != 0) continue;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (first + i >= p.top_k) continue;
            const long long entry = (long long)token * p.top_k + first + i;
            const float g = row[i] < 0 ? 0.f : sums[i];
            if (p.wide_weights) static_cast<float *>(p.grad_weights)[entry] = g;
            else static_cast<T *>(p.grad_weights)[entry] = from_f32<T>(g);
        }
    }
}

// Rows of the gradient that no entry wrote are 0: those behind the last expert's, and of an order that was changed (entries taken out beyond an
// expert's capacity) any.  What `entry` holds of a row counts only if that entry's position is the row, so nothing has to be set before.  A
// warp looks at 32 rows and clears runs of them together.  149504 x 4 x 256 bf16: with the entries' stores 8 us of 132 (a row of zeros beforehand for
// each would be 306 MB, 48 us), 64 tokens 1 us.
constexpr int kClearBlocks = 8;
template <typename T, bool kRagged>
__global__ void __launch_bounds__(kThreads) clear_unwritten_kernel(const MoveArgs p) {
    wait_for_previous_kernel();
    const int lane = threadIdx.x % 32;
    const long long step = (long long)gridDim.x * kThreads;
    for (long long first = (long long)blockIdx.x * kThreads + threadIdx.x - lane; first < p.entries; first += step) {
        const long long row = first + lane;
        bool clear = row < p.entries;
        if (clear) {
            const int entry = p.entry[row];
            clear = entry < 0 || entry >= p.entries || p.position[entry] != row;
        }
        unsigned rows = __ballot_sync(kAll, clear);
        while (rows) {
            const int from = __ffs(rows) - 1, n = __ffs(~(rows >> from)) - 1;  // n is -1 where all 32 are
            const int run = n < 0 ? 32 : n;
            clear_rows<T, kRagged>(static_cast<T *>(p.out), p.width, first + from, first + from + run, lane, 32);
            rows = from + run < 32 ? rows >> (from + run) << (from + run) : 0;
        }
    }
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

// 7 us for 598016 entries: latency of two rounds of loads and of the launch.
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

// Over the blocks, 32 experts at a time: 32 runs of blocks side by side, a run's counts in registers (6 us, latency; 7.6 with two passes).
__global__ void __launch_bounds__(1024) sort_scan_kernel(const SortArgs p) {
    __shared__ int sums[32][33];
    wait_for_previous_kernel();
    constexpr int kRun = (kMostChunks + 31) / 32;
    const int lane = threadIdx.x % 32, run = threadIdx.x / 32, e = blockIdx.x * 32 + lane;
    int n[kRun], s = 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const int c = run * kRun + i;
        n[i] = e < p.n_experts && c < p.chunks ? p.counts[(size_t)c * p.n_experts + e] : 0;
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i) s += n[i];
    sums[run][lane] = s;
    __syncthreads();
    // a warp adds up an expert's runs, then each run has those before it
    const int own = sums[lane][run], upto = fda_linear::warp_scan_sum(own);
    if (lane == 31 && blockIdx.x * 32 + run < p.n_experts) p.total[blockIdx.x * 32 + run] = upto;
    __syncthreads();
    sums[lane][run] = upto - own;
    __syncthreads();
    int before = sums[run][lane];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const int c = run * kRun + i;
        if (e < p.n_experts && c < p.chunks) p.counts[(size_t)c * p.n_experts + e] = before;
        before += n[i];
    }
}

// How a block of the moving kernel learns how many entries of each expert there are, and how many before its own.
enum Counted {
    kByItself,  // it counts all entries
    kPerBlock,  // counts of each block: it adds them up, of up to kFewExperts
    kScanned    // added up by sort_scan_kernel
};

constexpr int kPart = 2048;  // entries of a block that are placed at a time
constexpr int kMoveThreads = 512, kMoveWarps = kMoveThreads / 32;
constexpr int kFewExperts = 32;
static_assert(kFewExperts <= kMoveThreads, "a thread takes one expert");

constexpr int kAheadBytes = 256 * 1024;  // of a block: together they fit L2

// Dynamic shared memory: next[kMoveWarps][n_experts], then total[n_experts], then start[n_experts + 1], then place[kPart].
inline int move_shared(int n_experts) { return ((kMoveWarps + 2) * n_experts + 1 + kPart) * (int)sizeof(int); }

// A block takes a chunk of entries (tokens), and of their rows the columns of one of gridDim.y slices.  Two blocks to an SM, a part of 2048
// entries at a time: smaller chunks learn their place more often (80000 entries of 256 bf16: 19 us, with twice the blocks 24).  Four tokens of a
// team are on their way at once.  149504 x 4 x 256 bf16: 81 us of 90 with the launches before, 4.7 TB/s, four fifths of it writes; while entries
// are placed, some 10 us, DRAM idles.
template <typename T, int kLanes, bool kRagged, int kCounted>
__global__ void __launch_bounds__(kMoveThreads, 2) dispatch_kernel(const SortArgs p, const MoveArgs m) {
    extern __shared__ int shared[];
    __shared__ int carry[kMoveWarps];
    wait_for_previous_kernel();
    const int E = p.n_experts, warp = threadIdx.x / 32;
    int *next = shared, *total = shared + kMoveWarps * E, *start = total + E, *place = start + E + 1;
    const long long first = (long long)blockIdx.x * p.chunk, last = min(first + p.chunk, p.entries);
    if (kCounted != kByItself) {  // the rows of the first entries come to L2 while these are placed
        const char *from = static_cast<const char *>(m.x) + first / m.top_k * m.width * sizeof(T);
        const long long bytes = (min(last, first + kPart) - first) / m.top_k * m.width * (long long)sizeof(T);
        for (long long i = threadIdx.x * 128ll; i < min(bytes, (long long)kAheadBytes); i += kMoveThreads * 128)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(from + i));
    }
    // next[0][e]: entries of expert e before the block's; total[e]: all
    for (int i = threadIdx.x; i < (kMoveWarps + 1) * E; i += kMoveThreads) next[i] = 0;
    __syncthreads();
    if (kCounted == kByItself) {
#pragma unroll 4
        for (long long i = threadIdx.x; i < p.entries; i += kMoveThreads) {
            const int e = expert_of(p, i, p.entries);
            if (e >= 0) atomicAdd(i < first ? &next[e] : &total[e], 1);
        }
        __syncthreads();
        for (int e = threadIdx.x; e < E; e += kMoveThreads) total[e] += next[e];
    } else if (kCounted == kPerBlock) {
        // threads side by side take neighbouring experts of one block; there are few experts
        const int e = threadIdx.x % E, row = threadIdx.x / E, rows = kMoveThreads / E;
        int all = 0, before = 0;
        if (row < rows) {
#pragma unroll 8
            for (int c = row; c < p.chunks; c += rows) {
                const int n = p.counts[(size_t)c * E + e];
                all += n;
                if (c < (int)blockIdx.x) before += n;
            }
            atomicAdd(&total[e], all);
            atomicAdd(&next[e], before);
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

    constexpr int W = kWidthOf<T>;
    const Rows<T> x(m.x, m.tokens, m.width), rows(m.out, p.entries, m.width);
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
        // the rows of the part's tokens: kLanes lanes to a token and pass; of few tokens several passes at a time (64 x 8 x 4096: 13 us without)
        constexpr int kTeams = kMoveThreads / kLanes, kAtOnce = 4;
        const int token0 = (int)(part / m.top_k), tokens = (int)((end - part) / m.top_k), tl = threadIdx.x % kLanes;
        int aside = 1;
        while (aside < m.passes && 2 * aside * tokens <= kTeams) aside *= 2;
        const int team = threadIdx.x / kLanes / aside, teams = kTeams / aside;
        for (int pass = blockIdx.y * aside; pass < m.passes; pass += gridDim.y * aside) {
            const int column = slot_of<kLanes, kRagged>(pass + threadIdx.x / kLanes % aside, tl) * W;  // may be behind the row
            for (int base = 0; base < tokens; base += teams * kAtOnce) {
                if constexpr (!kRagged) {
                    uint4 v[kAtOnce];
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        const int t = base + i * teams + team;
                        v[i] = x.template fetch<false>(token0 + t, column, t < tokens);
                    }
                    for (int j = 0; j < m.top_k; ++j) {
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i) {
                            const int t = base + i * teams + team;
                            const int at = t < tokens ? place[t * m.top_k + j] : -1;
                            if (at >= 0) rows.template store<false>(at, column, v[i]);
                        }
                    }
                } else {
                    for (int j = 0; j < m.top_k; ++j) {
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i) {
                            const int t = base + i * teams + team;
                            const int at = t < tokens ? place[t * m.top_k + j] : -1;
                            const int own = column - rows.lead(max(at, 0));
                            const uint4 v = x.template fetch<true>(token0 + (at >= 0 ? t : 0), own, at >= 0);
                            if (at >= 0 && takes<kLanes, kRagged>(tl)) rows.template store<true>(at, own, v);
                        }
                    }
                }
            }
        }
        __syncthreads();
    }
    clear_rows<T, kRagged>(rows.base, m.width, start[E], p.entries, ((long long)blockIdx.y * gridDim.x + blockIdx.x) * kMoveThreads + threadIdx.x,
                           (long long)gridDim.x * gridDim.y * kMoveThreads);
}

// ---- host --------------------------------------------------------------------------------------------------------------------
// Lanes that take a token, and passes over its vectors: the fewest lanes' turns, wider teams where these are nearly as few.
template <typename T>
void set_passes(MoveArgs &p, int &lanes, bool &ragged) {
    constexpr int W = kWidthOf<T>;
    ragged = p.width % W != 0;
    const long long slots = ragged ? (p.width + 2 * W - 2) / W : p.width / W;  // vectors that a row can touch
    long long least = 0;
    for (int l = 32; l >= 4; l /= 2) {
        const long long passes = ceil_div(slots, l - (ragged ? 1 : 0)), turns = passes * l;
        if (l < 32 && turns * 8 > least * 7) continue;
        least = turns;
        lanes = l;
        p.passes = (int)passes;
    }
}

template <typename T, int kLanes, bool kRagged, int kAtOnce>
int run_combine(const MoveArgs &p, bool backward, cudaStream_t st) {
    long long units = p.tokens * p.passes, most = kCombineBlocks * kSms;
    auto kernel = combine_kernel<T, kLanes, kRagged, kAtOnce>;
    MoveArgs q = p;
    if (backward) {
        units = p.tokens;
        most = (kRagged ? 8 : kCombineBackwardBlocks<kRagged, kAtOnce>) * kSms;
        kernel = combine_backward_kernel<T, kLanes, kRagged, kAtOnce>;
        // wide rows of few tokens: a block to a token
        if (p.passes > 1 && p.tokens < 8 * kSms * kWarps) {
            q.passes = (int)ceil_div((long long)p.passes * kLanes, kThreads - (kRagged ? kWarps : 0));
            units *= kThreads / kLanes;
            kernel = combine_backward_kernel<T, 0, kRagged, kAtOnce>;
        }
    }
    const unsigned blocks = (unsigned)std::min<long long>(ceil_div(units, kThreads / kLanes), most);
    if (const int rc = launched(launch_early(kernel, blocks, kThreads, 0, st, 1, q))) return rc;
    if (!backward || !p.out) return FDA_OK;
    const unsigned clears = (unsigned)std::min<long long>(ceil_div(p.entries, kThreads), kClearBlocks * kSms);
    return launched(launch_early(clear_unwritten_kernel<T, kRagged>, clears, kThreads, 0, st, 1, q));
}

template <typename T, bool kRagged, int kAtOnce>
int run_combine(const MoveArgs &p, int lanes, bool backward, cudaStream_t st) {
    if (lanes == 4) return run_combine<T, 4, kRagged, kAtOnce>(p, backward, st);
    if (lanes == 8) return run_combine<T, 8, kRagged, kAtOnce>(p, backward, st);
    if (lanes == 16) return run_combine<T, 16, kRagged, kAtOnce>(p, backward, st);
    return run_combine<T, 32, kRagged, kAtOnce>(p, backward, st);
}

template <typename T>
int run_combine(MoveArgs p, bool backward, cudaStream_t st) {
    int lanes;
    bool ragged;
    set_passes<T>(p, lanes, ragged);
    if (p.top_k <= 2) return ragged ? run_combine<T, true, 2>(p, lanes, backward, st) : run_combine<T, false, 2>(p, lanes, backward, st);
    return ragged ? run_combine<T, true, 4>(p, lanes, backward, st) : run_combine<T, false, 4>(p, lanes, backward, st);
}

int run_combine(const MoveArgs &p, int dtype, bool backward, cudaStream_t st) {
    if (dtype == FDA_DTYPE_F32) return run_combine<float>(p, backward, st);
    if (dtype == FDA_DTYPE_F16) return run_combine<__half>(p, backward, st);
    return run_combine<__nv_bfloat16>(p, backward, st);
}

// Entries that every block counts by itself.  9003 by 131 experts take 10.7 us so and 13.9 by the launches before (16 experts: 10.4 and 11.5);
// 16000 by 64 take longer.
constexpr long long kFewEntries = 10240;

// Entries of a block, and blocks along them.
void set_chunks(SortArgs &s, int top_k, int passes, unsigned &slices) {
    const long long tokens = s.entries / top_k;
    const bool few = s.entries <= kFewEntries;
    // few: a token to a warp and pass, and slices of columns until every SM has a block; never more than two blocks to an SM along the tokens
    const long long per = std::max<long long>(ceil_div(tokens, kMostChunks), few ? std::max(1, kMoveWarps / passes) : 1);
    s.chunk = (int)(per * top_k);
    s.chunks = (int)ceil_div(tokens, per);
    slices = few ? (unsigned)std::min<long long>(passes, std::max<long long>(1, kSms / s.chunks)) : 1;
}
Counted counted(const SortArgs &s) {
    if (s.entries <= kFewEntries) return kByItself;
    // blocks add up a few experts' counts while a third launch would start: 147456 entries by 16 experts 25.6 us so and 27.4 with a scan, 80000
    // by 64 experts 19.5 and 18.7
    return s.n_experts <= kFewExperts ? kPerBlock : kScanned;
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
    set_passes<T>(p, lanes, ragged);
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
size_t counts_bytes(int n_experts) { return fda_linear::round256((size_t)kMostChunks * n_experts * sizeof(int)); }

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
    p.x = x; p.out = rows; p.tokens = tokens; p.top_k = top_k; p.entries = s.entries; p.width = features;
    if (dtype == FDA_DTYPE_F32) return run_dispatch<float>(s, p, st);
    if (dtype == FDA_DTYPE_F16) return run_dispatch<__half>(s, p, st);
    return run_dispatch<__nv_bfloat16>(s, p, st);
}

int fda_combine_rows(const void *rows, const int64_t *position, const void *weights, const void *residual, void *y, long long tokens, int top_k,
                     int features, int dtype, int weight_dtype, void *stream) {
    if (const int rc = check_rows(tokens, top_k, features, dtype)) return rc;
    if (weights && weight_dtype != dtype && weight_dtype != FDA_DTYPE_F32) return FDA_ERR_BAD_DTYPE;
    if (tokens == 0) return FDA_OK;
    if (!rows || !position || !y) return FDA_ERR_NULL_POINTER;
    if (misaligned16(rows) || misaligned16(residual) || misaligned16(y)) return FDA_ERR_MISALIGNED;
    MoveArgs p{};
    p.rows = rows; p.position = position; p.weights = weights; p.residual = residual; p.out = y; p.tokens = tokens; p.top_k = top_k;
    p.entries = tokens * top_k; p.width = features; p.wide_weights = weight_dtype == FDA_DTYPE_F32;
    return run_combine(p, dtype, false, static_cast<cudaStream_t>(stream));
}

size_t fda_combine_rows_backward_workspace_bytes(long long tokens, int top_k) {
    if (tokens <= 0 || top_k < 1 || top_k > kMostChoices || tokens > INT32_MAX / top_k) return 0;
    return fda_linear::round256((size_t)tokens * top_k * sizeof(int));
}

int fda_combine_rows_backward(const void *rows, const int64_t *position, const void *weights, const void *grad_y, void *grad_rows,
                              void *grad_weights, void *workspace, size_t workspace_bytes, long long tokens, int top_k, int features, int dtype,
                              int weight_dtype, void *stream) {
    if (const int rc = check_rows(tokens, top_k, features, dtype)) return rc;
    if ((weights || grad_weights) && weight_dtype != dtype && weight_dtype != FDA_DTYPE_F32) return FDA_ERR_BAD_DTYPE;
    if (tokens == 0 || (!grad_rows && !grad_weights)) return FDA_OK;
    if (!position || !grad_y || (grad_weights && !rows)) return FDA_ERR_NULL_POINTER;
    if (grad_rows && (!workspace || workspace_bytes < fda_combine_rows_backward_workspace_bytes(tokens, top_k))) return FDA_ERR_WORKSPACE;
    if (misaligned16(rows) || misaligned16(grad_y) || misaligned16(grad_rows) || (grad_rows && misaligned16(workspace))) return FDA_ERR_MISALIGNED;
    MoveArgs p{};
    p.rows = rows; p.position = position; p.entry = static_cast<int *>(workspace); p.weights = weights; p.grad = grad_y; p.out = grad_rows; p.grad_weights = grad_weights;
    p.tokens = tokens; p.top_k = top_k; p.entries = tokens * top_k; p.width = features; p.wide_weights = weight_dtype == FDA_DTYPE_F32;
    return run_combine(p, dtype, true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

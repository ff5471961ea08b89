// Rows sorted by expert, and back.
//
//     entry i = token * top_k + choice;  an entry whose expert is outside 0 .. n_experts - 1 belongs to none
//     position[i] = entries of lower experts + entries of its own expert before it, -1 for none;  start[e] = entries of lower experts
//     dispatch   rows[position[i]] = x[token]                                 rows behind the last expert's are 0
//     combine    y[token] = sum over choices of weight * rows[position] + residual
//     its gradients   drows[position] = weight * dy[token],   dweight = <rows[position], dy[token]>,   dresidual = dy
//     dispatch's      dx[token] = sum over choices of drows[position]  (a combine without weights)
//
// A counting sort by chunks of entries: counts of each chunk, their sums over the chunks before it, then each entry's place among
// its expert's.  The order is that of the entries, whatever the blocks do.  Moving the rows is bound by DRAM: dispatch reads a row of x once
// and writes it top_k times, its opposite the other way round, both without atomics.
#include "fda_rows.cuh"

#include <algorithm>

namespace {

using namespace fda_rows;

constexpr unsigned kAll = 0xffffffffu;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMostExperts = 1024, kMostChoices = 32;
constexpr int kChunk = 2048;  // entries of a block

struct SortArgs {
    const int64_t *experts;
    int64_t *start, *position;
    int *counts;  // [chunks][n_experts]: of a chunk, then of those before it
    int *total;   // [n_experts]
    long long entries;
    int n_experts, chunks;
};

__device__ __forceinline__ int expert_of(const SortArgs &p, long long i) {
    if (i >= p.entries) return -1;
    const int64_t e = p.experts[i];
    return e >= 0 && e < p.n_experts ? (int)e : -1;
}

__global__ void __launch_bounds__(kThreads) sort_count_kernel(const SortArgs p) {
    __shared__ int count[kMostExperts];
    wait_for_previous_kernel();
    for (int e = threadIdx.x; e < p.n_experts; e += kThreads) count[e] = 0;
    __syncthreads();
    const long long first = (long long)blockIdx.x * kChunk;
    for (int i = threadIdx.x; i < kChunk; i += kThreads) {
        const int e = expert_of(p, first + i);
        if (e >= 0) atomicAdd(&count[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.n_experts; e += kThreads) p.counts[(size_t)blockIdx.x * p.n_experts + e] = count[e];
}

// Over the chunks, 32 experts a block: 32 runs of chunks side by side.
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

// start[0 .. n_experts] from the totals, by one block, into shared memory.
__device__ __forceinline__ void scan_totals(const SortArgs &p, int *start) {
    __shared__ int carry[kWarps];
    constexpr int kEach = kMostExperts / kThreads;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int n[kEach], sum = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int e = threadIdx.x * kEach + k;
        n[k] = e < p.n_experts ? p.total[e] : 0;
        sum += n[k];
    }
    const int upto = fda_linear::warp_scan_sum(sum);
    if (lane == 31) carry[warp] = upto;
    __syncthreads();
    int at = upto - sum;
    for (int w = 0; w < warp; ++w) at += carry[w];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int e = threadIdx.x * kEach + k;
        if (e <= p.n_experts) start[e] = at;
        at += n[k];
    }
    if (threadIdx.x == kThreads - 1 && p.n_experts == kMostExperts) start[kMostExperts] = at;
    __syncthreads();
}

__global__ void __launch_bounds__(kThreads) sort_place_kernel(const SortArgs p) {
    extern __shared__ int shared[];  // next[kWarps][n_experts], then start[n_experts + 1]
    wait_for_previous_kernel();
    const int E = p.n_experts, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int *next = shared, *start = shared + kWarps * E;
    scan_totals(p, start);
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= E; e += kThreads) p.start[e] = start[e];
    // a warp takes a run of the chunk; first its counts
    constexpr int kRun = kChunk / kWarps, kSteps = kRun / 32;
    const long long first = (long long)blockIdx.x * kChunk + warp * kRun;
    for (int i = threadIdx.x; i < kWarps * E; i += kThreads) next[i] = 0;
    __syncthreads();
    int expert[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        expert[k] = expert_of(p, first + k * 32 + lane);
        if (expert[k] >= 0) atomicAdd(&next[warp * E + expert[k]], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kThreads) {
        int at = start[e] + p.counts[(size_t)blockIdx.x * E + e];
        for (int w = 0; w < kWarps; ++w) {
            const int n = next[w * E + e];
            next[w * E + e] = at;
            at += n;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        const long long i = first + k * 32 + lane;
        const unsigned same = __match_any_sync(kAll, expert[k]);
        const int before = __popc(same & ((1u << lane) - 1));
        int at = -1;
        if (expert[k] >= 0) at = next[warp * E + expert[k]] + before;
        __syncwarp();
        if (expert[k] >= 0 && before == 0) next[warp * E + expert[k]] += __popc(same);
        __syncwarp();
        if (i < p.entries) p.position[i] = at;
    }
}

// ---- rows --------------------------------------------------------------------------------------------------------------------
struct MoveArgs {
    const void *rows, *x, *weights, *residual, *grad;
    const int64_t *position, *end;  // end: where the last expert's rows end
    void *out, *grad_weights;
    long long tokens;
    int top_k, width, weight_dtype;
};

// Vectors of kWidth elements, or single ones (kWidth 1) where rows do not start on 16-byte boundaries.
template <typename T, int kWidth>
struct Piece {
    Raw<T, kWidth> raw;
    __device__ __forceinline__ void load(const T *p) { raw.load(p); }
    __device__ __forceinline__ void store(T *p) const { raw.store(p); }
    __device__ __forceinline__ void get(float *v) const { raw.get(v); }
    __device__ __forceinline__ void set(const float *v) { raw.set(v); }
    __device__ __forceinline__ void clear() { raw.clear(); }
};
template <typename T>
struct Piece<T, 1> {
    T raw;
    __device__ __forceinline__ void load(const T *p) { raw = *p; }
    __device__ __forceinline__ void store(T *p) const { *p = raw; }
    __device__ __forceinline__ void get(float *v) const { v[0] = to_f32(raw); }
    __device__ __forceinline__ void set(const float *v) { raw = from_f32<T>(v[0]); }
    __device__ __forceinline__ void clear() { raw = from_f32<T>(0.f); }
};

// A position that leads nowhere counts as none.
__device__ __forceinline__ long long row_of(const MoveArgs &p, long long entry) {
    const int64_t at = p.position[entry];
    return at >= 0 && at < p.tokens * p.top_k ? at : -1;
}

// Rows behind the last expert's are 0: every warp of the grid clears some.
template <typename T, int kWidth>
__device__ __forceinline__ void clear_rest(const MoveArgs &p, T *rows) {
    const long long all = p.tokens * p.top_k, end = min(max((long long)*p.end, 0ll), all);
    const int lane = threadIdx.x % 32;
    Piece<T, kWidth> zero;
    zero.clear();
    for (long long row = end + (long long)blockIdx.x * kWarps + threadIdx.x / 32; row < all; row += (long long)gridDim.x * kWarps)
        for (int c = lane * kWidth; c < p.width; c += 32 * kWidth) zero.store(rows + row * p.width + c);
}

template <typename T, int kWidth>
__global__ void __launch_bounds__(kThreads) dispatch_kernel(const MoveArgs p) {
    wait_for_previous_kernel();
    const int lane = threadIdx.x % 32;
    T *rows = static_cast<T *>(p.out);
    for (long long token = (long long)blockIdx.x * kWarps + threadIdx.x / 32; token < p.tokens; token += (long long)gridDim.x * kWarps) {
        const long long mine = lane < p.top_k ? row_of(p, token * p.top_k + lane) : -1;
        for (int c = lane * kWidth; c - lane * kWidth < p.width; c += 32 * kWidth) {
            Piece<T, kWidth> v;
            if (c < p.width) v.load(static_cast<const T *>(p.x) + token * p.width + c);
            for (int j = 0; j < p.top_k; ++j) {
                const long long at = __shfl_sync(kAll, mine, j);
                if (at >= 0 && c < p.width) v.store(rows + at * p.width + c);
            }
        }
    }
    clear_rest<T, kWidth>(p, rows);
}

template <typename T, int kWidth>
__global__ void __launch_bounds__(kThreads) combine_kernel(const MoveArgs p) {
    wait_for_previous_kernel();
    const int lane = threadIdx.x % 32;
    const T *rows = static_cast<const T *>(p.rows);
    for (long long token = (long long)blockIdx.x * kWarps + threadIdx.x / 32; token < p.tokens; token += (long long)gridDim.x * kWarps) {
        const long long entry = token * p.top_k + lane;
        const long long mine = lane < p.top_k ? row_of(p, entry) : -1;
        const float weight = mine >= 0 && p.weights ? load_as_f32(p.weights, p.weight_dtype, entry) : 1.f;
        for (int c = lane * kWidth; c - lane * kWidth < p.width; c += 32 * kWidth) {
            float sum[kWidth];
            Piece<T, kWidth> v;
#pragma unroll
            for (int i = 0; i < kWidth; ++i) sum[i] = 0.f;
            for (int j = 0; j < p.top_k; ++j) {
                const long long at = __shfl_sync(kAll, mine, j);
                const float w = __shfl_sync(kAll, weight, j);
                if (at < 0 || c >= p.width) continue;
                v.load(rows + at * p.width + c);
                float e[kWidth];
                v.get(e);
#pragma unroll
                for (int i = 0; i < kWidth; ++i) sum[i] += w * e[i];
            }
            if (c >= p.width) continue;
            if (p.residual) {
                v.load(static_cast<const T *>(p.residual) + token * p.width + c);
                float e[kWidth];
                v.get(e);
#pragma unroll
                for (int i = 0; i < kWidth; ++i) sum[i] += e[i];
            }
            v.set(sum);
            v.store(static_cast<T *>(p.out) + token * p.width + c);
        }
    }
}

template <typename T, int kWidth>
__global__ void __launch_bounds__(kThreads) combine_backward_kernel(const MoveArgs p) {
    wait_for_previous_kernel();
    const int lane = threadIdx.x % 32;
    const T *rows = static_cast<const T *>(p.rows), *grad = static_cast<const T *>(p.grad);
    T *out = static_cast<T *>(p.out);
    for (long long token = (long long)blockIdx.x * kWarps + threadIdx.x / 32; token < p.tokens; token += (long long)gridDim.x * kWarps) {
        const long long entry = token * p.top_k + lane;
        const long long mine = lane < p.top_k ? row_of(p, entry) : -1;
        const float weight = mine >= 0 && p.weights ? load_as_f32(p.weights, p.weight_dtype, entry) : 1.f;
        float dweight = 0.f;
        for (int j = 0; j < p.top_k; ++j) {
            const long long at = __shfl_sync(kAll, mine, j);
            const float w = __shfl_sync(kAll, weight, j);
            float dot = 0.f;
            if (at >= 0)
                for (int c = lane * kWidth; c < p.width; c += 32 * kWidth) {
                    Piece<T, kWidth> v;
                    float dy[kWidth], e[kWidth];
                    v.load(grad + token * p.width + c);
                    v.get(dy);
                    if (p.grad_weights) {
                        v.load(rows + at * p.width + c);
                        v.get(e);
#pragma unroll
                        for (int i = 0; i < kWidth; ++i) dot += dy[i] * e[i];
                    }
                    if (out) {
#pragma unroll
                        for (int i = 0; i < kWidth; ++i) dy[i] *= w;
                        v.set(dy);
                        v.store(out + at * p.width + c);
                    }
                }
            if (p.grad_weights) {
                dot = lanes_sum<32>(dot);
                if (lane == j) dweight = dot;
            }
        }
        if (p.grad_weights && lane < p.top_k) store_from_f32(p.grad_weights, p.weight_dtype, entry, dweight);
    }
    if (out) clear_rest<T, kWidth>(p, out);
}

enum Move { kDispatch, kCombine, kCombineBackward };

template <typename T, int kWidth>
int run_move(Move move, const MoveArgs &p, cudaStream_t st) {
    const unsigned blocks = (unsigned)std::min<long long>(ceil_div(p.tokens, kWarps), 8 * kSms);
    const auto kernel = move == kDispatch ? dispatch_kernel<T, kWidth> : move == kCombine ? combine_kernel<T, kWidth> : combine_backward_kernel<T, kWidth>;
    return launched(launch_early(kernel, blocks, kThreads, 0, st, 1, p));
}

template <typename T>
int run_move(Move move, const MoveArgs &p, cudaStream_t st) {
    constexpr int W = 16 / (int)sizeof(T);
    return p.width % W == 0 ? run_move<T, W>(move, p, st) : run_move<T, 1>(move, p, st);
}

int run_move(Move move, const MoveArgs &p, int dtype, cudaStream_t st) {
    if (dtype == FDA_DTYPE_F32) return run_move<float>(move, p, st);
    if (dtype == FDA_DTYPE_F16) return run_move<__half>(move, p, st);
    return run_move<__nv_bfloat16>(move, p, st);
}

int check_rows(long long tokens, int top_k, int width, int dtype) {
    if (!known_dtype(dtype)) return FDA_ERR_BAD_DTYPE;
    if (tokens < 0 || top_k < 1 || width < 1 || width >= 1 << 26) return FDA_ERR_BAD_SHAPE;
    if (top_k > kMostChoices) return FDA_ERR_TOO_LARGE_STATIC;
    if (tokens > INT32_MAX / top_k) return FDA_ERR_BAD_SHAPE;
    return FDA_OK;
}

size_t counts_bytes(long long entries, int n_experts) { return fda_linear::round256((size_t)ceil_div(entries, kChunk) * n_experts * sizeof(int)); }

}  // namespace

extern "C" {

size_t fda_dispatch_workspace_bytes(long long tokens, int top_k, int n_experts) {
    if (tokens <= 0 || top_k < 1 || top_k > kMostChoices || tokens > INT32_MAX / top_k || n_experts < 1 || n_experts > kMostExperts) return 0;
    return counts_bytes(tokens * top_k, n_experts) + fda_linear::round256((size_t)n_experts * sizeof(int));
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
    if (!workspace || workspace_bytes < fda_dispatch_workspace_bytes(tokens, top_k, n_experts)) return FDA_ERR_WORKSPACE;
    if ((uintptr_t)workspace % 256 || misaligned16(x) || misaligned16(rows)) return FDA_ERR_MISALIGNED;
    SortArgs s{};
    s.experts = experts; s.start = group_start_index; s.position = position;
    s.entries = tokens * top_k; s.n_experts = n_experts; s.chunks = (int)ceil_div(s.entries, kChunk);
    s.counts = static_cast<int *>(workspace);
    s.total = reinterpret_cast<int *>(static_cast<char *>(workspace) + counts_bytes(s.entries, n_experts));
    if (const int rc = launched(launch_early(sort_count_kernel, s.chunks, kThreads, 0, st, 1, s))) return rc;
    if (const int rc = launched(launch_early(sort_scan_kernel, (unsigned)ceil_div(n_experts, 32), 1024, 0, st, 1, s))) return rc;
    const int shared = ((kWarps + 1) * n_experts + 1) * (int)sizeof(int);
    if (const int rc = launched(launch_early(sort_place_kernel, s.chunks, kThreads, shared, st, 1, s))) return rc;
    MoveArgs p{};
    p.x = x; p.position = position; p.end = group_start_index + n_experts; p.out = rows; p.tokens = tokens; p.top_k = top_k; p.width = features;
    return run_move(kDispatch, p, dtype, st);
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
    return run_move(kCombine, p, dtype, static_cast<cudaStream_t>(stream));
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
    return run_move(kCombineBackward, p, dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

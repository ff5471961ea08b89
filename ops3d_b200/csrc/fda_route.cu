// Routing of tokens to experts, forward and backward.
//
//     score = softmax(logits) or sigmoid(logits),   select = score + bias                                     per token
//     the top_k largest of select, largest first, among the experts of the top_groups best groups (n_groups consecutive runs of
//     experts; a group is worth its largest select, or the sum of its two largest); ties go to the lower index
//     weight_j = scale * score_j / sum of the chosen scores, or scale * score_j
//
// A warp takes a token, a lane kPer neighbouring experts, so that of equal values the lowest lane's comes first.  What is chosen is what
// exact scores choose.  Where select is a monotone function of one logit (no bias, no sum over a group) the logits themselves are
// compared.  Elsewhere scores in fp32 are compared as long as their distance is beyond what they can be off by; a token for
// which it is not is decided by scores in 64 bits, so that no choice depends on how an exponential rounds.  A NaN counts as minus
// infinity in comparisons, and stays one in the weights.
#include "fda_rows.cuh"

#include <algorithm>

namespace {

using namespace fda_rows;

constexpr unsigned kAll = 0xffffffffu;
constexpr int kThreads = 256;
constexpr int kMostExperts = 1024, kMostChoices = 32, kMostExpertGroups = 32;

struct RouteArgs {
    const void *logits;
    const float *bias;  // may be nullptr
    float *weights;
    int64_t *experts;
    const float *grad_weights;
    void *grad_logits;
    long long tokens;
    int n_experts, top_k, sigmoid, n_groups, top_groups, top2, renormalise, dtype;
    float scale;
};

// Numbers in the order of unsigned integers, all above 0; -0 as 0, NaN as minus infinity.
__device__ __forceinline__ unsigned order_of(float v) {
    if (!(v == v)) v = -INFINITY;
    const unsigned u = __float_as_uint(v + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_of(double v) {
    if (!(v == v)) v = -INFINITY;
    const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ unsigned warp_max(unsigned v) { return __reduce_max_sync(kAll, v); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        const unsigned long long o = __shfl_xor_sync(kAll, v, d);
        v = o > v ? o : v;
    }
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) v = fmaxf(v, __shfl_xor_sync(kAll, v, d));
    return v;
}
template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(kAll, v, d);
    return v;
}

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
// 1 / (1 + e^-v)
template <typename F>
__device__ __forceinline__ F sigmoid_of(F v) { return (F)1 / ((F)1 + exp_of(-v)); }

// By how much a score in fp32 can be off, relative to itself: e^(l - max) by the rounding of l - max (2^-24 |l - max|, at most 104 before
// it is 0) and the exponential (2 units), their sum by kPer + 5 additions, the quotient; 1 / (1 + e^-l) by less.
constexpr float kScoreError = 1.f / 65536.f;
// The same for the additions, relative to the larger of two values that are compared: the smaller one, where it is below minus that, is
// further away than it can be off by.
constexpr float kSumError = 1.f / 2097152.f;
constexpr float kSmallest = 1e-37f;           // scores below the normal range have an absolute error

// The top_k experts of a token whose select values are v (float or double): lane j gets the j-th.  allowed: bit i of a lane
// for its expert i.
template <typename K, int kPer>
__device__ __forceinline__ int choose(const K (&key)[kPer], unsigned allowed, int top_k) {
    const int lane = threadIdx.x % 32;
    int mine = 0;
    unsigned left = allowed;
    for (int j = 0; j < top_k; ++j) {
        K best = 0;
        int slot = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if ((left >> i & 1) && key[i] > best) { best = key[i]; slot = i; }
        const K top = warp_max(best);
        const int winner = __ffs(__ballot_sync(kAll, best == top)) - 1;
        if (lane == winner) left &= ~(1u << slot);
        const int expert = __shfl_sync(kAll, lane * kPer + slot, winner);
        if (lane == j) mine = expert;
    }
    return mine;
}

// Which experts of a lane are in the top_groups best groups.  values [n_experts]: select values of the token in shared memory.
// unsure: set where the border between the groups is closer than the values' errors (`error` of one value).
template <typename F, int kPer>
__device__ __forceinline__ unsigned allowed_experts(const RouteArgs &p, const F *values, F error, bool &unsure) {
    const int lane = threadIdx.x % 32, size = p.n_experts / p.n_groups;
    unsigned experts = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (lane * kPer + i < p.n_experts) experts |= 1u << i;
    if (p.top_groups == p.n_groups) return experts;
    // 32 / (a power of two of groups) lanes to a group
    int share = 32;
    while (32 / share < p.n_groups) share /= 2;
    const int group = lane / share;
    F first = -INFINITY, second = -INFINITY;
    if (group < p.n_groups)
        for (int i = lane % share; i < size; i += share) {
            F v = values[group * size + i];
            if (!(v == v)) v = -INFINITY;
            if (v > first) { second = first; first = v; }
            else if (v > second) second = v;
        }
    for (int d = 1; d < share; d *= 2) {
        const F a = __shfl_xor_sync(kAll, first, d), b = __shfl_xor_sync(kAll, second, d);
        if (a > first) { second = first > b ? first : b; first = a; }
        else second = a > second ? a : second;
    }
    F worth = p.top2 && size > 1 ? first + second : first;
    if (!(worth == worth)) worth = -INFINITY;
    // a group's place: how many are better
    int place = 0;
    for (int g = 0; g < p.n_groups; ++g) {
        const F other = __shfl_sync(kAll, worth, g * share);
        if (other > worth || (other == worth && g < group)) ++place;
    }
    const bool chosen = group < p.n_groups && place < p.top_groups;
    if (error >= 0) {
        F low = chosen ? worth : (F)INFINITY, high = group < p.n_groups && !chosen ? worth : -(F)INFINITY;
        for (int d = 16; d > 0; d /= 2) {
            const F a = __shfl_xor_sync(kAll, low, d), b = __shfl_xor_sync(kAll, high, d);
            low = a < low ? a : low;
            high = b > high ? b : high;
        }
        if (!(low - high > error) && low > -(F)INFINITY) unsure = true;
    }
    const unsigned groups = __ballot_sync(kAll, chosen && lane % share == 0);
    unsigned allowed = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if ((experts >> i & 1) && (groups >> ((lane * kPer + i) / size * share) & 1)) allowed |= 1u << i;
    return allowed;
}

template <typename T>
__device__ __forceinline__ float logit(const RouteArgs &p, long long token, int expert) {
    return to_f32(static_cast<const T *>(p.logits)[token * p.n_experts + expert]);
}

// Softmax's shift and the inverse of its sum; a row without a finite logit has no score.
template <typename F, int kPer>
__device__ __forceinline__ void softmax_of(const float (&l)[kPer], int n_experts, F &shift, F &inverse) {
    const int lane = threadIdx.x % 32;
    float top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (lane * kPer + i < n_experts) {
            top = fmaxf(top, l[i]);
            nan |= !(l[i] == l[i]);
        }
    shift = warp_max(top);
    if (__any_sync(kAll, nan)) shift = NAN;
    if (shift == -(F)INFINITY) {
        shift = 0;
        inverse = 0;
        return;
    }
    F sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (lane * kPer + i < n_experts) sum += exp_of((F)l[i] - shift);
    inverse = (F)1 / warp_sum(sum);
}

// A score as every comparison of a token computes it: no contraction with what follows.
__device__ __forceinline__ float score_of(const RouteArgs &p, float l, float shift, float inverse) {
    if (p.sigmoid) return sigmoid_of(l);
    return inverse == 0.f ? 0.f : __fmul_rn(expf(l - shift), inverse);
}

// The choice by scores in 64 bits; values: [n_experts] numbers of the warp in shared memory.
template <typename T, int kPer>
__device__ __noinline__ int choose_exactly(const RouteArgs &p, long long token, double *values) {
    const int lane = threadIdx.x % 32;
    float l[kPer];
    for (int i = 0; i < kPer; ++i) l[i] = lane * kPer + i < p.n_experts ? logit<T>(p, token, lane * kPer + i) : -INFINITY;
    double shift = 0, inverse = 1;
    if (!p.sigmoid) softmax_of<double, kPer>(l, p.n_experts, shift, inverse);
    unsigned long long key[kPer];
    __syncwarp();
    for (int i = 0; i < kPer; ++i) {
        const int e = lane * kPer + i;
        if (e >= p.n_experts) { key[i] = 0; continue; }
        double v = p.sigmoid ? sigmoid_of((double)l[i]) : exp((double)l[i] - shift) * inverse;
        if (p.bias) v += (double)p.bias[e];
        values[e] = v;
        key[i] = order_of(v);
    }
    __syncwarp();
    bool unsure = false;
    return choose<unsigned long long, kPer>(key, allowed_experts<double, kPer>(p, values, -1.0, unsure), p.top_k);
}

// Score of a chosen expert (lane j's), before scaling, and what the weights are divided by.
struct Chosen {
    float score, total;
};
template <int kPer>
__device__ __forceinline__ Chosen chosen_scores(const RouteArgs &p, float logit, float shift, float inverse) {
    const bool there = (int)(threadIdx.x % 32) < p.top_k;
    Chosen c;
    if (p.sigmoid) {
        c.score = there ? sigmoid_of(logit) : 0.f;
        c.total = p.renormalise ? warp_sum(c.score) : 1.f;
    } else if (p.renormalise) {  // softmax over the chosen
        const float nan = there && !(logit == logit) ? logit : 0.f;
        const float top = warp_max(there ? logit : -INFINITY);
        c.score = !there ? 0.f : top == -INFINITY && nan == 0.f ? 0.f : expf(logit - top);
        c.total = warp_sum(c.score);
    } else {
        c.score = there ? (inverse == 0.f ? 0.f : expf(logit - shift) * inverse) : 0.f;
        c.total = 1.f;
    }
    return c;
}

template <typename T, int kPer>
__global__ void __launch_bounds__(kThreads) route_forward_kernel(const RouteArgs p) {
    extern __shared__ double shared[];
    wait_for_previous_kernel();
    const int lane = threadIdx.x % 32, E = p.n_experts;
    double *values64 = shared + (threadIdx.x / 32) * E;
    float *values = reinterpret_cast<float *>(values64);
    const bool grouped = p.top_groups < p.n_groups;
    // what is compared: logits, or scores
    const bool sums = grouped && p.top2 && E > p.n_groups;
    const bool by_score = p.bias || sums;
    const bool need_softmax = !p.sigmoid && (by_score || !p.renormalise);
    for (long long token = (long long)blockIdx.x * (kThreads / 32) + threadIdx.x / 32; token < p.tokens; token += (long long)gridDim.x * (kThreads / 32)) {
        float l[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) l[i] = lane * kPer + i < E ? logit<T>(p, token, lane * kPer + i) : -INFINITY;
        float shift = 0.f, inverse = 1.f;
        if (need_softmax) softmax_of<float, kPer>(l, E, shift, inverse);
        unsigned key[kPer];
        float v[kPer], score[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = lane * kPer + i;
            score[i] = 0.f;
            v[i] = l[i];
            if (by_score && e < E) {
                score[i] = score_of(p, l[i], shift, inverse);
                v[i] = p.bias ? __fadd_rn(score[i], p.bias[e]) : score[i];
            }
            key[i] = e < E ? order_of(p.bias ? v[i] : l[i]) : 0;
        }
        bool unsure = false;
        unsigned allowed = kPer == 32 ? kAll : (1u << kPer) - 1;
        if (grouped) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (lane * kPer + i < E) values[lane * kPer + i] = v[i];
            __syncwarp();
            // a group is worth up to two values, and two groups are compared
            float error = 0.f;
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (fabsf(v[i]) < INFINITY) error = fmaxf(error, score[i] * kScoreError + fabsf(v[i]) * kSumError);
            allowed = allowed_experts<float, kPer>(p, values, by_score ? 4.f * (warp_max(error) + kSmallest) : -1.f, unsure);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (lane * kPer + i >= E) allowed &= ~(1u << i);
        }
        int mine = choose<unsigned, kPer>(key, allowed, p.top_k);
        if (p.bias && !unsure) {
            // the chosen among themselves, and the rest against the last of them
            const bool there = lane < p.top_k;
            const float ml = there ? logit<T>(p, token, mine) : 0.f, mb = there ? p.bias[mine] : 0.f;
            const float ms = there ? score_of(p, ml, shift, inverse) : 0.f, mv = __fadd_rn(ms, mb);
            const float nl = __shfl_down_sync(kAll, ml, 1), nb = __shfl_down_sync(kAll, mb, 1), ns = __shfl_down_sync(kAll, ms, 1),
                        nv = __shfl_down_sync(kAll, mv, 1);
            bool close = lane + 1 < p.top_k && !(mv - nv > (ms + ns) * kScoreError + fabsf(mv) * kSumError + kSmallest) &&
                         !(ml == nl && mb == nb);
            const int last = p.top_k - 1;
            const float ll = __shfl_sync(kAll, ml, last), lb = __shfl_sync(kAll, mb, last), ls = __shfl_sync(kAll, ms, last),
                        lv = __shfl_sync(kAll, mv, last);
            const unsigned lk = order_of(lv);
            const int le = __shfl_sync(kAll, mine, last);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int e = lane * kPer + i;
                // those before the last in the order are chosen
                if (!(allowed >> i & 1) || key[i] > lk || (key[i] == lk && e <= le)) continue;
                if (!(lv - v[i] > (ls + score[i]) * kScoreError + fabsf(lv) * kSumError + kSmallest) &&
                    !(l[i] == ll && p.bias[e] == lb))
                    close = true;
            }
            unsure = __any_sync(kAll, close);
        }
        if (unsure) mine = choose_exactly<T, kPer>(p, token, values64);
        const float ml = lane < p.top_k ? logit<T>(p, token, mine) : -INFINITY;
        const Chosen c = chosen_scores<kPer>(p, ml, shift, inverse);
        if (lane < p.top_k) {
            p.weights[token * p.top_k + lane] = c.total == 0.f ? 0.f : p.scale * c.score / c.total;
            p.experts[token * p.top_k + lane] = mine;
        }
    }
}

// grad_logits from grad_weights: with s the scores of the chosen and S their sum,
//     softmax, renormalised    dl_j = w_j (dw_j - sum of dw w / scale)           (a softmax over the chosen alone)
//     softmax                  dl_i = scale p_i ([i chosen] dw_i - sum of dw p)
//     sigmoid                  dl_j = ds_j s_j (1 - s_j),  ds_j = scale (dw_j - sum of dw s / S) / S  or  scale dw_j
// An expert outside 0 .. n_experts - 1 gets none.  No atomics: a row is put together in shared memory.
template <typename T, int kPer>
__global__ void __launch_bounds__(kThreads) route_backward_kernel(const RouteArgs p) {
    extern __shared__ float rows[];
    wait_for_previous_kernel();
    const int lane = threadIdx.x % 32, E = p.n_experts;
    float *row = rows + (threadIdx.x / 32) * E;
    const bool dense = !p.sigmoid && !p.renormalise;
    for (long long token = (long long)blockIdx.x * (kThreads / 32) + threadIdx.x / 32; token < p.tokens; token += (long long)gridDim.x * (kThreads / 32)) {
        const int64_t chosen = lane < p.top_k ? p.experts[token * p.top_k + lane] : -1;
        const bool there = chosen >= 0 && chosen < E;
        const float dw = there ? p.grad_weights[token * p.top_k + lane] * p.scale : 0.f;
        const float ml = there ? logit<T>(p, token, (int)chosen) : -INFINITY;
        float l[kPer], shift = 0.f, inverse = 1.f;
        if (dense) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) l[i] = lane * kPer + i < E ? logit<T>(p, token, lane * kPer + i) : -INFINITY;
            softmax_of<float, kPer>(l, E, shift, inverse);
        }
        const Chosen c = chosen_scores<kPer>(p, ml, shift, inverse);
        const float s = c.score;
        float dl = 0.f, along = 0.f;
        if (p.sigmoid) {
            along = p.renormalise ? (c.total == 0.f ? 0.f : warp_sum(dw * s) / c.total) : 0.f;
            dl = c.total == 0.f ? 0.f : (dw - along) / c.total * s * (1.f - s);
        } else if (p.renormalise) {
            const float q = c.total == 0.f ? 0.f : s / c.total;
            dl = q * (dw - warp_sum(dw * q));
        } else {
            along = warp_sum(dw * s);
            dl = s * dw;
        }
        __syncwarp();
        for (int i = lane; i < E; i += 32) row[i] = 0.f;
        __syncwarp();
        if (there) row[chosen] = dl;
        __syncwarp();
        T *out = static_cast<T *>(p.grad_logits) + token * E;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = lane * kPer + i;
            if (e >= E) continue;
            float v = row[e];
            if (dense) v -= inverse == 0.f ? 0.f : expf(l[i] - shift) * inverse * along;
            out[e] = from_f32<T>(v);
        }
    }
}

template <typename T, int kPer>
int launch_route(bool backward, const RouteArgs &p, cudaStream_t st) {
    const unsigned blocks = (unsigned)std::min<long long>(ceil_div(p.tokens, kThreads / 32), 16 * kSms);
    const int shared = (kThreads / 32) * p.n_experts * (int)(backward ? sizeof(float) : sizeof(double));
    const auto kernel = backward ? route_backward_kernel<T, kPer> : route_forward_kernel<T, kPer>;
    if (shared > 48 * 1024)
        if (const int rc = launched(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared))) return rc;
    return launched(launch_early(kernel, blocks, kThreads, shared, st, 1, p));
}

template <typename T>
int launch_route(bool backward, const RouteArgs &p, cudaStream_t st) {
    if (p.n_experts <= 32) return launch_route<T, 1>(backward, p, st);
    if (p.n_experts <= 64) return launch_route<T, 2>(backward, p, st);
    if (p.n_experts <= 128) return launch_route<T, 4>(backward, p, st);
    if (p.n_experts <= 256) return launch_route<T, 8>(backward, p, st);
    if (p.n_experts <= 512) return launch_route<T, 16>(backward, p, st);
    return launch_route<T, 32>(backward, p, st);
}

int launch_route(bool backward, const RouteArgs &p, cudaStream_t st) {
    if (p.dtype == FDA_DTYPE_F32) return launch_route<float>(backward, p, st);
    if (p.dtype == FDA_DTYPE_F16) return launch_route<__half>(backward, p, st);
    return launch_route<__nv_bfloat16>(backward, p, st);
}

int check_route(long long tokens, int n_experts, int top_k, int score, int n_groups, int top_groups, int group_score, int dtype) {
    if (!known_dtype(dtype)) return FDA_ERR_BAD_DTYPE;
    if (tokens < 0 || tokens > INT32_MAX || n_experts < 1 || top_k < 1 || n_groups < 1 || top_groups < 1 || top_groups > n_groups ||
        n_experts % n_groups != 0 || top_k > n_experts / n_groups * top_groups)
        return FDA_ERR_BAD_SHAPE;
    if (n_experts > kMostExperts || top_k > kMostChoices || n_groups > kMostExpertGroups) return FDA_ERR_TOO_LARGE_STATIC;
    if (score < FDA_SCORE_SOFTMAX || score > FDA_SCORE_SIGMOID || group_score < FDA_GROUP_MAX || group_score > FDA_GROUP_TOP2)
        return FDA_ERR_BAD_SCORE;
    return FDA_OK;
}

}  // namespace

extern "C" {

int fda_route_forward(const void *logits, const float *bias, float *weights, int64_t *experts, long long tokens, int n_experts, int top_k,
                      int score, int n_groups, int top_groups, int group_score, int renormalise, float scale, int dtype, void *stream) {
    if (const int rc = check_route(tokens, n_experts, top_k, score, n_groups, top_groups, group_score, dtype)) return rc;
    if (tokens == 0) return FDA_OK;
    if (!logits || !weights || !experts) return FDA_ERR_NULL_POINTER;
    RouteArgs p{};
    p.logits = logits; p.bias = bias; p.weights = weights; p.experts = experts; p.tokens = tokens; p.n_experts = n_experts; p.top_k = top_k;
    p.sigmoid = score == FDA_SCORE_SIGMOID; p.n_groups = n_groups; p.top_groups = top_groups; p.top2 = group_score == FDA_GROUP_TOP2;
    p.renormalise = renormalise; p.dtype = dtype; p.scale = scale;
    return launch_route(false, p, static_cast<cudaStream_t>(stream));
}

int fda_route_backward(const void *logits, const int64_t *experts, const float *grad_weights, void *grad_logits, long long tokens, int n_experts,
                       int top_k, int score, int renormalise, float scale, int dtype, void *stream) {
    if (const int rc = check_route(tokens, n_experts, top_k, score, 1, 1, FDA_GROUP_MAX, dtype)) return rc;
    if (tokens == 0) return FDA_OK;
    if (!logits || !experts || !grad_weights || !grad_logits) return FDA_ERR_NULL_POINTER;
    RouteArgs p{};
    p.logits = logits; p.experts = const_cast<int64_t *>(experts); p.grad_weights = grad_weights; p.grad_logits = grad_logits;
    p.tokens = tokens; p.n_experts = n_experts; p.top_k = top_k; p.sigmoid = score == FDA_SCORE_SIGMOID; p.renormalise = renormalise;
    p.dtype = dtype; p.scale = scale;
    return launch_route(true, p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

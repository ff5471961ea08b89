// Routing of tokens to experts, forward and backward.
//
//     score = softmax(logits) or sigmoid(logits),   select = score + bias                                     per token
//     the top_k largest of select, largest first, among the experts of the top_groups best groups (n_groups consecutive runs of
//     experts; a group is worth its largest select, or the sum of its two largest); ties go to the lower index
//     weight_j = scale * score_j / sum of the chosen scores, or scale * score_j
//
// What is chosen is what exact scores choose.  Where select is a monotone function of one logit (no bias, no sum over a group) the
// logits themselves are compared.  Elsewhere scores in fp32 are compared as long as their distance is beyond what they can be off by;
// a token for which it is not is decided by scores in 64 bits, so that no choice depends on how an exponential rounds.  A NaN
// counts as minus infinity in comparisons, and stays one in the weights.
//
// kLanes lanes take a token: 4 up to 64 experts, 8 up to 512, 16 beyond, so that a warp's instructions serve eight, four or two.  A lane
// holds octets of neighbouring experts, octet o of the token belonging to lane o mod kLanes.  Their values lie in shared memory, their
// largest in a register: a step of the choice takes the largest of these over the lanes, then eight lanes (four that look at two each) look at
// the octet that has it.  Bound by instructions, no pipe of which is full (comparisons and selections 50 %, shuffles and shared memory 56 %,
// issue slots 61 %); beyond 128 experts 64 registers (128 beyond 256) spill some 300 bytes a thread.  149504 tokens x 256 experts, 8 chosen, bf16:
// 60 us by logits, 83 by biased softmax scores, of which the bytes would take 14; 37376 x 64 in 8 groups 17 us.
//
// How many tokens are decided in 64 bits depends on the logits: an error is taken relative to the token's largest score, so that low scores of a
// peaked softmax, or scores of saturated sigmoids, count as equal.  149504 x 256 f32 with a bias of zeros, by the logits' standard deviation
// (1.5, 4, 6, 8): softmax 90, 109, 189, 296 us, sigmoid 89, 239, 609, 628 us; every token so 660 us.
#include "fda_rows.cuh"

#include <algorithm>

namespace {

using namespace fda_rows;

constexpr unsigned kAll = 0xffffffffu;
constexpr int kThreads = 128, kWarps = kThreads / 32;
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
__device__ __forceinline__ unsigned long long order_of(double v) {
    if (!(v == v)) v = -INFINITY;
    const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        const unsigned long long o = __shfl_xor_sync(kAll, v, d);
        v = o > v ? o : v;
    }
    return v;
}
template <int kLanes>
__device__ __forceinline__ float most(float v) {  // NaN only where every lane has one
#pragma unroll
    for (int d = kLanes / 2; d > 0; d /= 2) v = fmaxf(v, __shfl_xor_sync(kAll, v, d));
    return v;
}
template <int kLanes>
__device__ __forceinline__ int least(int v) {
#pragma unroll
    for (int d = kLanes / 2; d > 0; d /= 2) v = min(v, __shfl_xor_sync(kAll, v, d));
    return v;
}
template <int kLanes, typename F>
__device__ __forceinline__ F total(F v) {
#pragma unroll
    for (int d = kLanes / 2; d > 0; d /= 2) v += __shfl_xor_sync(kAll, v, d);
    return v;
}

// 2^v for comparisons: off by 2^-22 of itself, 0 below the normal range.
__device__ __forceinline__ float quick_exp2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// By how much a score in fp32 can be off.  A softmax's, relative to the token's largest: 2^-24 (1.5 |d| + 4) e^d, d = l - max, is at most
// 5 * 2^-24; the sum, by octets and then over up to 8 of them and 16 lanes, adds 20 * 2^-24, quotient and product 4.  A sigmoid's: (1.5 |l| + 4)
// s (1 - s) 2^-24 is at most 1.1 * 2^-24, sum and quotient add 3.
constexpr float kSoftmaxError = 1.f / 524288.f, kSigmoidError = 1.f / 2097152.f;
// For the addition of the bias, relative to the larger of two values that are compared: a smaller one that is below minus that is further
// away than it can be off by.
constexpr float kSumError = 1.f / 2097152.f;
constexpr float kSmallest = 1e-37f;  // scores below the normal range have an absolute error

template <typename T>
__device__ __forceinline__ float logit(const RouteArgs &p, long long token, int expert) {
    return to_f32(static_cast<const T *>(p.logits)[token * p.n_experts + expert]);
}

// ---- in 64 bits, a warp to a token ---------------------------------------------------------------------------------------------
// Bit i of a lane: its expert kPer * lane + i is in one of the top_groups best groups.  values: the token's in shared memory.
template <int kPer>
__device__ unsigned exactly_allowed(const RouteArgs &p, const double *values) {
    const int lane = threadIdx.x % 32, size = p.n_experts / p.n_groups;
    unsigned groups = kAll;
    if (p.top_groups < p.n_groups) {  // a lane takes a group
        double first = -INFINITY, second = -INFINITY;
        if (lane < p.n_groups)
            for (int i = 0; i < size; ++i) {
                double v = values[lane * size + i];
                if (!(v == v)) v = -INFINITY;
                if (v > first) { second = first; first = v; }
                else if (v > second) second = v;
            }
        double worth = p.top2 && size > 1 ? first + second : first;
        if (!(worth == worth)) worth = -INFINITY;
        int better = 0;
        for (int g = 0; g < p.n_groups; ++g) {
            const double other = __shfl_sync(kAll, worth, g);
            if (other > worth || (other == worth && g < lane)) ++better;
        }
        groups = __ballot_sync(kAll, lane < p.n_groups && better < p.top_groups);
    }
    unsigned allowed = 0;
    for (int i = 0; i < kPer; ++i) {
        const int e = lane * kPer + i;
        if (e < p.n_experts && (groups >> (e / size) & 1 || p.top_groups == p.n_groups)) allowed |= 1u << i;
    }
    return allowed;
}

// The choice by scores in 64 bits into chosen[top_k]; values: room for [n_experts] numbers.  One token of a call is enough to wait for it, so
// logits and bias are read once and each exponential is taken once.
template <typename T, int kPer>
__device__ __noinline__ void choose_exactly(const RouteArgs &p, long long token, double *values, int *chosen) {
    const int lane = threadIdx.x % 32;
    float l[kPer], bias[kPer], top = -INFINITY;
    double v[kPer], inverse = 1;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane * kPer + i;
        l[i] = e < p.n_experts ? logit<T>(p, token, e) : -INFINITY;
        bias[i] = e < p.n_experts && p.bias ? p.bias[e] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        top = fmaxf(top, l[i]);
        nan |= !(l[i] == l[i]);
    }
    if (p.sigmoid) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = 1 / (1 + exp(-(double)l[i]));
    } else {
        double shift = most<32>(top), sum = 0;
        if (__any_sync(kAll, nan)) shift = NAN;
        if (shift == -INFINITY) shift = 0;  // every score is 0
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            v[i] = exp((double)l[i] - shift);
            sum += v[i];
        }
        sum = total<32>(sum);
        inverse = sum == 0 ? 0 : 1 / sum;
    }
    unsigned long long key[kPer];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane * kPer + i;
        key[i] = 0;
        if (e >= p.n_experts) continue;
        if (!p.sigmoid) v[i] *= inverse;
        if (p.bias) v[i] += (double)bias[i];
        values[e] = v[i];
        key[i] = order_of(p.bias ? v[i] : (double)l[i]);  // without a bias experts are compared by their logits, only groups by sums of scores
    }
    __syncwarp();
    unsigned left = exactly_allowed<kPer>(p, values);
    for (int j = 0; j < p.top_k; ++j) {
        unsigned long long best = 0;
        int slot = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if ((left >> i & 1) && key[i] > best) { best = key[i]; slot = i; }
        const unsigned long long top = warp_max(best);
        const int winner = __ffs(__ballot_sync(kAll, best == top)) - 1;  // neighbouring experts are a lane's: the lowest lane's come first
        if (lane != winner) continue;
        left &= ~(1u << slot);
        chosen[j] = lane * kPer + slot;
    }
    __syncwarp();
}

// ---- in fp32, kLanes lanes to a token ------------------------------------------------------------------------------------------
// v[q][i] = the logit of expert (q kLanes + lane) 8 + i; minus infinity beyond the last one.
template <typename T, int kLanes, int kOctets, bool kVector>
__device__ __forceinline__ void load_logits(const RouteArgs &p, long long token, int lane, float (&v)[kOctets][8]) {
    const T *row = static_cast<const T *>(p.logits) + token * p.n_experts;
#pragma unroll
    for (int q = 0; q < kOctets; ++q) {
        const int first = (q * kLanes + lane) * 8;
        if (kVector && first < p.n_experts) {  // their number is a multiple of 8
            Raw<T, 8> raw;
            raw.load(row + first);
            raw.get(v[q]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[q][i] = !kVector && first + i < p.n_experts ? to_f32(row[first + i]) : -INFINITY;
        }
    }
}

// e^(l - shift) in place of the logits, `quick` for comparisons; shift is the largest logit.  The inverse of their sum; 0 for a token without
// a finite logit, which has no score.
template <int kLanes, int kOctets>
__device__ __forceinline__ void softmax_of(float (&v)[kOctets][8], bool quick, float &shift, float &inverse) {
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int q = 0; q < kOctets; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, v[q][i]);
    shift = most<kLanes>(top);
    if (shift == -INFINITY) shift = 0.f;  // every term is 0 then, or NaN
    const Pair minus(-shift), scale(1.44269504088896341f);
#pragma unroll
    for (int q = 0; q < kOctets; ++q) {
        if (quick) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const Pair d = (Pair(v[q][i], v[q][i + 1]) + minus) * scale;
                d.get(v[q][i], v[q][i + 1]);
                v[q][i] = quick_exp2(v[q][i]);
                v[q][i + 1] = quick_exp2(v[q][i + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[q][i] = expf(v[q][i] - shift);
        }
        Pair half[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) half[i] = Pair(v[q][2 * i], v[q][2 * i + 1]);
        sum += ((half[0] + half[1]) + (half[2] + half[3])).sum();
    }
    sum = total<kLanes>(sum);
    inverse = sum == 0.f ? 0.f : 1.f / sum;
}

// The largest of a token's chosen logits, 0 where there is none above minus infinity.
template <int kLanes, int kMine>
__device__ __forceinline__ float largest_chosen(const float (&l)[kMine], const bool (&there)[kMine]) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMine; ++i)
        if (there[i]) top = fmaxf(top, l[i]);
    top = most<kLanes>(top);
    return top == -INFINITY ? 0.f : top;
}

// Scores of the chosen experts with the logits l (kMine of them in a lane; those that are not there have there[i] false), before
// scaling, and what the weights are divided by.  Renormalised scores are ratios, which stay what they are where the scores themselves leave fp32's
// range: a softmax is taken over the chosen alone, and with m = min(0, largest chosen logit) a sigmoid's share of them is
//     e^(l - m) / (1 + e^(l - m) e^m)   for l < 0,     1 / (1 + e^-l)   else (m is 0 then)
// which is the score divided by e^m.
template <int kLanes, int kMine>
__device__ __forceinline__ float chosen_scores(const RouteArgs &p, const float (&l)[kMine], const bool (&there)[kMine], float shift, float inverse,
                                               float (&score)[kMine]) {
    float sum = 0.f;
    if (p.sigmoid) {
        const float m = p.renormalise ? fminf(largest_chosen<kLanes>(l, there), 0.f) : 0.f, scale = expf(m);
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            score[i] = 0.f;
            if (i * kLanes >= p.top_k) continue;
            if (there[i]) {
                const bool low = l[i] < 0.f;
                const float e = expf(low ? l[i] - m : -l[i]);
                score[i] = (low ? e : 1.f) / (1.f + (low ? e * scale : e));
            }
            sum += score[i];
        }
    } else {
        if (p.renormalise) {
            shift = largest_chosen<kLanes>(l, there);
            inverse = 1.f;
        }
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            score[i] = 0.f;
            if (i * kLanes >= p.top_k) continue;
            if (there[i] && inverse != 0.f) score[i] = expf(l[i] - shift) * inverse;
            sum += score[i];
        }
    }
    return p.renormalise ? total<kLanes>(sum) : 1.f;
}

// Of a warp, in shared memory.
template <int kLanes, int kOctets>
struct WarpShared {
    static constexpr int kTokens = 32 / kLanes, kExperts = kLanes * kOctets * 8;
    float values[kTokens][kExperts];
    union {
        struct {  // while groups are chosen
            float2 largest[kTokens][kExperts / 8];  // two of each octet
            float worth[kTokens][kMostExpertGroups];
        };
        struct {  // after it
            float chosen_value[kTokens][kMostChoices];
            int chosen[kTokens][kMostChoices];
        };
    };
};

__device__ __forceinline__ float2 two_largest(float2 a, float2 b) {  // of two pairs, each largest first
    return make_float2(fmaxf(a.x, b.x), fmaxf(fminf(a.x, b.x), fmaxf(a.y, b.y)));
}

// Takes the experts of other than the top_groups best groups out of v (NaN).  `worths` are the values that groups are compared by, v those of
// experts.  Returns false where the border between the groups is closer than `error`.
template <int kLanes, int kOctets>
__device__ __forceinline__ bool keep_best_groups(const RouteArgs &p, WarpShared<kLanes, kOctets> &s, int segment, int lane, float error,
                                                 const float (&worths)[kOctets][8], float (&v)[kOctets][8]) {
    const int size = p.n_experts / p.n_groups;
    const bool sums = p.top2 && size > 1, octets = size % 8 == 0;  // octets: groups are runs of whole octets
    float *worth = s.worth[segment];
    __syncwarp();
#pragma unroll
    for (int q = 0; q < kOctets; ++q) {
        if (octets) {
            float2 best[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                best[i] = make_float2(fmaxf(worths[q][2 * i], worths[q][2 * i + 1]), fminf(worths[q][2 * i], worths[q][2 * i + 1]));
            s.largest[segment][q * kLanes + lane] = two_largest(two_largest(best[0], best[1]), two_largest(best[2], best[3]));
        } else {
            float4 *at = reinterpret_cast<float4 *>(s.values[segment] + (q * kLanes + lane) * 8);
            at[0] = make_float4(worths[q][0], worths[q][1], worths[q][2], worths[q][3]);
            at[1] = make_float4(worths[q][4], worths[q][5], worths[q][6], worths[q][7]);
        }
    }
    __syncwarp();
    int share = kLanes;  // lanes to a group
    while (share > 1 && kLanes / share < p.n_groups) share /= 2;
    for (int base = 0; base < p.n_groups; base += kLanes / share) {
        const int g = base + lane / share;
        float2 best = make_float2(-INFINITY, -INFINITY);
        if (g < p.n_groups) {
            if (octets) {
                for (int i = lane % share; i < size / 8; i += share) best = two_largest(best, s.largest[segment][g * (size / 8) + i]);
            } else {
                for (int i = lane % share; i < size; i += share) best = two_largest(best, make_float2(s.values[segment][g * size + i], -INFINITY));
            }
        }
        for (int d = 1; d < share; d *= 2)
            best = two_largest(best, make_float2(__shfl_xor_sync(kAll, best.x, d), __shfl_xor_sync(kAll, best.y, d)));
        if (g < p.n_groups && lane % share == 0) worth[g] = fmaxf(sums ? best.x + best.y : best.x, -INFINITY);
    }
    __syncwarp();
    unsigned groups = 0;
    float low = INFINITY, high = -INFINITY;
    for (int g = lane; g < p.n_groups; g += kLanes) {
        const float mine = worth[g];
        int better = 0;
        for (int o = 0; o < p.n_groups; ++o) {
            const float other = worth[o];
            if (other > mine || (other == mine && o < g)) ++better;
        }
        if (better < p.top_groups) {
            groups |= 1u << g;
            low = fminf(low, mine);
        } else {
            high = fmaxf(high, mine);
        }
    }
#pragma unroll
    for (int d = kLanes / 2; d > 0; d /= 2) groups |= __shfl_xor_sync(kAll, groups, d);
    low = -most<kLanes>(-low);
    high = most<kLanes>(high);
    const unsigned inverse_size = ((1u << 20) + size - 1) / size;  // e / size for e < 1024
#pragma unroll
    for (int q = 0; q < kOctets; ++q) {
        const unsigned e = (q * kLanes + lane) * 8;
        if (octets) {
            const bool keep = groups >> (e * inverse_size >> 20 & 31) & 1;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[q][i] = keep ? v[q][i] : NAN;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(groups >> ((e + i) * inverse_size >> 20 & 31) & 1)) v[q][i] = NAN;
        }
    }
    return error < 0.f || low - high > error || low == -INFINITY;
}

// NaN for experts beyond the last, which are no candidates; with `sanitise` minus infinity for other NaN.
template <int kLanes, int kOctets>
__device__ __forceinline__ void only_candidates(int n_experts, int lane, bool sanitise, float (&v)[kOctets][8]) {
    if (sanitise) {
#pragma unroll
        for (int q = 0; q < kOctets; ++q)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[q][i] = fmaxf(v[q][i], -INFINITY);
    }
    if (n_experts < kLanes * kOctets * 8) {
#pragma unroll
        for (int q = 0; q < kOctets; ++q)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((q * kLanes + lane) * 8 + i >= n_experts) v[q][i] = NAN;
    }
}

// Whether a lane finds a NaN among its share of a token's logits.  Few tokens ask: not inlined, so that others keep their registers.
template <typename T>
__device__ __noinline__ bool has_nan(const RouteArgs &p, long long token, int lane, int lanes) {
    bool nan = false;
    for (int e = lane; e < p.n_experts; e += lanes) {
        const float x = logit<T>(p, token, e);
        nan |= x != x;
    }
    return nan;
}

template <typename T, int kLanes, int kOctets, bool kVector>
__global__ void __launch_bounds__(kThreads, kOctets <= 4 ? 8 : 4) route_forward_kernel(const RouteArgs p) {
    using Shared = WarpShared<kLanes, kOctets>;
    __shared__ alignas(16) Shared warps[kWarps];
    __shared__ alignas(16) float bias[Shared::kExperts];
    wait_for_previous_kernel();
    constexpr int kMine = kMostChoices / kLanes;
    const int lane = threadIdx.x % kLanes, segment = threadIdx.x % 32 / kLanes, E = p.n_experts;
    Shared &s = warps[threadIdx.x / 32];
    float *values = s.values[segment];
    if (p.bias) {
        for (int e = threadIdx.x; e < Shared::kExperts; e += kThreads) bias[e] = e < E ? fmaxf(p.bias[e], -INFINITY) : 0.f;
        __syncthreads();
    }
    const bool grouped = p.top_groups < p.n_groups, sums = grouped && p.top2 && E > p.n_groups;
    const bool by_score = p.bias || sums;  // what is compared: scores, or logits
    const bool need_softmax = !p.sigmoid && (by_score || !p.renormalise);
    const long long step = (long long)gridDim.x * kWarps * Shared::kTokens;
    for (long long base = ((long long)blockIdx.x * kWarps + threadIdx.x / 32) * Shared::kTokens; base < p.tokens; base += step) {
        const bool active = base + segment < p.tokens;
        const long long token = active ? base + segment : base;
        float v[kOctets][8], shift = 0.f, inverse = 1.f, largest = 1.f;
        load_logits<T, kLanes, kOctets, kVector>(p, token, lane, v);
        if (need_softmax) {
            softmax_of<kLanes, kOctets>(v, p.renormalise, shift, inverse);
            largest = inverse;
            if (by_score) {
#pragma unroll
                for (int q = 0; q < kOctets; ++q)
#pragma unroll
                    for (int i = 0; i < 8; i += 2) (Pair(v[q][i], v[q][i + 1]) * Pair(inverse)).get(v[q][i], v[q][i + 1]);
            } else {
                load_logits<T, kLanes, kOctets, kVector>(p, token, lane, v);
            }
        } else if (by_score) {
#pragma unroll
            for (int q = 0; q < kOctets; ++q)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[q][i] = __fdividef(1.f, 1.f + quick_exp2(v[q][i] * -1.44269504088896341f));
        }
        const float score_error = p.sigmoid ? kSigmoidError : largest * kSoftmaxError;
        if (p.bias) {
#pragma unroll
            for (int q = 0; q < kOctets; ++q) {
                const float4 *at = reinterpret_cast<const float4 *>(bias + (q * kLanes + lane) * 8);
                const float4 a = at[0], b = at[1];
                const Pair add[4] = {Pair(a.x, a.y), Pair(a.z, a.w), Pair(b.x, b.y), Pair(b.z, b.w)};
#pragma unroll
                for (int i = 0; i < 4; ++i) (Pair(v[q][2 * i], v[q][2 * i + 1]) + add[i]).get(v[q][2 * i], v[q][2 * i + 1]);
            }
        }
        // a NaN is never the largest; where nothing else is left the choice is made again below
        only_candidates<kLanes, kOctets>(E, lane, grouped, v);
        bool sure = true;
        __syncwarp();
        if (grouped) {
            float error = -1.f;
            if (by_score) {  // a group is worth up to two values, and two groups are compared
                float far = 0.f;
#pragma unroll
                for (int q = 0; q < kOctets; ++q)
#pragma unroll
                    for (int i = 0; i < 8; ++i) far = fabsf(v[q][i]) < INFINITY ? fmaxf(far, fabsf(v[q][i])) : far;
                error = 4.f * (score_error + kSmallest + kSumError * most<kLanes>(far));
            }
            if (by_score && !p.bias) {  // the groups by sums of scores, experts by their logits
                float l[kOctets][8];
                load_logits<T, kLanes, kOctets, kVector>(p, token, lane, l);
                only_candidates<kLanes, kOctets>(E, lane, true, l);
                sure = keep_best_groups<kLanes, kOctets>(p, s, segment, lane, error, v, l);
#pragma unroll
                for (int q = 0; q < kOctets; ++q)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[q][i] = l[q][i];
            } else {
                sure = keep_best_groups<kLanes, kOctets>(p, s, segment, lane, error, v, v);
            }
        }
        float head[kOctets];  // largest of each octet
#pragma unroll
        for (int q = 0; q < kOctets; ++q) {
            float4 *at = reinterpret_cast<float4 *>(values + (q * kLanes + lane) * 8);
            at[0] = make_float4(v[q][0], v[q][1], v[q][2], v[q][3]);
            at[1] = make_float4(v[q][4], v[q][5], v[q][6], v[q][7]);
            head[q] = NAN;
#pragma unroll
            for (int i = 0; i < 8; ++i) head[q] = fmaxf(head[q], v[q][i]);
        }
        __syncwarp();
        const auto largest_of_lane = [&]() {
            float top = head[0];
#pragma unroll
            for (int q = 1; q < kOctets; ++q) top = fmaxf(top, head[q]);
            return top;
        };
        // The first expert of the largest value leaves: every lane of the token gets its value (NaN where none is left) and its number (-1).
        // The octet that it is in is looked at by a lane an expert, always the same one, so that no lane reads here what another has written.
        const auto take = [&](float &top) {
            const float own = largest_of_lane();
            top = most<kLanes>(own);
            constexpr unsigned kSegment = (unsigned)((1ull << kLanes) - 1);
            const unsigned have = __ballot_sync(kAll, own == top) >> (segment * kLanes) & kSegment;
            int octet = INT32_MAX;
#pragma unroll
            for (int q = kOctets - 1; q >= 0; --q)
                if (head[q] == top) octet = q * kLanes + lane;
            if (__any_sync(kAll, have & (have - 1))) octet = least<kLanes>(octet);  // several lanes have it
            else octet = __shfl_sync(kAll, octet, __ffs(have) - 1, kLanes);
            const bool any = have != 0;
            // a lane looks at one or two of its experts
            constexpr int kLooks = kLanes >= 8 ? 1 : 8 / kLanes;
            float x[kLooks], rest = NAN;
            int slot = -1;
#pragma unroll
            for (int i = 0; i < kLooks; ++i) {
                x[i] = any && (kLanes <= 8 || lane < 8) ? values[octet * 8 + i * kLanes + lane] : NAN;
                const unsigned equal = __ballot_sync(kAll, x[i] == top) >> (segment * kLanes) & kSegment;
                if (slot < 0 && equal) slot = i * kLanes + __ffs(equal) - 1;
            }
#pragma unroll
            for (int i = 0; i < kLooks; ++i) rest = fmaxf(rest, slot == i * kLanes + lane ? NAN : x[i]);
            rest = most<kLanes>(rest);
            if (!any) return -1;
            if (slot % kLanes == lane) values[octet * 8 + slot] = NAN;
#pragma unroll
            for (int q = 0; q < kOctets; ++q)
                if (octet == q * kLanes + lane) head[q] = rest;
            return octet * 8 + slot;
        };
        for (int j = 0; j < p.top_k; ++j) {
            float top;
            const int e = take(top);
            if (e < 0) sure = false;
            if (lane == 0) {
                s.chosen[segment][j] = e;
                s.chosen_value[segment][j] = top;
            }
        }
        __syncwarp();
        // A NaN counts as minus infinity, of which the lower index is chosen; without groups it is no candidate here, and one before the last
        // chosen minus infinity is a choice.
        if (!grouped && s.chosen_value[segment][p.top_k - 1] == -INFINITY && has_nan<T>(p, token, lane, kLanes)) sure = false;
        if (p.bias) {
            // the chosen among themselves, and the last of them against what is left
            const float margin = 2.f * score_error + kSmallest, last = s.chosen_value[segment][p.top_k - 1];
            const auto same = [&](int a, int b) {
                return min(a, b) >= 0 && logit<T>(p, token, a) == logit<T>(p, token, b) && bias[a] == bias[b];
            };
            for (int j = lane; j + 1 < p.top_k; j += kLanes) {
                const float a = s.chosen_value[segment][j], b = s.chosen_value[segment][j + 1];
                if (!(a - b > margin + fabsf(a) * kSumError) && !same(s.chosen[segment][j], s.chosen[segment][j + 1])) sure = false;
            }
            // of equal experts the lower ones are chosen: all that is left within the margin has to be equal to the last
            const int last_chosen = s.chosen[segment][p.top_k - 1];
            const float next = most<kLanes>(largest_of_lane()), reach = margin + fabsf(last) * kSumError;
            const bool open = next == next && !(last - next > reach);
            if (__any_sync(kAll, open)) {
                for (int e = lane; e < E; e += kLanes) {  // what is taken or no candidate is NaN
                    const float x = values[e];
                    if (open && x == x && !(last - x > reach) && !same(last_chosen, e)) sure = false;
                }
            }
        }
        const unsigned unsure = __ballot_sync(kAll, active && !sure);
        if (unsure) {
            for (int t = 0; t < Shared::kTokens; ++t)
                if (unsure >> (t * kLanes) & ((1ull << kLanes) - 1))
                    choose_exactly<T, Shared::kExperts / 32>(p, base + t, reinterpret_cast<double *>(s.values), s.chosen[t]);
            __syncwarp();
        }
        int mine[kMine];
        float l[kMine], score[kMine];
        bool there[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            there[i] = lane + i * kLanes < p.top_k;
            mine[i] = 0;
            l[i] = 0.f;
            if (there[i]) {
                mine[i] = s.chosen[segment][lane + i * kLanes];
                l[i] = logit<T>(p, token, mine[i]);
            }
        }
        const float sum = chosen_scores<kLanes, kMine>(p, l, there, shift, inverse, score);
        if (!active) continue;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            if (!there[i]) continue;
            const long long at = token * p.top_k + lane + i * kLanes;
            p.weights[at] = sum == 0.f ? 0.f : p.scale * score[i] / sum;
            p.experts[at] = mine[i];
        }
    }
}

// A warp sets n <= kMost elements to 0, in vectors but for the ends.
template <int kMost, typename T>
__device__ __forceinline__ void clear_run(T *begin, int n, int lane) {
    constexpr int W = 16 / (int)sizeof(T);
    const int head = min((int)(-(reinterpret_cast<uintptr_t>(begin) / sizeof(T)) % W), n), vectors = (n - head) / W, tail = head + vectors * W;
    if (lane < head) begin[lane] = from_f32<T>(0.f);
#pragma unroll
    for (int i = 0; i < kMost / W; i += 32)
        if (i + lane < vectors) reinterpret_cast<uint4 *>(begin + head)[i + lane] = make_uint4(0, 0, 0, 0);
    if (tail + lane < n) begin[tail + lane] = from_f32<T>(0.f);
}

// grad_logits from grad_weights: with s the scores of the chosen and S their sum,
//     softmax, renormalised    dl_j = w_j (dw_j - sum of dw w / scale)           (a softmax over the chosen alone)
//     softmax                  dl_i = scale p_i ([i chosen] dw_i - sum of dw p)
//     sigmoid                  dl_j = ds_j s_j (1 - s_j),  ds_j = scale (dw_j - sum of dw s / S) / S  or  scale dw_j
// An expert outside 0 .. n_experts - 1 gets none.  A token's row is one team's, so there are no atomics.  149504 x 256 bf16: 27 us (3.4 TB/s)
// renormalised, 39 (4.3 TB/s) for the dense softmax; bound by the chain from a choice to its logit.  A lane has kMine choices, no more than top_k
// needs (149504 x 64 f32, 2 chosen: 11 us, with room for 32 18).  The rows of a warp's tokens lie one behind the other and are zeroed as one run
// (100000 x 131 bf16 10.5 us, row by row 45; 20000 x 1000 f32 16 and 21; 149504 x 256 bf16 26.7 and 26.0).
template <typename T, int kLanes, int kOctets, bool kVector, bool kDense, int kMine>
__global__ void __launch_bounds__(kThreads) route_backward_kernel(const RouteArgs p) {
    constexpr int kTokens = 32 / kLanes, kExperts = kLanes * kOctets * 8;
    __shared__ alignas(16) float rows[kDense ? kWarps : 1][kTokens][kDense ? kExperts : 1];
    wait_for_previous_kernel();
    const int lane = threadIdx.x % kLanes, segment = threadIdx.x % 32 / kLanes, E = p.n_experts;
    float *row = rows[kDense ? threadIdx.x / 32 : 0][segment];
    const long long step = (long long)gridDim.x * kWarps * kTokens;
    // Choices and their weights' gradients of the next token are on their way while one is worked on; eight of them in a lane have no registers
    // for that (149504 x 64: 18 us with, 14 without; four, 149504 x 256 29.5 with, 32.4 without).
    constexpr bool kAhead = kMine <= 4;
    long long next_chosen[kMine];
    float next_dw[kMine];
    const auto read_choices = [&](long long t) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int j = lane + i * kLanes;
            next_chosen[i] = -1;
            next_dw[i] = 0.f;
            if (t < p.tokens && j < p.top_k) {
                next_chosen[i] = p.experts[t * p.top_k + j];
                next_dw[i] = p.grad_weights[t * p.top_k + j];
            }
        }
    };
    const long long start = ((long long)blockIdx.x * kWarps + threadIdx.x / 32) * kTokens;
    if (kAhead) read_choices(start + segment);
    for (long long base = start; base < p.tokens; base += step) {
        const bool active = base + segment < p.tokens;
        const long long token = active ? base + segment : base;
        if (!kAhead) read_choices(base + segment);
        int chosen[kMine];
        float dw[kMine], l[kMine], score[kMine];
        bool there[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            there[i] = (unsigned long long)next_chosen[i] < (unsigned long long)E;
            chosen[i] = there[i] ? (int)next_chosen[i] : 0;
            dw[i] = there[i] ? next_dw[i] * p.scale : 0.f;
        }
        if (kAhead) read_choices(base + step + segment);
        float v[kOctets][8], shift = 0.f, inverse = 1.f;
        if (kDense) {  // softmax without renormalising: every expert's logit has a gradient
            load_logits<T, kLanes, kOctets, kVector>(p, token, lane, v);
            softmax_of<kLanes, kOctets>(v, false, shift, inverse);
        }
#pragma unroll
        for (int i = 0; i < kMine; ++i) l[i] = there[i] ? logit<T>(p, token, chosen[i]) : 0.f;
        const float sum = chosen_scores<kLanes, kMine>(p, l, there, shift, inverse, score);
        const float over = sum == 0.f ? 0.f : 1.f / sum;
        float along = 0.f;
#pragma unroll
        for (int i = 0; i < kMine; ++i) along += dw[i] * score[i] * over;
        along = total<kLanes>(along);
        T *out = static_cast<T *>(p.grad_logits) + token * E;
        float dl[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            dl[i] = score[i] * over * (p.renormalise ? dw[i] - along : dw[i]);
            if (p.sigmoid && there[i]) dl[i] *= 1.f / (1.f + expf(l[i]));  // 1 - s, without its cancellation near 1
        }
        if constexpr (!kDense) {  // zeros, and the chosen behind them
            clear_run<kTokens * kExperts>(static_cast<T *>(p.grad_logits) + base * E, (int)min((long long)kTokens, p.tokens - base) * E, threadIdx.x % 32);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kMine; ++i)
                if (active && there[i]) out[chosen[i]] = from_f32<T>(dl[i]);
        } else {
            __syncwarp();
#pragma unroll
            for (int q = 0; q < kOctets; ++q) {
                float4 *at = reinterpret_cast<float4 *>(row + (q * kLanes + lane) * 8);
                at[0] = at[1] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kMine; ++i)
                if (there[i]) row[chosen[i]] = dl[i];
            __syncwarp();
            if (!active) continue;
            const float each = inverse * along;
#pragma unroll
            for (int q = 0; q < kOctets; ++q) {
                const int first = (q * kLanes + lane) * 8;
                if (first >= E) continue;
                const float4 *at = reinterpret_cast<const float4 *>(row + first);
                const float4 a = at[0], b = at[1];
                float d[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] -= v[q][i] * each;
                if (kVector) {
                    Raw<T, 8> raw;
                    raw.set(d);
                    raw.store(out + first);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (first + i < E) out[first + i] = from_f32<T>(d[i]);
                }
            }
        }
    }
}

template <typename T, int kLanes, int kOctets, int kMine>
auto route_backward_kernel_of(bool vector, bool dense) {
    if (!dense) return route_backward_kernel<T, kLanes, kOctets, false, false, kMine>;  // without vectors of a token's row
    return vector ? route_backward_kernel<T, kLanes, kOctets, true, true, kMine> : route_backward_kernel<T, kLanes, kOctets, false, true, kMine>;
}

template <typename T, int kLanes, int kOctets>
int launch_route(bool backward, const RouteArgs &p, cudaStream_t st) {
    const unsigned blocks = (unsigned)std::min<long long>(ceil_div(p.tokens, kWarps * 32 / kLanes), 16 * kSms);
    // rows of octets that start on 16-byte boundaries
    const bool vector = p.n_experts % 8 == 0 && !misaligned16(p.logits) && !misaligned16(p.grad_logits);
    const bool dense = !p.sigmoid && !p.renormalise;
    auto kernel = vector ? route_forward_kernel<T, kLanes, kOctets, true> : route_forward_kernel<T, kLanes, kOctets, false>;
    if (backward) {
        kernel = p.top_k <= kLanes       ? route_backward_kernel_of<T, kLanes, kOctets, 1>(vector, dense)
                 : p.top_k <= 2 * kLanes ? route_backward_kernel_of<T, kLanes, kOctets, 2>(vector, dense)
                                         : route_backward_kernel_of<T, kLanes, kOctets, kMostChoices / kLanes>(vector, dense);
    }
    return launched(launch_early(kernel, blocks, kThreads, 0, st, 1, p));
}

template <typename T>
int launch_route(bool backward, const RouteArgs &p, cudaStream_t st) {
    // four lanes up to 64 experts (149504 x 64 f32 forward: 20 us, eight lanes 25), not beyond (x 256 bf16: 95 us, eight lanes 88)
    if (p.n_experts <= 32) return launch_route<T, 4, 1>(backward, p, st);
    if (p.n_experts <= 64) return launch_route<T, 4, 2>(backward, p, st);
    if (p.n_experts <= 128) return launch_route<T, 8, 2>(backward, p, st);
    if (p.n_experts <= 256) return launch_route<T, 8, 4>(backward, p, st);
    if (p.n_experts <= 512) return launch_route<T, 8, 8>(backward, p, st);
    return launch_route<T, 16, 8>(backward, p, st);
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

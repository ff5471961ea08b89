// Row access shared by the kernels around the linear operators (layer norm, routing to experts, rows sorted by expert): 16-byte
// vectors in the tensors' type, values in fp32, sums over the lanes that share a row.
#pragma once

#include "fda_linear.cuh"

namespace fda {
void record_cuda_error(int e);  // fda_api.cu
}

namespace fda_rows {

using fda_linear::ceil_div;
using fda_linear::from_f32;
using fda_linear::kSms;
using fda_linear::launch_early;
using fda_linear::to_f32;
using fda_linear::wait_for_previous_kernel;

inline int launched(cudaError_t e) {
    if (e == cudaSuccess) return FDA_OK;
    fda::record_cuda_error((int)e);
    return FDA_ERR_CUDA;
}

inline size_t type_size(int dtype) { return dtype == FDA_DTYPE_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype >= FDA_DTYPE_F32 && dtype <= FDA_DTYPE_BF16; }
inline bool misaligned16(const void *p) { return (uintptr_t)p % 16 != 0; }

// Two 16-bit numbers of a word, the lower one first.
template <typename T> __device__ __forceinline__ void unpack(unsigned u, float &a, float &b);
template <> __device__ __forceinline__ void unpack<__nv_bfloat16>(unsigned u, float &a, float &b) {
    a = __uint_as_float(u << 16);
    b = __uint_as_float(u & 0xffff0000u);
}
template <> __device__ __forceinline__ void unpack<__half>(unsigned u, float &a, float &b) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u));
    a = f.x;
    b = f.y;
}
template <typename T> __device__ __forceinline__ unsigned pack(float a, float b);
template <> __device__ __forceinline__ unsigned pack<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&v);
}
template <> __device__ __forceinline__ unsigned pack<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&v);
}

// Two fp32 numbers that one instruction works on.
struct Pair {
    unsigned long long bits;
    __device__ __forceinline__ Pair() {}
    __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(a), "f"(b)); }
    __device__ __forceinline__ explicit Pair(float a) : Pair(a, a) {}
    __device__ __forceinline__ void get(float &a, float &b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(bits)); }
    __device__ __forceinline__ float sum() const {
        float a, b;
        get(a, b);
        return a + b;
    }
};
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
    return r;
}

// kWidth neighbouring elements as they lie in memory: 16 or 32 bytes.
template <typename T, int kWidth>
struct Raw {
    static constexpr int kUnits = kWidth * (int)sizeof(T) / 16;
    uint4 u[kUnits];

    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) u[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) reinterpret_cast<uint4 *>(p)[i] = u[i];
    }
    // Element j, known when this is compiled.
    __device__ __forceinline__ T element(int j) const {
        const uint4 &a = u[j * (int)sizeof(T) / 16];
        const int k = j * (int)sizeof(T) / 4 % 4;
        const unsigned w = k == 0 ? a.x : k == 1 ? a.y : k == 2 ? a.z : a.w;
        if constexpr (sizeof(T) == 4) return __uint_as_float(w);
        else {
            const unsigned short h = (unsigned short)(j % 2 ? w >> 16 : w);
            return *reinterpret_cast<const T *>(&h);
        }
    }
    __device__ __forceinline__ void get(float *v) const {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const unsigned w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 4) v[4 * i + j] = __uint_as_float(w[j]);
                else unpack<T>(w[j], v[8 * i + 2 * j], v[8 * i + 2 * j + 1]);
            }
        }
    }
    __device__ __forceinline__ void get(Pair *v) const {
        float f[kWidth];
        get(f);
#pragma unroll
        for (int j = 0; j < kWidth / 2; ++j) v[j] = Pair(f[2 * j], f[2 * j + 1]);
    }
    __device__ __forceinline__ void set(const Pair *v) {
        float f[kWidth];
#pragma unroll
        for (int j = 0; j < kWidth / 2; ++j) v[j].get(f[2 * j], f[2 * j + 1]);
        set(f);
    }
    __device__ __forceinline__ void set(const float *v) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            unsigned w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v[4 * i + j]);
                else w[j] = pack<T>(v[8 * i + 2 * j], v[8 * i + 2 * j + 1]);
            }
            u[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
};

// A parameter of either type, as fp32.
__device__ __forceinline__ float load_as_f32(const void *p, int dtype, size_t i) {
    if (dtype == FDA_DTYPE_F32) return static_cast<const float *>(p)[i];
    if (dtype == FDA_DTYPE_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_from_f32(void *p, int dtype, size_t i, float v) {
    if (dtype == FDA_DTYPE_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == FDA_DTYPE_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

template <int kLanes>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int d = kLanes / 2; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// Three sums over a warp: halves and quarters of it take different ones, which needs 9 exchanges instead of 15.
__device__ __forceinline__ void warp_sum3(float (&v)[3]) {
    const bool upper = threadIdx.x & 16, odd = threadIdx.x & 8;
    float a = (upper ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[1], 16);
    const float b = v[2] + __shfl_xor_sync(0xffffffffu, v[2], 16);
    a = (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
    for (int d = 4; d > 0; d /= 2) a += __shfl_xor_sync(0xffffffffu, a, d);
    v[0] = __shfl_sync(0xffffffffu, a, 0);
    v[1] = __shfl_sync(0xffffffffu, a, 16);
    v[2] = __shfl_sync(0xffffffffu, a, 8);
}
template <int kLanes, int kCount>
__device__ __forceinline__ void lanes_sums(float (&v)[kCount]) {
    if constexpr (kLanes == 32 && kCount == 3) {
        warp_sum3(v);
    } else {
#pragma unroll
        for (int k = 0; k < kCount; ++k) v[k] = lanes_sum<kLanes>(v[k]);
    }
}

// The threads that share a row: kLanes lanes of a warp, or (0) the block.  sum() leaves the same numbers in all of them.
template <int kLanes>
struct Team {
    __device__ __forceinline__ int lane() const { return threadIdx.x % kLanes; }
    __device__ __forceinline__ int size() const { return kLanes; }
    template <int kCount>
    __device__ __forceinline__ void sum(float (&v)[kCount]) {
        lanes_sums<kLanes>(v);
    }
};
template <>
struct Team<0> {
    static constexpr int kMost = 3, kWarps = 32;
    float (*shared)[kMost][kWarps];  // [2], 0 for warps that are not there; a buffer is written again only after everyone has passed the barrier
                                     // behind the other
    int buffer = 0;
    __device__ __forceinline__ int lane() const { return threadIdx.x; }
    __device__ __forceinline__ int size() const { return blockDim.x; }
    template <int kCount>
    __device__ __forceinline__ void sum(float (&v)[kCount]) {
        static_assert(kCount <= kMost, "");
        lanes_sums<32>(v);
        if (threadIdx.x % 32 == 0) {
#pragma unroll
            for (int k = 0; k < kCount; ++k) shared[buffer][k][threadIdx.x / 32] = v[k];
        }
        __syncthreads();
        if (blockDim.x <= 128) {
#pragma unroll
            for (int k = 0; k < kCount; ++k) {
                const float4 s = *reinterpret_cast<const float4 *>(shared[buffer][k]);
                v[k] = (s.x + s.y) + (s.z + s.w);
            }
        } else {
#pragma unroll
            for (int k = 0; k < kCount; ++k) v[k] = shared[buffer][k][threadIdx.x % 32];
            lanes_sums<32>(v);
        }
        buffer ^= 1;
    }
};

}  // namespace fda_rows

// Building blocks of the tensor-core linear kernels: barriers with bounded waits, tiled copies, tcgen05 and its descriptors.
#pragma once

#include <cuda.h>

#include "fda_linear.cuh"

namespace fda_linear {

// Waits that ran out since the library was loaded, on this device (fda_linear_timeouts).
static __device__ unsigned int g_timeouts;

__device__ __forceinline__ uint32_t smem_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ unsigned long long time_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

struct Barrier {
    unsigned long long word;
    __device__ __forceinline__ void init(int count) {
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_address(this)), "r"(count) : "memory");
    }
    __device__ __forceinline__ void arrive() {
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_address(this)) : "memory");
    }
    __device__ __forceinline__ void arrive_expect(unsigned bytes) {
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_address(this)), "r"(bytes) : "memory");
    }
    __device__ __forceinline__ bool passed(unsigned parity) {
        unsigned ok;
        asm volatile(
            "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
            : "=r"(ok)
            : "r"(smem_address(this)), "r"(parity)
            : "memory");
        return ok;
    }
    // False when the phase did not end within two seconds or another wait of the block ran out before: the caller leaves.
    __device__ __noinline__ bool wait_slowly(unsigned parity, volatile int *failed) {
        const unsigned long long begin = time_ns();
        for (;;) {
            for (int i = 0; i < 64; ++i)
                if (passed(parity)) return true;
            if (*failed) return false;
            if (time_ns() - begin > 2000000000ull) {
                *failed = 1;
                return false;
            }
        }
    }
    __device__ __forceinline__ bool wait(unsigned parity, volatile int *failed) {
        return passed(parity) || passed(parity) || wait_slowly(parity, failed);
    }
};

// A place in a ring of kStages, with the parity of its current round.
template <int kStages>
struct Ring {
    int stage = 0;
    unsigned round = 0;
    __device__ __forceinline__ void next() {
        if (++stage == kStages) { stage = 0; round ^= 1; }
    }
};

__device__ __forceinline__ void tma_2d(const CUtensorMap *map, void *dst, Barrier *bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
                     smem_address(dst)),
                 "l"(map), "r"(smem_address(bar)), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void tma_3d(const CUtensorMap *map, void *dst, Barrier *bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                     smem_address(dst)),
                 "l"(map), "r"(smem_address(bar)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// ---- tcgen05 ----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, int columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(slot)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t address, int columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
}
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool accumulate) {
    asm volatile(
        "{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b),
        "r"(instruction), "r"((unsigned)accumulate)
        : "memory");
}
// Arrives on the barrier when every tcgen05 operation issued so far by this thread has ended.
__device__ __forceinline__ void mma_commit(Barrier *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_address(bar)) : "memory");
}
// 32 lanes x 32 columns of fp32: register j of a lane is column j of its row.
__device__ __forceinline__ void tmem_load(uint32_t address, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
        "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
          "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(address));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory operand descriptors, 128-byte swizzle (layout code 2, descriptor version 1).  A swizzle atom is 8 lines of 128
// bytes.  Contraction along a line ("K-major"): `stride` bytes between atoms of 8 rows; a step of 16 elements is 32 bytes further.
// Rows along a line ("MN-major"): an atom is 64 rows x 8 contraction indices, `stride` bytes between atoms along the
// contraction, `leading` bytes between blocks of 64 rows; a step of 16 is two atoms further.
__device__ __forceinline__ uint64_t operand(const void *p, uint32_t leading, uint32_t stride) {
    return (uint64_t)((smem_address(p) & 0x3ffff) >> 4) | ((uint64_t)((leading & 0x3ffff) >> 4) << 16) |
           ((uint64_t)((stride & 0x3ffff) >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
constexpr uint32_t kAtom = 1024;       // bytes of a swizzle atom
constexpr uint32_t kLineElements = 64; // 16-bit elements of a line

// Instruction descriptor of kind::f16 with fp32 accumulators.
template <typename T> struct MmaType;
template <> struct MmaType<__half> { static constexpr uint32_t kCode = 0; };
template <> struct MmaType<__nv_bfloat16> { static constexpr uint32_t kCode = 1; };
template <typename T>
__host__ __device__ constexpr uint32_t instruction(int m, int n, bool a_mn_major, bool b_mn_major) {
    return (1u << 4) | (MmaType<T>::kCode << 7) | (MmaType<T>::kCode << 10) | ((uint32_t)a_mn_major << 15) | ((uint32_t)b_mn_major << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// ---- 16-bit rows in registers -------------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

__device__ __forceinline__ void load_32_bytes(const void *p, uint32_t *v) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "l"(p));
}
__device__ __forceinline__ void store_32_bytes(void *p, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// 32 elements of a 16-bit row, of which `count` exist; `vector` is what the row's address is a multiple of (32, 16 or less, in bytes).
template <typename T>
__device__ __forceinline__ void load_row(const T *p, int count, int vector, uint32_t (&v)[16]) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = 0;
    if (vector == 32 && count == 32) {
        load_32_bytes(p, v);
        load_32_bytes(p + 16, v + 8);
    } else if (vector >= 16) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (8 * j < count) {
                const uint4 q = *reinterpret_cast<const uint4 *>(p + 8 * j);
                v[4 * j] = q.x; v[4 * j + 1] = q.y; v[4 * j + 2] = q.z; v[4 * j + 3] = q.w;
            }
    } else {
        const unsigned short *s = reinterpret_cast<const unsigned short *>(p);
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j < count) v[j / 2] |= (uint32_t)s[j] << (16 * (j & 1));
    }
}
template <typename T>
__device__ __forceinline__ void store_row(T *p, int count, int vector, const uint32_t (&v)[16]) {
    if (vector == 32 && count == 32) {
        store_32_bytes(p, v);
        store_32_bytes(p + 16, v + 8);
    } else if (vector >= 16) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (8 * j < count) *reinterpret_cast<uint4 *>(p + 8 * j) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    } else {
        unsigned short *s = reinterpret_cast<unsigned short *>(p);
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j < count) s[j] = (unsigned short)(v[j / 2] >> (16 * (j & 1)));
    }
}

}  // namespace fda_linear

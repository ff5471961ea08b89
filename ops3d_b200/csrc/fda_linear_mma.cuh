// Building blocks of the tensor-core linear kernels: barriers with bounded waits, tiled copies, tcgen05 and its descriptors.
#pragma once

#include <cuda.h>

#include "fda_linear.cuh"

namespace fda_linear {

// Waits that ran out since the library was loaded, on this device (fda_linear_timeouts).
static __device__ unsigned int g_timeouts;

__device__ __forceinline__ uint32_t smem_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// Limit of a wait: about two seconds of the SM's clock.  A stretch between two looks at the clock counts a sixteenth of it at most: what lies
// beyond is time in which the block was not running (another process had the SM), and no sign of a fault.
constexpr long long kWaitCycles = 4000000000ll, kMostBetweenLooks = kWaitCycles / 16;

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
        long long waited = 0, last = clock64();
        for (;;) {
            for (int i = 0; i < 64; ++i)
                if (passed(parity)) return true;
            if (*failed) return false;
            const long long now = clock64();
            waited += min(now - last, kMostBetweenLooks);
            last = now;
            if (waited > kWaitCycles) {
                *failed = 1;
                return false;
            }
        }
    }
    __device__ __forceinline__ bool wait(unsigned parity, volatile int *failed) {
        return passed(parity) || passed(parity) || passed(parity) || passed(parity) || wait_slowly(parity, failed);
    }
};

// The address in another block of the cluster that corresponds to one of this block's.
__device__ __forceinline__ uint32_t cluster_address(const void *p, unsigned rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_address(p)), "r"(rank));
    return r;
}
// Relaxed: what it announces are reads of tensor memory, which tcgen05.wait::ld has ended and tcgen05.fence orders.  A release across the
// cluster would wait for the caller's global stores besides (per tile of 256 x 256: 9 us instead of 6).
__device__ __forceinline__ void arrive_at(uint32_t cluster_barrier) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_barrier) : "memory");
}
__device__ __forceinline__ void release_at(uint32_t cluster_barrier) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_barrier) : "memory");
}
// Behind a wait for release_at: a barrier's own wait acquires what this block's threads have released, not what the other's have.
__device__ __forceinline__ void acquire_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }
__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Between this thread's accesses to shared memory and those of copies and products to the same places, either way round.
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A place in a ring, with the parity of its current round.
struct Ring {
    int stages, stage = 0;
    unsigned round = 0;
    __device__ __forceinline__ explicit Ring(int stages) : stages(stages) {}
    __device__ __forceinline__ void next() {
        if (++stage == stages) { stage = 0; round ^= 1; }
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
// The same for a pair of blocks: the copy goes to this block's memory and signals a barrier of either.
__device__ __forceinline__ void tma_2d_pair(const CUtensorMap *map, void *dst, uint32_t bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
                     smem_address(dst)),
                 "l"(map), "r"(bar), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void tma_3d_pair(const CUtensorMap *map, void *dst, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            smem_address(dst)),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
// A box of a matrix into L2.
__device__ __forceinline__ void prefetch_2d(const CUtensorMap *map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
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
// One lane of a converged warp.  The issuing loops keep the whole warp together around it: their operands then stay in uniform
// registers, where a loop of one lane moves each of them there for every product.
__device__ __forceinline__ bool elected() {
    unsigned is;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(is));
    return is;
}
// A descriptor's upper half is the same for all slices of an operand, its lower half holds the address.
template <bool kPair>
__device__ __forceinline__ void mma_f16(uint32_t d, uint32_t a, uint32_t a_high, uint32_t b, uint32_t b_high, uint32_t instruction, bool accumulate) {
    if (kPair)
        asm volatile(
            "{ .reg .pred p; .reg .b64 a, b; mov.b64 a, {%1, %2}; mov.b64 b, {%3, %4}; setp.ne.u32 p, %6, 0; "
            "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %5, p; }" ::"r"(d), "r"(a), "r"(a_high), "r"(b), "r"(b_high), "r"(instruction),
            "r"((unsigned)accumulate)
            : "memory");
    else
        asm volatile(
            "{ .reg .pred p; .reg .b64 a, b; mov.b64 a, {%1, %2}; mov.b64 b, {%3, %4}; setp.ne.u32 p, %6, 0; "
            "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p; }" ::"r"(d), "r"(a), "r"(a_high), "r"(b), "r"(b_high), "r"(instruction),
            "r"((unsigned)accumulate)
            : "memory");
}
// Arrives on the barrier when every tcgen05 operation issued so far by this thread has ended.
__device__ __forceinline__ void mma_commit(Barrier *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_address(bar)) : "memory");
}
// The same for a pair of blocks (cta_group::2): both allocate and free, the first issues the products, a commit arrives in both.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t *slot, int columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(slot)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t address, int columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
}
template <bool kPair>
__device__ __forceinline__ void commit(Barrier *bar);
__device__ __forceinline__ void mma_commit_pair(Barrier *bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     smem_address(bar)),
                 "h"((unsigned short)3)
                 : "memory");
}
template <> __device__ __forceinline__ void commit<false>(Barrier *bar) { mma_commit(bar); }
template <> __device__ __forceinline__ void commit<true>(Barrier *bar) { mma_commit_pair(bar); }
// 32 lanes x 16 or 32 columns of fp32: register j of a lane is column j of its row.
__device__ __forceinline__ void tmem_load(uint32_t address, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(address));
}
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
__device__ __forceinline__ uint32_t operand_low(const void *p, uint32_t leading) {
    return ((smem_address(p) & 0x3ffff) >> 4) | ((leading & 0x3ffff) >> 4) << 16;
}
__host__ __device__ constexpr uint32_t operand_high(uint32_t stride) { return ((stride & 0x3ffff) >> 4) | 1u << 14 | 2u << 29; }
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

// ---- activations beside 16-bit outputs --------------------------------------------------------------------------------------------
// A tile of 128 x 256 has 256 elements a lane of an SM, and its bytes pass in about 5500 cycles: more than some 20 instructions
// an element and the epilogue, not memory, sets the pace (erff, expf and a division took 5.7 us a tile forward and 9.4 backward).
// So: one exp2 and one reciprocal of the special-function unit each, the rest on pairs of elements where the instruction set has
// the pair's form.  Errors stay below 1e-6 of 1 + |v|: an absolute bound, as 1 + erf(v) in fp32 has one.  In gelu's negative tail, where the
// value itself is small, that can be more than a rounding of it (0.16 % of the value at -5, 0.36 % at -6, 3 % of the 5e-15 at -8; bf16's
// half step is up to 0.39 %).
struct Pair {
    unsigned long long bits;
    __device__ __forceinline__ Pair() {}
    __device__ __forceinline__ Pair(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(lo), "f"(hi)); }
    __device__ __forceinline__ explicit Pair(float both) : Pair(both, both) {}
    __device__ __forceinline__ void split(float &lo, float &hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(bits)); }
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
__device__ __forceinline__ Pair exp2_2(Pair v) {
    float lo, hi;
    v.split(lo, hi);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(lo));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(hi));
    return Pair(lo, hi);
}
__device__ __forceinline__ Pair reciprocal_2(Pair v) {
    float lo, hi;
    v.split(lo, hi);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(lo));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(hi));
    return Pair(lo, hi);
}
__device__ __forceinline__ float max_keeping_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The normal density at a >= 0 and the tail above a: density times a polynomial in 1 / (1 + p a), Abramowitz and Stegun 26.2.17, off by
// at most 7.5e-8.
__device__ __forceinline__ Pair normal_tail(Pair a, Pair &density) {
    const Pair t = reciprocal_2(fma2(a, Pair(0.2316419f), Pair(1.f)));
    density = exp2_2(fma2(a * a, Pair(-0.72134752f), Pair(-1.32574806f)));  // e^(-a^2 / 2) / sqrt(2 pi)
    Pair q = fma2(t, Pair(1.330274429f), Pair(-1.821255978f));
    q = fma2(t, q, Pair(1.781477937f));
    q = fma2(t, q, Pair(-0.356563782f));
    q = fma2(t, q, Pair(0.319381530f));
    return density * (t * q);
}
// (1 + tanh(u)) / 2 = 1 / (1 + e^(-2u)), u = sqrt(2/pi) (v + 0.044715 v^3)
__device__ __forceinline__ Pair tanh_gate(Pair v) {
    return reciprocal_2(exp2_2(v * fma2(v * v, Pair(-0.102943240f), Pair(-2.302208198f))) + Pair(1.f));
}
__device__ __forceinline__ Pair sigmoid_2(Pair v) { return reciprocal_2(exp2_2(v * Pair(-1.44269504f)) + Pair(1.f)); }

template <int kAct>
__device__ __forceinline__ Pair activate_2(Pair v) {
    if (kAct == FDA_ACT_GELU) {
        // v Phi(v) = max(v, 0) - |v| tail(|v|).  From 30 on the tail is 0 (and must not meet an infinite |v|).
        float lo, hi, tail_lo, tail_hi;
        v.split(lo, hi);
        const float a_lo = fminf(fabsf(lo), 30.f), a_hi = fminf(fabsf(hi), 30.f);
        Pair density;
        normal_tail(Pair(a_lo, a_hi), density).split(tail_lo, tail_hi);
        return Pair(fmaf(-a_lo, tail_lo, max_keeping_nan(lo, 0.f)), fmaf(-a_hi, tail_hi, max_keeping_nan(hi, 0.f)));
    }
    if (kAct == FDA_ACT_GELU_TANH) return v * tanh_gate(v);
    if (kAct == FDA_ACT_SILU) return v * sigmoid_2(v);
    if (kAct == FDA_ACT_RELU) {
        float lo, hi;
        v.split(lo, hi);
        return Pair(max_keeping_nan(lo, 0.f), max_keeping_nan(hi, 0.f));
    }
    return v;
}
template <int kAct>
__device__ __forceinline__ Pair activate_backward_2(Pair v, Pair dy) {
    float lo, hi;
    v.split(lo, hi);
    if (kAct == FDA_ACT_GELU) {
        Pair density;
        float h_lo, h_hi;
        fma2(normal_tail(Pair(fabsf(lo), fabsf(hi)), density), Pair(-1.f), Pair(0.5f)).split(h_lo, h_hi);
        const Pair cdf = Pair(copysignf(h_lo, lo), copysignf(h_hi, hi)) + Pair(0.5f);
        return dy * fma2(v, density, cdf);
    }
    if (kAct == FDA_ACT_GELU_TANH) {
        // beyond 12 the gate is 0 or 1 to the last bit, and the slope's polynomial would overflow for very large v
        const Pair s = tanh_gate(v), c(fminf(fmaxf(lo, -12.f), 12.f), fminf(fmaxf(hi, -12.f), 12.f));
        return dy * fma2(c * (s * fma2(s, Pair(-1.f), Pair(1.f))), fma2(c * c, Pair(0.214064437f), Pair(1.595769122f)), s);
    }
    if (kAct == FDA_ACT_SILU) {
        const Pair s = sigmoid_2(v);
        return dy * (s * fma2(v, fma2(s, Pair(-1.f), Pair(1.f)), Pair(1.f)));
    }
    if (kAct == FDA_ACT_RELU) {
        float dlo, dhi;
        dy.split(dlo, dhi);
        return Pair(activate_backward<kAct>(lo, dlo), activate_backward<kAct>(hi, dhi));
    }
    return dy;
}

// ---- 16-bit rows in registers -------------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <typename T> __device__ __forceinline__ uint32_t pack2(Pair v) {
    float lo, hi;
    v.split(lo, hi);
    return pack2<T>(lo, hi);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T> __device__ __forceinline__ Pair unpack2(uint32_t v);
template <> __device__ __forceinline__ Pair unpack2<__half>(uint32_t v) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&v));
    return Pair(f.x, f.y);
}
template <> __device__ __forceinline__ Pair unpack2<__nv_bfloat16>(uint32_t v) {
    return Pair(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// A warp's 32 rows x 32 elements of a 16-bit matrix, between global memory and registers (lane = row, two elements a register).
// The transfer to or from global memory is coalesced, four lanes a row of 64 bytes where the rows' addresses are multiples of 16
// bytes (kVector), else one lane an element; rows change hands in shared memory, 16 of them at a time.  (Each lane writing its
// own row in sectors: 122 instead of 113 us for 598016 x 256 x 256.)  `count` of the columns and the first `rows` rows exist; p
// is the first row's address.
using Stage = uint4[16 * 4];

// Unit u (16 bytes) of row r: eight lanes with rows of their own and four lanes of a row both meet every bank once.
__device__ __forceinline__ int stage_unit(int r, int u) { return r * 4 + (u ^ ((r >> 1) & 3)); }
__device__ __forceinline__ unsigned short *stage_element(Stage &stage, int r, int c) {
    return reinterpret_cast<unsigned short *>(&stage[stage_unit(r, c / 8)]) + c % 8;
}

// What a lane holds of the rows between its loads and the exchange: rows lane / 4 + 8 i, unit lane % 4.
struct Fetched {
    uint4 part[4];
};
template <typename T>
__device__ __forceinline__ void fetch_rows(const T *p, unsigned pitch, int rows, int count, Fetched &f) {
    const int lane = threadIdx.x % 32, unit = lane % 4;
    const T *mine = p + ((size_t)((lane / 4) * pitch) + 8 * unit);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f.part[i] = make_uint4(0, 0, 0, 0);
        if (lane / 4 + 8 * i < rows && 8 * unit < count) f.part[i] = __ldg(reinterpret_cast<const uint4 *>(mine + (size_t)(8 * i * pitch)));
    }
}
__device__ __forceinline__ void own_row_from(Stage &stage, int half, uint32_t (&v)[16]) {
    const int lane = threadIdx.x % 32;
    if (lane / 16 == half)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint4 q = stage[stage_unit(lane % 16, u)];
            v[4 * u] = q.x; v[4 * u + 1] = q.y; v[4 * u + 2] = q.z; v[4 * u + 3] = q.w;
        }
}
__device__ __forceinline__ void rows_of_fetched(const Fetched &f, Stage &stage, uint32_t (&v)[16]) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        __syncwarp();
        stage[stage_unit(lane / 4, lane % 4)] = f.part[2 * half];
        stage[stage_unit(lane / 4 + 8, lane % 4)] = f.part[2 * half + 1];
        __syncwarp();
        own_row_from(stage, half, v);
    }
}
// Rows that no vector access reaches, an element a lane.  All loads are on their way before the first is used.
template <typename T>
__device__ __forceinline__ void load_elements(const T *p, unsigned pitch, int rows, int count, Stage &stage, uint32_t (&v)[16]) {
    const int lane = threadIdx.x % 32;
    const unsigned short *s = reinterpret_cast<const unsigned short *>(p);
    unsigned short e[32];
#pragma unroll
    for (int r = 0; r < 32; ++r) e[r] = (r < rows && lane < count) ? s[(size_t)(r * pitch) + lane] : 0;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        __syncwarp();
#pragma unroll
        for (int r = 0; r < 16; ++r) *stage_element(stage, r, lane) = e[16 * half + r];
        __syncwarp();
        own_row_from(stage, half, v);
    }
}
template <bool kVector, typename T>
__device__ __forceinline__ void store_rows(T *p, unsigned pitch, int rows, int count, Stage &stage, const uint32_t (&v)[16]) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        __syncwarp();
        if (lane / 16 == half)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                stage[stage_unit(lane % 16, u)] = make_uint4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
        __syncwarp();
        if (kVector) {
            T *mine = p + ((size_t)((16 * half + lane / 4) * pitch) + 8 * (lane % 4));
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (16 * half + lane / 4 + 8 * i < rows && 8 * (lane % 4) < count)
                    *reinterpret_cast<uint4 *>(mine + (size_t)(8 * i * pitch)) = stage[stage_unit(lane / 4 + 8 * i, lane % 4)];
        } else {
            unsigned short *s = reinterpret_cast<unsigned short *>(p);
#pragma unroll 4
            for (int r = 0; r < 16; ++r)
                if (16 * half + r < rows && lane < count) s[(size_t)((16 * half + r) * pitch) + lane] = *stage_element(stage, r, lane);
        }
    }
}

// NaN instead of results that a warp could not wait for: up to 32 rows of `count` elements, and their sums where there are any.
template <typename T>
__device__ __noinline__ void store_nan(T *p, unsigned pitch, int rows, int count, float *sums) {
    const float nan = __int_as_float(0x7fffffff);
    for (int r = 0; r < min(rows, 32); ++r)
        for (int c = threadIdx.x % 32; c < count; c += 32) p[(size_t)r * pitch + c] = from_f32<T>(nan);
    if (sums && rows > 0)
        for (int c = threadIdx.x % 32; c < count; c += 32) sums[c] = nan;
}

}  // namespace fda_linear

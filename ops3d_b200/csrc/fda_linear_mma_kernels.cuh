// The linear operators' products on the tensor cores, for 16-bit types: tcgen05.mma over operands that the copy engine brings into
// swizzled shared memory, accumulators in tensor memory, everything after the product from there.
//
// One block per SM walks the output tiles.  Warp 0 keeps a ring of operand slices filled, warp 1 issues the products, warps 4 and up
// take finished sums out of tensor memory: accumulators are doubled, so that a tile's epilogue runs beside the next tile's
// products.  Every wait is bounded: a role that waited in vain leaves, the others follow, the epilogue writes NaN where it has no sums,
// and the block counts the event.
//
// Included by one translation unit per type.
#pragma once

#include <algorithm>

#include "fda_config.h"
#include "fda_linear_mma.cuh"

namespace fda_linear {

namespace {

constexpr int kTileRows = kMmaTileRows;            // rows of an accumulator: one per lane of tensor memory
constexpr int kSliceK = kMmaSlice;                 // contraction indices per slice: one swizzled line
constexpr int kBytesA = kTileRows * kSliceK * 2;
constexpr int kRingBytes = 192 * 1024;

template <int BN>
struct Shape {
    static constexpr int kBytesB = BN * kSliceK * 2;
    static constexpr int kBytes = kBytesA + kBytesB;
    static constexpr int kStages = kRingBytes / kBytes;  // 4, 6, 8
    // Warps 0 and 1 work on operands, 2 and 3 idle (an epilogue warp's number modulo 4 decides which lanes of tensor memory it can
    // read), then four for each part of the columns.
    static constexpr int kPart = BN == 256 ? 64 : 32, kParts = BN / kPart;
    static constexpr int kEpilogueWarps = 4 * kParts, kThreads = 32 * (4 + kEpilogueWarps);
};
constexpr int kFirstEpilogueWarp = 4;

// Common to both kernels: the ring, the accumulators' barriers, tensor memory.
template <int kStages>
struct Pipeline {
    Barrier full[kStages], empty[kStages], sums_full[2], sums_empty[2], weight_empty, drained;
    Barrier mask_go, masked;  // of pairs
    uint32_t tmem;
    volatile int failed;
};

template <bool kPair, int kStages>
__device__ __forceinline__ void pipeline_begin(Pipeline<kStages> &p, int columns, int epilogue_warps) {
    if (threadIdx.x == 32) {
        for (int i = 0; i < kStages; ++i) {
            p.full[i].init(1);
            p.empty[i].init(1);
        }
        for (int i = 0; i < 2; ++i) {
            p.sums_full[i].init(1);
            p.sums_empty[i].init(epilogue_warps * (kPair ? 2 : 1));
        }
        p.mask_go.init(1);
        p.masked.init(1);
        p.weight_empty.init(1);
        p.drained.init(1);
        p.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (threadIdx.x < 32) {
        if (kPair) tmem_alloc_pair(&p.tmem, columns);
        else tmem_alloc(&p.tmem, columns);
    }
    fence_before_sync();
}

// After every role has left.  In a sound run nothing is in flight any more (the epilogue has waited for every product, and so
// for every copy); after a wait that ran out, copies and products still running are waited for, again with a limit.
template <bool kPair, int kStages>
__device__ __forceinline__ void pipeline_end(Pipeline<kStages> &p, int columns, const Ring &issued, bool any) {
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (threadIdx.x == 0 && p.failed) {
        atomicAdd(&g_timeouts, 1u);
        volatile int again = 0;
        if (any)
            for (int i = 0; i < issued.stages; ++i) {
                // the ring's next place is `issued`: a place before it was last filled in the current round, the others in the one before
                const unsigned parity = i < issued.stage ? issued.round : issued.round ^ 1;
                p.full[i].wait(parity, &again);
            }
    }
    if (threadIdx.x == 32 && p.failed) {
        volatile int again = 0;
        if (!kPair) mma_commit(&p.drained);
        else if (cluster_rank() == 0) mma_commit_pair(&p.drained);
        p.drained.wait(0, &again);
    }
    __syncthreads();
    if (kPair) cluster_sync();  // nothing of the other block may be touched once it has left
    if (threadIdx.x < 32) {
        if (kPair) tmem_free_pair(p.tmem, columns);
        else tmem_free(p.tmem, columns);
    }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Products over rows: forward, gradient of the pre-activation, gradient of x
// ---------------------------------------------------------------------------------------------------------------------------
template <typename T>
struct RowsArgs {
    const T *bias, *extra;
    T *out;
    unsigned extra_pitch, out_pitch;  // 32 of them fit 32 bits (the host has checked)
    int depth, cols;
    bool resident;
    float *sums;  // MmaRows::sums
    Groups g;
};

// A resident weight: where all slices of a column tile fit (kResidentBytes), a block keeps them and only rows stream through the
// ring.  The grid is a multiple of the column tiles, so a block's column stays and its weight changes with the group or not at all;
// at any time the blocks work on neighbouring rows (a contiguous range of rows each was slower: 172 instead of 131 us for
// 149504 x 256 x 1024 with a residual).
// Per 128 x 256 tile of 256 inputs 64 KB instead of 192 pass from L2, whose 9 TB/s had been the bound (149504 x 256 x 1024: 107 us).
constexpr int kResidentStages = 4;
constexpr int kResidentBytes = kRingBytes - kResidentStages * kBytesA;

constexpr int kForwardPlain = 3;  // kForward without a residual

// Sums over the 32 lanes of 16 values each: lane l returns that of value l / 2 (bits reversed: sum_column).
__device__ __forceinline__ float sums_over_lanes(float (&v)[16]) {
    const unsigned lane = threadIdx.x % 32;
#pragma unroll
    for (int n = 8; n > 0; n /= 2) {  // lanes 2 n apart share out 2 n values
        const bool upper = lane & (2 * n);
#pragma unroll
        for (int j = 0; j < n; ++j) {
            const float keep = upper ? v[j + n] : v[j], give = upper ? v[j] : v[j + n];
            v[j] = keep + __shfl_xor_sync(0xffffffffu, give, 2 * n);
        }
    }
    return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1);
}
__device__ __forceinline__ int sum_column() {
    const int lane = threadIdx.x % 32;
    return (lane & 16) / 2 + (lane & 8) / 2 + (lane & 4) / 2 + (lane & 2) / 2;
}

// 16 columns of a lane's row: `row` comes as the extra elements and leaves as the results.  `bias` is in shared memory, the same
// address for the whole warp.  kPreGrad with `sums`: the sums of the results over the first `rows` lanes go there, in fp32: the bias's
// gradient is made of them, and of results rounded to 16 bits it would be off by up to twice the rounding of the sum itself.
template <typename T, int kMode, int kAct>
__device__ __forceinline__ void finish_columns(const uint32_t (&v)[16], const float *bias, uint32_t *row, float *sums, int rows, int columns) {
    float kept[kMode == kPreGrad ? 16 : 1];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        Pair r(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
        if (kMode != kGradX) {
            const float2 b = *reinterpret_cast<const float2 *>(bias + 2 * j);
            r = r + Pair(b.x, b.y);
            if (kMode == kPreGrad) {
                r = activate_backward_2<kAct>(r, unpack2<T>(row[j]));
                r.split(kept[(2 * j) % (sizeof(kept) / 4)], kept[(2 * j + 1) % (sizeof(kept) / 4)]);
            } else {
                r = activate_2<kAct>(r);
                if (kMode == kForward) r = r + unpack2<T>(row[j]);
            }
        }
        row[j] = pack2<T>(r);
    }
    if constexpr (kMode == kPreGrad)
        if (sums) {
            const int lane = threadIdx.x % 32;
#pragma unroll
            for (int j = 0; j < 16; ++j) kept[j] = lane < rows ? kept[j] : 0.f;  // what lies beyond may be anything
            const float sum = sums_over_lanes(kept);
            const int c = sum_column();
            if (lane % 2 == 0 && c < columns) sums[c] = sum;
        }
}

// kVector: the rows of out and of extra start on 16-byte boundaries.
template <typename T, int kMode, int kAct, int BN, bool kVector>
__global__ void __launch_bounds__(Shape<BN>::kThreads, 1)
    linear_rows_mma_kernel(const RowsArgs<T> p, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                           const __grid_constant__ CUtensorMap map_extra) {
    constexpr int kStages = Shape<BN>::kStages, kColumns = 2 * BN;
    constexpr bool kWeightMn = kMode == kGradX;  // the weight's lines run along the output columns
    constexpr bool kExtra = kMode == kForward || kMode == kPreGrad;
    extern __shared__ char dynamic[];
    __shared__ RowTable table;
    __shared__ Pipeline<kStages> pipe;
    __shared__ __align__(16) float bias_of[Shape<BN>::kEpilogueWarps][Shape<BN>::kPart];
    __shared__ __align__(16) Stage stages[Shape<BN>::kEpilogueWarps];
    char *const ring = reinterpret_cast<char *>(((uintptr_t)dynamic + kAtom - 1) & ~(uintptr_t)(kAtom - 1));
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        prefetch_map(&map_a);
        prefetch_map(&map_w);
    }
    pipeline_begin<false>(pipe, kColumns, Shape<BN>::kEpilogueWarps);
    wait_for_previous_kernel();
    build_row_table(p.g, kTileRows, kMode != kPreGrad, table);
    __syncthreads();
    fence_after_sync();
    const unsigned columns = (p.cols + BN - 1) / BN;
    const unsigned tiles = (unsigned)table.unit_begin[p.g.groups + 2] * p.g.batch * columns;  // the host has checked that they fit
    const int slices = (p.depth + kSliceK - 1) / kSliceK;
    char *const weight = p.resident ? ring + kResidentStages * kBytesA : ring + kBytesA;  // of the first slice or the first stage
    const int stage_bytes = p.resident ? kBytesA : Shape<BN>::kBytes, weight_step = p.resident ? Shape<BN>::kBytesB : 0;
    volatile int *const failed = &pipe.failed;
    Ring ring_at(p.resident ? kResidentStages : kStages);
    bool any = false;

    if (warp == 0) {
        if (lane == 0) {
            bool sound = true;
            int weight_group = -1, weight_col = -1;
            unsigned changes = 0;
            for (unsigned tile = blockIdx.x; tile < tiles && sound; tile += gridDim.x) {
                const RowUnit u = row_unit(p.g, table, kTileRows, tile / columns);
                if (u.group < 0) continue;
                const int col0 = (int)(tile % columns * BN);
                if (kExtra && kVector)  // on their way to L2 while the tile's products run: the epilogue's loads then wait for L2 only
#pragma unroll
                    for (int i = 0; i < BN / 64; ++i) prefetch_2d(&map_extra, col0 + 64 * i, (int)u.row);
                const bool fresh = !p.resident || u.group != weight_group || col0 != weight_col;
                if (p.resident && fresh) {  // the products with the weight before have to be through
                    if (changes++) sound = pipe.weight_empty.wait(changes & 1, failed);
                    if (!sound) break;
                    weight_group = u.group;
                    weight_col = col0;
                }
                for (int s = 0; s < slices; ++s) {
                    sound = pipe.empty[ring_at.stage].wait(ring_at.round ^ 1, failed);
                    if (!sound) break;
                    char *a = ring + ring_at.stage * stage_bytes;
                    Barrier *bar = &pipe.full[ring_at.stage];
                    bar->arrive_expect(kBytesA + (fresh ? Shape<BN>::kBytesB : 0));
                    tma_2d(&map_a, a, bar, s * kSliceK, (int)u.row);
                    if (fresh) {
                        char *b = weight + (p.resident ? s * weight_step : ring_at.stage * stage_bytes);
                        if (kWeightMn) {
#pragma unroll
                            for (int i = 0; i < BN / 64; ++i)
                                tma_3d(&map_w, b + i * (64 * kSliceK * 2), bar, col0 + 64 * i, s * kSliceK, u.group);
                        } else {
                            tma_3d(&map_w, b, bar, s * kSliceK, col0, u.group);
                        }
                    }
                    ring_at.next();
                    any = true;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        constexpr uint32_t kInstruction = instruction<T>(kTileRows, BN, false, kWeightMn);
        constexpr uint32_t kHigh = operand_high(kAtom), kStepB = kWeightMn ? 2 * kAtom / 16 : 2;  // of 16 contraction indices
        const uint32_t a0 = operand_low(ring, 16), b0 = operand_low(weight, kWeightMn ? 64 * kSliceK * 2 : 16);
        Ring sums(2);
        bool sound = true;
        int weight_group = -1, weight_col = -1;
        for (unsigned tile = blockIdx.x; tile < tiles && sound; tile += gridDim.x) {
            const RowUnit u = row_unit(p.g, table, kTileRows, tile / columns);
            if (u.group < 0) continue;
            const int tile_col = (int)(tile % columns * BN);
            if (p.resident && (u.group != weight_group || tile_col != weight_col)) {
                if (weight_group >= 0 && elected()) commit<false>(&pipe.weight_empty);
                weight_group = u.group;
                weight_col = tile_col;
            }
            sound = __all_sync(0xffffffffu, pipe.sums_empty[sums.stage].wait(sums.round ^ 1, failed));
            if (!sound) break;
            fence_after_sync();
            const uint32_t d = pipe.tmem + sums.stage * BN;
            for (int s = 0; s < slices; ++s) {
                sound = __all_sync(0xffffffffu, pipe.full[ring_at.stage].wait(ring_at.round, failed));
                if (!sound) break;
                fence_after_sync();
                const uint32_t at = ring_at.stage * (stage_bytes / 16);
                const uint32_t a = a0 + at, b = b0 + (p.resident ? s * (weight_step / 16) : at);
                if (elected()) {
#pragma unroll
                    for (int k = 0; k < kSliceK / 16; ++k)
                        mma_f16<false>(d, a + 2 * k, kHigh, b + kStepB * k, kHigh, kInstruction, s > 0 || k > 0);
                    commit<false>(&pipe.empty[ring_at.stage]);
                }
                ring_at.next();
            }
            if (!sound) break;
            if (elected()) commit<false>(&pipe.sums_full[sums.stage]);
            sums.next();
        }
        __syncwarp();
    } else if (warp >= kFirstEpilogueWarp) {
        // Each warp owns the 32 lanes of tensor memory that its number allows it, and a part of the columns.  What it needs from
        // global memory it asks for before it waits for the sums: loads chunk by chunk, each waited for, cost a tile of
        // 128 x 256 two of its five microseconds.
        constexpr int kPart = Shape<BN>::kPart, kChunks = kPart / 32;
        const int quarter = warp % 4, part = (warp - kFirstEpilogueWarp) / 4;
        float *const bias = bias_of[warp - kFirstEpilogueWarp];
        Stage &stage = stages[warp - kFirstEpilogueWarp];
        for (int i = lane; i < kPart; i += 32) bias[i] = 0.f;
        int bias_group = -1, bias_col = -1;
        Ring sums(2);
        struct Place {
            long long first;  // row of the warp's part of a tile
            int rows, col0, group;
        };
        const auto place = [&](unsigned tile) {
            const RowUnit u = row_unit(p.g, table, kTileRows, tile / columns);
            Place at;
            at.first = u.row + quarter * 32;
            at.rows = u.count - quarter * 32;  // none or fewer where not positive
            at.col0 = (int)(tile % columns * BN) + part * kPart;
            at.group = u.group;
            return at;
        };
        Fetched fetched;  // the extra rows of the chunk to come
        const auto fetch = [&](const Place &at, int c) {
            if (kExtra && kVector)
                fetch_rows(p.extra + (size_t)at.first * p.extra_pitch + at.col0 + 32 * c, p.extra_pitch, at.rows, p.cols - at.col0 - 32 * c, fetched);
        };
        const auto give_up = [&](unsigned tile) {  // NaN for what the warp still owes
            for (; tile < tiles; tile += gridDim.x) {
                const Place at = place(tile);
                float *const sums_row =
                    kMode == kPreGrad && p.sums ? p.sums + ((size_t)(tile / columns) * (kTileRows / kSumRows) + quarter) * p.cols + at.col0 : nullptr;
                store_nan(p.out + (size_t)at.first * p.out_pitch + at.col0, p.out_pitch, at.rows, min(kPart, p.cols - at.col0), sums_row);
            }
        };
        Place next;
        if (blockIdx.x < tiles) {
            next = place(blockIdx.x);
            fetch(next, 0);
        }
        for (unsigned tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            const Place u = next;
            if (tile + gridDim.x < tiles) next = place(tile + gridDim.x);
            const int rows = u.rows, col0 = u.col0;
            T *const out_rows = p.out + (size_t)u.first * p.out_pitch + col0;
            const auto extra_of = [&](int c, int count, uint32_t(&v)[16]) {  // chunk c of the extra rows, lane by row; asks for the one after
                if (kExtra && kVector) {
                    rows_of_fetched(fetched, stage, v);
                    if (c + 1 < kChunks && count > 32) fetch(u, c + 1);
                    else if (tile + gridDim.x < tiles) fetch(next, 0);
                }
            };
            // (tiles of which no vector access reaches the rows have one chunk a warp)
            uint32_t elements[16] = {};
            static_assert(kVector || kChunks == 1, "");
            if (kExtra && !kVector)
                load_elements(p.extra + (size_t)u.first * p.extra_pitch + col0, p.extra_pitch, rows, p.cols - col0, stage, elements);
            if (col0 >= p.cols) {  // no column of this part: nothing is fetched or stored, but the tile counts
                if (tile + gridDim.x < tiles) fetch(next, 0);
            }
            if (kMode != kGradX) {
                if (p.bias && u.group >= 0 && (u.group != bias_group || col0 != bias_col)) {
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < kPart / 32; ++i)
                        if (col0 + 32 * i + lane < p.cols) bias[32 * i + lane] = to_f32<T>(p.bias[(size_t)u.group * p.cols + col0 + 32 * i + lane]);
                    bias_group = u.group;
                    bias_col = col0;
                    __syncwarp();
                }
            }
            if (u.group < 0) {  // no product: the residual, or zeros
#pragma unroll 1
                for (int c = 0; c < kChunks; ++c)
                    if (col0 + 32 * c < p.cols) {
                        uint32_t row[16] = {};
                        if (kVector) extra_of(c, p.cols - col0 - 32 * c, row);
                        store_rows<kVector>(out_rows + 32 * c, p.out_pitch, rows, p.cols - col0 - 32 * c, stage, kVector ? row : elements);
                    }
                continue;
            }
            if (!__all_sync(0xffffffffu, pipe.sums_full[sums.stage].wait(sums.round, failed))) {
                give_up(tile);
                break;
            }
            fence_after_sync();
            const uint32_t address = pipe.tmem + sums.stage * BN + part * kPart + ((uint32_t)(quarter * 32) << 16);
            float *const sums_row =
                kMode == kPreGrad && p.sums && rows > 0 ? p.sums + ((size_t)(tile / columns) * (kTileRows / kSumRows) + quarter) * p.cols + col0 : nullptr;
#pragma unroll 1
            for (int c = 0; c < kChunks; ++c) {
                const int count = p.cols - col0 - 32 * c;
                if (count <= 0) break;
                uint32_t row[16];
                if (kVector) {
                    extra_of(c, count, row);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) row[j] = elements[j];
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t v[16];
                    __syncwarp();
                    tmem_load(address + 32 * c + 16 * h, v);
                    tmem_load_wait();
                    finish_columns<T, kMode, kAct>(v, bias + 32 * c + 16 * h, row + 8 * h, sums_row ? sums_row + 32 * c + 16 * h : nullptr, rows,
                                                   count - 16 * h);
                }
                store_rows<kVector>(out_rows + 32 * c, p.out_pitch, rows, count, stage, row);
            }
            fence_before_sync();
            __syncwarp();
            if (lane == 0) pipe.sums_empty[sums.stage].arrive();
            sums.next();
        }
    }
    pipeline_end<false>(pipe, kColumns, ring_at, any);
}

// ---------------------------------------------------------------------------------------------------------------------------
// Products over rows by pairs of blocks
// ---------------------------------------------------------------------------------------------------------------------------
// Two blocks of a cluster make one tile of 256 x 256 (cta_group::2): each brings its own 128 rows and its half of the weight's 256
// columns and keeps 128 rows of sums, so per block half the weight passes from L2 and lies in shared memory.  Where there are
// extra rows, what that leaves holds a buffer of 32 rows x 64 columns for each of the 16 epilogue warps, which the copy engine
// fills a tile ahead; otherwise it makes the ring longer.
//
// The first block issues all products; the barriers that these wait for are its own, and the second block's copies and epilogue
// warps signal them across the cluster.
constexpr int kPairRows = 256, kPairColumns = 256, kPairEpilogueWarps = 16;
constexpr int kPairThreads = 32 * (kFirstEpilogueWarp + kPairEpilogueWarps);
constexpr int kPairBytesB = kPairColumns / 2 * kSliceK * 2;  // a block's half of a weight slice
constexpr int kPairMaxStages = 8, kPairLeastStages = 4;
constexpr int kPairOperands = 192 * 1024, kBufferBytes = 32 * 64 * 2;
__host__ __device__ constexpr int pair_ring(bool extra) { return kPairOperands - (extra ? kPairEpilogueWarps * kBufferBytes : 0); }
constexpr int kPairSmem = kPairOperands + kAtom;

struct PairPipeline {
    Barrier full[kPairMaxStages], empty[kPairMaxStages], sums_full[2], sums_empty[2], weight_empty, drained;
    Barrier extra_full[kPairEpilogueWarps], extra_empty[kPairEpilogueWarps];
    uint32_t tmem;
    volatile int failed;
};

// Unit u (16 bytes) of row r in a buffer, as the copy engine's 128-byte swizzle has it.
__device__ __forceinline__ const uint4 *buffer_unit(const char *buffer, int r, int u) {
    return reinterpret_cast<const uint4 *>(buffer + r * 128 + ((u ^ (r & 7)) * 16));
}

template <typename T, int kMode, int kAct>
__global__ void __launch_bounds__(kPairThreads, 1)
    linear_rows_pair_kernel(const RowsArgs<T> p, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                            const __grid_constant__ CUtensorMap map_extra) {
    constexpr bool kWeightMn = kMode == kGradX;
    constexpr bool kExtra = kMode == kForward || kMode == kPreGrad;
    constexpr int kColumns = 512;
    extern __shared__ char dynamic[];
    __shared__ RowTable table;
    __shared__ PairPipeline pipe;
    __shared__ __align__(16) float bias_of[kPairEpilogueWarps][64];
    __shared__ __align__(16) Stage stages_of[kPairEpilogueWarps];
    char *const ring = reinterpret_cast<char *>(((uintptr_t)dynamic + kAtom - 1) & ~(uintptr_t)(kAtom - 1));
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const unsigned rank = cluster_rank();
    if (threadIdx.x == 32) {
        for (int i = 0; i < kPairMaxStages; ++i) {
            pipe.full[i].init(1);
            pipe.empty[i].init(1);
        }
        for (int i = 0; i < 2; ++i) {
            pipe.sums_full[i].init(1);
            pipe.sums_empty[i].init(2 * kPairEpilogueWarps);
        }
        pipe.weight_empty.init(1);
        pipe.drained.init(1);
        for (int i = 0; i < kPairEpilogueWarps; ++i) {
            pipe.extra_full[i].init(1);
            pipe.extra_empty[i].init(32);
        }
        pipe.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 0) tmem_alloc_pair(&pipe.tmem, kColumns);
    wait_for_previous_kernel();
    build_row_table(p.g, kPairRows, kMode != kPreGrad, table);
    fence_before_sync();
    __syncthreads();
    cluster_sync();
    fence_after_sync();
    const unsigned columns = (p.cols + kPairColumns - 1) / kPairColumns, pairs = gridDim.x / 2, pair = blockIdx.x / 2;
    const unsigned tiles = (unsigned)table.unit_begin[p.g.groups + 2] * p.g.batch * columns;
    const int slices = (p.depth + kSliceK - 1) / kSliceK;
    // as many stages as fit beside the weight, if that stays
    const int stage_bytes = p.resident ? kBytesA : kBytesA + kPairBytesB, weight_step = p.resident ? kPairBytesB : 0;
    const int stages = min(kPairMaxStages, (pair_ring(kExtra) - slices * weight_step) / stage_bytes);
    char *const weight = p.resident ? ring + stages * kBytesA : ring + kBytesA;  // of the first slice or the first stage
    volatile int *const failed = &pipe.failed;
    Ring ring_at(stages);

    if (warp == 0) {
        if (lane == 0) {
            bool sound = true;
            int weight_group = -1, weight_col = -1;
            unsigned changes = 0;
            for (unsigned tile = pair; tile < tiles && sound; tile += pairs) {
                const RowUnit u = row_unit(p.g, table, kPairRows, tile / columns);
                if (u.group < 0) continue;
                const int tile_col = (int)(tile % columns * kPairColumns), col0 = tile_col + (int)rank * (kPairColumns / 2);
                const int row0 = (int)u.row + (int)rank * kTileRows;
                if (kExtra)  // on their way to L2 while the tile's products run
#pragma unroll
                    for (int i = 0; i < 4 * (kPairColumns / 64); ++i) prefetch_2d(&map_extra, tile_col + 64 * (i / 4), row0 + 32 * (i % 4));
                const bool fresh = !p.resident || u.group != weight_group || col0 != weight_col;
                if (p.resident && fresh) {  // the products with the weight before have to be through
                    if (changes++) sound = pipe.weight_empty.wait(changes & 1, failed);
                    if (!sound) break;
                    weight_group = u.group;
                    weight_col = col0;
                }
                for (int s = 0; s < slices; ++s) {
                    sound = pipe.empty[ring_at.stage].wait(ring_at.round ^ 1, failed);
                    if (!sound) break;
                    char *a = ring + ring_at.stage * stage_bytes;
                    // the first block's barrier counts the bytes of both
                    const uint32_t bar = cluster_address(&pipe.full[ring_at.stage], 0);
                    if (rank == 0) pipe.full[ring_at.stage].arrive_expect(2 * (kBytesA + (fresh ? kPairBytesB : 0)));
                    tma_2d_pair(&map_a, a, bar, s * kSliceK, row0);
                    if (fresh) {
                        char *b = weight + (p.resident ? s * weight_step : ring_at.stage * stage_bytes);
                        if (kWeightMn) {
#pragma unroll
                            for (int i = 0; i < kPairColumns / 128; ++i)
                                tma_3d_pair(&map_w, b + i * (64 * kSliceK * 2), bar, col0 + 64 * i, s * kSliceK, u.group);
                        } else {
                            tma_3d_pair(&map_w, b, bar, s * kSliceK, col0, u.group);
                        }
                    }
                    ring_at.next();
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            constexpr uint32_t kInstruction = instruction<T>(kPairRows, kPairColumns, false, kWeightMn);
            constexpr uint32_t kHigh = operand_high(kAtom), kStepB = kWeightMn ? 2 * kAtom / 16 : 2;  // of 16 contraction indices
            const uint32_t a0 = operand_low(ring, 16), b0 = operand_low(weight, kWeightMn ? 64 * kSliceK * 2 : 16);
            Ring sums(2);
            bool sound = true;
            int weight_group = -1, weight_col = -1;
            for (unsigned tile = pair; tile < tiles && sound; tile += pairs) {
                const RowUnit u = row_unit(p.g, table, kPairRows, tile / columns);
                if (u.group < 0) continue;
                const int tile_col = (int)(tile % columns * kPairColumns);
                if (p.resident && (u.group != weight_group || tile_col != weight_col)) {
                    if (weight_group >= 0 && elected()) commit<true>(&pipe.weight_empty);
                    weight_group = u.group;
                    weight_col = tile_col;
                }
                sound = __all_sync(0xffffffffu, pipe.sums_empty[sums.stage].wait(sums.round ^ 1, failed));
                if (!sound) break;
                fence_after_sync();
                const uint32_t d = pipe.tmem + sums.stage * kPairColumns;
                for (int s = 0; s < slices; ++s) {
                    sound = __all_sync(0xffffffffu, pipe.full[ring_at.stage].wait(ring_at.round, failed));
                    if (!sound) break;
                    fence_after_sync();
                    const uint32_t at = ring_at.stage * (stage_bytes / 16);
                    const uint32_t a = a0 + at, b = b0 + (p.resident ? s * (weight_step / 16) : at);
                    if (elected()) {
#pragma unroll
                        for (int k = 0; k < kSliceK / 16; ++k)
                            mma_f16<true>(d, a + 2 * k, kHigh, b + kStepB * k, kHigh, kInstruction, s > 0 || k > 0);
                        commit<true>(&pipe.empty[ring_at.stage]);
                    }
                    ring_at.next();
                }
                if (!sound) break;
                if (elected()) commit<true>(&pipe.sums_full[sums.stage]);
                sums.next();
            }
        }
        __syncwarp();
    } else if (warp >= kFirstEpilogueWarp) {
        const int mine = warp - kFirstEpilogueWarp, quarter = warp % 4, part = mine / 4;
        char *const buffer = ring + pair_ring(true) + mine * kBufferBytes;
        float *const bias = bias_of[mine];
        Stage &stage = stages_of[mine];
        for (int i = lane; i < 64; i += 32) bias[i] = 0.f;
        int bias_group = -1, bias_col = -1;
        const uint32_t sums_empty[2] = {cluster_address(&pipe.sums_empty[0], 0), cluster_address(&pipe.sums_empty[1], 0)};
        Ring sums(2);
        struct Place {
            long long first;  // row of the warp's part of a tile
            int rows, col0, group;
        };
        const auto place = [&](unsigned tile) {
            const RowUnit u = row_unit(p.g, table, kPairRows, tile / columns);
            const int above = (int)rank * kTileRows + quarter * 32;
            Place at;
            at.first = u.row + above;
            at.rows = u.count - above;  // none where not positive
            at.col0 = (int)(tile % columns * kPairColumns) + part * 64;
            at.group = u.group;
            return at;
        };
        const auto works = [&](const Place &at) { return at.rows > 0 && at.col0 < p.cols; };
        // A place's extra rows into the buffer.  Its readers are ordinary loads and its next writer is the copy engine, which no barrier
        // alone orders behind them: an arrival right behind the reads let the copy overtake some.  So each lane arrives at extra_empty
        // when it has stored what it made of its rows (its loads have ended) and has put a fence between the two kinds of access.
        unsigned asked = 0, loads = 0;
        const auto request = [&](const Place &at) {
            if (!kExtra || !works(at)) return;
            ++asked;
            if (lane == 0 && pipe.extra_empty[mine].wait(asked & 1, failed)) {
                pipe.extra_full[mine].arrive_expect(kBufferBytes);
                tma_2d(&map_extra, buffer, &pipe.extra_full[mine], at.col0, (int)at.first);
            }
        };
        const auto give_up = [&](unsigned tile) {  // NaN for what the warp still owes
            for (; tile < tiles; tile += pairs) {
                const Place at = place(tile);
                float *const sums_row =
                    kMode == kPreGrad && p.sums
                        ? p.sums + ((size_t)(tile / columns) * (kPairRows / kSumRows) + rank * (kTileRows / kSumRows) + quarter) * p.cols + at.col0
                        : nullptr;
                store_nan(p.out + (size_t)at.first * p.out_pitch + at.col0, p.out_pitch, at.rows, min(64, p.cols - at.col0), sums_row);
            }
        };
        Place next;
        if (pair < tiles) {
            next = place(pair);
            request(next);
        }
        for (unsigned tile = pair; tile < tiles; tile += pairs) {
            const Place u = next;
            const bool more = tile + pairs < tiles;
            if (more) next = place(tile + pairs);
            if (kMode != kGradX && p.bias && u.group >= 0 && (u.group != bias_group || u.col0 != bias_col)) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (u.col0 + 32 * i + lane < p.cols) bias[32 * i + lane] = to_f32<T>(p.bias[(size_t)u.group * p.cols + u.col0 + 32 * i + lane]);
                bias_group = u.group;
                bias_col = u.col0;
                __syncwarp();
            }
            if (u.group >= 0) {
                if (!__all_sync(0xffffffffu, pipe.sums_full[sums.stage].wait(sums.round, failed))) {
                    give_up(tile);
                    break;
                }
                fence_after_sync();
            }
            if (works(u)) {
                if (kExtra) {
                    if (!__all_sync(0xffffffffu, pipe.extra_full[mine].wait(loads & 1, failed))) {
                        give_up(tile);
                        break;
                    }
                    ++loads;
                }
                const uint32_t address = pipe.tmem + sums.stage * kPairColumns + part * 64 + ((uint32_t)(quarter * 32) << 16);
                T *const out = p.out + (size_t)u.first * p.out_pitch + u.col0;
                float *const sums_row =
                    kMode == kPreGrad && p.sums
                        ? p.sums + ((size_t)(tile / columns) * (kPairRows / kSumRows) + rank * (kTileRows / kSumRows) + quarter) * p.cols + u.col0
                        : nullptr;
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    uint32_t row[16] = {};
                    if (kExtra) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint4 q = *buffer_unit(buffer, lane, 4 * c + j);
                            row[4 * j] = q.x; row[4 * j + 1] = q.y; row[4 * j + 2] = q.z; row[4 * j + 3] = q.w;
                        }
                    }
                    if (u.group >= 0)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t v[16];
                            __syncwarp();
                            tmem_load(address + 32 * c + 16 * h, v);
                            tmem_load_wait();
                            finish_columns<T, kMode, kAct>(v, bias + 32 * c + 16 * h, row + 8 * h,
                                                           sums_row ? sums_row + 32 * c + 16 * h : nullptr, u.rows,
                                                           p.cols - u.col0 - 32 * c - 16 * h);
                        }
                    store_rows<true>(out + 32 * c, p.out_pitch, u.rows, p.cols - u.col0 - 32 * c, stage, row);
                }
                if (kExtra) {
                    fence_async();
                    pipe.extra_empty[mine].arrive();
                }
            }
            if (more) request(next);
            if (u.group >= 0) {
                fence_before_sync();
                __syncwarp();
                if (lane == 0) arrive_at(sums_empty[sums.stage]);
                sums.next();
            }
        }
        if (kExtra && asked != loads && lane == 0) {  // only after a wait that ran out: a copy may still be on its way
            volatile int again = 0;
            pipe.extra_full[mine].wait((asked - 1) & 1, &again);
        }
        __syncwarp();
    }

    // As in pipeline_end; nothing of the other block may be touched once it has left.
    fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 32 && rank == 0 && pipe.failed) {
        volatile int again = 0;
        mma_commit_pair(&pipe.drained);
        pipe.drained.wait(0, &again);
    }
    if (threadIdx.x == 0 && pipe.failed) {
        atomicAdd(&g_timeouts, 1u);
        volatile int again = 0;
        if (rank == 0)
            for (int i = 0; i < stages; ++i) pipe.full[i].wait(i < ring_at.stage ? ring_at.round : ring_at.round ^ 1, &again);
    }
    __syncthreads();
    cluster_sync();
    fence_after_sync();
    if (warp == 0) tmem_free_pair(pipe.tmem, kColumns);
}

// ---------------------------------------------------------------------------------------------------------------------------
// Gradient of the weight
// ---------------------------------------------------------------------------------------------------------------------------
// An accumulator holds 128 outputs x BN inputs of g^T x over a piece of a group's rows; both operands have their lines across
// the contraction.  The bias's gradient is one more narrow product of the same g with ones.
//
// kPair: two blocks make 256 outputs x 256 inputs, each with its own 128 outputs and half of the inputs, so that 32 instead of 48 KB
// pass from L2 for 64 rows (73728 rows, 256 -> 1024: 51 -> 45 us).
constexpr int kOnesColumns = 16;
constexpr int kOnesBytes = kOnesColumns * kSliceK * 2;

template <int BN, bool kPair>
struct WeightShape {
    static constexpr int kOutputs = kPair ? 2 * kTileRows : kTileRows, kColumnsB = kPair ? BN / 2 : BN;
    static constexpr int kBytes = kBytesA + kColumnsB * kSliceK * 2, kStages = kRingBytes / kBytes;
};

template <typename T>
struct WeightGradArgs {
    T *grad_weight, *grad_bias;
    float *slots, *bias_slots;
    int in_features, out_features;
    int piece;
    Groups g;
};

template <typename T, int BN, bool kVector, bool kPair>
__global__ void __launch_bounds__(Shape<BN>::kThreads, 1)
    linear_weight_grad_mma_kernel(const WeightGradArgs<T> p, const __grid_constant__ CUtensorMap map_g,
                                  const __grid_constant__ CUtensorMap map_x) {
    using W = WeightShape<BN, kPair>;
    constexpr int kStages = W::kStages, kColumns = 512;
    extern __shared__ char dynamic[];
    __shared__ PieceTable table;
    __shared__ Pipeline<kStages> pipe;
    __shared__ __align__(16) Stage stages[Shape<BN>::kEpilogueWarps];
    char *const ring = reinterpret_cast<char *>(((uintptr_t)dynamic + kAtom - 1) & ~(uintptr_t)(kAtom - 1));
    char *const ones = ring + kStages * W::kBytes;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        prefetch_map(&map_g);
        prefetch_map(&map_x);
    }
    pipeline_begin<kPair>(pipe, kColumns, Shape<BN>::kEpilogueWarps);
    for (int i = threadIdx.x; i < kOnesBytes / 4; i += Shape<BN>::kThreads) reinterpret_cast<uint32_t *>(ones)[i] = pack2<T>(1.f, 1.f);
    fence_async();
    wait_for_previous_kernel();
    build_piece_table(p.g, kSliceK, p.piece, table);
    __syncthreads();
    if (kPair) cluster_sync();
    fence_after_sync();
    const unsigned rank = kPair ? cluster_rank() : 0, worker = kPair ? blockIdx.x / 2 : blockIdx.x, workers = kPair ? gridDim.x / 2 : gridDim.x;
    const int out_tiles = (p.out_features + W::kOutputs - 1) / W::kOutputs, in_tiles = (p.in_features + BN - 1) / BN;
    const int per_piece = out_tiles * in_tiles;
    const long long items = (long long)table.piece_begin[p.g.groups] * per_piece;
    volatile int *const failed = &pipe.failed;
    Ring ring_at(kStages);
    bool any = false;

    struct Item {
        int group, piece, out0, in0, first, last, step;  // blocks first, first + step, ... of the group, below last
    };
    const auto item_at = [&](long long i) {
        Item it;
        const int piece = (int)(i / per_piece), t = (int)(i % per_piece);
        it.group = find_section(table.piece_begin, p.g.groups, piece);
        it.piece = piece - table.piece_begin[it.group];
        it.out0 = (t / in_tiles) * W::kOutputs + (int)rank * kTileRows;  // this block's
        it.in0 = (t % in_tiles) * BN;
        // the pieces of a group take its blocks in turn, so that at any time they read neighbouring rows
        it.first = it.piece;
        it.step = table.piece_begin[it.group + 1] - table.piece_begin[it.group];
        it.last = group_blocks(p.g, table.start, it.group, kSliceK);
        return it;
    };

    // An item's blocks one after the other, without a division for each (with one the 512 blocks of 4736 x 8192 x 1024 took 166 us, 154
    // without).
    struct Walk {
        int row, count;  // of the current block: its first row over all batch elements, its rows
        int left;        // blocks to come, this one among them
        int index, per, length, rows, step, base;
        __device__ __forceinline__ void place() {
            row = base + index * kSliceK;
            count = min(kSliceK, length - index * kSliceK);
        }
        __device__ __forceinline__ void next() {
            if (--left <= 0) return;
            for (index += step; index >= per; index -= per) base += rows;
            place();
        }
    };
    const auto walk = [&](const Item &it) {
        Walk w;
        const int start = table.start[it.group];
        w.length = table.start[it.group + 1] - start;
        w.per = (int)(((long long)w.length + kSliceK - 1) / kSliceK);
        w.left = it.first < it.last ? (it.last - it.first + it.step - 1) / it.step : 0;
        w.rows = p.g.rows;
        w.step = it.step;
        if (w.left > 0) {
            w.index = it.first % w.per;
            w.base = start + it.first / w.per * p.g.rows;
            w.place();
        }
        return w;
    };

    if (warp == 0) {
        if (lane == 0) {
            bool sound = true;
            for (long long i = worker; i < items && sound; i += workers) {
                const Item it = item_at(i);
                for (Walk at = walk(it); at.left > 0; at.next()) {
                    const int row = at.row;
                    sound = pipe.empty[ring_at.stage].wait(ring_at.round ^ 1, failed);
                    if (!sound) break;
                    char *a = ring + ring_at.stage * W::kBytes, *b = a + kBytesA;
                    Barrier *bar = &pipe.full[ring_at.stage];
                    if (rank == 0) bar->arrive_expect(W::kBytes * (kPair ? 2 : 1));
                    const int in0 = it.in0 + (int)rank * W::kColumnsB;
                    if (kPair) {  // the first block's barrier counts the bytes of both
                        const uint32_t first = cluster_address(bar, 0);
#pragma unroll
                        for (int k = 0; k < kTileRows / 64; ++k)
                            tma_2d_pair(&map_g, a + k * (64 * kSliceK * 2), first, it.out0 + 64 * k, row);
#pragma unroll
                        for (int k = 0; k < W::kColumnsB / 64; ++k)
                            tma_2d_pair(&map_x, b + k * (64 * kSliceK * 2), first, in0 + 64 * k, row);
                    } else {
#pragma unroll
                        for (int k = 0; k < kTileRows / 64; ++k) tma_2d(&map_g, a + k * (64 * kSliceK * 2), bar, it.out0 + 64 * k, row);
#pragma unroll
                        for (int k = 0; k < W::kColumnsB / 64; ++k) tma_2d(&map_x, b + k * (64 * kSliceK * 2), bar, in0 + 64 * k, row);
                    }
                    ring_at.next();
                    any = true;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        constexpr uint32_t kInstruction = instruction<T>(W::kOutputs, BN, true, true);
        constexpr uint32_t kOnesInstruction = instruction<T>(W::kOutputs, kOnesColumns, true, false);
        // Lines of the next group's rows (or of nothing) go out of both operands, for 0 times NaN is NaN.  A line of 128 bytes is one
        // row of a block of 64 columns, wherever the swizzle has its parts.
        const auto clear_lines = [&](char *a, int count) {
            constexpr int kBlocks = kTileRows / 64 + W::kColumnsB / 64;
            const int lines = kSliceK - count;
            for (int l = lane; l < kBlocks * lines * 8; l += 32) {
                const int block = l / (lines * 8), rest = l - block * lines * 8;
                reinterpret_cast<uint4 *>(a + block * (64 * kSliceK * 2) + count * 128)[rest] = make_uint4(0, 0, 0, 0);
            }
            fence_async();
            __syncwarp();
        };
        constexpr uint32_t kHigh = operand_high(kAtom);
        const uint32_t a0 = operand_low(ring, 64 * kSliceK * 2), b0 = operand_low(ring + kBytesA, 64 * kSliceK * 2), ones0 = operand_low(ones, 16);
        const uint32_t pipe_tmem = pipe.tmem;
        unsigned round = 0, masks = 0;
        bool sound = true;
        for (long long i = worker; i < items && sound; i += workers) {
            const Item it = item_at(i);
            if (it.first >= it.last) continue;
            const bool bias = it.in0 == 0 && p.grad_bias;
            if (rank == 0) {
                sound = __all_sync(0xffffffffu, pipe.sums_empty[0].wait(round ^ 1, failed));
                if (!sound) break;
                fence_after_sync();
            }
            bool more = false;
            for (Walk at = walk(it); at.left > 0; at.next()) {
                const int count = at.count;
                char *a = ring + ring_at.stage * W::kBytes;
                if (rank != 0) {  // the second block clears its lines when the first has seen the copies of both
                    if (count < kSliceK) {
                        sound = __all_sync(0xffffffffu, pipe.mask_go.wait(masks++ & 1, failed));
                        if (!sound) break;
                        acquire_cluster();  // the copies that the zeros overwrite
                        clear_lines(a, count);
                        if (lane == 0) release_at(cluster_address(&pipe.masked, 0));
                    }
                    ring_at.next();
                    continue;
                }
                sound = __all_sync(0xffffffffu, pipe.full[ring_at.stage].wait(ring_at.round, failed));
                if (!sound) break;
                if (count < kSliceK) {
                    if (kPair && lane == 0) release_at(cluster_address(&pipe.mask_go, 1));
                    clear_lines(a, count);
                    if (kPair) {
                        sound = __all_sync(0xffffffffu, pipe.masked.wait(masks++ & 1, failed));
                        if (!sound) break;
                        acquire_cluster();
                    }
                }
                fence_after_sync();
                if (elected()) {
                    const uint32_t at = ring_at.stage * (W::kBytes / 16);
#pragma unroll
                    for (int k = 0; k < kSliceK / 16; ++k) {
                        const bool sum = more || k > 0;
                        const uint32_t ak = a0 + at + 2 * kAtom / 16 * k;
                        mma_f16<kPair>(pipe_tmem, ak, kHigh, b0 + at + 2 * kAtom / 16 * k, kHigh, kInstruction, sum);
                        if (bias) mma_f16<kPair>(pipe_tmem + BN, ak, kHigh, ones0 + 2 * k, kHigh, kOnesInstruction, sum);
                    }
                    commit<kPair>(&pipe.empty[ring_at.stage]);
                }
                more = true;
                __syncwarp();
                ring_at.next();
            }
            if (!sound) break;
            if (rank == 0 && elected()) commit<kPair>(&pipe.sums_full[0]);
            __syncwarp();
            round ^= 1;
        }
        __syncwarp();
    } else if (warp >= kFirstEpilogueWarp) {
        constexpr int kPart = Shape<BN>::kPart, kChunks = kPart / 32;
        const int quarter = warp % 4, part = (warp - kFirstEpilogueWarp) / 4;
        Stage &stage = stages[warp - kFirstEpilogueWarp];
        unsigned round = 0;
        const auto give_up = [&](long long i) {  // NaN for what the warp still owes
            const float nan = __int_as_float(0x7fffffff);
            for (; i < items; i += workers) {
                const Item it = item_at(i);
                const bool whole = table.slot_begin[it.group + 1] == table.slot_begin[it.group];
                const size_t slot = whole ? (size_t)it.group : (size_t)table.slot_begin[it.group] + it.piece;
                const int first = it.out0 + quarter * 32, in0 = it.in0 + part * kPart, count = min(kPart, p.in_features - in0);
                for (int out = first; out < min(first + 32, p.out_features); ++out) {
                    const size_t at = slot * p.out_features + out;
                    for (int k = lane; k < count && p.grad_weight; k += 32) {
                        if (whole) p.grad_weight[at * p.in_features + in0 + k] = from_f32<T>(nan);
                        else p.slots[at * p.in_features + in0 + k] = nan;
                    }
                    if (lane == 0 && part == 0 && it.in0 == 0 && p.grad_bias) {
                        if (whole) p.grad_bias[at] = from_f32<T>(nan);
                        else p.bias_slots[at] = nan;
                    }
                }
            }
        };
        for (long long i = worker; i < items; i += workers) {
            const Item it = item_at(i);
            const bool none = it.first >= it.last;
            const bool whole = table.slot_begin[it.group + 1] == table.slot_begin[it.group];
            const size_t slot = whole ? (size_t)it.group : (size_t)table.slot_begin[it.group] + it.piece;
            const int out = it.out0 + quarter * 32 + lane;
            if (!none) {
                if (!__all_sync(0xffffffffu, pipe.sums_full[0].wait(round, failed))) {
                    give_up(i);
                    break;
                }
                fence_after_sync();
            }
            const uint32_t address = pipe.tmem + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
            for (int c = 0; c < kChunks; ++c) {
                const int in0 = it.in0 + part * kPart + 32 * c;
                const int count = min(32, p.in_features - in0);
                if (count <= 0 || !p.grad_weight) break;
                uint32_t v[32];
                __syncwarp();
                if (none) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = 0;
                } else {
                    tmem_load(address + part * kPart + 32 * c, v);
                    tmem_load_wait();
                }
                const size_t at = (slot * p.out_features + out) * p.in_features + in0;
                if (whole) {
                    uint32_t packed[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) packed[j] = pack2<T>(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
                    store_rows<kVector>(p.grad_weight + at - (size_t)lane * p.in_features, p.in_features, p.out_features - (out - lane), count,
                                        stage, packed);
                } else if (out >= p.out_features) {
                } else if (kVector) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (4 * j < count)
                            *reinterpret_cast<uint4 *>(p.slots + at + 4 * j) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (j < count) p.slots[at + j] = __uint_as_float(v[j]);
                }
            }
            __syncwarp();
            if (part == 0 && it.in0 == 0 && p.grad_bias) {
                uint32_t sum = 0;
                if (!none) {
                    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(sum) : "r"(address + BN));
                    tmem_load_wait();
                }
                if (out < p.out_features) {
                    const size_t at = slot * p.out_features + out;
                    if (whole) p.grad_bias[at] = from_f32<T>(__uint_as_float(sum));
                    else p.bias_slots[at] = __uint_as_float(sum);
                }
            }
            if (!none) {
                fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (kPair) arrive_at(cluster_address(&pipe.sums_empty[0], 0));
                    else pipe.sums_empty[0].arrive();
                }
                round ^= 1;
            }
        }
    }
    pipeline_end<kPair>(pipe, kColumns, ring_at, any && rank == 0);
}

// ---------------------------------------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found);
        return e == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(p) : nullptr;
    }();
    return fn;
}

// Rows of `line` elements, `pitch` apart, in a box of 64 x box_rows; with `planes` a third axis.  What a box has beyond the
// tensor's extents arrives as zeros.
int make_map(CUtensorMap &map, int dtype, const void *base, long long line, long long rows, long long pitch, int box_rows, long long planes) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) {
        fda::record_cuda_error((int)cudaErrorNotSupported);
        return FDA_ERR_CUDA;
    }
    const cuuint64_t extent[3] = {(cuuint64_t)line, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t stride[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)pitch * 2 * (cuuint64_t)rows};
    const cuuint32_t box[3] = {kLineElements, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
    const CUresult r = encode(&map, dtype == FDA_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                              planes > 0 ? 3 : 2, const_cast<void *>(base), extent, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return FDA_OK;
    fda::record_cuda_error((int)cudaErrorInvalidValue);
    return FDA_ERR_CUDA;
}

bool whole_vectors(const void *base, long long pitch) { return ((uintptr_t)base | (uintptr_t)(pitch * 2)) % 16 == 0; }

int status(cudaError_t e) {
    if (e == cudaSuccess) return FDA_OK;
    fda::record_cuda_error((int)e);
    return FDA_ERR_CUDA;
}

// The attribute belongs to the current device, so every call sets it.  It comes before make_map: on a thread that has not used
// the device yet (autograd's, say) it is also what makes the device's context current, which the driver's encoder needs.
template <typename Kernel>
int allow_shared(Kernel kernel, int bytes) {
    return status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
}

// Whether a block (or pair) of `most` meets the same group and column tile several times in a row; otherwise slices of the weight
// stream with the rows, which waits for no tile to end.
bool weight_stays(long long tiles, long long columns, int groups, int most) {
    return columns <= most / 8 && (groups == 1 || tiles >= 2ll * groups * most);
}

template <int BN>
bool single_keeps(int depth, long long tiles, long long columns, int groups) {
    return ceil_div(depth, kSliceK) * Shape<BN>::kBytesB <= kResidentBytes && weight_stays(tiles, columns, groups, kSms);
}

// Blocks (or pairs) for `tiles`: a multiple of the column tiles where the weight is resident.
unsigned row_grid(long long tiles, long long columns, unsigned most, bool resident) {
    if (tiles <= most) return (unsigned)tiles;
    return resident ? most - most % (unsigned)columns : most;
}

template <typename T, int kMode, int kAct, int BN, bool kVector>
int launch_rows(RowsArgs<T> a, const MmaRows &p, long long units, cudaStream_t st) {
    constexpr int kSmem = Shape<BN>::kStages * Shape<BN>::kBytes + kAtom;
    const auto kernel = linear_rows_mma_kernel<T, kMode, kAct, BN, kVector>;
    if (const int rc = allow_shared(kernel, kSmem)) return rc;
    CUtensorMap map_a, map_w, map_extra;
    const long long rows = (long long)p.g.batch * p.g.rows;
    if (const int rc = make_map(map_a, p.dtype, p.a, a.depth, rows, p.a_pitch, kTileRows, 0)) return rc;
    if (const int rc = make_map(map_w, p.dtype, p.w, p.in_features, p.out_features, p.w_pitch, kMode == kGradX ? kSliceK : BN, p.g.groups))
        return rc;
    if (a.extra && kVector) {
        if (const int rc = make_map(map_extra, p.dtype, p.extra, a.cols, rows, p.extra_pitch, kTileRows, 0)) return rc;
    } else {
        map_extra = map_a;
    }
    const long long tiles = units * ceil_div(a.cols, BN);
    a.resident = single_keeps<BN>(a.depth, tiles, ceil_div(a.cols, BN), p.g.groups);
    if (tiles >= (1ll << 31)) return FDA_ERR_BAD_SHAPE;
    return status(launch_early(kernel, row_grid(tiles, ceil_div(a.cols, BN), kSms, a.resident), Shape<BN>::kThreads, kSmem, st, 1, a, map_a,
                               map_w, map_extra));
}

template <typename T, int kMode, int kAct>
int launch_pair(RowsArgs<T> a, const MmaRows &p, long long units, cudaStream_t st) {
    const auto kernel = linear_rows_pair_kernel<T, kMode, kAct>;
    if (const int rc = allow_shared(kernel, kPairSmem)) return rc;
    CUtensorMap map_a, map_w, map_extra;
    const long long rows = (long long)p.g.batch * p.g.rows;
    if (const int rc = make_map(map_a, p.dtype, p.a, a.depth, rows, p.a_pitch, kTileRows, 0)) return rc;
    if (const int rc = make_map(map_w, p.dtype, p.w, p.in_features, p.out_features, p.w_pitch, kMode == kGradX ? kSliceK : kPairColumns / 2,
                                p.g.groups))
        return rc;
    map_extra = map_a;
    if (a.extra)
        if (const int rc = make_map(map_extra, p.dtype, p.extra, a.cols, rows, p.extra_pitch, 32, 0)) return rc;
    const long long tiles = units * ceil_div(a.cols, kPairColumns);
    a.resident = pair_ring(kMode == kForward || kMode == kPreGrad) - ceil_div(a.depth, kSliceK) * kPairBytesB >= kPairLeastStages * kBytesA &&
                 weight_stays(tiles, ceil_div(a.cols, kPairColumns), p.g.groups, kSms / 2);
    if (tiles >= (1ll << 31)) return FDA_ERR_BAD_SHAPE;
    return status(launch_early(kernel, 2 * row_grid(tiles, ceil_div(a.cols, kPairColumns), kSms / 2, a.resident), kPairThreads, kPairSmem, st,
                               2, a, map_a, map_w, map_extra));
}

// Tiles enough for every pair of blocks, and groups not so short that much of the pairs' units would be empty.
bool pairs_fit(const Groups &g, int cols, long long pair_units) {
    return cols > 128 && pair_units * ceil_div(cols, kPairColumns) >= kSms / 2 && (!g.starts || g.rows / g.groups >= 2 * kPairRows);
}

int pre_grad_unit(const MmaRows &p) {
    const bool vectors = whole_vectors(p.out, p.out_pitch) && whole_vectors(p.extra, p.extra_pitch);
    return vectors && pairs_fit(p.g, p.out_features, most_units(p.g.batch, p.g.rows, p.g.groups, kPairRows, false)) ? kPairRows : kTileRows;
}

template <typename T, int kMode, int kAct>
int rows_of(const MmaRows &p, cudaStream_t st) {
    RowsArgs<T> a;
    a.bias = static_cast<const T *>(p.bias);
    a.extra = static_cast<const T *>(p.extra);
    a.out = static_cast<T *>(p.out);
    a.extra_pitch = (unsigned)p.extra_pitch;
    a.out_pitch = (unsigned)p.out_pitch;
    a.depth = kMode == kGradX ? p.out_features : p.in_features;
    a.cols = kMode == kGradX ? p.in_features : p.out_features;
    a.sums = p.sums;
    a.g = p.g;
    // the widest tile that still gives every SM one
    const long long units = most_units(p.g.batch, p.g.rows, p.g.groups, kTileRows, kMode != kPreGrad && p.g.starts);
    if (!whole_vectors(p.out, p.out_pitch) || (p.extra && !whole_vectors(p.extra, p.extra_pitch))) {
        if (a.cols > 64 && units * ceil_div(a.cols, 128) >= kSms) return launch_rows<T, kMode, kAct, 128, false>(a, p, units, st);
        return launch_rows<T, kMode, kAct, 64, false>(a, p, units, st);
    }
    // Pairs where they pay: extra rows (73728 x 256 x 1024 with a residual 68 us against 86 by single blocks) or weights that a single
    // block cannot keep, for their length or because they change with the tile (149504 x 1024 x 256: 74 against 82); else single
    // blocks, whose epilogues wait for no other (598016 x 256 x 256: 105 against 117).
    const bool extra = kMode == kForward || kMode == kPreGrad;
    const bool pays = extra || !single_keeps<256>(a.depth, units * ceil_div(a.cols, 256), ceil_div(a.cols, 256), p.g.groups);
    const long long pair_units = most_units(p.g.batch, p.g.rows, p.g.groups, kPairRows, kMode != kPreGrad && p.g.starts);
    if (pays && pairs_fit(p.g, a.cols, pair_units)) return launch_pair<T, kMode, kAct>(a, p, pair_units, st);
    if (a.cols > 128 && units * ceil_div(a.cols, 256) >= kSms) return launch_rows<T, kMode, kAct, 256, true>(a, p, units, st);
    if (a.cols > 64 && units * ceil_div(a.cols, 128) >= kSms) return launch_rows<T, kMode, kAct, 128, true>(a, p, units, st);
    return launch_rows<T, kMode, kAct, 64, true>(a, p, units, st);
}

template <typename T, int kMode>
int rows_of(const MmaRows &p, cudaStream_t st) {
    switch (p.activation) {
        case FDA_ACT_NONE: return rows_of<T, kMode, FDA_ACT_NONE>(p, st);
        case FDA_ACT_RELU: return rows_of<T, kMode, FDA_ACT_RELU>(p, st);
        case FDA_ACT_GELU: return rows_of<T, kMode, FDA_ACT_GELU>(p, st);
        case FDA_ACT_GELU_TANH: return rows_of<T, kMode, FDA_ACT_GELU_TANH>(p, st);
        default: return rows_of<T, kMode, FDA_ACT_SILU>(p, st);
    }
}

template <typename T>
int rows_of(int mode, const MmaRows &p, cudaStream_t st) {
    if (mode == kForward) return p.extra ? rows_of<T, kForward>(p, st) : rows_of<T, kForwardPlain>(p, st);
    if (mode == kPreGrad) return rows_of<T, kPreGrad>(p, st);
    return rows_of<T, kGradX, FDA_ACT_NONE>(p, st);
}

template <typename T, int BN, bool kVector, bool kPair = false>
int launch_weight_grad(const MmaWeightGrad &p, cudaStream_t st) {
    WeightGradArgs<T> a;
    a.grad_weight = static_cast<T *>(p.grad_weight);
    a.grad_bias = static_cast<T *>(p.grad_bias);
    a.slots = p.slots;
    a.bias_slots = p.bias_slots;
    a.in_features = p.in_features;
    a.out_features = p.out_features;
    a.piece = p.cut.piece;
    a.g = p.g;
    using W = WeightShape<BN, kPair>;
    constexpr int kSmem = W::kStages * W::kBytes + kOnesBytes + kAtom;
    const auto kernel = linear_weight_grad_mma_kernel<T, BN, kVector, kPair>;
    if (const int rc = allow_shared(kernel, kSmem)) return rc;
    CUtensorMap map_g, map_x;
    const long long rows = (long long)p.g.batch * p.g.rows;
    if (const int rc = make_map(map_g, p.dtype, p.grad, p.out_features, rows, p.grad_pitch, kSliceK, 0)) return rc;
    if (const int rc = make_map(map_x, p.dtype, p.x, p.in_features, rows, p.x_pitch, kSliceK, 0)) return rc;
    const long long items = p.cut.pieces * ceil_div(p.out_features, W::kOutputs) * ceil_div(p.in_features, BN);
    const unsigned workers = (unsigned)std::min<long long>(items, kPair ? kSms / 2 : kSms);
    return status(launch_early(kernel, kPair ? 2 * workers : workers, Shape<BN>::kThreads, kSmem, st, kPair ? 2 : 1, a, map_g, map_x));
}

template <typename T, bool kVector>
int weight_grad_of(const MmaWeightGrad &p, cudaStream_t st) {
    if (p.pair) return launch_weight_grad<T, 256, kVector, true>(p, st);
    switch (p.tile) {
        case 256: return launch_weight_grad<T, 256, kVector>(p, st);
        case 128: return launch_weight_grad<T, 128, kVector>(p, st);
        default: return launch_weight_grad<T, 64, kVector>(p, st);
    }
}

template <typename T>
int weight_grad_of(const MmaWeightGrad &p, cudaStream_t st) {
    return whole_vectors(p.grad_weight, p.in_features) ? weight_grad_of<T, true>(p, st) : weight_grad_of<T, false>(p, st);
}

int timeouts() {
    unsigned int n = 0;
    return cudaMemcpyFromSymbol(&n, g_timeouts, sizeof(n)) == cudaSuccess ? (int)n : -1;
}

}  // namespace

}  // namespace fda_linear

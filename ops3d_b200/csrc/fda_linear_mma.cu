// The linear operators' products on the tensor cores, for 16-bit types: tcgen05.mma over operands that the copy engine brings into
// swizzled shared memory, accumulators in tensor memory, everything after the product from there.
//
// One block per SM walks the output tiles.  Warp 0 keeps a ring of operand slices filled, warp 1 issues the products, warps 2-9
// take finished sums out of tensor memory: accumulators are doubled, so that a tile's epilogue runs beside the next tile's
// products.  Every wait is bounded: a role that waited in vain leaves, the others follow, and the block counts the event.
#include <algorithm>

#include "fda_config.h"
#include "fda_linear_mma.cuh"

namespace fda_linear {

namespace {

constexpr int kTileRows = 128;                     // rows of an accumulator: one per lane of tensor memory
constexpr int kSliceK = 64;                        // contraction indices per slice: one swizzled line
constexpr int kBytesA = kTileRows * kSliceK * 2;
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 32 * (2 + kEpilogueWarps);
constexpr int kRingBytes = 192 * 1024;

template <int BN>
struct Shape {
    static constexpr int kBytesB = BN * kSliceK * 2;
    static constexpr int kBytes = kBytesA + kBytesB;
    static constexpr int kStages = kRingBytes / kBytes;  // 4, 6, 8
};

// Common to both kernels: the ring, the accumulators' barriers, tensor memory.
template <int kStages>
struct Pipeline {
    Barrier full[kStages], empty[kStages], sums_full[2], sums_empty[2], drained;
    uint32_t tmem;
    volatile int failed;
};

template <int kStages>
__device__ __forceinline__ void pipeline_begin(Pipeline<kStages> &p, int columns) {
    if (threadIdx.x == 32) {
        for (int i = 0; i < kStages; ++i) {
            p.full[i].init(1);
            p.empty[i].init(1);
        }
        for (int i = 0; i < 2; ++i) {
            p.sums_full[i].init(1);
            p.sums_empty[i].init(kEpilogueWarps);
        }
        p.drained.init(1);
        p.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (threadIdx.x < 32) tmem_alloc(&p.tmem, columns);
    fence_before_sync();
}

// After every role has left.  In a sound run nothing is in flight any more (the epilogue has waited for every product, and so
// for every copy); after a wait that ran out, copies and products still running are waited for, again with a limit.
template <int kStages>
__device__ __forceinline__ void pipeline_end(Pipeline<kStages> &p, int columns, const Ring<kStages> &issued, bool any) {
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (threadIdx.x == 0 && p.failed) {
        atomicAdd(&g_timeouts, 1u);
        volatile int again = 0;
        if (any)
            for (int i = 0; i < kStages; ++i) {
                // the ring's next place is `issued`: a place before it was last filled in the current round, the others in the one before
                const unsigned parity = i < issued.stage ? issued.round : issued.round ^ 1;
                p.full[i].wait(parity, &again);
            }
    }
    if (threadIdx.x == 32 && p.failed) {
        volatile int again = 0;
        mma_commit(&p.drained);
        p.drained.wait(0, &again);
    }
    __syncthreads();
    if (threadIdx.x < 32) tmem_free(p.tmem, columns);
}

// ---------------------------------------------------------------------------------------------------------------------------
// Products over rows: forward, gradient of the pre-activation, gradient of x
// ---------------------------------------------------------------------------------------------------------------------------
template <typename T>
struct RowsArgs {
    const T *bias, *extra;
    T *out;
    long long extra_pitch, out_pitch;
    int depth, cols;
    int bias_vector, extra_vector, out_vector;  // bytes that the rows' addresses are multiples of: 32, 16 or less
    int activation;
    Groups g;
};

template <typename T, int kMode, int kAct>
__device__ __forceinline__ void finish_chunk(uint32_t (&v)[32], const uint32_t (&bias)[16], const uint32_t (&extra)[16], uint32_t (&out)[16]) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float2 b = unpack2<T>(bias[j]), e = unpack2<T>(extra[j]);
        float lo = __uint_as_float(v[2 * j]) + b.x, hi = __uint_as_float(v[2 * j + 1]) + b.y;
        if (kMode == kForward) {
            lo = activate<kAct>(lo) + e.x;
            hi = activate<kAct>(hi) + e.y;
        } else if (kMode == kPreGrad) {
            lo = activate_backward<kAct>(lo, e.x);
            hi = activate_backward<kAct>(hi, e.y);
        }
        out[j] = pack2<T>(lo, hi);
    }
}

template <typename T, int kMode, int BN>
__global__ void __launch_bounds__(kThreads, 1)
    linear_rows_mma_kernel(const RowsArgs<T> p, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w) {
    constexpr int kStages = Shape<BN>::kStages, kColumns = 2 * BN;
    constexpr bool kWeightMn = kMode == kGradX;  // the weight's lines run along the output columns
    extern __shared__ char dynamic[];
    __shared__ RowTable table;
    __shared__ Pipeline<kStages> pipe;
    char *const ring = reinterpret_cast<char *>(((uintptr_t)dynamic + kAtom - 1) & ~(uintptr_t)(kAtom - 1));
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        prefetch_map(&map_a);
        prefetch_map(&map_w);
    }
    pipeline_begin(pipe, kColumns);
    build_row_table(p.g, kTileRows, kMode != kPreGrad, table);
    __syncthreads();
    fence_after_sync();
    const int column_tiles = (p.cols + BN - 1) / BN, slices = (p.depth + kSliceK - 1) / kSliceK;
    const long long tiles = (long long)table.unit_begin[p.g.groups + 2] * p.g.batch * column_tiles;
    volatile int *const failed = &pipe.failed;
    Ring<kStages> ring_at;
    bool any = false;

    if (warp == 0) {
        if (lane == 0) {
            bool sound = true;
            for (long long tile = blockIdx.x; tile < tiles && sound; tile += gridDim.x) {
                const RowUnit u = row_unit(p.g, table, kTileRows, (unsigned)(tile / column_tiles));
                if (u.group < 0) continue;
                const int col0 = (int)(tile % column_tiles) * BN;
                for (int s = 0; s < slices; ++s) {
                    sound = pipe.empty[ring_at.stage].wait(ring_at.round ^ 1, failed);
                    if (!sound) break;
                    char *a = ring + ring_at.stage * Shape<BN>::kBytes, *b = a + kBytesA;
                    Barrier *bar = &pipe.full[ring_at.stage];
                    bar->arrive_expect(Shape<BN>::kBytes);
                    tma_2d(&map_a, a, bar, s * kSliceK, (int)u.row);
                    if (kWeightMn) {
#pragma unroll
                        for (int i = 0; i < BN / 64; ++i) tma_3d(&map_w, b + i * (64 * kSliceK * 2), bar, col0 + 64 * i, s * kSliceK, u.group);
                    } else {
                        tma_3d(&map_w, b, bar, s * kSliceK, col0, u.group);
                    }
                    ring_at.next();
                    any = true;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t kInstruction = instruction<T>(kTileRows, BN, false, kWeightMn);
            Ring<2> sums;
            bool sound = true;
            for (long long tile = blockIdx.x; tile < tiles && sound; tile += gridDim.x) {
                const RowUnit u = row_unit(p.g, table, kTileRows, (unsigned)(tile / column_tiles));
                if (u.group < 0) continue;
                sound = pipe.sums_empty[sums.stage].wait(sums.round ^ 1, failed);
                if (!sound) break;
                fence_after_sync();
                const uint32_t d = pipe.tmem + sums.stage * BN;
                for (int s = 0; s < slices; ++s) {
                    sound = pipe.full[ring_at.stage].wait(ring_at.round, failed);
                    if (!sound) break;
                    fence_after_sync();
                    const char *a = ring + ring_at.stage * Shape<BN>::kBytes, *b = a + kBytesA;
#pragma unroll
                    for (int k = 0; k < kSliceK / 16; ++k) {
                        const uint64_t da = operand(a + 32 * k, 16, kAtom);
                        const uint64_t db = kWeightMn ? operand(b + 2 * kAtom * k, 64 * kSliceK * 2, kAtom) : operand(b + 32 * k, 16, kAtom);
                        mma_f16(d, da, db, kInstruction, s > 0 || k > 0);
                    }
                    mma_commit(&pipe.empty[ring_at.stage]);
                    ring_at.next();
                }
                if (!sound) break;
                mma_commit(&pipe.sums_full[sums.stage]);
                sums.next();
            }
        }
        __syncwarp();
    } else {
        // Each warp owns the 32 lanes of tensor memory that its number allows it, and half of the columns.
        constexpr int kChunks = BN / 64;  // of 32 columns
        const int quarter = warp % 4, half = (warp - 2) / 4;
        Ring<2> sums;
        for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            const RowUnit u = row_unit(p.g, table, kTileRows, (unsigned)(tile / column_tiles));
            const int col0 = (int)(tile % column_tiles) * BN + half * (BN / 2);
            const int r = quarter * 32 + lane;
            const bool mine = r < u.count;
            const T *extra_row = p.extra ? p.extra + (size_t)(u.row + r) * p.extra_pitch + col0 : nullptr;
            T *out_row = p.out + (size_t)(u.row + r) * p.out_pitch + col0;
            if (u.group >= 0) {
                if (!__all_sync(0xffffffffu, pipe.sums_full[sums.stage].wait(sums.round, failed))) break;
                fence_after_sync();
            }
            const uint32_t address = pipe.tmem + sums.stage * BN + half * (BN / 2) + ((uint32_t)(quarter * 32) << 16);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int count = min(32, p.cols - col0 - 32 * c);
                if (count <= 0) break;
                uint32_t v[32], extra[16], bias[16], out[16];
                __syncwarp();
                if (u.group >= 0) {
                    tmem_load(address + 32 * c, v);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = 0;
                }
                if (kMode != kGradX && extra_row && mine) {
                    load_row(extra_row + 32 * c, count, p.extra_vector, extra);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) extra[j] = 0;
                }
                if (kMode != kGradX && p.bias && u.group >= 0) {
                    load_row(p.bias + (size_t)u.group * p.cols + col0 + 32 * c, count, p.bias_vector, bias);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) bias[j] = 0;
                }
                tmem_load_wait();
                switch (kMode == kGradX || u.group < 0 ? FDA_ACT_NONE : p.activation) {
                    case FDA_ACT_NONE: finish_chunk<T, kMode, FDA_ACT_NONE>(v, bias, extra, out); break;
                    case FDA_ACT_RELU: finish_chunk<T, kMode, FDA_ACT_RELU>(v, bias, extra, out); break;
                    case FDA_ACT_GELU: finish_chunk<T, kMode, FDA_ACT_GELU>(v, bias, extra, out); break;
                    case FDA_ACT_GELU_TANH: finish_chunk<T, kMode, FDA_ACT_GELU_TANH>(v, bias, extra, out); break;
                    default: finish_chunk<T, kMode, FDA_ACT_SILU>(v, bias, extra, out); break;
                }
                if (mine) store_row(out_row + 32 * c, count, p.out_vector, out);
            }
            if (u.group >= 0) {
                fence_before_sync();
                __syncwarp();
                if (lane == 0) pipe.sums_empty[sums.stage].arrive();
                sums.next();
            }
        }
    }
    pipeline_end(pipe, kColumns, ring_at, any);
}

// ---------------------------------------------------------------------------------------------------------------------------
// Gradient of the weight
// ---------------------------------------------------------------------------------------------------------------------------
// An accumulator holds 128 outputs x BN inputs of g^T x over a piece of a group's rows; both operands have their lines across
// the contraction.  The bias's gradient is one more narrow product of the same g with ones.
constexpr int kOnesColumns = 16;
constexpr int kOnesBytes = kOnesColumns * kSliceK * 2;

template <typename T>
struct WeightGradArgs {
    T *grad_weight, *grad_bias;
    float *slots, *bias_slots;
    int in_features, out_features;
    int piece;
    bool weight_vector;  // rows of grad_weight and of the slots start on 16-byte boundaries
    Groups g;
};

template <typename T, int BN>
__global__ void __launch_bounds__(kThreads, 1)
    linear_weight_grad_mma_kernel(const WeightGradArgs<T> p, const __grid_constant__ CUtensorMap map_g,
                                  const __grid_constant__ CUtensorMap map_x) {
    constexpr int kStages = Shape<BN>::kStages, kColumns = 512;
    extern __shared__ char dynamic[];
    __shared__ PieceTable table;
    __shared__ Pipeline<kStages> pipe;
    char *const ring = reinterpret_cast<char *>(((uintptr_t)dynamic + kAtom - 1) & ~(uintptr_t)(kAtom - 1));
    char *const ones = ring + kStages * Shape<BN>::kBytes;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        prefetch_map(&map_g);
        prefetch_map(&map_x);
    }
    pipeline_begin(pipe, kColumns);
    for (int i = threadIdx.x; i < kOnesBytes / 4; i += kThreads) reinterpret_cast<uint32_t *>(ones)[i] = pack2<T>(1.f, 1.f);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    build_piece_table(p.g, kSliceK, p.piece, table);
    __syncthreads();
    fence_after_sync();
    const int out_tiles = (p.out_features + kTileRows - 1) / kTileRows, in_tiles = (p.in_features + BN - 1) / BN;
    const int per_piece = out_tiles * in_tiles;
    const long long items = (long long)table.piece_begin[p.g.groups] * per_piece;
    volatile int *const failed = &pipe.failed;
    Ring<kStages> ring_at;
    bool any = false;

    struct Item {
        int group, piece, out0, in0, first, last;  // blocks first .. last - 1 of the group
    };
    const auto item_at = [&](long long i) {
        Item it;
        const int piece = (int)(i / per_piece), t = (int)(i % per_piece);
        it.group = find_section(table.piece_begin, p.g.groups, piece);
        it.piece = piece - table.piece_begin[it.group];
        it.out0 = (t / in_tiles) * kTileRows;
        it.in0 = (t % in_tiles) * BN;
        it.first = it.piece * p.piece;
        it.last = min(group_blocks(p.g, table.start, it.group, kSliceK), it.first + p.piece);
        return it;
    };

    if (warp == 0) {
        if (lane == 0) {
            bool sound = true;
            for (long long i = blockIdx.x; i < items && sound; i += gridDim.x) {
                const Item it = item_at(i);
                for (int j = it.first; j < it.last; ++j) {
                    long long row;
                    int count;
                    block_rows(p.g, table.start, it.group, kSliceK, j, row, count);
                    sound = pipe.empty[ring_at.stage].wait(ring_at.round ^ 1, failed);
                    if (!sound) break;
                    char *a = ring + ring_at.stage * Shape<BN>::kBytes, *b = a + kBytesA;
                    Barrier *bar = &pipe.full[ring_at.stage];
                    bar->arrive_expect(Shape<BN>::kBytes);
#pragma unroll
                    for (int k = 0; k < kTileRows / 64; ++k) tma_2d(&map_g, a + k * (64 * kSliceK * 2), bar, it.out0 + 64 * k, (int)row);
#pragma unroll
                    for (int k = 0; k < BN / 64; ++k) tma_2d(&map_x, b + k * (64 * kSliceK * 2), bar, it.in0 + 64 * k, (int)row);
                    ring_at.next();
                    any = true;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        constexpr uint32_t kInstruction = instruction<T>(kTileRows, BN, true, true);
        constexpr uint32_t kOnesInstruction = instruction<T>(kTileRows, kOnesColumns, true, false);
        unsigned round = 0;
        bool sound = true;
        for (long long i = blockIdx.x; i < items && sound; i += gridDim.x) {
            const Item it = item_at(i);
            if (it.first >= it.last) continue;
            const bool bias = it.in0 == 0 && p.grad_bias;
            sound = __all_sync(0xffffffffu, pipe.sums_empty[0].wait(round ^ 1, failed));
            if (!sound) break;
            fence_after_sync();
            for (int j = it.first; j < it.last; ++j) {
                long long row;
                int count;
                block_rows(p.g, table.start, it.group, kSliceK, j, row, count);
                sound = __all_sync(0xffffffffu, pipe.full[ring_at.stage].wait(ring_at.round, failed));
                if (!sound) break;
                char *a = ring + ring_at.stage * Shape<BN>::kBytes, *b = a + kBytesA;
                if (count < kSliceK) {
                    // lines of the next group's rows (or of nothing): out of both operands, for 0 times NaN is NaN.  A line of 128
                    // bytes is one row of a block of 64 columns, wherever the swizzle has its parts.
                    constexpr int kBlocks = kTileRows / 64 + BN / 64;
                    const int lines = kSliceK - count;
                    for (int l = lane; l < kBlocks * lines * 8; l += 32) {
                        const int block = l / (lines * 8), rest = l - block * lines * 8;
                        reinterpret_cast<uint4 *>(a + block * (64 * kSliceK * 2) + count * 128)[rest] = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                fence_after_sync();
                if (lane == 0) {
#pragma unroll
                    for (int k = 0; k < kSliceK / 16; ++k) {
                        const uint64_t da = operand(a + 2 * kAtom * k, 64 * kSliceK * 2, kAtom);
                        mma_f16(pipe.tmem, da, operand(b + 2 * kAtom * k, 64 * kSliceK * 2, kAtom), kInstruction, j > it.first || k > 0);
                        if (bias) mma_f16(pipe.tmem + BN, da, operand(ones + 32 * k, 16, kAtom), kOnesInstruction, j > it.first || k > 0);
                    }
                    mma_commit(&pipe.empty[ring_at.stage]);
                }
                __syncwarp();
                ring_at.next();
            }
            if (!sound) break;
            if (lane == 0) mma_commit(&pipe.sums_full[0]);
            __syncwarp();
            round ^= 1;
        }
        __syncwarp();
    } else {
        constexpr int kChunks = BN / 64;
        const int quarter = warp % 4, half = (warp - 2) / 4;
        unsigned round = 0;
        for (long long i = blockIdx.x; i < items; i += gridDim.x) {
            const Item it = item_at(i);
            const bool none = it.first >= it.last;
            const bool whole = table.slot_begin[it.group + 1] == table.slot_begin[it.group];
            const size_t slot = whole ? (size_t)it.group : (size_t)table.slot_begin[it.group] + it.piece;
            const int out = it.out0 + quarter * 32 + lane;
            if (!none) {
                if (!__all_sync(0xffffffffu, pipe.sums_full[0].wait(round, failed))) break;
                fence_after_sync();
            }
            const uint32_t address = pipe.tmem + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
            for (int c = 0; c < kChunks; ++c) {
                const int in0 = it.in0 + half * (BN / 2) + 32 * c;
                const int count = min(32, p.in_features - in0);
                if (count <= 0 || !p.grad_weight) break;
                uint32_t v[32];
                __syncwarp();
                if (none) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = 0;
                } else {
                    tmem_load(address + half * (BN / 2) + 32 * c, v);
                    tmem_load_wait();
                }
                const size_t at = (slot * p.out_features + out) * p.in_features + in0;
                if (out >= p.out_features) {
                } else if (whole) {
                    uint32_t packed[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) packed[j] = pack2<T>(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
                    store_row(p.grad_weight + at, count, p.weight_vector ? 16 : 2, packed);
                } else if (p.weight_vector) {
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
            if (half == 0 && it.in0 == 0 && p.grad_bias) {
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
                if (lane == 0) pipe.sums_empty[0].arrive();
                round ^= 1;
            }
        }
    }
    pipeline_end(pipe, kColumns, ring_at, any);
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

int vector_bytes(const void *base, long long pitch_elements) {
    const uintptr_t bits = (uintptr_t)base | (uintptr_t)(pitch_elements * 2);
    return bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : 2;
}

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

template <typename T, int kMode, int BN>
int launch_rows(const RowsArgs<T> &a, const MmaRows &p, long long units, cudaStream_t st) {
    constexpr int kSmem = Shape<BN>::kStages * Shape<BN>::kBytes + kAtom;
    const auto kernel = linear_rows_mma_kernel<T, kMode, BN>;
    if (const int rc = allow_shared(kernel, kSmem)) return rc;
    CUtensorMap map_a, map_w;
    const long long rows = (long long)p.g.batch * p.g.rows;
    if (const int rc = make_map(map_a, p.dtype, p.a, a.depth, rows, p.a_pitch, kTileRows, 0)) return rc;
    if (const int rc = make_map(map_w, p.dtype, p.w, p.in_features, p.out_features, p.w_pitch, kMode == kGradX ? kSliceK : BN, p.g.groups))
        return rc;
    const long long tiles = units * ceil_div(a.cols, BN);
    kernel<<<(unsigned)std::min<long long>(tiles, kSms), kThreads, kSmem, st>>>(a, map_a, map_w);
    return status(cudaGetLastError());
}

template <typename T, int kMode>
int rows_of(const MmaRows &p, cudaStream_t st) {
    RowsArgs<T> a;
    a.bias = static_cast<const T *>(p.bias);
    a.extra = static_cast<const T *>(p.extra);
    a.out = static_cast<T *>(p.out);
    a.extra_pitch = p.extra_pitch;
    a.out_pitch = p.out_pitch;
    a.depth = kMode == kGradX ? p.out_features : p.in_features;
    a.cols = kMode == kGradX ? p.in_features : p.out_features;
    a.bias_vector = vector_bytes(p.bias, a.cols);
    a.extra_vector = vector_bytes(p.extra, p.extra_pitch);
    a.out_vector = vector_bytes(p.out, p.out_pitch);
    a.activation = p.activation;
    a.g = p.g;
    // the widest tile that still gives every SM one
    const long long units = most_units(p.g.batch, p.g.rows, p.g.groups, kTileRows, kMode != kPreGrad && p.g.starts);
    if (a.cols > 128 && units * ceil_div(a.cols, 256) >= kSms) return launch_rows<T, kMode, 256>(a, p, units, st);
    if (a.cols > 64 && units * ceil_div(a.cols, 128) >= kSms) return launch_rows<T, kMode, 128>(a, p, units, st);
    return launch_rows<T, kMode, 64>(a, p, units, st);
}

template <typename T>
int rows_of(int mode, const MmaRows &p, cudaStream_t st) {
    if (mode == kForward) return rows_of<T, kForward>(p, st);
    if (mode == kPreGrad) return rows_of<T, kPreGrad>(p, st);
    return rows_of<T, kGradX>(p, st);
}

int weight_tile(int in_features) { return in_features > 128 ? 256 : in_features > 64 ? 128 : 64; }

template <typename T, int BN>
int launch_weight_grad(const MmaWeightGrad &p, cudaStream_t st) {
    WeightGradArgs<T> a;
    a.grad_weight = static_cast<T *>(p.grad_weight);
    a.grad_bias = static_cast<T *>(p.grad_bias);
    a.slots = p.slots;
    a.bias_slots = p.bias_slots;
    a.in_features = p.in_features;
    a.out_features = p.out_features;
    a.piece = p.cut.piece;
    a.weight_vector = vector_bytes(p.grad_weight, p.in_features) >= 16;
    a.g = p.g;
    constexpr int kSmem = Shape<BN>::kStages * Shape<BN>::kBytes + kOnesBytes + kAtom;
    const auto kernel = linear_weight_grad_mma_kernel<T, BN>;
    if (const int rc = allow_shared(kernel, kSmem)) return rc;
    CUtensorMap map_g, map_x;
    const long long rows = (long long)p.g.batch * p.g.rows;
    if (const int rc = make_map(map_g, p.dtype, p.grad, p.out_features, rows, p.grad_pitch, kSliceK, 0)) return rc;
    if (const int rc = make_map(map_x, p.dtype, p.x, p.in_features, rows, p.x_pitch, kSliceK, 0)) return rc;
    const long long items = p.cut.pieces * ceil_div(p.out_features, kTileRows) * ceil_div(p.in_features, BN);
    kernel<<<(unsigned)std::min<long long>(items, kSms), kThreads, kSmem, st>>>(a, map_g, map_x);
    return status(cudaGetLastError());
}

template <typename T>
int weight_grad_of(const MmaWeightGrad &p, cudaStream_t st) {
    switch (weight_tile(p.in_features)) {
        case 256: return launch_weight_grad<T, 256>(p, st);
        case 128: return launch_weight_grad<T, 128>(p, st);
        default: return launch_weight_grad<T, 64>(p, st);
    }
}

}  // namespace

int mma_rows(int mode, const MmaRows &p, cudaStream_t st) {
    return p.dtype == FDA_DTYPE_F16 ? rows_of<__half>(mode, p, st) : rows_of<__nv_bfloat16>(mode, p, st);
}

Cut mma_cut(int batch, int rows, int groups, int in_features, int out_features) {
    return cut_rows(batch, rows, groups, ceil_div(out_features, kTileRows) * ceil_div(in_features, weight_tile(in_features)), kSliceK, 8);
}

int mma_weight_grad(const MmaWeightGrad &p, cudaStream_t st) {
    return p.dtype == FDA_DTYPE_F16 ? weight_grad_of<__half>(p, st) : weight_grad_of<__nv_bfloat16>(p, st);
}

int mma_timeouts() {
    unsigned int n = 0;
    if (cudaMemcpyFromSymbol(&n, g_timeouts, sizeof(n)) != cudaSuccess) return -1;
    return (int)n;
}

}  // namespace fda_linear

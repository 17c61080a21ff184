// linear_tc.cu — C = A B^T on the tensor cores for 16-bit operands, with the linear layer's epilogue.
//
// Two CTAs of a cluster make one tile of 256 x TN values: each holds 128 rows of A and half of B's rows in
// shared memory (TMA, 64 values of K a stage), the leader's warp 9 issues products over both (cta_group::2),
// and each CTA has the sums of its own 128 rows in its tensor memory, twice, so that one tile's epilogue runs
// under the next one's products. Rows of an operand may run along K or across it (the gradients' products
// read weight, x and v_z across): the tensor cores take either from shared memory.
//
//   warps 0-7: epilogue, a thread a row and half of the columns
//   warp 8:    asks for the CTA's part of the tiles, on the leader's barriers
//   warp 9:    allocates tensor memory; in the leader issues the products
#include <cuda.h>

#include <algorithm>

#include "sx_linear.h"
#include "sx_tcgen05.cuh"

namespace sx {

__device__ uint32_t g_linear_status;

uint32_t linear_status() {
    uint32_t st = 0;
    const uint32_t zero = 0;
    cuda_check(cudaDeviceSynchronize(), "linear_status");
    cuda_check(cudaMemcpyFromSymbol(&st, g_linear_status, sizeof(st)), "linear_status");
    if (st) cuda_check(cudaMemcpyToSymbol(g_linear_status, &zero, sizeof(zero)), "linear_status");
    return st;
}

namespace {

constexpr int kRows = 128, kTileM = 2 * kRows, kDepth = 64;
constexpr int kPanel = kDepth * 128;  // bytes of 64 values of K for 64 rows that lie across K
constexpr int kEpilogueWarps = 8, kThreads = 320;
constexpr long long kLanding = 4000000;  // cycles in which any copy has landed (2 ms)

struct LinearMaps {
    CUtensorMap a, b;
};

template <int TN>
struct Smem {
    static constexpr int kA = kRows * 128, kB = TN / 2 * 128, kStage = kA + kB;
    static constexpr int kStages = TN == 256 ? 6 : 8;
    static constexpr int kBias = kStages * kStage;                     // [warps][TN / 2] floats
    static constexpr int kTurn = kBias + kEpilogueWarps * TN / 2 * 4;  // [warps][32][17] floats
    static constexpr int kBars = kTurn + kEpilogueWarps * 32 * 17 * 4;
    static constexpr int kBytes = kBars + (2 * kStages + 5) * 8 + 16;
    static_assert(kBytes <= 232448, "shared memory");
};

template <int STAGES>
struct Bars {
    uint32_t base;
    __device__ uint32_t full(int s) const { return base + s * 8; }                     // the leader's
    __device__ uint32_t empty(int s) const { return base + (STAGES + s) * 8; }         // each CTA's
    __device__ uint32_t acc_full(int i) const { return base + (2 * STAGES + i) * 8; }  // each CTA's
    __device__ uint32_t acc_empty(int i) const { return base + (2 * STAGES + 2 + i) * 8; }  // the leader's
    __device__ uint32_t drained() const { return base + (2 * STAGES + 4) * 8; }
};

// ---- what a pair of CTAs needs ----
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {  // the same place in a CTA of the cluster
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void arrive_in(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// A box of a 2-axis map into this CTA's shared memory, counted on a barrier of either CTA.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t cluster_bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(cluster_bar)
        : "memory");
}
__device__ __forceinline__ void pair_alloc(uint32_t to_smem, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to_smem), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_free(uint32_t tmem, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
__device__ __forceinline__ void pair_mma(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(shape), "r"(static_cast<uint32_t>(add)), "r"(one)
        : "memory");
}
// Arrives on the barrier at this place in both CTAs once every product issued before is complete.
__device__ __forceinline__ void pair_commit(uint32_t one, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t.reg .b16 m;\n\tsetp.ne.u32 q, %1, 0;\n\tmov.b16 m, 3;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}" ::"r"(bar), "r"(one)
        : "memory");
}
// 256 x n product of T with 32-bit sums; whether the operands' rows in shared memory run across K.
template <typename T>
__host__ __device__ constexpr uint32_t pair_shape(int n, bool a_across, bool b_across) {
    return 1u << 4 | tc::Format<T>::code << 7 | tc::Format<T>::code << 10 | (a_across ? 1u << 15 : 0u) | (b_across ? 1u << 16 : 0u) |
           static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(kTileM >> 4) << 24;
}

// The columns that a tile's products have: half of them where the product's last ones need no more.
template <int TN>
__device__ __forceinline__ int columns(const LinearProduct& p, const LinearTile& tile) {
    if constexpr (TN == 256) return p.n - static_cast<int64_t>(tile.n) * TN <= TN / 2 ? TN / 2 : TN;
    return TN;
}

// ---- loads ----
template <int ROWS, bool ACROSS>  // ROWS rows from `row` and 64 values of K from `k`
__device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap* map, int row, int k, uint32_t bar) {
    if constexpr (ACROSS) {
#pragma unroll
        for (int i = 0; i < ROWS / 64; ++i) load_box(dst + i * kPanel, map, row + i * 64, k, bar);
    } else {
        load_box(dst, map, k, row, bar);
    }
}

// ---- epilogue ----
template <typename T>
__device__ __forceinline__ void load_values(const T* p, bool wide, float (&x)[16]) {  // 16-byte aligned, `wide`: 32
    uint32_t w[8];
    if (wide) {
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : SX_R8(w, 0) : "l"(p) : "memory");
    } else {
        *reinterpret_cast<uint4*>(w) = reinterpret_cast<const uint4*>(p)[0];
        *reinterpret_cast<uint4*>(w + 4) = reinterpret_cast<const uint4*>(p)[1];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const auto v = *reinterpret_cast<const Pack<T, 2>*>(&w[i]);
        x[2 * i] = to_f32(v.v[0]), x[2 * i + 1] = to_f32(v.v[1]);
    }
}
template <typename T>
__device__ __forceinline__ void store_values(T* p, bool wide, const float (&x)[16]) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = tc::pack2<T>(x[2 * i], x[2 * i + 1]);
    if (wide) {
        tc::store32(p, w);
    } else {
        reinterpret_cast<uint4*>(p)[0] = *reinterpret_cast<uint4*>(w);
        reinterpret_cast<uint4*>(p)[1] = *reinterpret_cast<uint4*>(w + 4);
    }
}
template <int ACT>
__device__ __forceinline__ void activate(float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) act_pair<ACT>(x[i], x[i + 1]);
}

// How the rows of y, pre and residual are reached: 32 or 16 bytes at a time, or value by value.
struct Reach {
    bool vectors, wide;
};

// 16 columns of the thread's row, whole, at addresses of 16 bytes.
template <typename T>
__device__ __forceinline__ void finish_row(const LinearProduct& p, Reach reach, int64_t row, int64_t col, float (&x)[16]) {
    if (p.pre) store_values(static_cast<T*>(p.pre) + row * p.pre_stride + col, reach.wide, x);
    switch (p.act) {
        case SXCUDA_ACT_RELU: activate<SXCUDA_ACT_RELU>(x); break;
        case SXCUDA_ACT_SILU: activate<SXCUDA_ACT_SILU>(x); break;
        case SXCUDA_ACT_GELU: activate<SXCUDA_ACT_GELU>(x); break;
        case SXCUDA_ACT_GELU_TANH: activate<SXCUDA_ACT_GELU_TANH>(x); break;
        default: break;
    }
    if (p.residual) {
        float r[16];
        load_values(static_cast<const T*>(p.residual) + row * p.residual_stride + col, reach.wide, r);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] += r[i];
    }
    store_values(static_cast<T*>(p.y) + row * p.y_stride + col, reach.wide, x);
}

// 16 columns of the warp's 32 rows, value by value: turned in shared memory, so that lanes stand side by side
// in a row.
template <typename T>
__device__ __forceinline__ void finish_turned(const LinearProduct& p, float (*turn)[17], int64_t row0, int64_t col0, int lane, const float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) turn[lane][i] = x[i];
    __syncwarp();
    const int64_t col = col0 + lane % 16;
    for (int i = lane / 16; i < 32; i += 2) {
        const int64_t row = row0 + i;
        if (row >= p.m || col >= p.n) continue;
        const float z = turn[i][lane % 16];
        if (p.pre) static_cast<T*>(p.pre)[row * p.pre_stride + col] = from_f32<T>(z);
        float y = act_of<T>(p.act, z);
        if (p.residual) y += to_f32(static_cast<const T*>(p.residual)[row * p.residual_stride + col]);
        static_cast<T*>(p.y)[row * p.y_stride + col] = from_f32<T>(y);
    }
    __syncwarp();
}

// 32 columns of a tile's row: the epilogue, or what is left of a part of the tile.
template <typename T>
__device__ __forceinline__ void finish(const LinearProduct& p, Reach reach, const float* bias, float (*turn)[17], int64_t row, int64_t col0,
                                       int lane, const uint32_t (&r)[32]) {
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
        const int64_t col = col0 + h;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const float4 b = *reinterpret_cast<const float4*>(bias + h + i);
            x[i] = __uint_as_float(r[h + i]) + b.x, x[i + 1] = __uint_as_float(r[h + i + 1]) + b.y;
            x[i + 2] = __uint_as_float(r[h + i + 2]) + b.z, x[i + 3] = __uint_as_float(r[h + i + 3]) + b.w;
        }
        if (reach.vectors && col + 16 <= p.n) {
            if (row < p.m) finish_row<T>(p, reach, row, col, x);
        } else if (col < p.n) {
            finish_turned<T>(p, turn, row - lane, col, lane, x);
        }
    }
}
__device__ __forceinline__ void leave(const LinearProduct& p, int slot, int row, int col, uint32_t (&r)[32]) {
    float* part = p.parts + slot * p.plan.slot_values() + row * p.plan.tile_n + col;
#pragma unroll
    for (int i = 0; i < 4; ++i) tc::store32(part + 8 * i, *reinterpret_cast<uint32_t(*)[8]>(r + 8 * i));
}

template <typename T, int TN, bool A_ACROSS, bool B_ACROSS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    linear_tc_kernel(const __grid_constant__ LinearProduct p, const __grid_constant__ LinearMaps maps, Reach reach) {
    using S = Smem<TN>;
    constexpr int kStages = S::kStages;
    extern __shared__ __align__(1024) uint8_t smem[];
    const Bars<kStages> bars{tc::smem_addr(smem) + S::kBars};
    volatile uint32_t* failed = reinterpret_cast<uint32_t*>(smem + S::kBars + (2 * kStages + 5) * 8);
    uint32_t* tmem_at = const_cast<uint32_t*>(failed) + 1;
    const uint32_t base = tc::smem_addr(smem);
    const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1;
    LinearWalk walk(p.plan, blockIdx.x / 2);
    LinearPiece piece;
    int asked = 0;  // stages that this warp has asked for

    if (warp == 8 && lane == 0) {
        tc::prefetch_map(&maps.a);
        tc::prefetch_map(&maps.b);
        for (int s = 0; s < kStages; ++s) tc::bar_init(bars.full(s), 1), tc::bar_init(bars.empty(s), 1);
        for (int i = 0; i < 2; ++i) tc::bar_init(bars.acc_full(i), 1), tc::bar_init(bars.acc_empty(i), 2 * kEpilogueWarps);
        tc::bar_init(bars.drained(), 1);
        tc::bar_init_fence();
        *failed = 0;
    }
    __syncwarp();
    if (warp == 9) pair_alloc(tc::smem_addr(tmem_at), 2 * TN);
    tc::fence_before();
    __syncthreads();
    cluster_sync();
    tc::fence_after();
    const uint32_t tmem = __shfl_sync(kFullMask, *tmem_at, 0);

    if (warp == 8) {
        int slot = 0;
        uint32_t parity = 0;
        bool ok = true;
        while (ok && walk.next(p.plan, piece)) {
            const LinearTile tile = linear_tile(p.plan, piece.tile);
            const int m = tile.m * kTileM + static_cast<int>(rank) * kRows, n = tile.n * TN + static_cast<int>(rank) * (columns<TN>(p, tile) / 2);
            for (int k = piece.k0; k < piece.k1; ++k) {
                if (asked >= kStages) ok = tc::bar_wait(bars.empty(slot), parity ^ 1, failed);
                if (!ok) break;
                if (lane == 0) {
                    const uint32_t to = base + slot * S::kStage, bar = in_cta(bars.full(slot), 0);
                    if (rank == 0) tc::bar_expect(bars.full(slot), 2 * S::kStage);
                    load_operand<kRows, A_ACROSS>(to, &maps.a, m, k * kDepth, bar);
                    load_operand<TN / 2, B_ACROSS>(to + S::kA, &maps.b, n, k * kDepth, bar);
                }
                __syncwarp();
                ++asked;
                if (++slot == kStages) slot = 0, parity ^= 1;
            }
        }
        // the products' last arrivals, without which this CTA's memory must not go
        for (int i = max(0, asked - kStages); ok && i < asked; ++i) ok = tc::bar_wait(bars.empty(i % kStages), (i / kStages) & 1, failed);
    } else if (warp == 9) {
        if (rank == 0) {
            const uint32_t one = tc::elect();
            int slot = 0, count = 0;
            uint32_t parity = 0;
            bool ok = true;
            for (; ok && walk.next(p.plan, piece); ++count) {
                const uint32_t d = tmem + (count & 1) * TN;
                const uint32_t shape = pair_shape<T>(columns<TN>(p, linear_tile(p.plan, piece.tile)), A_ACROSS, B_ACROSS);
                if (count >= 2) ok = tc::bar_wait(bars.acc_empty(count & 1), ((count >> 1) & 1) ^ 1, failed);
                tc::fence_after();
                for (int k = piece.k0; ok && k < piece.k1; ++k) {
                    ok = tc::bar_wait(bars.full(slot), parity, failed);
                    if (!ok) break;
                    const uint32_t a = base + slot * S::kStage, b = a + S::kA;
#pragma unroll
                    for (int i = 0; i < kDepth / 16; ++i)
                        pair_mma(one, d, A_ACROSS ? tc::operand(a + i * 2048, kPanel) : tc::operand(a + i * 32, 16),
                                 B_ACROSS ? tc::operand(b + i * 2048, kPanel) : tc::operand(b + i * 32, 16), shape, k > piece.k0 || i > 0);
                    pair_commit(one, bars.empty(slot));
                    if (++slot == kStages) slot = 0, parity ^= 1;
                }
                if (ok) pair_commit(one, bars.acc_full(count & 1));
            }
        }
    } else {
        constexpr int kCols = TN / 2;
        const int half = warp >> 2, in_tile = static_cast<int>(rank) * kRows + (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        float* bias = reinterpret_cast<float*>(smem + S::kBias) + warp * kCols;
        float(*turn)[17] = reinterpret_cast<float(*)[17]>(smem + S::kTurn) + warp * 32;
        bool ok = true;
        for (int count = 0; ok && walk.next(p.plan, piece); ++count) {
            const LinearTile tile = linear_tile(p.plan, piece.tile);
            const int64_t row = static_cast<int64_t>(tile.m) * kTileM + in_tile, n0 = static_cast<int64_t>(tile.n) * TN + half * kCols;
            __syncwarp();
            for (int i = lane; i < kCols; i += 32) bias[i] = n0 + i < p.n ? linear_param(p.bias, p.bias_dtype, n0 + i) : 0.f;
            __syncwarp();
            ok = tc::bar_wait(bars.acc_full(count & 1), (count >> 1) & 1, failed);
            if (!ok) break;
            tc::fence_after();
            const uint32_t at = tmem + lanes + (count & 1) * TN + half * kCols;
#pragma unroll 1
            for (int c = 0; c < kCols; c += 32) {
                uint32_t r[32];
                __syncwarp();
                tc::tmem_load32(r, at + c);
                tc::wait_ld(r);
                if (c + 32 == kCols) {
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_in(in_cta(bars.acc_empty(count & 1), 0));
                }
                if (n0 + c >= p.n) continue;  // the same for the whole warp
                if (piece.slot < 0) finish<T>(p, reach, bias + c, turn, row, n0 + c, lane, r);
                else if (row < p.m) leave(p, piece.slot, in_tile, half * kCols + c, r);
            }
        }
    }

    tc::fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *failed) {
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(in_cta(tc::smem_addr(const_cast<uint32_t*>(failed)), rank ^ 1)), "r"(1) : "memory");
    }
    cluster_sync();
    if (*failed) {  // nothing may land in the pair's memory after it has gone
        if (warp == 8) {
            if (rank == 0)
                for (int i = max(0, asked - kStages); i < asked; ++i) tc::bar_drain(bars.full(i % kStages), (i / kStages) & 1);
            for (const long long start = clock64(); clock64() - start < kLanding;) {
            }
        } else if (warp == 9 && rank == 0) {
            const uint32_t one = tc::elect();
            asm volatile(
                "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
                "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bars.drained()), "r"(one)
                : "memory");
            tc::bar_drain(bars.drained(), 0);
        }
        __syncthreads();
        cluster_sync();
        if (threadIdx.x == 0) atomicOr(&g_linear_status, 1u);
    }
    if (warp == 9) pair_free(tmem, 2 * TN);
}

// ---- host ----
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
    static const EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        cuda_check(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found), "cuTensorMapEncodeTiled");
        if (!p || found != cudaDriverEntryPointSuccess) throw RuntimeError("linear: the driver has no cuTensorMapEncodeTiled");
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// The operand's memory as [outer][inner], inner contiguous: K is the inner axis, or the rows are (across). Boxes
// of 64 inner values; what lies beyond the operand reads as zero.
CUtensorMap make_map(const LinearOperand& o, int64_t rows, int64_t k, int box_rows, int32_t dtype) {
    CUtensorMap m;
    const int64_t inner = o.across ? rows : k, outer = o.across ? k : rows;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
    // one row may have any stride: a length that fits stands for it
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(2 * (outer > 1 ? o.stride : (inner + 7) / 8 * 8))};
    const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(o.across ? kDepth : box_rows)}, step[2] = {1, 1};
    const CUresult r = encode_fn()(&m, dtype == SXCUDA_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                                   const_cast<void*>(o.data), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw RuntimeError("linear: cuTensorMapEncodeTiled failed with " + std::to_string(static_cast<int>(r)));
    return m;
}

Reach reach_of(const LinearProduct& p) {
    const auto fits = [&](const void* x, int64_t stride, int64_t bytes) {
        return !x || (reinterpret_cast<uintptr_t>(x) % bytes == 0 && (p.m <= 1 || stride * 2 % bytes == 0));
    };
    const auto all = [&](int64_t bytes) {
        return fits(p.y, p.y_stride, bytes) && fits(p.pre, p.pre_stride, bytes) && fits(p.residual, p.residual_stride, bytes);
    };
    return {all(16), all(32)};
}

template <typename T, int TN, bool A_ACROSS, bool B_ACROSS>
void launch_tile(const LinearProduct& p, cudaStream_t s) {
    const auto kernel = linear_tc_kernel<T, TN, A_ACROSS, B_ACROSS>;
    smem_limit_once(reinterpret_cast<const void*>(kernel), Smem<TN>::kBytes, "linear");
    const LinearMaps maps{make_map(p.a, p.m, p.k, kRows, p.dtype), make_map(p.b, p.n, p.k, TN / 2, p.dtype)};
    SX_LAUNCH(kernel, static_cast<unsigned>(2 * p.plan.workers), kThreads, Smem<TN>::kBytes, s, p, maps, reach_of(p));
}
template <typename T, int TN>
void launch_across(const LinearProduct& p, cudaStream_t s) {
    if (p.a.across) launch_tile<T, TN, true, true>(p, s);  // the weight's gradient
    else if (p.b.across) launch_tile<T, TN, false, true>(p, s);
    else launch_tile<T, TN, false, false>(p, s);
}

}  // namespace

bool linear_tc_takes(const void* data, int64_t stride, int64_t rows) {
    return reinterpret_cast<uintptr_t>(data) % 16 == 0 && (rows <= 1 || (stride % 8 == 0 && stride < (1ll << 38)));
}

LinearPlan linear_tc_plan(int64_t m, int64_t n, int64_t k) {
    const int64_t pairs = sm_count() / 2;
    const int64_t tiles = (m + kTileM - 1) / kTileM * ((n + 255) / 256);
    const bool narrow = n <= 128 || (tiles < pairs && tiles * ((k + kDepth - 1) / kDepth) < 16 * pairs);
    return linear_plan(m, n, k, kTileM, narrow ? 128 : 256, kDepth, pairs, 4, 24);
}

void launch_linear_tc(const LinearProduct& p, cudaStream_t s) {
    const auto type = [&](auto t) {
        if (p.plan.tile_n == 128) launch_across<decltype(t), 128>(p, s);
        else launch_across<decltype(t), 256>(p, s);
    };
    if (p.dtype == SXCUDA_F16) type(__half{});
    else type(__nv_bfloat16{});
}

}  // namespace sx

// linear_tc.cu — C = A B^T on the tensor cores for 16-bit operands, with the linear layer's epilogue.
//
// Two CTAs of a cluster make one tile of 256 x TN values: each holds 128 rows of A and half of B's rows in
// shared memory (TMA, 64 values of K a stage), one warp of the leader issues products over both (cta_group::2),
// and each CTA has the sums of its own 128 rows in its tensor memory, twice, so that one tile's epilogue runs
// under the next one's products. Rows of an operand may run along K or across it (the gradients' products
// read weight, x and v_z across): the tensor cores take either from shared memory.
//
//   the first warps: epilogue, a thread a row and its share of the columns
//   the loader:      asks for the CTA's part of the tiles, on the leader's barriers
//   the issuer:      allocates tensor memory; in the leader issues the products
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
    return st | rotary_status();
}

namespace {

constexpr int kRows = 128, kTileM = 2 * kRows, kDepth = 64;
constexpr int kPanel = kDepth * 128;  // bytes of 64 values of K for 64 rows that lie across K
constexpr int kPatches = 16;      // of a CTA

constexpr int kTurnPitch = 9;    // words of 16 values' row, and one
constexpr int kPatchCols = 32;   // a warp's unit of the epilogue: 32 rows and so many columns
constexpr int kPatch = 32 * kPatchCols * 2;
constexpr long long kLanding = 4000000;  // cycles in which any copy has landed (2 ms)

struct LinearMaps {
    CUtensorMap a, b, y, pre, residual;
};

template <int TN>
struct Smem {
    static constexpr int kA = kRows * 128, kB = TN / 2 * 128, kStage = kA + kB;
    static constexpr int kStages = TN == 256 ? 6 : 8;
    static constexpr int kPatchesAt = kStages * kStage;
    static constexpr int kBias = kPatchesAt + kPatches * kPatch;  // [2][TN] floats
    static constexpr int kBars = kBias + 2 * TN * 4;
    static constexpr int kBytes = kBars + (2 * kStages + 9 + kPatches) * 8 + 16;
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
    __device__ uint32_t bias(int part) const { return base + (2 * STAGES + 5 + part) * 8; }
    static constexpr int kCount = 2 * STAGES + 9 + kPatches;
    static __device__ bool is_acc_empty(int i) { return i / 2 == STAGES + 1; }
    static __device__ bool is_bias(int i) { return i >= 2 * STAGES + 5 && i < 2 * STAGES + 9; }
    __device__ uint32_t residual(int warp) const { return base + (2 * STAGES + 9 + warp) * 8; }
};

// ---- what a pair of CTAs needs ----
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {  // the same place in a CTA of the cluster
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// Without a release of its own, which would wait for the CTA's memory: what has to be seen is fenced where it is written.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.relaxed;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void arrive_in(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// A box of a 2-axis map into this CTA's shared memory, counted on a barrier of either CTA.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t cluster_bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(cluster_bar)
        : "memory");
}
__device__ __forceinline__ void load_own(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void store_box(const CUtensorMap* map, int x, int y, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
}
__device__ __forceinline__ void stores_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>  // all but the last N groups of the thread's stores have left shared memory
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
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
__device__ __forceinline__ void tmem_load16(uint32_t (&r)[16], uint32_t at) {  // 16 consecutive columns of the thread's lane
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : SX_R8(r, 0), SX_R8(r, 8)
        : "r"(at));
}
__device__ __forceinline__ void wait_ld16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    asm volatile("" : SX_T8(r, 0), SX_T8(r, 8));
}
template <typename T>
__device__ __forceinline__ void unpack(const uint32_t (&w)[8], float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const auto v = *reinterpret_cast<const Pack<T, 2>*>(&w[i]);
        x[2 * i] = to_f32(v.v[0]), x[2 * i + 1] = to_f32(v.v[1]);
    }
}
template <typename T>
__device__ __forceinline__ void pack(const float (&x)[16], uint32_t (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = tc::pack2<T>(x[2 * i], x[2 * i + 1]);
}
template <int ACT>
__device__ __forceinline__ void activate(float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) act_pair<ACT>(x[i], x[i + 1]);
}

template <typename T>
__device__ __forceinline__ void epilogue_act(int32_t act, float (&x)[16]) {
    switch (act) {
        case SXCUDA_ACT_RELU: activate<SXCUDA_ACT_RELU>(x); break;
        case SXCUDA_ACT_SILU: activate<SXCUDA_ACT_SILU>(x); break;
        case SXCUDA_ACT_GELU: activate<SXCUDA_ACT_GELU>(x); break;
        case SXCUDA_ACT_GELU_TANH: activate<SXCUDA_ACT_GELU_TANH>(x); break;
        default: break;
    }
}
__device__ __forceinline__ void add_bias(const uint32_t* r, const float* bias, float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        const float4 b = *reinterpret_cast<const float4*>(bias + i);
        x[i] = __uint_as_float(r[i]) + b.x, x[i + 1] = __uint_as_float(r[i + 1]) + b.y;
        x[i + 2] = __uint_as_float(r[i + 2]) + b.z, x[i + 3] = __uint_as_float(r[i + 3]) + b.w;
    }
}

// A patch in shared memory as the copies have its rows, with their swizzle: 16 bytes of a lane's row.
__device__ __forceinline__ uint4* patch_at(uint8_t* patch, int lane, int i) {
    return reinterpret_cast<uint4*>(patch + lane * 64 + ((i ^ (lane >> 1 & 3)) << 4));
}
__device__ __forceinline__ void to_patch(uint8_t* patch, int lane, int i, const uint32_t (&w)[8]) {
    *patch_at(patch, lane, i) = uint4{w[0], w[1], w[2], w[3]};
    *patch_at(patch, lane, i + 1) = uint4{w[4], w[5], w[6], w[7]};
}
__device__ __forceinline__ void from_patch(uint8_t* patch, int lane, int i, uint32_t (&w)[8]) {
    const uint4 a = *patch_at(patch, lane, i), b = *patch_at(patch, lane, i + 1);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
}

// The epilogue of 16 columns of a patch, those from 16 h on, a thread a row: r are its sums. The residual is
// in the patch; pre goes to it (if it is wanted, y to `w` alone), or y does.
template <typename T>
__device__ __forceinline__ void finish_patch(const LinearProduct& p, const uint32_t (&r)[16], const float* bias, uint8_t* patch, int lane, int h,
                                             uint32_t (&w)[8]) {
    float x[16];
    add_bias(r, bias, x);
    uint32_t z[8];
    if (p.residual) from_patch(patch, lane, 2 * h, z);
    if (p.pre) {
        pack<T>(x, w);
        to_patch(patch, lane, 2 * h, w);
    }
    epilogue_act<T>(p.act, x);
    if (p.residual) {
        float v[16];
        unpack<T>(z, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] += v[i];
    }
    pack<T>(x, w);
    if (!p.pre) to_patch(patch, lane, 2 * h, w);
}

// The same where copies do not reach the rows of y, pre or residual: 16 columns at a time are turned in shared
// memory, so that lanes stand side by side in a row, and go value by value.
struct Turn {
    int lane, rows, cols;  // rows and columns that there are
    uint32_t* words;       // [32][kTurnPitch]
};
template <typename T>
__device__ __forceinline__ void put(const Turn& at, T* first, int64_t stride, const float (&x)[16]) {
    uint32_t w[8];
    pack<T>(x, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) at.words[at.lane * kTurnPitch + i] = w[i];
    __syncwarp();
    const int half = at.lane / 16, col = at.lane % 16;
    const T* from = reinterpret_cast<const T*>(at.words) + half * 2 * kTurnPitch + col;
    T* to = first + half * stride + col;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (2 * i + half < at.rows && col < at.cols) to[2 * i * stride] = from[2 * i * 2 * kTurnPitch];
    __syncwarp();
}
template <typename T>
__device__ __forceinline__ void get(const Turn& at, const T* first, int64_t stride, float (&x)[16]) {
    const int half = at.lane / 16, col = at.lane % 16;
    const T* from = first + half * stride + col;
    T* to = reinterpret_cast<T*>(at.words) + half * 2 * kTurnPitch + col;
    T v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 2 * i + half < at.rows && col < at.cols ? from[2 * i * stride] : from_f32<T>(0.f);
#pragma unroll
    for (int i = 0; i < 16; ++i) to[2 * i * 2 * kTurnPitch] = v[i];
    __syncwarp();
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = at.words[at.lane * kTurnPitch + i];
    __syncwarp();
    unpack<T>(w, x);
}
template <typename T>
__device__ __forceinline__ void finish_turned(const LinearProduct& p, const uint32_t (&r)[16], const float* bias, uint32_t* words, int lane, int rows,
                                              int64_t row, int64_t col) {
    const Turn at{lane, rows, static_cast<int>(min(p.n - col, static_cast<int64_t>(16))), words};
    if (at.cols <= 0) return;
    float x[16];
    add_bias(r, bias, x);
    if (p.pre) put(at, static_cast<T*>(p.pre) + row * p.pre_stride + col, p.pre_stride, x);
    epilogue_act<T>(p.act, x);
    if (p.residual) {
        float y[16];
        get(at, static_cast<const T*>(p.residual) + row * p.residual_stride + col, p.residual_stride, y);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] += y[i];
    }
    put(at, static_cast<T*>(p.y) + row * p.y_stride + col, p.y_stride, x);
}

// Part of a cut tile, as [columns / 8][rows][8]: a warp's rows side by side.
__device__ __forceinline__ void leave(const LinearProduct& p, int slot, int row, int col, uint32_t (&r)[16]) {
    float* part = linear_part(p, slot, row, col);
#pragma unroll
    for (int i = 0; i < 2; ++i) tc::store32(part + i * kTileM * 8, *reinterpret_cast<uint32_t(*)[8]>(r + 8 * i));
}

// The warps of the epilogue: sixteen where there is an activation, a residual, a second result; eight for the
// gradients, whose epilogue only rounds (measured in us, eight and sixteen: 32768 x 1024 x 4096 with gelu and pre
// 245 and 230, without either 177 and 182).
template <bool B_ACROSS>
constexpr int kEpilogueWarps = B_ACROSS ? 8 : 16;
template <bool B_ACROSS>
constexpr int kThreads = 32 * (kEpilogueWarps<B_ACROSS> + 2);

template <typename T, int TN, bool A_ACROSS, bool B_ACROSS, bool COPIES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads<B_ACROSS>, 1)
    linear_tc_kernel(const __grid_constant__ LinearProduct p, const __grid_constant__ LinearMaps maps) {
    using S = Smem<TN>;
    constexpr int kStages = S::kStages, kWarps = kEpilogueWarps<B_ACROSS>, kLoader = kWarps, kIssuer = kWarps + 1;
    extern __shared__ __align__(1024) uint8_t smem[];
    const Bars<kStages> bars{tc::smem_addr(smem) + S::kBars};
    volatile uint32_t* failed = reinterpret_cast<uint32_t*>(smem + S::kBytes - 16);
    uint32_t* tmem_at = const_cast<uint32_t*>(failed) + 1;
    const uint32_t base = tc::smem_addr(smem);
    const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1;
    LinearWalk walk(p.plan, blockIdx.x / 2);
    LinearPiece piece;
    int asked = 0;  // stages that this warp has asked for

    if (warp == kLoader) {
        if (lane == 0) {
            tc::prefetch_map(&maps.a);
            tc::prefetch_map(&maps.b);
            *failed = 0;
        }
        for (int i = lane; i < Bars<kStages>::kCount; i += 32)
            tc::bar_init(bars.base + i * 8, Bars<kStages>::is_acc_empty(i) ? 2 * kWarps : Bars<kStages>::is_bias(i) ? 4 : 1);
        tc::bar_init_fence();
    }
    __syncwarp();
    if (warp == kIssuer) pair_alloc(tc::smem_addr(tmem_at), 2 * TN);
    tc::fence_before();
    __syncthreads();
    cluster_sync();
    tc::fence_after();
    const uint32_t tmem = __shfl_sync(kFullMask, *tmem_at, 0);

    if (warp == kLoader) {
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
    } else if (warp == kIssuer) {
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
            // the other CTA's last arrivals, without which this CTA's memory must not go
            for (int i = max(0, count - 2); ok && i < count; ++i) ok = tc::bar_wait(bars.acc_empty(i & 1), (i >> 1) & 1, failed);
        }
    } else {
        constexpr int kCols = TN / (kWarps / 4), kOwn = kPatches / kWarps;  // columns and patches of a warp
        const int part = warp >> 2, in_tile = static_cast<int>(rank) * kRows + (warp & 3) * 32;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        uint8_t* patch = smem + S::kPatchesAt + warp * kOwn * kPatch;
        uint32_t patch_in = tc::smem_addr(patch);
        // two patches in turn where a patch holds nothing else
        const bool in_turn = kOwn == 2 && !p.residual && !p.pre;
        uint32_t turn = 0;  // parity of the residuals' barrier
        bool due = false;   // a residual's copy is on its way
        const auto ask = [&](int row, int col) {
            if (lane == 0) {
                stores_read<0>();
                tc::bar_expect(bars.residual(warp), kPatch);
                load_own(patch_in, &maps.residual, col, row, bars.residual(warp));
            }
            due = true;
            __syncwarp();
        };
        const auto send = [&](const CUtensorMap* map, int row, int col) {
            tc::fence_smem_to_async();
            __syncwarp();
            if (lane == 0) {
                store_box(map, col, row, patch_in);
                stores_commit();
            }
        };
        // where a piece is, and its bias: taken a tile ahead. Four warps have the same columns.
        struct Place {
            int row, col, rows, slot;
            float bias;
        };
        const int bias_at = part * kCols + (warp & 3) * (kCols / 4) + lane;
        const auto place = [&]() {
            const LinearTile tile = linear_tile(p.plan, piece.tile);
            Place r{tile.m * kTileM + in_tile, tile.n * TN + part * kCols, 0, piece.slot, 0.f};
            r.rows = static_cast<int>(max(min(p.m - r.row, static_cast<int64_t>(32)), static_cast<int64_t>(0)));
            const int col = tile.n * TN + bias_at;
            if (lane < kCols / 4 && col < p.n) r.bias = linear_param(p.bias, p.bias_dtype, col);
            return r;
        };
        bool more = walk.next(p.plan, piece), ok = true;
        Place next{};
        if (more) next = place();
        for (int count = 0; ok && more; ++count) {
            const Place here = next;
            const int row = here.row, n0 = here.col, rows = here.rows;
            const bool finishes = here.slot < 0 && rows > 0;
            float* bias = reinterpret_cast<float*>(smem + S::kBias) + (count & 1) * TN;
            if (lane < kCols / 4) bias[bias_at] = here.bias;
            bias += part * kCols;
            __syncwarp();
            if (lane == 0) tc::bar_arrive(bars.bias(part));
            ok = tc::bar_wait(bars.bias(part), count & 1, failed);  // a warp may have given up: no barrier without a limit
            if (!ok) break;
            more = walk.next(p.plan, piece);
            if (more) next = place();
            if (COPIES && finishes && p.residual && n0 < p.n) ask(row, n0);
            ok = tc::bar_wait(bars.acc_full(count & 1), (count >> 1) & 1, failed);
            if (!ok) break;
            tc::fence_after();
            const uint32_t at = tmem + lanes + (count & 1) * TN + part * kCols;
            uint32_t sums[2][16];  // 16 columns, and the next ones on their way
            tmem_load16(sums[0], at);
            const auto take = [&](int col) {  // those from `col` on are there, the next ones asked for, or all are read
                wait_ld16(sums[col / 16 & 1]);
                if (col + 16 < kCols) {
                    __syncwarp();
                    tmem_load16(sums[(col / 16 & 1) ^ 1], at + col + 16);
                } else {
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_in(in_cta(bars.acc_empty(count & 1), 0));
                }
            };
#pragma unroll 1
            for (int c = 0; c < kCols; c += kPatchCols) {
                const bool some = n0 + c < p.n && rows > 0;  // the same for the whole warp
                const bool patched = COPIES && some && finishes;
                if (patched) {
                    if (p.residual) {
                        ok = tc::bar_wait(bars.residual(warp), turn, failed);
                        if (!ok) break;
                        turn ^= 1;
                        due = false;
                    } else if (lane == 0) {
                        if (in_turn) stores_read<1>();
                        else stores_read<0>();
                    }
                    __syncwarp();
                }
                uint32_t y[2][8];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    take(c + 16 * h);
                    uint32_t(&r)[16] = sums[h];
                    if (!some) continue;
                    if (!finishes) {
                        if (lane < rows) leave(p, here.slot, in_tile + lane, part * kCols + c + 16 * h, r);
                    } else if constexpr (COPIES) {
                        finish_patch<T>(p, r, bias + c + 16 * h, patch, lane, h, y[h]);
                    } else {
                        finish_turned<T>(p, r, bias + c + 16 * h, reinterpret_cast<uint32_t*>(patch), lane, rows, row, n0 + c + 16 * h);
                    }
                }
                if (!patched) continue;
                if (p.pre) {
                    send(&maps.pre, row, n0 + c);
                    if (lane == 0) stores_read<0>();
                    __syncwarp();
#pragma unroll
                    for (int h = 0; h < 2; ++h) to_patch(patch, lane, 2 * h, y[h]);
                }
                send(&maps.y, row, n0 + c);
                if (in_turn) {
                    const int to = patch_in == tc::smem_addr(smem + S::kPatchesAt + warp * kOwn * kPatch) ? kPatch : -kPatch;
                    patch += to, patch_in += to;
                }
                if (p.residual && c + kPatchCols < kCols && n0 + c + kPatchCols < p.n) ask(row, n0 + c + kPatchCols);
            }
        }
        if (due) tc::bar_drain(bars.residual(warp), turn);
        if (lane == 0) stores_read<0>();
    }

    tc::fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *failed) {
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(in_cta(tc::smem_addr(const_cast<uint32_t*>(failed)), rank ^ 1)), "r"(1) : "memory");
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
    }
    cluster_sync();
    if (*failed) {  // nothing may land in the pair's memory after it has gone
        if (warp == kLoader) {
            if (rank == 0)
                for (int i = max(0, asked - kStages); i < asked; ++i) tc::bar_drain(bars.full(i % kStages), (i / kStages) & 1);
            for (const long long start = clock64(); clock64() - start < kLanding;) {
            }
        } else if (warp == kIssuer && rank == 0) {
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
    if (warp == kIssuer) pair_free(tmem, 2 * TN);
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

void encode(CUtensorMap* m, int32_t dtype, const void* data, const cuuint64_t (&dims)[2], const cuuint64_t (&strides)[1], int cols, int rows,
            CUtensorMapSwizzle swizzle) {
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(cols), static_cast<cuuint32_t>(rows)}, step[2] = {1, 1};
    const CUresult r = encode_fn()(m, dtype == SXCUDA_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                                   const_cast<void*>(data), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw RuntimeError("linear: cuTensorMapEncodeTiled failed with " + std::to_string(static_cast<int>(r)));
}

// The operand's memory as [outer][inner], inner contiguous: K is the inner axis, or the rows are (across). Boxes
// of 64 inner values; what lies beyond the operand reads as zero.
CUtensorMap make_map(const LinearOperand& o, int64_t rows, int64_t k, int box_rows, int32_t dtype) {
    CUtensorMap m;
    const int64_t inner = o.across ? rows : k, outer = o.across ? k : rows;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
    // one row may have any stride: a length that fits stands for it
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(2 * (outer > 1 ? o.stride : (inner + 7) / 8 * 8))};
    encode(&m, dtype, o.data, dims, strides, 64, o.across ? kDepth : box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
    return m;
}

// The epilogue's patches of y, pre and residual.
CUtensorMap patch_map(const LinearProduct& p, const void* data, int64_t stride) {
    CUtensorMap m{};
    if (!data) return m;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.n), static_cast<cuuint64_t>(p.m)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(2 * (p.m > 1 ? stride : (p.n + 7) / 8 * 8))};
    encode(&m, p.dtype, data, dims, strides, kPatchCols, 32, CU_TENSOR_MAP_SWIZZLE_64B);
    return m;
}

template <typename T, int TN, bool A_ACROSS, bool B_ACROSS>
void launch_tile(const LinearProduct& p, cudaStream_t s) {
    LinearMaps maps{make_map(p.a, p.m, p.k, kRows, p.dtype), make_map(p.b, p.n, p.k, TN / 2, p.dtype), {}, {}, {}};
    const auto run = [&](auto kernel) {
        smem_limit_once(reinterpret_cast<const void*>(kernel), Smem<TN>::kBytes, "linear");
        SX_LAUNCH(kernel, static_cast<unsigned>(2 * p.plan.workers), kThreads<B_ACROSS>, Smem<TN>::kBytes, s, p, maps);
    };
    const auto reached = [&](const void* x, int64_t stride) { return !x || linear_tc_takes(x, stride, p.m); };
    // a copy to memory ends on 16 bytes (measured): with any other length of row it also writes behind the row
    if (p.n % 8 == 0 && reached(p.y, p.y_stride) && reached(p.pre, p.pre_stride) && reached(p.residual, p.residual_stride)) {
        maps.y = patch_map(p, p.y, p.y_stride);
        maps.pre = patch_map(p, p.pre, p.pre_stride);
        maps.residual = patch_map(p, p.residual, p.residual_stride);
        run(linear_tc_kernel<T, TN, A_ACROSS, B_ACROSS, true>);
    } else {
        run(linear_tc_kernel<T, TN, A_ACROSS, B_ACROSS, false>);
    }
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

// Tiles of 256 or of 128 columns, cut or not: by what they take. Measured with all pairs at work: 64 values of K 0.38 and
// 0.23 us, an epilogue that nothing hides 3.1 and 1.6 us, a cut (the parts' way through memory and the second
// kernel) some 6 us. 5001 x 333 x 777 with a residual, 128 and 256: 25 and 37 us.
LinearPlan linear_tc_plan(int64_t m, int64_t n, int64_t k) {
    const int64_t pairs = sm_count() / 2;
    const auto time = [&](const LinearPlan& p, double block, double least) {
        const double tile = std::max(static_cast<double>(p.kblocks) * block, least);
        const int64_t turns = (p.whole + pairs - 1) / pairs;
        return static_cast<double>(turns) * tile + (p.cut() ? static_cast<double>(p.share) * block + 6. : 0.);
    };
    const LinearPlan narrow = linear_plan(m, n, k, kTileM, 128, kDepth, pairs, 4, 26);
    if (n <= 128) return narrow;
    const LinearPlan wide = linear_plan(m, n, k, kTileM, 256, kDepth, pairs, 4, 16);
    return time(narrow, 0.23, 1.6) < time(wide, 0.38, 3.1) ? narrow : wide;
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

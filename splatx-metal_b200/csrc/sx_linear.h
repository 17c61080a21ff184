// sx_linear.h — what the kernels of the linear layer share: a product's arguments, how its tiles are
// divided among workers, and what follows the sums.
#pragma once

#include "sx_internal.h"
#include "sx_network.h"

namespace sx {

// Rows of an operand: element (row, k) at data[row * row_stride + k * k_stride]; one of the strides is 1.
struct LinearOperand {
    const void* data;
    int64_t row_stride, k_stride;
};

// How a product's output tiles are worked on. Tiles below `whole` go round the workers; the K blocks of
// the others are one line of units that is cut into as many equal pieces as there are workers, so that all
// of them end together. A tile that a cut goes through is left in parts in the workspace, 32-bit sums,
// which a second kernel adds in order.
struct LinearPlan {
    int32_t tile_m = 0, tile_n = 0;
    int64_t tiles_m = 0, tiles_n = 0, kblocks = 0;
    int64_t whole = 0, units = 0;
    int32_t workers = 0;
    __host__ __device__ int64_t tiles() const { return tiles_m * tiles_n; }
    __host__ __device__ bool cut() const { return units > 0; }
    __host__ __device__ int64_t start(int64_t worker) const { return worker * units / workers; }
    __host__ __device__ int64_t worker_of(int64_t unit) const { return ((unit + 1) * workers - 1) / units; }
    // Every worker may leave a part that begins in its tile's middle (slot 2 w) and one that begins at its
    // tile's start (slot 2 w + 1).
    __host__ __device__ int64_t slot_values() const { return static_cast<int64_t>(tile_m) * tile_n; }
    size_t workspace() const { return cut() ? static_cast<size_t>(2 * workers * slot_values()) * 4 : 0; }
};

// A product C = A B^T over K, [m, n], and its epilogue y = act(C + bias) + residual.
struct LinearProduct {
    LinearOperand a, b;  // rows of A: m of them, of B: n
    int64_t m, n, k;
    int32_t dtype, bias_dtype, act;
    const void* bias;
    const void* residual;
    int64_t residual_stride;
    void* y;
    int64_t y_stride;
    void* pre;
    int64_t pre_stride;
    float* parts;
    LinearPlan plan;
};

// One stretch of a tile's K blocks; slot: of the part it is left in, -1 where it is the whole tile.
struct LinearPiece {
    int64_t tile;
    int32_t k0, k1;
    int64_t slot;
};

// The pieces of one worker, in order.
struct LinearWalk {
    int64_t tile, unit, end;
    int32_t worker;
    __device__ LinearWalk(const LinearPlan& p, int32_t w) : tile(w), unit(p.cut() ? p.start(w) : 0), end(p.cut() ? p.start(w + 1) : 0), worker(w) {}
    __device__ bool next(const LinearPlan& p, LinearPiece& piece) {
        if (tile < p.whole) {
            piece = {tile, 0, static_cast<int32_t>(p.kblocks), -1};
            tile += p.workers;
            return true;
        }
        if (unit >= end) return false;
        const int64_t t = unit / p.kblocks, k0 = unit - t * p.kblocks;
        const int64_t k1 = k0 + end - unit < p.kblocks ? k0 + end - unit : p.kblocks;
        const bool all = k0 == 0 && k1 == p.kblocks;
        piece = {p.whole + t, static_cast<int32_t>(k0), static_cast<int32_t>(k1), all ? -1 : 2 * static_cast<int64_t>(worker) + (k0 == 0)};
        unit += k1 - k0;
        return true;
    }
};

// Which tile a number stands for: bands of kBand rows of tiles, in each the rows fastest, so that the tiles
// that are worked on at the same time share their operands in L2.
constexpr int kLinearBand = 8;
struct LinearTile {
    int64_t m, n;
};
__host__ __device__ inline LinearTile linear_tile(const LinearPlan& p, int64_t t) {
    const int64_t band = t / (kLinearBand * p.tiles_n), first = band * kLinearBand;
    const int64_t rows = p.tiles_m - first < kLinearBand ? p.tiles_m - first : kLinearBand, r = t - first * p.tiles_n;
    return {first + r % rows, r / rows};
}

__device__ __forceinline__ float linear_param(const void* w, int32_t dtype, int64_t i) {
    if (!w) return 0.f;
    if (dtype == SXCUDA_F32) return static_cast<const float*>(w)[i];
    if (dtype == SXCUDA_F16) return __half2float(static_cast<const __half*>(w)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// ---- activations in 32 bits ----
constexpr float kGeluTanh = 1.5957691216057308f;  // 2 sqrt(2 / pi): (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
constexpr float kGeluCube = 0.044715f;
// 1 / (1 + exp(-z)) and what it lacks to 1, neither by a difference that would lose a small one's digits.
struct Gate {
    float on, off;
};
__device__ __forceinline__ Gate gate_f32(float z) {
    const float e = expf(-fabsf(z)), large = 1.f / (1.f + e), small = e * large;
    return z < 0.f ? Gate{small, large} : Gate{large, small};
}
__device__ __forceinline__ float tanh_gate_at(float z) { return kGeluTanh * fmaf(kGeluCube * z * z, z, z); }
__device__ __forceinline__ float linear_act(int32_t act, float z) {
    switch (act) {
        case SXCUDA_ACT_RELU: return z < 0.f ? 0.f : z;  // NaN stays
        case SXCUDA_ACT_SILU: return z * gate_f32(z).on;
        case SXCUDA_ACT_GELU: return z * normcdff(z);
        case SXCUDA_ACT_GELU_TANH: return z * gate_f32(tanh_gate_at(z)).on;
        default: return z;
    }
}
__device__ __forceinline__ float linear_slope(int32_t act, float z) {
    z = fabsf(z) > 1e4f ? copysignf(1e4f, z) : z;  // the slope has its limit long before; 0 * inf would be NaN
    switch (act) {
        case SXCUDA_ACT_RELU: return z > 0.f ? 1.f : z != z ? z : 0.f;
        case SXCUDA_ACT_SILU: {
            const Gate g = gate_f32(z);
            return g.on * fmaf(z, g.off, 1.f);
        }
        case SXCUDA_ACT_GELU: return fmaf(z * 0.3989422804014327f, expf(-0.5f * z * z), normcdff(z));
        case SXCUDA_ACT_GELU_TANH: {
            const Gate g = gate_f32(tanh_gate_at(z));
            return fmaf(z * g.on * g.off, kGeluTanh * fmaf(3.f * kGeluCube * z, z, 1.f), g.on);
        }
        default: return 1.f;
    }
}

}  // namespace sx

// sx_linear.h — what the kernels of the linear layer share: a product's arguments, how its tiles are
// divided among workers, and what follows the sums.
#pragma once

#include <type_traits>

#include "sx_internal.h"
#include "sx_network.h"
#include "sx_two.cuh"

namespace sx {

// An operand of a product: element (row, k) at data[row * stride + k], or, with its rows across K, at
// data[k * stride + row].
struct LinearOperand {
    const void* data;
    int64_t stride;
    bool across;
};

// How a product's output tiles are worked on. Tiles below `whole` go round the workers. The `rest`, fewer
// than there are workers, are cut along K so that all workers end together: worker t + j rest takes the K
// blocks [j share, (j + 1) share) of rest tile t for each j < main, so that those who run at the same time
// read the same K blocks; the tails behind main * share make one line of rest * tail blocks that the
// other workers divide, tail_share each. A cut tile is left in parts in the workspace, 32-bit sums, which a
// second kernel adds in the order of K.
struct LinearPlan {
    int32_t tile_m = 0, tile_n = 0, tiles_m = 0, tiles_n = 0, kblocks = 0, whole = 0, workers = 0;
    int32_t rest = 0, main = 0, share = 0, tail = 0, tail_share = 1, slots = 0;  // slots: of a tile's parts
    __host__ __device__ int32_t tiles() const { return tiles_m * tiles_n; }
    __host__ __device__ bool cut() const { return rest > 0; }
    __host__ __device__ int32_t first_tail(int32_t t) const { return t * tail / tail_share; }
    __host__ __device__ int32_t parts(int32_t t) const { return main + (tail ? ((t + 1) * tail - 1) / tail_share - first_tail(t) + 1 : 0); }
    __host__ __device__ int64_t slot_values() const { return static_cast<int64_t>(tile_m) * tile_n; }
    size_t workspace() const { return static_cast<size_t>(rest) * slots * slot_values() * 4; }
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

// Where a part of a tile lies: [columns / 8][rows][8].
__device__ __forceinline__ float* linear_part(const LinearProduct& p, int slot, int row, int col) {
    return p.parts + slot * p.plan.slot_values() + (col / 8 * p.plan.tile_m + row) * 8 + col % 8;
}

// One stretch of a tile's K blocks; slot: of the part it is left in, -1 where it is the whole tile.
struct LinearPiece {
    int32_t tile, k0, k1, slot;
};

// The pieces of one worker, in order.
struct LinearWalk {
    int32_t tile, main, unit, end;  // main: the piece of a rest tile that is this worker's, -1: none left
    __device__ LinearWalk(const LinearPlan& p, int32_t w) : tile(w), main(-1), unit(0), end(0) {
        if (!p.cut()) return;
        if (w < p.main * p.rest) main = w;
        else unit = (w - p.main * p.rest) * p.tail_share, end = min(unit + p.tail_share, p.rest * p.tail);
    }
    __device__ bool next(const LinearPlan& p, LinearPiece& piece) {
        if (tile < p.whole) {
            piece = {tile, 0, p.kblocks, -1};
            tile += p.workers;
            return true;
        }
        if (main >= 0) {
            const int32_t t = main % p.rest, j = main / p.rest;
            piece = {p.whole + t, j * p.share, (j + 1) * p.share, t * p.slots + j};
            main = -1;
            return true;
        }
        if (unit >= end) return false;
        const int32_t t = unit / p.tail, at = unit - t * p.tail, n = min(end - unit, p.tail - at), k0 = p.main * p.share + at;
        piece = {p.whole + t, k0, k0 + n, t * p.slots + p.main + unit / p.tail_share - p.first_tail(t)};
        unit += n;
        return true;
    }
};

// Which tile a number stands for: bands of kLinearBand rows of tiles, in each the rows fastest, so that the
// tiles that are worked on at the same time share their operands in L2.
constexpr int kLinearBand = 8;
struct LinearTile {
    int32_t m, n;
};
__device__ inline LinearTile linear_tile(const LinearPlan& p, int32_t t) {
    const int32_t band = t / (kLinearBand * p.tiles_n), first = band * kLinearBand;
    const int32_t rows = min(p.tiles_m - first, kLinearBand), r = t - first * p.tiles_n;
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
// The normal distribution function and exp(-z^2 / 2), within 2^-20 of their values as far as these are normal numbers,
// without branches: 1 / 2 plus an odd polynomial for |z| < 1 (fit 2e-8), beyond it by the tail t P(t) exp(-a^2 / 2),
// t = 1 / (1 + 0.325 a) (1.1e-8). What z^2 lost to its rounding multiplies the exponential afterwards: by itself it is
// 2^-18 at |z| = 12. (Held from below, as an infinite z^2 leaves no rest.)
struct Normal {
    float below, bell;
};
__device__ __forceinline__ Normal normal_f32(float z) {
    const float a = fabsf(z), w = z * z, lost = fmaxf(fmaf(z, z, -w), -1.f), about = expf(-0.5f * w);
    const float bell = fmaf(-0.5f * lost, about, about), t = __frcp_rn(fmaf(0.325f, a, 1.f));
    float s = fmaf(0x1.8be0acp-14f, w, -0x1.329e2cp-10f);
    s = fmaf(s, w, 0x1.469c80p-7f);
    s = fmaf(s, w, -0x1.10576cp-4f);
    s = fmaf(s, w, 0x1.988452p-2f);
    float p = fmaf(0x1.5ad578p-5f, t, -0x1.22280ep-3f);
    p = fmaf(p, t, 0x1.f823d2p-4f);
    p = fmaf(p, t, -0x1.97cd8ep-12f);
    p = fmaf(p, t, 0x1.a958fcp-4f);
    p = fmaf(p, t, 0x1.cff48ap-4f);
    p = fmaf(p, t, 0x1.0a12b0p-3f);
    p = fmaf(p, t, 0x1.098388p-3f);
    const float tail = p * t * bell;
    return {a < 1.f ? fmaf(s, z, 0.5f) : z < 0.f ? tail : 1.f - tail, bell};
}
__device__ __forceinline__ float linear_act(int32_t act, float z) {
    switch (act) {
        case SXCUDA_ACT_RELU: return z < 0.f ? 0.f : z;  // NaN stays
        case SXCUDA_ACT_SILU: return z * gate_f32(z).on;
        case SXCUDA_ACT_GELU: return z * normal_f32(z).below;
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
        case SXCUDA_ACT_GELU: {
            const Normal n = normal_f32(z);
            return fmaf(z * 0.3989422804014327f, n.bell, n.below);
        }
        case SXCUDA_ACT_GELU_TANH: {
            const Gate g = gate_f32(tanh_gate_at(z));
            return fmaf(z * g.on * g.off, kGeluTanh * fmaf(3.f * kGeluCube * z, z, 1.f), g.on);
        }
        default: return 1.f;
    }
}

// ---- the same for 16-bit results: within 2^-15 of the value (2^-16.0 at worst, far out where a rounding of the exponential's
// argument counts most; 2^-16.7 for |z| < 4), at two instructions of the special-function unit ----
// The normal distribution's tail: Phi(-a) = t P(t) exp(-a^2 / 2) with t = 1 / (1 + 0.3 a); P fitted for the least
// relative error over a = 0..14 (8.2e-6).
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2Of = 1.4426950408889634f;  // of e
__device__ __forceinline__ float normal_fast(float z) {  // Phi(z)
    const float a = fabsf(z), t = rcp_fast(fmaf(0.3f, a, 1.f)), e = exp2_fast(-0.5f * kLog2Of * a * a);
    float p = fmaf(-0x1.3bca6ap-4f, t, 0x1.ba7182p-3f);
    p = fmaf(p, t, -0x1.15ac44p-6f);
    p = fmaf(p, t, 0x1.27505cp-3f);
    p = fmaf(p, t, 0x1.d1e316p-4f);
    p = fmaf(p, t, 0x1.ebd2f4p-4f);
    const float tail = p * t * e;
    return z < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float gate_fast(float z) { return rcp_fast(1.f + exp2_fast(-kLog2Of * z)); }
template <int ACT>
__device__ __forceinline__ float act_fast(float z) {
    if constexpr (ACT == SXCUDA_ACT_RELU) return z < 0.f ? 0.f : z;
    if constexpr (ACT == SXCUDA_ACT_SILU) return z * gate_fast(z);
    if constexpr (ACT == SXCUDA_ACT_GELU) return fmaxf(z, -64.f) * normal_fast(z);  // -inf gives its limit, as in act_pair
    if constexpr (ACT == SXCUDA_ACT_GELU_TANH) return z * gate_fast(tanh_gate_at(z));
    return z;
}
// act_fast of two values, by instructions that work on two where there are such.
template <int ACT>
__device__ __forceinline__ void act_pair(float& x, float& y) {
    using namespace tc;
    if constexpr (ACT == SXCUDA_ACT_GELU) {
        // max(z, 0) - |z| Phi(-|z|). Beyond 64 the tail is zero, which infinity must not multiply; a NaN comes
        // back by exp(-z^2 / 2) alone. One reciprocal for two: of 1 .. 20.2, so that their product is as good.
        const Two a = two(fminf(fabsf(x), 64.f), fminf(fabsf(y), 64.f));
        float u, v;
        split(fma2(a, two(0.3f, 0.3f), two(1.f, 1.f)), u, v);
        const float both = rcp_fast(u * v);
        const Two t = mul2(two(both, both), two(v, u)), z = two(x, y);
        split(mul2(mul2(z, two(-0.5f * kLog2Of, -0.5f * kLog2Of)), z), u, v);
        const Two e = two(exp2_fast(u), exp2_fast(v));
        Two p = fma2(two(0x1.3bca6ap-4f, 0x1.3bca6ap-4f), t, two(-0x1.ba7182p-3f, -0x1.ba7182p-3f));
        p = fma2(p, t, two(0x1.15ac44p-6f, 0x1.15ac44p-6f));
        p = fma2(p, t, two(-0x1.27505cp-3f, -0x1.27505cp-3f));
        p = fma2(p, t, two(-0x1.d1e316p-4f, -0x1.d1e316p-4f));
        p = fma2(p, t, two(-0x1.ebd2f4p-4f, -0x1.ebd2f4p-4f));  // all signs turned
        split(fma2(mul2(mul2(p, t), a), e, two(fmaxf(x, 0.f), fmaxf(y, 0.f))), x, y);
    } else if constexpr (ACT == SXCUDA_ACT_SILU || ACT == SXCUDA_ACT_GELU_TANH) {
        const Two z = two(x, y);
        Two u = z;
        if constexpr (ACT == SXCUDA_ACT_GELU_TANH) u = mul2(z, fma2(mul2(z, z), two(kGeluCube, kGeluCube), two(1.f, 1.f)));
        constexpr float k = ACT == SXCUDA_ACT_SILU ? -kLog2Of : -kLog2Of * kGeluTanh;
        float a, b;
        split(mul2(u, two(k, k)), a, b);
        split(add2(two(exp2_fast(a), exp2_fast(b)), two(1.f, 1.f)), a, b);
        split(mul2(z, two(rcp_fast(a), rcp_fast(b))), x, y);
    } else {
        x = act_fast<ACT>(x), y = act_fast<ACT>(y);
    }
}
template <typename T>
__device__ __forceinline__ float act_of(int32_t act, float z) {
    if constexpr (sizeof(T) == 4) return linear_act(act, z);
    switch (act) {
        case SXCUDA_ACT_RELU: return act_fast<SXCUDA_ACT_RELU>(z);
        case SXCUDA_ACT_SILU: return act_fast<SXCUDA_ACT_SILU>(z);
        case SXCUDA_ACT_GELU: return act_fast<SXCUDA_ACT_GELU>(z);
        case SXCUDA_ACT_GELU_TANH: return act_fast<SXCUDA_ACT_GELU_TANH>(z);
        default: return z;
    }
}
// The slopes at two values, within 2^-20 (of 1): their products with v_y are also summed to the bias' gradient, which
// may be held in 32 bits. So P has its 8th power (2.8e-8, with t = 1 / (1 + 0.26 a)). Beyond 1e4 the slopes have
// their limits long since, and infinity times zero would be NaN.
template <int ACT>
__device__ __forceinline__ void slope_pair(float& x, float& y) {
    using namespace tc;
    const Two one = two(1.f, 1.f);
    if constexpr (ACT == SXCUDA_ACT_RELU) {
        x = x > 0.f ? 1.f : x != x ? x : 0.f, y = y > 0.f ? 1.f : y != y ? y : 0.f;
    } else {
        x = fabsf(x) > 1e4f ? copysignf(1e4f, x) : x, y = fabsf(y) > 1e4f ? copysignf(1e4f, y) : y;
        const Two z = two(x, y);
        float u, v;
        if constexpr (ACT == SXCUDA_ACT_GELU) {
            split(fma2(two(fabsf(x), fabsf(y)), two(0.26f, 0.26f), one), u, v);
            const Two t = two(rcp_fast(u), rcp_fast(v));
            split(mul2(mul2(z, two(-0.5f * kLog2Of, -0.5f * kLog2Of)), z), u, v);
            const Two e = two(exp2_fast(u), exp2_fast(v));
            Two p = two(0x1.ef4a64p-6f, 0x1.ef4a64p-6f);
            p = fma2(p, t, two(-0x1.364252p-3f, -0x1.364252p-3f));
            p = fma2(p, t, two(0x1.fd6710p-3f, 0x1.fd6710p-3f));
            p = fma2(p, t, two(-0x1.2eab5ap-3f, -0x1.2eab5ap-3f));
            p = fma2(p, t, two(0x1.4522c6p-3f, 0x1.4522c6p-3f));
            p = fma2(p, t, two(0x1.a9b2fep-5f, 0x1.a9b2fep-5f));
            p = fma2(p, t, two(0x1.a505a4p-4f, 0x1.a505a4p-4f));
            p = fma2(p, t, two(0x1.a618cap-4f, 0x1.a618cap-4f));
            p = fma2(p, t, two(0x1.a8fd20p-4f, 0x1.a8fd20p-4f));
            const Two tail = mul2(mul2(p, t), e);
            float a, b;
            split(tail, a, b);
            split(fma2(tail, two(-1.f, -1.f), one), u, v);
            split(fma2(mul2(z, two(0.3989422804014327f, 0.3989422804014327f)), e, two(x < 0.f ? a : u, y < 0.f ? b : v)), x, y);
        } else {
            const Two w = mul2(z, z);
            Two at = z, steep = one;
            if constexpr (ACT == SXCUDA_ACT_GELU_TANH) {
                at = mul2(z, fma2(w, two(kGeluTanh * kGeluCube, kGeluTanh * kGeluCube), two(kGeluTanh, kGeluTanh)));
                steep = fma2(w, two(3.f * kGeluTanh * kGeluCube, 3.f * kGeluTanh * kGeluCube), two(kGeluTanh, kGeluTanh));
            }
            // g = 1 / (1 + e), and 1 - g = e g, which loses no digits; e stays finite, and a NaN comes back by z
            split(mul2(at, two(-kLog2Of, -kLog2Of)), u, v);
            const Two e = two(fminf(exp2_fast(u), 1e30f), fminf(exp2_fast(v), 1e30f));
            split(add2(e, one), u, v);
            const Two g = two(rcp_fast(u), rcp_fast(v)), off = mul2(e, g);
            split(fma2(mul2(mul2(z, g), off), steep, g), x, y);
        }
    }
}
// Times the slopes at z, for N values.
template <typename T, int N>
__device__ __forceinline__ void times_slopes(int32_t act, const float (&z)[N], float (&x)[N]) {
    float s[N + 1];
#pragma unroll
    for (int i = 0; i < N + 1; ++i) s[i] = i < N ? z[i] : 0.f;
    const auto pairs = [&](auto a) {
#pragma unroll
        for (int i = 0; i < N; i += 2) slope_pair<decltype(a)::value>(s[i], s[i + 1]);
    };
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = linear_slope(act, s[i]);
    } else if (act == SXCUDA_ACT_RELU) {
        pairs(std::integral_constant<int, SXCUDA_ACT_RELU>{});
    } else if (act == SXCUDA_ACT_SILU) {
        pairs(std::integral_constant<int, SXCUDA_ACT_SILU>{});
    } else if (act == SXCUDA_ACT_GELU) {
        pairs(std::integral_constant<int, SXCUDA_ACT_GELU>{});
    } else {
        pairs(std::integral_constant<int, SXCUDA_ACT_GELU_TANH>{});
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= s[i];
}

// ---- products on the tensor cores (linear_tc.cu), of operands that tensor maps take ----
bool linear_tc_takes(const void* data, int64_t stride, int64_t rows);
LinearPlan linear_tc_plan(int64_t m, int64_t n, int64_t k);
void launch_linear_tc(const LinearProduct& p, cudaStream_t s);

// Cuts the last turn's tiles where that saves at least `gain` K blocks of it: the cut costs a launch and
// its parts' way through memory. A piece has at least `least` K blocks.
LinearPlan linear_plan(int64_t m, int64_t n, int64_t k, int tile_m, int tile_n, int depth, int64_t workers, int64_t least,
                       int64_t gain);

}  // namespace sx

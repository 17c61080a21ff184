// layer_norm.cu — layer norm forward and backward over the last axis.
//
// Forward: mean = sum x / C, d = x - mean, rstd = 1 / sqrt(sum d^2 / C + eps), y = d rstd w + b.
// Backward, with xhat = d rstd and g = v_y w:
//   v_x = rstd (g - sum g / C - xhat sum(g xhat) / C),  v_w = sum_rows v_y xhat,  v_b = sum_rows v_y.
// Both are bound by memory: the row is read once into registers, and the variance is taken there
// about the mean (the difference of two sums would lose the digits of a mean that is large beside
// the spread).
//
// A row belongs to W warps, each thread holding NV packs of V values. The grid is what the SMs
// hold at once; each row group keeps its columns' weights in registers and takes every n-th row,
// so weights are read once per group and the backward's column sums stay in registers until the
// group is done. They then go, one partial row per CTA, to the workspace, and a second kernel
// adds the partial rows in order: the result does not depend on timing.
#include "sx_internal.h"
#include "sx_network.h"

namespace sx {
namespace {

constexpr int kNormThreads = 256;

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, V>*>(p);
}

__device__ __forceinline__ float param_at(const void* p, int32_t dtype, int64_t i, float none) {
    if (!p) return none;
    if (dtype == SXCUDA_F32) return static_cast<const float*>(p)[i];
    if (dtype == SXCUDA_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void param_to(void* p, int32_t dtype, int64_t i, float x) {
    if (dtype == SXCUDA_F32) static_cast<float*>(p)[i] = x;
    else if (dtype == SXCUDA_F16) static_cast<__half*>(p)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

// Sums of K values over the W warps of a row group; every thread gets them. `buf` holds
// kNormThreads / 32 * K floats per phase, two phases in turn, so one barrier a reduction is enough.
template <int W, int K>
__device__ __forceinline__ void group_sum(float (&x)[K], float* buf, int& phase) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) x[k] += __shfl_xor_sync(kFullMask, x[k], o);
    if constexpr (W > 1) {
        float* b = buf + phase * (kNormThreads / 32) * 2;
        phase ^= 1;
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) b[warp * 2 + k] = x[k];
        const int group = warp / W;
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(W * 32) : "memory");
#pragma unroll
        for (int k = 0; k < K; ++k) x[k] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int k = 0; k < K; ++k) x[k] += b[(group * W + w) * 2 + k];
    }
}

struct NormArgs {
    const void* x;
    const void* w;
    const void* b;
    const void* g;  // v_y
    void* y;        // y, or v_x
    float* mean;
    float* rstd;
    float* part;  // backward: [gridDim.x][2][C]
    int64_t rows, x_stride, g_stride, y_stride;
    int32_t cols, param_dtype;
    float eps;
};

template <typename T, int V, int NV, int W>
__global__ void __launch_bounds__(kNormThreads) norm_fwd_kernel(const NormArgs a) {
    constexpr int G = kNormThreads / (W * 32), E = V * NV;
    __shared__ float buf[2 * (kNormThreads / 32) * 2];
    int phase = 0;
    const int group = threadIdx.x / (W * 32), tid = threadIdx.x % (W * 32);
    float w[E], b[E];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int c = (j * W * 32 + tid) * V + e;
            w[j * V + e] = c < a.cols ? param_at(a.w, a.param_dtype, c, 1.f) : 0.f;
            b[j * V + e] = c < a.cols ? param_at(a.b, a.param_dtype, c, 0.f) : 0.f;
        }
    const float inv_c = 1.f / static_cast<float>(a.cols);
    const int64_t stride = static_cast<int64_t>(gridDim.x) * G;
    Pack<T, V> next[NV];
    auto fetch = [&](int64_t row) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * W * 32 + tid) * V;
            if (c < a.cols) next[j] = load_pack<T, V>(x + c);
        }
    };
    int64_t row = static_cast<int64_t>(blockIdx.x) * G + group;
    if (row < a.rows) fetch(row);
    for (; row < a.rows; row += stride) {
        float x[E];
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) x[j * V + e] = to_f32(next[j].v[e]);
        if (row + stride < a.rows) fetch(row + stride);
        float s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if ((j * W * 32 + tid) * V < a.cols)
#pragma unroll
                for (int e = 0; e < V; ++e) s[0] += x[j * V + e];
        group_sum<W, 1>(s, buf, phase);
        const float mean = s[0] * inv_c;
        s[0] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if ((j * W * 32 + tid) * V < a.cols)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x[j * V + e] -= mean;
                    s[0] = fmaf(x[j * V + e], x[j * V + e], s[0]);
                }
        group_sum<W, 1>(s, buf, phase);
        const float rstd = 1.f / sqrtf(fmaf(s[0], inv_c, a.eps));
        T* y = static_cast<T*>(a.y) + row * a.y_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * W * 32 + tid) * V;
            if (c < a.cols) {
                Pack<T, V> o;
#pragma unroll
                for (int e = 0; e < V; ++e) o.v[e] = from_f32<T>(fmaf(x[j * V + e] * rstd, w[j * V + e], b[j * V + e]));
                *reinterpret_cast<Pack<T, V>*>(y + c) = o;
            }
        }
        if (a.mean && tid == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

template <typename T, int V, int NV, int W>
__global__ void __launch_bounds__(kNormThreads) norm_bwd_kernel(const NormArgs a) {
    constexpr int G = kNormThreads / (W * 32), E = V * NV;
    __shared__ float buf[2 * (kNormThreads / 32) * 2];
    extern __shared__ float cols_buf[];  // [G][C] when G > 1
    int phase = 0;
    const int group = threadIdx.x / (W * 32), tid = threadIdx.x % (W * 32);
    float w[E], dw[E], db[E];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int c = (j * W * 32 + tid) * V + e;
            w[j * V + e] = c < a.cols ? param_at(a.w, a.param_dtype, c, 1.f) : 0.f;
            dw[j * V + e] = db[j * V + e] = 0.f;
        }
    const float inv_c = 1.f / static_cast<float>(a.cols);
    const int64_t stride = static_cast<int64_t>(gridDim.x) * G;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * G + group; row < a.rows; row += stride) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* g = static_cast<const T*>(a.g) + row * a.g_stride;
        Pack<T, V> xp[NV], gp[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * W * 32 + tid) * V;
            if (c < a.cols) {
                xp[j] = load_pack<T, V>(x + c);
                gp[j] = load_pack<T, V>(g + c);
            }
        }
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if ((j * W * 32 + tid) * V < a.cols)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int k = j * V + e;
                    const float gy = to_f32(gp[j].v[e]), xhat = (to_f32(xp[j].v[e]) - mean) * rstd;
                    dw[k] = fmaf(gy, xhat, dw[k]);
                    db[k] += gy;
                    s[0] = fmaf(gy, w[k], s[0]);
                    s[1] = fmaf(gy * w[k], xhat, s[1]);
                }
        group_sum<W, 2>(s, buf, phase);
        const float m0 = s[0] * inv_c, m1 = s[1] * inv_c;
        T* y = static_cast<T*>(a.y) + row * a.y_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * W * 32 + tid) * V;
            if (c < a.cols) {
                Pack<T, V> o;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xhat = (to_f32(xp[j].v[e]) - mean) * rstd;
                    o.v[e] = from_f32<T>((fmaf(to_f32(gp[j].v[e]), w[j * V + e], -m0) - xhat * m1) * rstd);
                }
                *reinterpret_cast<Pack<T, V>*>(y + c) = o;
            }
        }
    }
    if (!a.part) return;
    // the CTA's groups added in order, then one partial row of each sum
    float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float(&mine)[E] = which ? db : dw;
        if (G > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int c = (j * W * 32 + tid) * V + e;
                    if (c < a.cols) cols_buf[group * a.cols + c] = mine[j * V + e];
                }
            __syncthreads();
            for (int c = threadIdx.x; c < a.cols; c += kNormThreads) {
                float sum = 0.f;
                for (int k = 0; k < G; ++k) sum += cols_buf[k * a.cols + c];
                part[which * a.cols + c] = sum;
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int c = (j * W * 32 + tid) * V + e;
                    if (c < a.cols) part[which * a.cols + c] = mine[j * V + e];
                }
        }
    }
}

// Columns too many for registers: a CTA per row, read again for each pass (from L2 as a rule), and
// the column sums by a thread per column over a slice of the rows.
template <typename T>
__device__ __forceinline__ float cta_sum(float x, float* buf, int& phase) {
    float s[1] = {x};
    group_sum<kNormThreads / 32, 1>(s, buf, phase);
    return s[0];
}
template <typename T>
__global__ void __launch_bounds__(kNormThreads) norm_fwd_wide_kernel(const NormArgs a) {
    __shared__ float buf[2 * (kNormThreads / 32) * 2];
    int phase = 0;
    const float inv_c = 1.f / static_cast<float>(a.cols);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        float s = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += kNormThreads) s += to_f32(x[c]);
        const float mean = cta_sum<T>(s, buf, phase) * inv_c;
        s = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += kNormThreads) {
            const float d = to_f32(x[c]) - mean;
            s = fmaf(d, d, s);
        }
        const float rstd = 1.f / sqrtf(fmaf(cta_sum<T>(s, buf, phase), inv_c, a.eps));
        T* y = static_cast<T*>(a.y) + row * a.y_stride;
        for (int c = threadIdx.x; c < a.cols; c += kNormThreads)
            y[c] = from_f32<T>(fmaf((to_f32(x[c]) - mean) * rstd, param_at(a.w, a.param_dtype, c, 1.f),
                                    param_at(a.b, a.param_dtype, c, 0.f)));
        if (a.mean && threadIdx.x == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}
template <typename T>
__global__ void __launch_bounds__(kNormThreads) norm_bwd_wide_kernel(const NormArgs a) {
    __shared__ float buf[2 * (kNormThreads / 32) * 2];
    int phase = 0;
    const float inv_c = 1.f / static_cast<float>(a.cols);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* g = static_cast<const T*>(a.g) + row * a.g_stride;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s[2] = {0.f, 0.f};
        for (int c = threadIdx.x; c < a.cols; c += kNormThreads) {
            const float gw = to_f32(g[c]) * param_at(a.w, a.param_dtype, c, 1.f);
            s[0] += gw;
            s[1] = fmaf(gw, (to_f32(x[c]) - mean) * rstd, s[1]);
        }
        group_sum<kNormThreads / 32, 2>(s, buf, phase);
        const float m0 = s[0] * inv_c, m1 = s[1] * inv_c;
        T* y = static_cast<T*>(a.y) + row * a.y_stride;
        for (int c = threadIdx.x; c < a.cols; c += kNormThreads) {
            const float xhat = (to_f32(x[c]) - mean) * rstd;
            y[c] = from_f32<T>((fmaf(to_f32(g[c]), param_at(a.w, a.param_dtype, c, 1.f), -m0) - xhat * m1) * rstd);
        }
    }
}
template <typename T>
__global__ void __launch_bounds__(kNormThreads) norm_cols_wide_kernel(const NormArgs a, int64_t slice) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kNormThreads + threadIdx.x;
    if (c >= a.cols) return;
    const int64_t r0 = blockIdx.y * slice, r1 = r0 + slice < a.rows ? r0 + slice : a.rows;
    float dw = 0.f, db = 0.f;
    for (int64_t row = r0; row < r1; ++row) {
        const float g = to_f32(static_cast<const T*>(a.g)[row * a.g_stride + c]);
        const float x = to_f32(static_cast<const T*>(a.x)[row * a.x_stride + c]);
        dw = fmaf(g, (x - a.mean[row]) * a.rstd[row], dw);
        db += g;
    }
    float* part = a.part + static_cast<int64_t>(blockIdx.y) * 2 * a.cols;
    part[c] = dw;
    part[a.cols + c] = db;
}

// Adds the partial rows of 32 columns: warp w takes every 8th row, then the warps are added in order.
__global__ void __launch_bounds__(256) norm_cols_kernel(const float* part, int64_t rows, int32_t cols, void* v_w,
                                                        void* v_b, int32_t param_dtype) {
    __shared__ float sums[8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;  // over both sums' columns
    float s = 0.f;
    if (c < 2 * static_cast<int64_t>(cols)) {
        int64_t r = warp;
        for (; r + 24 < rows; r += 32) {
            const float x0 = part[r * 2 * cols + c], x1 = part[(r + 8) * 2 * cols + c];
            const float x2 = part[(r + 16) * 2 * cols + c], x3 = part[(r + 24) * 2 * cols + c];
            s += (x0 + x1) + (x2 + x3);
        }
        for (; r < rows; r += 8) s += part[r * 2 * cols + c];
    }
    sums[warp][lane] = s;
    __syncthreads();
    if (warp || c >= 2 * static_cast<int64_t>(cols)) return;
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sums[w][lane];
    if (c < cols) {
        if (v_w) param_to(v_w, param_dtype, c, s);
    } else if (v_b) {
        param_to(v_b, param_dtype, c - cols, s);
    }
}

bool packs(const void* p, int64_t stride, int64_t rows, int64_t size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || stride * size % 16 == 0);
}

// The smallest row group whose threads hold a row in at most 32 values each, and the fewest packs
// a thread that cover it.
template <typename T, int V, typename F>
void by_shape(int32_t cols, F&& f) {
    using std::integral_constant;
    const int64_t packs_in_row = (cols + V - 1) / V;
    const auto with = [&](auto w) {
        constexpr int W = decltype(w)::value;
        constexpr int most = 32 / V;
        const int64_t need = (packs_in_row + W * 32 - 1) / (W * 32);
        if (need <= most / 4) f(integral_constant<int, V>{}, integral_constant<int, most / 4>{}, w);
        else if (need <= most / 2) f(integral_constant<int, V>{}, integral_constant<int, most / 2>{}, w);
        else f(integral_constant<int, V>{}, integral_constant<int, most>{}, w);
    };
    if (cols <= 1024) with(integral_constant<int, 1>{});
    else if (cols <= 2048) with(integral_constant<int, 2>{});
    else if (cols <= 4096) with(integral_constant<int, 4>{});
    else with(integral_constant<int, 8>{});
}
constexpr int kMostCols = 8192;

constexpr int kPartialsPerSm = 2;  // CTAs that leave a partial row, per SM
int64_t wide_slices(const SxLayerNormInputs& in) {
    return std::min<int64_t>(std::max<int64_t>(in.rows / 64, 1), 64);
}
int64_t partial_rows(const SxLayerNormInputs& in) {
    return in.cols > kMostCols ? wide_slices(in) : static_cast<int64_t>(kPartialsPerSm) * sm_count();
}

template <typename T, typename F>
void by_layout(const NormArgs& a, bool wide_ok, F&& f) {
    constexpr int V = 16 / sizeof(T);
    if (wide_ok) by_shape<T, V>(a.cols, f);
    else by_shape<T, 1>(a.cols, f);
}

}  // namespace

void launch_layer_norm_fwd(const SxLayerNormInputs& in, void* y, int64_t y_stride, float* mean,
                           float* rstd, cudaStream_t s) {
    if (in.rows == 0) return;
    const NormArgs a{in.x, in.weight, in.bias, nullptr, y, mean, rstd, nullptr, in.rows, in.x_stride,
                     0, y_stride, static_cast<int32_t>(in.cols), in.param_dtype, in.eps};
    by_dtype(in.dtype, [&](auto t) {
        using T = decltype(t);
        if (in.cols > kMostCols) {
            const auto kernel = norm_fwd_wide_kernel<T>;
            SX_LAUNCH(kernel, static_cast<unsigned>(std::min<int64_t>(in.rows, INT32_MAX)), kNormThreads, 0, s, a);
            return;
        }
        const int64_t e = sizeof(T);
        const bool vec = in.cols * e % 16 == 0 && packs(in.x, in.x_stride, in.rows, e) && packs(y, y_stride, in.rows, e);
        by_layout<T>(a, vec, [&](auto v, auto nv, auto w) {
            constexpr int W = decltype(w)::value, G = kNormThreads / (W * 32);
            const auto kernel = norm_fwd_kernel<T, decltype(v)::value, decltype(nv)::value, W>;
            const int64_t grid = std::min<int64_t>((in.rows + G - 1) / G, 2 * sm_count());
            SX_LAUNCH(kernel, static_cast<unsigned>(grid), kNormThreads, 0, s, a);
        });
    });
}

size_t layer_norm_bwd_workspace(const SxLayerNormInputs& in) {
    return static_cast<size_t>(partial_rows(in)) * 2 * in.cols * sizeof(float);
}

void launch_layer_norm_bwd(const SxLayerNormInputs& in, const SxLayerNormGradsIn& g,
                           const SxLayerNormGrads& out, void* ws, cudaStream_t s) {
    const bool cols_wanted = out.v_weight || out.v_bias;
    NormArgs a{in.x, in.weight, nullptr, g.v_y, out.v_x, const_cast<float*>(g.mean),
               const_cast<float*>(g.rstd), cols_wanted ? static_cast<float*>(ws) : nullptr, in.rows,
               in.x_stride, g.v_y_stride, out.v_x_stride, static_cast<int32_t>(in.cols), in.param_dtype, in.eps};
    int64_t parts = 0;
    if (in.rows) by_dtype(in.dtype, [&](auto t) {
        using T = decltype(t);
        if (in.cols > kMostCols) {
            const auto kernel = norm_bwd_wide_kernel<T>;
            SX_LAUNCH(kernel, static_cast<unsigned>(std::min<int64_t>(in.rows, INT32_MAX)), kNormThreads, 0, s, a);
            if (cols_wanted) {
                parts = wide_slices(in);
                const dim3 grid(blocks_for(in.cols, kNormThreads), static_cast<unsigned>(parts));
                const auto cols = norm_cols_wide_kernel<T>;
                SX_LAUNCH(cols, grid, kNormThreads, 0, s, a, (in.rows + parts - 1) / parts);
            }
            return;
        }
        const int64_t e = sizeof(T);
        const bool vec = in.cols * e % 16 == 0 && packs(in.x, in.x_stride, in.rows, e) &&
                         packs(g.v_y, g.v_y_stride, in.rows, e) && packs(out.v_x, out.v_x_stride, in.rows, e);
        by_layout<T>(a, vec, [&](auto v, auto nv, auto w) {
            constexpr int W = decltype(w)::value, G = kNormThreads / (W * 32);
            const auto kernel = norm_bwd_kernel<T, decltype(v)::value, decltype(nv)::value, W>;
            parts = std::min<int64_t>((in.rows + G - 1) / G, static_cast<int64_t>(kPartialsPerSm) * sm_count());
            const int smem = G > 1 ? static_cast<int>(G * in.cols * sizeof(float)) : 0;
            SX_LAUNCH(kernel, static_cast<unsigned>(parts), kNormThreads, smem, s, a);
        });
    });
    if (cols_wanted)
        SX_LAUNCH(norm_cols_kernel, blocks_for(2 * in.cols, 32), 256, 0, s, static_cast<const float*>(ws), parts,
                  static_cast<int32_t>(in.cols), out.v_weight, out.v_bias, in.param_dtype);
}

}  // namespace sx

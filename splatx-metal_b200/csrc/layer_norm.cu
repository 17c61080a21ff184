// layer_norm.cu — layer norm forward and backward over the last axis.
//
// Forward: mean = sum x / C, d = x - mean, rstd = 1 / sqrt(sum d^2 / C + eps), y = d rstd w + b.
// Backward, with xhat = d rstd and g = v_y w:
//   v_x = rstd (g - sum g / C - xhat sum(g xhat) / C),  v_w = sum_rows v_y xhat,  v_b = sum_rows v_y.
// Both are bound by memory: the row is read once into registers, and the variance is taken there
// about the mean (the difference of two sums would lose the digits of a mean that is large beside
// the spread).
//
// A row belongs to a group of lanes of one warp, or of whole warps, each thread holding NV packs of V
// values, and the next row is on its way while one is worked on. Beside memory it is instructions that
// cost: a thread holds 64 bytes of a row (half of that in the backward, whose column sums take two
// registers a value), so that the groups' sums are spread over many values; the arithmetic is done two
// values at a time; and the weights lie in shared memory, in the order the lanes read them, which
// leaves registers for more rows. bf16 32768 x 1024: forward 24.8 us (5.4 TB/s), backward 43.5 us
// (4.6 TB/s); with the weights in registers and 32 values a thread the forward took 47 us (8 warps an
// SM), with 8 values a thread 39 us (twice the instructions a row). Of the backward's time 37.8 us are
// the first kernel's without its partial rows (5.3 TB/s, with the rows that 128 registers a thread leave
// in flight), 5.7 us the partial rows and the second kernel.
// The grid is what the SMs hold; each group takes every n-th row, so the backward's column sums stay
// in registers until the group is done. They then go, one partial row per CTA, to the workspace, and a
// second kernel adds the partial rows in order: the result does not depend on timing.
#include "sx_internal.h"
#include "sx_network.h"
#include "sx_two.cuh"

namespace sx {
namespace {

constexpr int kNormThreads = 256;  // of the kernels for rows beyond the registers

// Threads of a CTA whose rows take LANES threads each, and the CTAs that an SM is to hold.
template <int LANES>
constexpr int kThreads = LANES > 256 ? LANES : 256;
template <int LANES>
constexpr int kFwdPerSm = 768 / kThreads<LANES>;
template <int LANES>
constexpr int kBwdPerSm = LANES > 256 ? 1 : 2;

// Where a thread's value k lies in the shared copy of the weights: pieces of 16 bytes, lane by lane.
template <int LANES>
__device__ __forceinline__ int weight_at(int tid, int k) {
    return (k / 4 * LANES + tid) * 4 + k % 4;
}

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

// Sums of K values over a row's LANES threads; every thread gets them. `buf` holds two values of each
// warp per phase, two phases in turn, so one barrier a reduction is enough.
template <int LANES, int K>
__device__ __forceinline__ void group_sum(float (&x)[K], float* buf, int& phase) {
#pragma unroll
    for (int o = (LANES < 32 ? LANES : 32) / 2; o; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) x[k] += __shfl_xor_sync(kFullMask, x[k], o);
    if constexpr (LANES > 32) {
        constexpr int W = LANES / 32;
        float* b = buf + phase * (kThreads<LANES> / 32) * 2;
        phase ^= 1;
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) b[warp * 2 + k] = x[k];
        const int group = warp / W;
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(LANES) : "memory");
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

using tc::Two;
__device__ __forceinline__ float2 widen(const float* p) { return float2{p[0], p[1]}; }
__device__ __forceinline__ float2 widen(const __half* p) { return __half22float2(*reinterpret_cast<const __half2*>(p)); }
__device__ __forceinline__ float2 widen(const __nv_bfloat16* p) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    return float2{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
}
__device__ __forceinline__ void narrow(float* p, float x, float y) { p[0] = x, p[1] = y; }
__device__ __forceinline__ void narrow(__half* p, float x, float y) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x, y); }
__device__ __forceinline__ void narrow(__nv_bfloat16* p, float x, float y) {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x, y);
}
// Values 2 i and 2 i + 1 of a thread's packs, and back.
template <typename T, int V, int NV>
__device__ __forceinline__ Two pair_of(const Pack<T, V> (&p)[NV], int i) {
    if constexpr (V == 1) return tc::two(to_f32(p[2 * i].v[0]), to_f32(p[2 * i + 1].v[0]));
    else {
        const float2 f = widen(p[2 * i / V].v + 2 * i % V);
        return tc::two(f.x, f.y);
    }
}
template <typename T, int V, int NV>
__device__ __forceinline__ void set_pair(Pack<T, V> (&p)[NV], int i, Two x) {
    float lo, hi;
    tc::split(x, lo, hi);
    if constexpr (V == 1) p[2 * i].v[0] = from_f32<T>(lo), p[2 * i + 1].v[0] = from_f32<T>(hi);
    else narrow(p[2 * i / V].v + 2 * i % V, lo, hi);
}
__device__ __forceinline__ float both(Two x) {
    float lo, hi;
    tc::split(x, lo, hi);
    return lo + hi;
}
__device__ __forceinline__ Two same(float x) { return tc::two(x, x); }

template <typename T, int V, int NV, int LANES>
__global__ void __launch_bounds__(kThreads<LANES>, kFwdPerSm<LANES>) norm_fwd_kernel(const NormArgs a) {
    constexpr int G = kThreads<LANES> / LANES, E = V * NV;
    __shared__ float buf[2 * (kThreads<LANES> / 32) * 2];
    extern __shared__ __align__(16) float weights[];  // [2][LANES * E]
    int phase = 0;
    const int group = threadIdx.x / LANES, tid = threadIdx.x % LANES;
    if (group == 0)
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const int c = (k / V * LANES + tid) * V + k % V, at = weight_at<LANES>(tid, k);
            weights[at] = c < a.cols ? param_at(a.w, a.param_dtype, c, 1.f) : 0.f;
            weights[LANES * E + at] = c < a.cols ? param_at(a.b, a.param_dtype, c, 0.f) : 0.f;
        }
    __syncthreads();
    const float inv_c = 1.f / static_cast<float>(a.cols);
    const int64_t stride = static_cast<int64_t>(gridDim.x) * G;
    Pack<T, V> next[NV] = {};
    const auto here = [&](int k) { return (k / V * LANES + tid) * V + k % V < a.cols; };  // value k is one of the row's
    const auto fetch = [&](int64_t row) {
        if (row >= a.rows) return;
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride + tid * V;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (here(j * V)) next[j] = load_pack<T, V>(x + j * LANES * V);
    };
    // a warp's groups go through the rows together: its shuffles are over all of it
    int64_t row = static_cast<int64_t>(blockIdx.x) * G + group;
    const int64_t in_warp = LANES < 32 ? group % (32 / LANES) : 0;
    fetch(row);
    for (; row - in_warp < a.rows; row += stride) {
        Two x[E / 2], t = same(0.f);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) x[i] = pair_of(next, i);  // zeros where the row has no value
        fetch(row + stride);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) t = tc::add2(t, x[i]);
        float s[1] = {both(t)};
        group_sum<LANES, 1>(s, buf, phase);
        const float mean = s[0] * inv_c;
        const Two minus_mean = same(-mean);
        t = same(0.f);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            x[i] = tc::add2(x[i], minus_mean);
            if constexpr (V == 1) {
                float lo, hi;
                tc::split(x[i], lo, hi);
                x[i] = tc::two(here(2 * i) ? lo : 0.f, here(2 * i + 1) ? hi : 0.f);
                t = tc::fma2(x[i], x[i], t);
            } else if (here(2 * i)) {
                t = tc::fma2(x[i], x[i], t);
            }
        }
        s[0] = both(t);
        group_sum<LANES, 1>(s, buf, phase);
        const float rstd = 1.f / sqrtf(fmaf(s[0], inv_c, a.eps));
        if (row >= a.rows) continue;
        T* y = static_cast<T*>(a.y) + row * a.y_stride + tid * V;
        const Two times = same(rstd);
        Pack<T, V> o[NV];
#pragma unroll
        for (int i = 0; i < E / 2; i += 2) {
            const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(weights + weight_at<LANES>(tid, 2 * i));
            const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(weights + LANES * E + weight_at<LANES>(tid, 2 * i));
            set_pair(o, i, tc::fma2(tc::mul2(x[i], times), Two{w.x}, Two{b.x}));
            set_pair(o, i + 1, tc::fma2(tc::mul2(x[i + 1], times), Two{w.y}, Two{b.y}));
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (here(j * V)) *reinterpret_cast<Pack<T, V>*>(y + j * LANES * V) = o[j];
        if (a.mean && tid == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

template <typename T, int V, int NV, int LANES>
__global__ void __launch_bounds__(kThreads<LANES>, kBwdPerSm<LANES>) norm_bwd_kernel(const NormArgs a) {
    constexpr int G = kThreads<LANES> / LANES, E = V * NV;
    __shared__ float buf[2 * (kThreads<LANES> / 32) * 2];
    extern __shared__ __align__(16) float weights[];  // [LANES * E]; at the end the groups' sums, [G][C]
    int phase = 0;
    const int group = threadIdx.x / LANES, tid = threadIdx.x % LANES;
    Two dw[E / 2], db[E / 2];
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int c = (k / V * LANES + tid) * V + k % V;
        if (group == 0) weights[weight_at<LANES>(tid, k)] = c < a.cols ? param_at(a.w, a.param_dtype, c, 1.f) : 0.f;
        dw[k / 2] = db[k / 2] = same(0.f);
    }
    __syncthreads();
    const float inv_c = 1.f / static_cast<float>(a.cols);
    const int64_t stride = static_cast<int64_t>(gridDim.x) * G;
    const auto here = [&](int k) { return (k / V * LANES + tid) * V + k % V < a.cols; };
    struct Row {
        Pack<T, V> x[NV] = {}, g[NV] = {};
        float mean = 0.f, rstd = 0.f;
    };
    Row next;
    const auto fetch = [&](int64_t row) {
        if (row >= a.rows) return;
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride + tid * V;
        const T* g = static_cast<const T*>(a.g) + row * a.g_stride + tid * V;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (here(j * V)) {
                next.x[j] = load_pack<T, V>(x + j * LANES * V);
                next.g[j] = load_pack<T, V>(g + j * LANES * V);
            }
        next.mean = a.mean[row];
        next.rstd = a.rstd[row];
    };
    int64_t row = static_cast<int64_t>(blockIdx.x) * G + group;
    const int64_t in_warp = LANES < 32 ? group % (32 / LANES) : 0;
    fetch(row);
    for (; row - in_warp < a.rows; row += stride) {
        const bool mine = row < a.rows;
        const Two rstd = same(next.rstd), shift = same(-next.mean);
        Two xhat[E / 2], gw[E / 2], t0 = same(0.f), t1 = same(0.f);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            xhat[i] = pair_of(next.x, i);
            gw[i] = mine ? pair_of(next.g, i) : same(0.f);
        }
        fetch(row + stride);
        // where the row has no value its gradient is zero, and so is all that it adds to
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            xhat[i] = tc::mul2(tc::add2(xhat[i], shift), rstd);
            dw[i] = tc::fma2(gw[i], xhat[i], dw[i]);
            db[i] = tc::add2(db[i], gw[i]);
            gw[i] = tc::mul2(gw[i], *reinterpret_cast<const Two*>(weights + weight_at<LANES>(tid, 2 * i)));
            t0 = tc::add2(t0, gw[i]);
            t1 = tc::fma2(gw[i], xhat[i], t1);
        }
        float s[2] = {both(t0), both(t1)};
        group_sum<LANES, 2>(s, buf, phase);
        if (!mine) continue;
        const Two m0 = same(-s[0] * inv_c), m1 = same(-s[1] * inv_c);
        T* y = static_cast<T*>(a.y) + row * a.y_stride + tid * V;
        Pack<T, V> o[NV];
#pragma unroll
        for (int i = 0; i < E / 2; ++i) set_pair(o, i, tc::mul2(tc::fma2(xhat[i], m1, tc::add2(gw[i], m0)), rstd));
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (here(j * V)) *reinterpret_cast<Pack<T, V>*>(y + j * LANES * V) = o[j];
    }
    if (!a.part) return;
    // the CTA's groups added in order, then one partial row of each sum
    float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const Two(&sums)[E / 2] = which ? db : dw;
        float mine[E];
#pragma unroll
        for (int i = 0; i < E / 2; ++i) tc::split(sums[i], mine[2 * i], mine[2 * i + 1]);
        float* to = G > 1 ? weights + group * a.cols : part + which * a.cols;
        if (G > 1) __syncthreads();
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (here(k)) to[(k / V * LANES + tid) * V + k % V] = mine[k];
        if (G > 1) {
            __syncthreads();
            for (int c = threadIdx.x; c < a.cols; c += kThreads<LANES>) {
                float sum = 0.f;
                for (int k = 0; k < G; ++k) sum += weights[k * a.cols + c];
                part[which * a.cols + c] = sum;
            }
        }
    }
}

// Columns too many for registers: a CTA per row, read again for each pass (from L2 as a rule), and
// the column sums by a thread per column over a slice of the rows.
__device__ __forceinline__ float cta_sum(float x, float* buf, int& phase) {
    float s[1] = {x};
    group_sum<kNormThreads, 1>(s, buf, phase);
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
        const float mean = cta_sum(s, buf, phase) * inv_c;
        s = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += kNormThreads) {
            const float d = to_f32(x[c]) - mean;
            s = fmaf(d, d, s);
        }
        const float rstd = 1.f / sqrtf(fmaf(cta_sum(s, buf, phase), inv_c, a.eps));
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
        group_sum<kNormThreads, 2>(s, buf, phase);
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

// Adds the partial rows of 32 columns: warp w takes every 32nd row, with eight in flight, then the
// warps are added in order.
__global__ void __launch_bounds__(1024) norm_cols_kernel(const float* part, int64_t rows, int32_t cols, void* v_w,
                                                         void* v_b, int32_t param_dtype) {
    __shared__ float sums[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane, width = 2 * static_cast<int64_t>(cols);
    float s = 0.f;
    if (c < width)
        for (int64_t r = warp; r < rows; r += 8 * 32) {
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = r + k * 32 < rows ? part[(r + k * 32) * width + c] : 0.f;
            s += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        }
    sums[warp][lane] = s;
    __syncthreads();
    s = sums[lane][warp];  // row `lane` of column `warp`
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 32 + warp;
    if (lane || at >= width) return;
    if (at < cols) {
        if (v_w) param_to(v_w, param_dtype, at, s);
    } else if (v_b) {
        param_to(v_b, param_dtype, at - cols, s);
    }
}

bool packs(const void* p, int64_t stride, int64_t rows, int64_t size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || stride * size % 16 == 0);
}

constexpr int kMostCols = 8192;

// The smallest row group whose threads hold a row, MOST values each at most: 8 lanes for up to 64
// values, then up to a warp with 8 values a lane, a warp with more, and groups of warps.
template <int V, int MOST, typename F>
void by_shape(int32_t cols, F&& f) {
    using std::integral_constant;
    const auto with = [&](auto lanes, auto values) {
        f(integral_constant<int, V>{}, integral_constant<int, decltype(values)::value / V>{}, lanes);
    };
    constexpr integral_constant<int, 8> k8{};
    constexpr integral_constant<int, 16> k16{};
    constexpr integral_constant<int, MOST> most{};
    static_assert(MOST >= 16, "packs");
    if (cols <= 64) with(integral_constant<int, 8>{}, k8);
    else if (cols <= 128) with(integral_constant<int, 16>{}, k8);
    else if (cols <= 256) with(integral_constant<int, 32>{}, k8);
    else if (cols <= 512) with(integral_constant<int, 32>{}, k16);
    else if (cols <= 32 * MOST) with(integral_constant<int, 32>{}, most);
    else if (cols <= 64 * MOST) with(integral_constant<int, 64>{}, most);
    else if (cols <= 128 * MOST) with(integral_constant<int, 128>{}, most);
    else if (cols <= 256 * MOST) with(integral_constant<int, 256>{}, most);
    else if constexpr (256 * MOST < kMostCols) with(integral_constant<int, kMostCols / MOST>{}, most);
}

constexpr int kPartialsPerSm = 2;  // the most CTAs that leave a partial row, per SM
int64_t wide_slices(const SxLayerNormInputs& in) {
    return std::min<int64_t>(std::max<int64_t>(in.rows / 64, 1), 64);
}
int64_t partial_rows(const SxLayerNormInputs& in) {
    return in.cols > kMostCols ? wide_slices(in) : static_cast<int64_t>(kPartialsPerSm) * sm_count();
}

template <typename T, int MOST, typename F>
void by_layout(const NormArgs& a, bool wide_ok, F&& f) {
    constexpr int V = 16 / sizeof(T);
    if (wide_ok) by_shape<V, MOST>(a.cols, f);
    else by_shape<1, MOST>(a.cols, f);
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
        by_layout<T, 64 / sizeof(T)>(a, vec, [&](auto v, auto nv, auto lanes) {
            constexpr int L = decltype(lanes)::value, V = decltype(v)::value, NV = decltype(nv)::value, G = kThreads<L> / L;
            const auto kernel = norm_fwd_kernel<T, V, NV, L>;
            constexpr int smem = 2 * L * V * NV * static_cast<int>(sizeof(float));
            if (smem > 48 * 1024) smem_limit_once(reinterpret_cast<const void*>(kernel), smem, "layer_norm_fwd");
            const int64_t grid = std::min<int64_t>((in.rows + G - 1) / G, static_cast<int64_t>(kFwdPerSm<L>) * sm_count());
            SX_LAUNCH(kernel, static_cast<unsigned>(grid), kThreads<L>, smem, s, a);
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
        by_layout<T, 16>(a, vec, [&](auto v, auto nv, auto lanes) {
            constexpr int L = decltype(lanes)::value, V = decltype(v)::value, NV = decltype(nv)::value, G = kThreads<L> / L;
            static_assert(kBwdPerSm<L> <= kPartialsPerSm, "workspace");
            const auto kernel = norm_bwd_kernel<T, V, NV, L>;
            parts = std::min<int64_t>((in.rows + G - 1) / G, static_cast<int64_t>(kBwdPerSm<L>) * sm_count());
            // the weights, and later a row of sums for each group
            const int smem = static_cast<int>(std::max<int64_t>(L * V * NV, G > 1 ? G * in.cols : 0) * sizeof(float));
            SX_LAUNCH(kernel, static_cast<unsigned>(parts), kThreads<L>, smem, s, a);
        });
    });
    if (cols_wanted)
        SX_LAUNCH(norm_cols_kernel, blocks_for(2 * in.cols, 32), 1024, 0, s, static_cast<const float*>(ws), parts,
                  static_cast<int32_t>(in.cols), out.v_weight, out.v_bias, in.param_dtype);
}

}  // namespace sx

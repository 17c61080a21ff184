// rotary.cu — norms of queries and keys per head and their rotation by the positions of their tokens, in
// one pass, and its gradients.
//
// Forward, per token and head: u = x rstd w with rstd = 1 / sqrt(mean x^2 + eps), then for every pair of
// values (u1, u2) -> (u1 c - u2 s, u1 s + u2 c), c and s of the angle position x frequency.
// Backward: g = the gradient rotated back; v_w = sum of g x rstd over tokens and heads;
// v_x = rstd (g w - xhat mean(g w xhat)), xhat = x rstd (taken anew from x: nothing is kept).
//
// Bound by memory: each value is read once and written once. A row (one head of one token) belongs to a
// group of lanes of a warp; a thread holds V first values of pairs and their V partners, so that the rotation
// needs no other lane, and 16-byte accesses where the pairs' layout allows them (V = 8 values of 16 bits).
// A warp takes one token at a time: its lanes share the token's sines and cosines (through shared memory,
// once for all heads), which then stay in registers, as the weights do for the whole kernel: a CTA works
// on queries only or on keys only. The next row and the next token's position are on their way meanwhile.
// Angles: position x frequency in turns in 64 bits, the nearest quarter turn taken off there; what is left
// is at most an eighth, and its 32 bits are exact to 2^-28 of a turn however far the position.
#include <algorithm>
#include <cmath>

#include "sx_internal.h"
#include "sx_network.h"

namespace sx {
namespace {

constexpr int kRotThreads = 128;
constexpr int kRotWarps = kRotThreads / 32;
constexpr int kRotMostPairs = 128;

struct RotHalf {  // the queries or the keys
    const void* x;
    const void* g;
    void* out;
    int64_t x_batch, x_token, x_head, g_batch, g_token, g_head, out_batch, out_token, out_head;
    const void* weight;
    float* part;  // [blocks, dim]: the CTAs' sums for the weight's gradient
    int32_t heads, chunk, chunks;  // heads; those of a unit of work; units a token
    int32_t blocks;
    int64_t units;
};

struct RotArgs {
    RotHalf half[2];
    const void* positions;
    int64_t pos_batch, pos_token, pos_axis;
    int64_t tokens;
    int32_t pos_dtype, param_dtype, axes, dim, pairs, slots, lanes;  // slots: V pairs each; lanes: of a row's group
    int32_t mode, norm;
    int32_t axis_dims[4];
    float eps, inv_dim;
    double turns[kRotMostPairs];  // frequency / 2 pi
    uint8_t axis[kRotMostPairs];
};

__device__ __forceinline__ float rot_param(const void* w, int32_t dtype, int64_t i) {
    if (!w) return 1.f;
    if (dtype == SXCUDA_F32) return static_cast<const float*>(w)[i];
    if (dtype == SXCUDA_F16) return __half2float(static_cast<const __half*>(w)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}
__device__ __forceinline__ void rot_param_to(void* w, int32_t dtype, int64_t i, float x) {
    if (dtype == SXCUDA_F32) static_cast<float*>(w)[i] = x;
    else if (dtype == SXCUDA_F16) static_cast<__half*>(w)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(w)[i] = __float2bfloat16_rn(x);
}

// Where a slot's V first values and their V partners (of neighbours: its 2 V values) start in a head;
// `second` is -1 where an odd value is left alone.
struct Slot {
    int first, second;
};
template <int V>
__device__ __forceinline__ Slot slot_at(const RotArgs& a, int slot) {
    const int j = slot * V, p = a.pairs;
    if (j >= p) {  // values that are not rotated
        const int r = j - p, rest = a.dim - 2 * p, half = (rest + 1) / 2;
        const Slot s = a.mode == SXCUDA_PAIRS_NEIGHBOURS ? Slot{2 * p + 2 * r, 2 * p + 2 * r + V} : Slot{2 * p + r, 2 * p + half + r};
        return {s.first, s.second < a.dim ? s.second : -1};
    }
    if (a.mode == SXCUDA_PAIRS_NEIGHBOURS) return {2 * j, 2 * j + V};
    if (a.mode == SXCUDA_PAIRS_WHOLE) return {j, j + p};
    int start = 0, axis = 0;
    while (axis < a.axes - 1 && j >= start + a.axis_dims[axis] / 2) start += a.axis_dims[axis++] / 2;
    return {start + j, start + j + a.axis_dims[axis] / 2};  // the run starts at value 2 start
}

template <typename T, int V, int NV>
struct Row {
    Pack<T, V> first[NV], second[NV];
};

// The thread's part of one kernel: which rows, pairs and weights are its own.
template <typename T, int V, bool NB, int NV>
struct Rot {
    static constexpr int W = V < 4 ? V : 4;  // values of a table access
    const RotArgs& a;
    const RotHalf& h;
    float* table;  // [2 V / W][slots][W]: cosines, then sines, in the order in which lanes read them
    const double* turns;
    const uint8_t* axis;
    int lane, group, in_group, rows;  // rows: groups of a warp
    Slot at[NV];
    bool mine[NV];

    __device__ Rot(const RotArgs& a, const RotHalf& h, float* table, const double* turns, const uint8_t* axis)
        : a(a), h(h), table(table), turns(turns), axis(axis), lane(threadIdx.x & 31) {
        group = lane / a.lanes;
        in_group = lane % a.lanes;
        rows = 32 / a.lanes;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int slot = in_group + n * a.lanes;
            mine[n] = slot < a.slots;
            at[n] = mine[n] ? slot_at<V>(a, slot) : Slot{0, -1};
        }
        for (int i = lane; i < a.slots * V; i += 32) *entry(i, 0) = 1.f, *entry(i, V) = 0.f;  // not rotated
        __syncwarp();
    }
    __device__ float* entry(int pair, int skip) const {
        const int slot = pair / V, e = pair % V + skip;
        return table + ((e / W) * a.slots + slot) * W + e % W;
    }
    // Lane i's position along axis i.
    __device__ double position(int64_t unit) const {
        if (lane >= a.axes || unit >= h.units) return 0.;
        const int64_t token = unit / h.chunks, b = token / a.tokens;
        const int64_t i = b * a.pos_batch + (token - b * a.tokens) * a.pos_token + lane * a.pos_axis;
        if (a.pos_dtype == SXCUDA_POS_F32) return static_cast<const float*>(a.positions)[i];
        if (a.pos_dtype == SXCUDA_POS_I32) return static_cast<const int32_t*>(a.positions)[i];
        return static_cast<double>(static_cast<const int64_t*>(a.positions)[i]);
    }
    __device__ void angles(double mine_position, float (&c)[NV][V], float (&s)[NV][V]) const {
        __syncwarp();
        for (int i = lane; i - lane < a.pairs; i += 32) {
            const int j = i < a.pairs ? i : 0;
            const double p = __shfl_sync(kFullMask, mine_position, axis[j]);
            const double t = p * turns[j], quarters = rint(4. * t);
            // of a product beyond 2^53 no digit of a turn is left: it stands at 0 (of an infinity NaN is left)
            float sine, cosine;
            sincospif(static_cast<float>(2. * fma(-0.25, quarters, t)), &sine, &cosine);
            const int q = static_cast<int>(static_cast<long long>(fabs(quarters) < 9e15 ? quarters : 0.) & 3);
            const float cc = q & 1 ? sine : cosine, ss = q & 1 ? cosine : sine;
            if (i < a.pairs) {
                *entry(i, 0) = q == 1 || q == 2 ? -cc : cc;
                *entry(i, V) = q >= 2 ? -ss : ss;
            }
        }
        __syncwarp();
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int slot = mine[n] ? in_group + n * a.lanes : 0;
#pragma unroll
            for (int e = 0; e < V; e += W) {
                const auto x = reinterpret_cast<const Pack<float, W>*>(table)[(e / W) * a.slots + slot];
                const auto y = reinterpret_cast<const Pack<float, W>*>(table)[((V + e) / W) * a.slots + slot];
#pragma unroll
                for (int k = 0; k < W; ++k) c[n][e + k] = x.v[k], s[n][e + k] = y.v[k];
            }
        }
    }
    // The group's head of a unit in its turn `it`; -1: none left.
    __device__ int head_of(int64_t unit, int it) const {
        const int in_chunk = it * rows + group, head = static_cast<int>(unit % h.chunks) * h.chunk + in_chunk;
        return unit < h.units && in_chunk < h.chunk && head < h.heads ? head : -1;
    }
    __device__ int64_t offset(int64_t unit, int head, int64_t batch, int64_t token, int64_t head_stride) const {
        const int64_t t = unit / h.chunks, b = t / a.tokens;
        return b * batch + (t - b * a.tokens) * token + head * head_stride;
    }
    __device__ void load(Row<T, V, NV>& r, const T* row, bool there) const {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            r.first[n] = r.second[n] = Pack<T, V>{};
            if (there && mine[n]) {
                r.first[n] = *reinterpret_cast<const Pack<T, V>*>(row + at[n].first);
                if (at[n].second >= 0) r.second[n] = *reinterpret_cast<const Pack<T, V>*>(row + at[n].second);
            }
        }
    }
    __device__ void store(T* row, const float (&p)[NV][V], const float (&q)[NV][V]) const {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            if (!mine[n]) continue;
            Pack<T, V> x, y;
#pragma unroll
            for (int e = 0; e < V; ++e) *value(x, y, e, 0) = from_f32<T>(p[n][e]), *value(x, y, e, 1) = from_f32<T>(q[n][e]);
            *reinterpret_cast<Pack<T, V>*>(row + at[n].first) = x;
            if (at[n].second >= 0) *reinterpret_cast<Pack<T, V>*>(row + at[n].second) = y;
        }
    }
    // The first (second) value of pair e among a slot's.
    template <typename P>
    static __device__ __forceinline__ auto* value(P& x, P& y, int e, int second) {
        if constexpr (NB) {
            const int i = 2 * e + second;
            return i < V ? &x.v[i] : &y.v[i - V];
        } else {
            return second ? &y.v[e] : &x.v[e];
        }
    }
    // The place in the head of the first (second) value of pair e of slot n.
    __device__ int place(int n, int e, int second) const {
        if constexpr (NB) {
            const int i = 2 * e + second;
            return i < V ? at[n].first + i : at[n].second < 0 ? -1 : at[n].second + i - V;
        } else {
            return second ? (at[n].second < 0 ? -1 : at[n].second + e) : at[n].first + e;
        }
    }
    __device__ void unpack(const Row<T, V, NV>& r, float (&p)[NV][V], float (&q)[NV][V]) const {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e)
                p[n][e] = to_f32(*value(r.first[n], r.second[n], e, 0)), q[n][e] = to_f32(*value(r.first[n], r.second[n], e, 1));
    }
    __device__ float group_sum(float x) const {
        for (int o = a.lanes / 2; o; o >>= 1) x += __shfl_xor_sync(kFullMask, x, o);
        return x;
    }
    __device__ void weights(float (&p)[NV][V], float (&q)[NV][V]) const {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int i = place(n, e, 0), j = place(n, e, 1);
                p[n][e] = mine[n] ? rot_param(h.weight, a.param_dtype, i) : 0.f;
                q[n][e] = mine[n] && j >= 0 ? rot_param(h.weight, a.param_dtype, j) : 0.f;
            }
    }
    __device__ float rstd(const float (&p)[NV][V], const float (&q)[NV][V]) const {
        float ss = 0.f;
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) ss = fmaf(p[n][e], p[n][e], fmaf(q[n][e], q[n][e], ss));
        return __frsqrt_rn(fmaf(group_sum(ss), a.inv_dim, a.eps));
    }
};

extern __shared__ double rot_smem[];

// The CTA's half, its number among that half's CTAs, and the tables in shared memory.
struct RotPlace {
    const RotHalf* half;
    int block;
    double* turns;
    uint8_t* axis;
    float* table;
};
__device__ __forceinline__ RotPlace rot_place(const RotArgs& a, int width) {
    const int k = blockIdx.x >= a.half[0].blocks;
    RotPlace p{&a.half[k], static_cast<int>(blockIdx.x) - (k ? a.half[0].blocks : 0), rot_smem, nullptr, nullptr};
    p.table = reinterpret_cast<float*>(rot_smem + (a.pairs + 1) / 2 * 2) + (threadIdx.x >> 5) * 2 * width;
    p.axis = reinterpret_cast<uint8_t*>(reinterpret_cast<float*>(rot_smem + (a.pairs + 1) / 2 * 2) + kRotWarps * 2 * width);
    for (int i = threadIdx.x; i < a.pairs; i += kRotThreads) p.turns[i] = a.turns[i], p.axis[i] = a.axis[i];
    __syncthreads();
    return p;
}
size_t rot_smem_bytes(const RotArgs& a, int v) {
    return (a.pairs + 1) / 2 * 2 * 8 + static_cast<size_t>(kRotWarps) * 2 * a.slots * v * 4 + a.pairs;
}

template <typename T, int V, bool NB, int NV>
__global__ void __launch_bounds__(kRotThreads) rotary_fwd_kernel(const __grid_constant__ RotArgs a) {
    const RotPlace at = rot_place(a, a.slots * V);
    const Rot<T, V, NB, NV> me(a, *at.half, at.table, at.turns, at.axis);
    const RotHalf& h = me.h;
    const int64_t step = static_cast<int64_t>(h.blocks) * kRotWarps;
    const int turns = (h.chunk + me.rows - 1) / me.rows;
    float w0[NV][V], w1[NV][V], c[NV][V], s[NV][V];
    me.weights(w0, w1);
    int64_t unit = static_cast<int64_t>(at.block) * kRotWarps + (threadIdx.x >> 5);
    int it = 0;
    const auto fetch = [&](Row<T, V, NV>& r, int64_t u, int i) {
        const int head = me.head_of(u, i);
        me.load(r, static_cast<const T*>(h.x) + (head < 0 ? 0 : me.offset(u, head, h.x_batch, h.x_token, h.x_head)), head >= 0);
    };
    Row<T, V, NV> row;
    fetch(row, unit, 0);
    double position = me.position(unit);
    while (unit < h.units) {
        const bool last = it + 1 == turns;
        const int64_t next_unit = last ? unit + step : unit;
        const int next_it = last ? 0 : it + 1;
        Row<T, V, NV> next;
        fetch(next, next_unit, next_it);
        if (it == 0) {
            me.angles(position, c, s);
            position = me.position(unit + step);
        }
        float p[NV][V], q[NV][V];
        me.unpack(row, p, q);
        const float r = a.norm ? me.rstd(p, q) : 1.f;
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float u1 = p[n][e] * r * w0[n][e], u2 = q[n][e] * r * w1[n][e];
                p[n][e] = fmaf(u1, c[n][e], -u2 * s[n][e]);
                q[n][e] = fmaf(u1, s[n][e], u2 * c[n][e]);
            }
        const int head = me.head_of(unit, it);
        if (head >= 0) me.store(static_cast<T*>(h.out) + me.offset(unit, head, h.out_batch, h.out_token, h.out_head), p, q);
        row = next;
        unit = next_unit;
        it = next_it;
    }
}

template <typename T, int V, bool NB, int NV>
__global__ void __launch_bounds__(kRotThreads) rotary_bwd_kernel(const __grid_constant__ RotArgs a) {
    const RotPlace at = rot_place(a, a.slots * V);
    const Rot<T, V, NB, NV> me(a, *at.half, at.table, at.turns, at.axis);
    const RotHalf& h = me.h;
    const int64_t step = static_cast<int64_t>(h.blocks) * kRotWarps;
    const int turns = (h.chunk + me.rows - 1) / me.rows;
    float w0[NV][V], w1[NV][V], c[NV][V], s[NV][V], sum0[NV][V] = {}, sum1[NV][V] = {};
    me.weights(w0, w1);
    int64_t unit = static_cast<int64_t>(at.block) * kRotWarps + (threadIdx.x >> 5);
    int it = 0;
    const auto fetch = [&](Row<T, V, NV>& x, Row<T, V, NV>& g, int64_t u, int i) {
        const int head = me.head_of(u, i);
        me.load(g, static_cast<const T*>(h.g) + (head < 0 ? 0 : me.offset(u, head, h.g_batch, h.g_token, h.g_head)), head >= 0);
        me.load(x, static_cast<const T*>(h.x) + (head < 0 ? 0 : me.offset(u, head, h.x_batch, h.x_token, h.x_head)),
                head >= 0 && a.norm);
    };
    Row<T, V, NV> x_row, g_row;
    fetch(x_row, g_row, unit, 0);
    double position = me.position(unit);
    while (unit < h.units) {
        const bool last = it + 1 == turns;
        const int64_t next_unit = last ? unit + step : unit;
        const int next_it = last ? 0 : it + 1;
        Row<T, V, NV> x_next, g_next;
        fetch(x_next, g_next, next_unit, next_it);
        if (it == 0) {
            me.angles(position, c, s);
            position = me.position(unit + step);
        }
        const int head = me.head_of(unit, it);
        float p[NV][V], q[NV][V];
        me.unpack(g_row, p, q);
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float g1 = p[n][e], g2 = q[n][e];
                p[n][e] = fmaf(g1, c[n][e], g2 * s[n][e]);
                q[n][e] = fmaf(g2, c[n][e], -g1 * s[n][e]);
            }
        if (a.norm) {
            float x0[NV][V], x1[NV][V];
            me.unpack(x_row, x0, x1);
            const float r = me.rstd(x0, x1);
            float dot = 0.f;
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x0[n][e] *= r, x1[n][e] *= r;
                    if (head >= 0) {  // of a group without a row r may be infinite
                        sum0[n][e] = fmaf(p[n][e], x0[n][e], sum0[n][e]);
                        sum1[n][e] = fmaf(q[n][e], x1[n][e], sum1[n][e]);
                    }
                    p[n][e] *= w0[n][e], q[n][e] *= w1[n][e];
                    dot = fmaf(p[n][e], x0[n][e], fmaf(q[n][e], x1[n][e], dot));
                }
            dot = me.group_sum(dot) * a.inv_dim;
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    p[n][e] = fmaf(-x0[n][e], dot, p[n][e]) * r;
                    q[n][e] = fmaf(-x1[n][e], dot, q[n][e]) * r;
                }
        }
        if (head >= 0) me.store(static_cast<T*>(h.out) + me.offset(unit, head, h.out_batch, h.out_token, h.out_head), p, q);
        x_row = x_next;
        g_row = g_next;
        unit = next_unit;
        it = next_it;
    }
    if (!h.part) return;
    // the warp's groups, then the CTA's warps, in order
    __syncthreads();
    float* sums = reinterpret_cast<float*>(rot_smem);  // [warps, dim], over the tables
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float x = sum0[n][e], y = sum1[n][e];
            for (int o = 16; o >= a.lanes; o >>= 1) x += __shfl_xor_sync(kFullMask, x, o), y += __shfl_xor_sync(kFullMask, y, o);
            if (me.group == 0 && me.mine[n]) {
                const int i = me.place(n, e, 0), j = me.place(n, e, 1);
                sums[(threadIdx.x >> 5) * a.dim + i] = x;
                if (j >= 0) sums[(threadIdx.x >> 5) * a.dim + j] = y;
            }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < a.dim; i += kRotThreads) {
        float x = 0.f;
        for (int w = 0; w < kRotWarps; ++w) x += sums[w * a.dim + i];
        h.part[static_cast<int64_t>(at.block) * a.dim + i] = x;
    }
}

// Adds the CTAs' sums of 32 values: warp w takes every 32nd row, then the warps are added in order.
__global__ void __launch_bounds__(1024) rotary_sums_kernel(const float* q_part, int64_t q_rows, const float* k_part, int64_t k_rows,
                                                           int32_t dim, void* v_qw, void* v_kw, int32_t param_dtype) {
    __shared__ float sums[32][33];
    const bool k = blockIdx.y;
    const float* part = k ? k_part : q_part;
    void* to = k ? v_kw : v_qw;
    if (!to) return;
    const int64_t rows = k ? k_rows : q_rows;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < dim)
        for (int64_t r = warp; r < rows; r += 8 * 32) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = r + i * 32 < rows ? part[(r + i * 32) * dim + c] : 0.f;
            s += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        }
    sums[warp][lane] = s;
    __syncthreads();
    s = sums[lane][warp];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
    const int i = blockIdx.x * 32 + warp;
    if (lane == 0 && i < dim) rot_param_to(to, param_dtype, i, s);
}

// ---- host ----
struct RotPlan {
    RotArgs a;
    int v = 1;
};

bool view_fits(const SxAttentionView& x, int64_t size, int64_t bytes) {
    const auto fits = [&](int64_t n) { return n * size % bytes == 0; };
    return reinterpret_cast<uintptr_t>(x.data) % bytes == 0 && fits(x.batch_stride) && fits(x.token_stride) && fits(x.head_stride);
}

// The most pairs a thread can take at once: runs of pairs, of their partners and of what is not rotated are
// multiples of it, and so are the views' strides and addresses.
int most_pairs(const SxRotaryInputs& in, std::initializer_list<SxAttentionView> views) {
    const int64_t size = dtype_bytes(in.dtype);
    int pairs = 0;
    for (int i = 0; i < in.axes; ++i) pairs += in.axis_dims[i] / 2;
    const int rest = in.head_dim - 2 * pairs;
    int v = in.dtype == SXCUDA_F32 ? 4 : 8;
    const auto holds = [&](int n) {
        if (rest % 2 || rest / 2 % n || pairs % n) return false;
        if (in.pairs == SXCUDA_PAIRS_AXIS)
            for (int i = 0; i < in.axes; ++i)
                if (in.axis_dims[i] / 2 % n) return false;
        return std::all_of(views.begin(), views.end(), [&](const SxAttentionView& x) { return view_fits(x, size, n * size); });
    };
    while (v > 1 && !holds(v)) v /= 2;
    return v;
}

RotArgs rot_args(const SxRotaryInputs& in, int v) {
    RotArgs a{};
    const double tau = 6.283185307179586476925286766559;
    a.positions = in.positions;
    a.pos_batch = in.pos_batch_stride, a.pos_token = in.pos_token_stride, a.pos_axis = in.pos_axis_stride;
    a.tokens = in.tokens;
    a.pos_dtype = in.pos_dtype, a.param_dtype = in.param_dtype;
    a.axes = in.axes, a.dim = in.head_dim, a.mode = in.pairs, a.norm = in.norm;
    a.eps = in.eps;
    a.inv_dim = 1.f / static_cast<float>(in.head_dim);
    for (int i = 0; i < in.axes; ++i) {
        a.axis_dims[i] = in.axis_dims[i];
        for (int j = 0; j < in.axis_dims[i] / 2; ++j, ++a.pairs) {
            a.turns[a.pairs] = in.freqs[a.pairs] / tau;
            a.axis[a.pairs] = static_cast<uint8_t>(i);
        }
    }
    a.slots = ((in.head_dim + 1) / 2 + v - 1) / v;
    for (a.lanes = 1; a.lanes < a.slots && a.lanes < 32;) a.lanes *= 2;
    const auto set = [&](RotHalf& h, const SxAttentionView& x, int heads, const void* weight) {
        h.x = x.data, h.x_batch = x.batch_stride, h.x_token = x.token_stride, h.x_head = x.head_stride;
        h.heads = heads;
        h.weight = weight;
    };
    set(a.half[0], in.q, in.q_heads, in.q_weight);
    if (in.k_heads) set(a.half[1], in.k, in.k_heads, in.k_weight);
    return a;
}

// Units of work and CTAs. A unit is a token with all its heads, so that its sines are taken once; where there
// are fewer tokens than half the warps that fit, a unit is as many heads as a warp has groups.
void rot_divide(RotArgs& a, int64_t tokens, int per_sm) {
    const int64_t most = static_cast<int64_t>(sm_count()) * per_sm;
    const int rows = 32 / a.lanes, heads = a.half[0].heads + a.half[1].heads;
    for (RotHalf& h : a.half) {
        if (!h.heads) continue;
        h.chunk = tokens * 2 >= most * kRotWarps ? h.heads : std::min(rows, h.heads);
        h.chunks = (h.heads + h.chunk - 1) / h.chunk;
        h.units = tokens * h.chunks;
        const int64_t share = std::max<int64_t>(most * h.heads / heads, 1);
        h.blocks = static_cast<int32_t>(std::min(share, (h.units + kRotWarps - 1) / kRotWarps));
    }
}

// Calls f(element, pairs a thread, neighbours, slots a thread).
template <typename F>
void by_layout(const SxRotaryInputs& in, int v, F&& f) {
    by_dtype(in.dtype, [&](auto t) {
        using T = decltype(t);
        const auto order = [&](auto n, auto slots) {
            if (in.pairs == SXCUDA_PAIRS_NEIGHBOURS) f(t, n, std::true_type{}, slots);
            else f(t, n, std::false_type{}, slots);
        };
        // up to 256 values are 16, 32, 64 and 128 slots for 32 lanes
        if constexpr (sizeof(T) == 2)
            if (v == 8) return order(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
        if (v == 4) return order(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
        if (v == 2) return order(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
        order(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
    });
}

constexpr int kRotFwdPerSm = 6, kRotBwdPerSm = 4;

}  // namespace

void launch_qk_norm_rotary_fwd(const SxRotaryInputs& in, const SxAttentionView& q_out, const SxAttentionView& k_out, cudaStream_t s) {
    const int64_t tokens = in.batch * in.tokens;
    if (tokens == 0) return;
    const int v = in.k_heads ? most_pairs(in, {in.q, in.k, q_out, k_out}) : most_pairs(in, {in.q, q_out});
    RotArgs a = rot_args(in, v);
    const auto set = [](RotHalf& h, const SxAttentionView& x) {
        h.out = x.data, h.out_batch = x.batch_stride, h.out_token = x.token_stride, h.out_head = x.head_stride;
    };
    set(a.half[0], q_out);
    if (in.k_heads) set(a.half[1], k_out);
    rot_divide(a, tokens, kRotFwdPerSm);
    by_layout(in, v, [&](auto t, auto n, auto nb, auto slots) {
        constexpr int V = decltype(n)::value, NV = decltype(slots)::value;
        const auto kernel = rotary_fwd_kernel<decltype(t), V, decltype(nb)::value, NV>;
        SX_LAUNCH(kernel, static_cast<unsigned>(a.half[0].blocks + a.half[1].blocks), kRotThreads, rot_smem_bytes(a, V), s, a);
    });
}

size_t qk_norm_rotary_bwd_workspace(const SxRotaryInputs& in) {
    return in.norm ? static_cast<size_t>(sm_count()) * kRotBwdPerSm * in.head_dim * 4 + 2 * in.head_dim * 4 : 0;
}

void launch_qk_norm_rotary_bwd(const SxRotaryInputs& in, const SxRotaryGrads& g, void* ws, cudaStream_t s) {
    const int64_t tokens = in.batch * in.tokens;
    const auto zero = [&](void* w) {
        if (w) cuda_check(cudaMemsetAsync(w, 0, in.head_dim * dtype_bytes(in.param_dtype), s), "qk_norm_rotary_bwd");
    };
    if (tokens == 0) {
        zero(g.v_q_weight);
        zero(g.v_k_weight);
        return;
    }
    SxRotaryInputs at = in;
    if (!in.norm) at.q = g.v_q_out, at.k = g.v_k_out;  // not read
    const int v = in.k_heads ? most_pairs(at, {at.q, at.k, g.v_q_out, g.v_k_out, g.v_q, g.v_k})
                             : most_pairs(at, {at.q, g.v_q_out, g.v_q});
    RotArgs a = rot_args(at, v);
    const auto set = [](RotHalf& h, const SxAttentionView& x, const SxAttentionView& y) {
        h.g = x.data, h.g_batch = x.batch_stride, h.g_token = x.token_stride, h.g_head = x.head_stride;
        h.out = y.data, h.out_batch = y.batch_stride, h.out_token = y.token_stride, h.out_head = y.head_stride;
    };
    set(a.half[0], g.v_q_out, g.v_q);
    if (in.k_heads) set(a.half[1], g.v_k_out, g.v_k);
    rot_divide(a, tokens, kRotBwdPerSm);
    float* part = static_cast<float*>(ws);
    if (g.v_q_weight) a.half[0].part = part;
    if (g.v_k_weight) a.half[1].part = part + static_cast<int64_t>(a.half[0].blocks) * in.head_dim;
    by_layout(in, v, [&](auto t, auto n, auto nb, auto slots) {
        constexpr int V = decltype(n)::value, NV = decltype(slots)::value;
        const auto kernel = rotary_bwd_kernel<decltype(t), V, decltype(nb)::value, NV>;
        const size_t smem = std::max<size_t>(rot_smem_bytes(a, V), static_cast<size_t>(kRotWarps) * in.head_dim * 4);
        SX_LAUNCH(kernel, static_cast<unsigned>(a.half[0].blocks + a.half[1].blocks), kRotThreads, smem, s, a);
    });
    if (g.v_q_weight || g.v_k_weight)
        SX_LAUNCH(rotary_sums_kernel, dim3(blocks_for(in.head_dim, 32), 2), 1024, 0, s, a.half[0].part, a.half[0].blocks,
                  a.half[1].part, a.half[1].blocks, in.head_dim, g.v_q_weight, g.v_k_weight, in.param_dtype);
}

}  // namespace sx

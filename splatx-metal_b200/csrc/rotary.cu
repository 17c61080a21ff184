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
// A warp takes one token at a time, its queries and then its keys: its lanes make the token's sines and
// cosines once for all heads, in shared memory, in the order in which lanes read them; the weights lie there
// in the same way. Groups of a warp read the same entries at the same time, so that a read is one pass of
// shared memory, and registers are left for warps and for rows that are on their way.
// Angles: position x frequency in turns in 64 bits, the nearest quarter turn taken off there; what is left
// is at most an eighth, and its 32 bits are exact to 2^-28 of a turn however far the position.
#include <algorithm>
#include <cmath>

#include "sx_internal.h"
#include "sx_network.h"
#include "sx_two.cuh"

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
    int32_t heads, turns;  // turns: of a warp's groups until all heads are done
};

struct RotArgs {
    RotHalf half[2];
    const void* positions;
    int64_t pos_batch, pos_token, pos_axis;
    int64_t tokens, units;
    int32_t chunk, chunks;  // turns of a unit of work, units of a token
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

// V values in pairs that one instruction works on.
template <int V>
struct Values {
    static constexpr int N = (V + 1) / 2;
    tc::Two v[N];
};

extern __shared__ double rot_smem[];

// The thread's part of a kernel.
template <typename T, int V, bool NB, int NV>
struct Rot {
    static constexpr int W = V < 4 ? V : 4;      // values of a table access
    static constexpr int N = Values<V>::N;
    const RotArgs& a;
    double* turns;
    float* weights;  // of queries, then of keys: [2][2 V / W][slots][W], first values and partners
    float* table;    // [2 V / W][slots][W]: cosines, then sines of the warp's token
    uint8_t* axis;
    int lane, group, in_group, rows;  // rows: groups of a warp
    Slot at[NV];
    bool mine[NV];

    __device__ explicit Rot(const RotArgs& a) : a(a), turns(rot_smem), lane(threadIdx.x & 31) {
        const int width = 2 * a.slots * V;
        weights = reinterpret_cast<float*>(rot_smem + (a.pairs + 1) / 2 * 2);
        table = weights + (2 + (threadIdx.x >> 5)) * width;
        axis = reinterpret_cast<uint8_t*>(weights + (2 + kRotWarps) * width);
        for (int i = threadIdx.x; i < a.pairs; i += kRotThreads) turns[i] = a.turns[i], axis[i] = a.axis[i];
        for (int i = threadIdx.x; i < 2 * a.slots * V; i += kRotThreads) {
            const int k = i >= a.slots * V, pair = i - k * a.slots * V;
            const Slot s = slot_at<V>(a, pair / V);
            const RotHalf& h = a.half[k];
            const int one = place(s, pair % V, 0), two = place(s, pair % V, 1);
            *entry(weights + k * width, pair, 0) = rot_param(h.weight, a.param_dtype, one);
            *entry(weights + k * width, pair, V) = two < 0 ? 0.f : rot_param(h.weight, a.param_dtype, two);
        }
        group = lane / a.lanes;
        in_group = lane % a.lanes;
        rows = 32 / a.lanes;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int slot = in_group + n * a.lanes;
            mine[n] = slot < a.slots;
            at[n] = mine[n] ? slot_at<V>(a, slot) : Slot{0, -1};
        }
        for (int i = lane; i < a.slots * V; i += 32) *entry(table, i, 0) = 1.f, *entry(table, i, V) = 0.f;  // not rotated
        __syncthreads();
    }
    static size_t smem_bytes(const RotArgs& a) {
        return (a.pairs + 1) / 2 * 2 * 8 + static_cast<size_t>(2 + kRotWarps) * 2 * a.slots * V * 4 + a.pairs;
    }
    __device__ float* entry(float* t, int pair, int skip) const {
        const int slot = pair / V, e = pair % V + skip;
        return t + ((e / W) * a.slots + slot) * W + e % W;
    }
    // The entries of the thread's slot n: V of them from `skip`.
    __device__ Values<V> entries(const float* t, int n, int skip) const {
        const int slot = mine[n] ? in_group + n * a.lanes : 0;
        Values<V> r;
#pragma unroll
        for (int e = 0; e < V; e += W) {
            const auto x = reinterpret_cast<const Pack<float, W>*>(t)[((skip + e) / W) * a.slots + slot];
            if constexpr (W == 1) {
                r.v[0] = tc::two(x.v[0], 0.f);
            } else {
#pragma unroll
                for (int k = 0; k < W; k += 2) r.v[(e + k) / 2] = tc::two(x.v[k], x.v[k + 1]);
            }
        }
        return r;
    }
    // Lane i's position along axis i.
    __device__ double position(int64_t unit) const {
        if (lane >= a.axes || unit >= a.units) return 0.;
        const Token t = token_of(unit);
        const int64_t i = t.batch * a.pos_batch + t.token * a.pos_token + lane * a.pos_axis;
        if (a.pos_dtype == SXCUDA_POS_F32) return static_cast<const float*>(a.positions)[i];
        if (a.pos_dtype == SXCUDA_POS_I32) return static_cast<const int32_t*>(a.positions)[i];
        return static_cast<double>(static_cast<const int64_t*>(a.positions)[i]);
    }
    __device__ void angles(double mine_position) const {
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
                *entry(table, i, 0) = q == 1 || q == 2 ? -cc : cc;
                *entry(table, i, V) = q >= 2 ? -ss : ss;
            }
        }
        __syncwarp();
    }
    struct Token {
        int64_t batch, token;
        int chunk;
    };
    __device__ Token token_of(int64_t unit) const {
        if (a.units <= INT32_MAX) {  // 64-bit divisions take some hundred instructions
            const uint32_t u = static_cast<uint32_t>(unit), t = u / static_cast<uint32_t>(a.chunks);
            const uint32_t n = static_cast<uint32_t>(a.tokens), b = t / n;
            return {b, t - b * n, static_cast<int>(u - t * a.chunks)};
        }
        const int64_t t = unit / a.chunks, b = t / a.tokens;
        return {b, t - b * a.tokens, static_cast<int>(unit - t * a.chunks)};
    }
    // A slot that is not the thread's own keeps the zeros it started with.
    __device__ void load(Row<T, V, NV>& r, const T* row, bool there) const {
#pragma unroll
        for (int n = 0; n < NV; ++n)
            if (there && mine[n]) {
                r.first[n] = *reinterpret_cast<const Pack<T, V>*>(row + at[n].first);
                if (V > 1 || at[n].second >= 0) r.second[n] = *reinterpret_cast<const Pack<T, V>*>(row + at[n].second);
            }
    }
    __device__ void store(T* row, const Values<V> (&p)[NV], const Values<V> (&q)[NV]) const {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            if (!mine[n]) continue;
            Pack<T, V> x, y;
            if constexpr (V == 1) {
                float lo, none;
                tc::split(p[n].v[0], lo, none);
                x.v[0] = from_f32<T>(lo);
                tc::split(q[n].v[0], lo, none);
                y.v[0] = from_f32<T>(lo);
            } else {
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    float a0, a1, b0, b1;
                    tc::split(p[n].v[e / 2], a0, a1);
                    tc::split(q[n].v[e / 2], b0, b1);
                    if constexpr (NB) {  // pair e is the values 2 e and 2 e + 1
                        two_to(2 * e < V ? x : y, 2 * e % V, a0, b0);
                        two_to(2 * e + 2 < V ? x : y, (2 * e + 2) % V, a1, b1);
                    } else {
                        two_to(x, e, a0, a1);
                        two_to(y, e, b0, b1);
                    }
                }
            }
            *reinterpret_cast<Pack<T, V>*>(row + at[n].first) = x;
            if (V > 1 || at[n].second >= 0) *reinterpret_cast<Pack<T, V>*>(row + at[n].second) = y;
        }
    }
    static __device__ __forceinline__ void two_to(Pack<T, V>& x, int i, float lo, float hi) {
        if constexpr (std::is_same_v<T, __half>) reinterpret_cast<__half2*>(x.v)[i / 2] = __floats2half2_rn(lo, hi);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) reinterpret_cast<__nv_bfloat162*>(x.v)[i / 2] = __floats2bfloat162_rn(lo, hi);
        else x.v[i] = lo, x.v[i + 1] = hi;
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
    // The place in the head of the first (second) value of a slot's pair e; -1: there is none.
    static __device__ int place(const Slot& s, int e, int second) {
        if constexpr (NB) {
            const int i = 2 * e + second;
            return i < V ? s.first + i : s.second < 0 ? -1 : s.second + i - V;
        } else {
            return second ? (s.second < 0 ? -1 : s.second + e) : s.first + e;
        }
    }
    static __device__ void unpack(const Row<T, V, NV>& r, Values<V> (&p)[NV], Values<V> (&q)[NV]) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const auto get = [&](int i, int second) { return i < V ? to_f32(*value(r.first[n], r.second[n], i, second)) : 0.f; };
                p[n].v[e / 2] = tc::two(get(e, 0), get(e + 1, 0));
                q[n].v[e / 2] = tc::two(get(e, 1), get(e + 1, 1));
            }
    }
    __device__ float group_sum(tc::Two x) const {
        float lo, hi;
        tc::split(x, lo, hi);
        lo += hi;
        for (int o = a.lanes / 2; o; o >>= 1) lo += __shfl_xor_sync(kFullMask, lo, o);
        return lo;
    }
    __device__ float rstd(const Values<V> (&p)[NV], const Values<V> (&q)[NV]) const {
        tc::Two ss = tc::two(0.f, 0.f);
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < N; ++e) ss = tc::fma2(p[n].v[e], p[n].v[e], tc::fma2(q[n].v[e], q[n].v[e], ss));
        return __frsqrt_rn(fmaf(group_sum(ss), a.inv_dim, a.eps));
    }
};

// Calls f(half, base of the token's rows as offsets, first turn, end) for the queries' and the keys' turns of a unit.
template <typename F>
__device__ __forceinline__ void rot_halves(const RotArgs& a, int chunk, F&& f) {
    const int begin = chunk * a.chunk, end = min(begin + a.chunk, a.half[0].turns + a.half[1].turns), q = a.half[0].turns;
    if (begin < q) f(std::integral_constant<int, 0>{}, begin, min(end, q));
    if (end > q) f(std::integral_constant<int, 1>{}, max(begin, q) - q, end - q);
}

constexpr int kFwdAhead = 4, kBwdAhead = 2;  // rows of a group that are asked for at once

template <typename T, int V, bool NB, int NV>
__global__ void __launch_bounds__(kRotThreads, V == 1 ? 2 : 5) rotary_fwd_kernel(const __grid_constant__ RotArgs a) {
    const Rot<T, V, NB, NV> me(a);
    using Me = Rot<T, V, NB, NV>;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRotWarps;
    const tc::Two minus = tc::two(-1.f, -1.f);
    Row<T, V, NV> row[kFwdAhead] = {};
    int64_t unit = static_cast<int64_t>(blockIdx.x) * kRotWarps + (threadIdx.x >> 5);
    double position = me.position(unit);
    for (; unit < a.units; unit += step) {
        const auto token = me.token_of(unit);
        bool made = false;
        rot_halves(a, token.chunk, [&](auto k, int turn, int end) {
            const RotHalf& h = a.half[k];
            const T* x = static_cast<const T*>(h.x) + token.batch * h.x_batch + token.token * h.x_token + (turn * me.rows + me.group) * h.x_head;
            T* out = static_cast<T*>(h.out) + token.batch * h.out_batch + token.token * h.out_token + (turn * me.rows + me.group) * h.out_head;
            const int64_t x_step = me.rows * h.x_head, out_step = me.rows * h.out_head;
            const float* weights = me.weights + k * 2 * a.slots * V;
            int left = h.heads - turn * me.rows - me.group;
            for (; turn < end; turn += kFwdAhead) {
#pragma unroll
                for (int i = 0; i < kFwdAhead; ++i, x += x_step) me.load(row[i], x, turn + i < end && left > i * me.rows);
                if (!made) {
                    me.angles(position);
                    position = me.position(unit + step);
                    made = true;
                }
#pragma unroll
                for (int i = 0; i < kFwdAhead; ++i, out += out_step) {
                    if (turn + i >= end) break;
                    Values<V> p[NV], q[NV];
                    Me::unpack(row[i], p, q);
                    if (a.norm) {
                        const float r = me.rstd(p, q);
                        const tc::Two rr = tc::two(r, r);
#pragma unroll
                        for (int n = 0; n < NV; ++n) {
                            const Values<V> w0 = me.entries(weights, n, 0), w1 = me.entries(weights, n, V);
#pragma unroll
                            for (int e = 0; e < Me::N; ++e) {
                                p[n].v[e] = tc::mul2(tc::mul2(p[n].v[e], rr), w0.v[e]);
                                q[n].v[e] = tc::mul2(tc::mul2(q[n].v[e], rr), w1.v[e]);
                            }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NV; ++n) {
                        const Values<V> c = me.entries(me.table, n, 0), s = me.entries(me.table, n, V);
#pragma unroll
                        for (int e = 0; e < Me::N; ++e) {
                            const tc::Two u1 = p[n].v[e], u2 = q[n].v[e];
                            p[n].v[e] = tc::fma2(u1, c.v[e], tc::mul2(tc::mul2(u2, minus), s.v[e]));
                            q[n].v[e] = tc::fma2(u1, s.v[e], tc::mul2(u2, c.v[e]));
                        }
                    }
                    if (left > i * me.rows) me.store(out, p, q);
                }
                left -= kFwdAhead * me.rows;
            }
        });
    }
}

template <typename T, int V, bool NB, int NV>
__global__ void __launch_bounds__(kRotThreads, V == 1 ? 2 : 4) rotary_bwd_kernel(const __grid_constant__ RotArgs a) {
    const Rot<T, V, NB, NV> me(a);
    using Me = Rot<T, V, NB, NV>;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRotWarps;
    const tc::Two minus = tc::two(-1.f, -1.f);
    Values<V> sum[2][2][NV];  // of queries and keys, first values and partners
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i)
#pragma unroll
        for (int e = 0; e < Me::N; ++e) sum[i / NV / 2][i / NV % 2][i % NV].v[e] = tc::two(0.f, 0.f);
    Row<T, V, NV> x_row[kBwdAhead] = {}, g_row[kBwdAhead] = {};
    int64_t unit = static_cast<int64_t>(blockIdx.x) * kRotWarps + (threadIdx.x >> 5);
    double position = me.position(unit);
    for (; unit < a.units; unit += step) {
        const auto token = me.token_of(unit);
        bool made = false;
        rot_halves(a, token.chunk, [&](auto k, int turn, int end) {
            const RotHalf& h = a.half[k];
            const int head = turn * me.rows + me.group;
            const T* x = static_cast<const T*>(h.x) + token.batch * h.x_batch + token.token * h.x_token + head * h.x_head;
            const T* g = static_cast<const T*>(h.g) + token.batch * h.g_batch + token.token * h.g_token + head * h.g_head;
            T* out = static_cast<T*>(h.out) + token.batch * h.out_batch + token.token * h.out_token + head * h.out_head;
            const int64_t x_step = me.rows * h.x_head, g_step = me.rows * h.g_head, out_step = me.rows * h.out_head;
            const float* weights = me.weights + k * 2 * a.slots * V;
            int left = h.heads - head;
            for (; turn < end; turn += kBwdAhead) {
#pragma unroll
                for (int i = 0; i < kBwdAhead; ++i, x += x_step, g += g_step) {
                    const bool there = turn + i < end && left > i * me.rows;
                    me.load(g_row[i], g, there);
                    me.load(x_row[i], x, there && a.norm);
                }
                if (!made) {
                    me.angles(position);
                    position = me.position(unit + step);
                    made = true;
                }
#pragma unroll
                for (int i = 0; i < kBwdAhead; ++i, out += out_step) {
                    if (turn + i >= end) break;
                    const bool there = left > i * me.rows;
                    Values<V> p[NV], q[NV];
                    Me::unpack(g_row[i], p, q);
#pragma unroll
                    for (int n = 0; n < NV; ++n) {
                        const Values<V> c = me.entries(me.table, n, 0), s = me.entries(me.table, n, V);
#pragma unroll
                        for (int e = 0; e < Me::N; ++e) {
                            const tc::Two g1 = p[n].v[e], g2 = q[n].v[e];
                            p[n].v[e] = tc::fma2(g1, c.v[e], tc::mul2(g2, s.v[e]));
                            q[n].v[e] = tc::fma2(g2, c.v[e], tc::mul2(tc::mul2(g1, minus), s.v[e]));
                        }
                    }
                    if (a.norm) {
                        Values<V> x0[NV], x1[NV];
                        Me::unpack(x_row[i], x0, x1);
                        const float r = me.rstd(x0, x1);
                        const tc::Two rr = tc::two(r, r);
                        tc::Two dot = tc::two(0.f, 0.f);
#pragma unroll
                        for (int n = 0; n < NV; ++n) {
                            const Values<V> w0 = me.entries(weights, n, 0), w1 = me.entries(weights, n, V);
#pragma unroll
                            for (int e = 0; e < Me::N; ++e) {
                                x0[n].v[e] = tc::mul2(x0[n].v[e], rr), x1[n].v[e] = tc::mul2(x1[n].v[e], rr);
                                if (there) {  // of a group without a row r may be infinite
                                    sum[k][0][n].v[e] = tc::fma2(p[n].v[e], x0[n].v[e], sum[k][0][n].v[e]);
                                    sum[k][1][n].v[e] = tc::fma2(q[n].v[e], x1[n].v[e], sum[k][1][n].v[e]);
                                }
                                p[n].v[e] = tc::mul2(p[n].v[e], w0.v[e]), q[n].v[e] = tc::mul2(q[n].v[e], w1.v[e]);
                                dot = tc::fma2(p[n].v[e], x0[n].v[e], tc::fma2(q[n].v[e], x1[n].v[e], dot));
                            }
                        }
                        const float m = -me.group_sum(dot) * a.inv_dim;
                        const tc::Two mm = tc::two(m, m);
#pragma unroll
                        for (int n = 0; n < NV; ++n)
#pragma unroll
                            for (int e = 0; e < Me::N; ++e) {
                                p[n].v[e] = tc::mul2(tc::fma2(x0[n].v[e], mm, p[n].v[e]), rr);
                                q[n].v[e] = tc::mul2(tc::fma2(x1[n].v[e], mm, q[n].v[e]), rr);
                            }
                    }
                    if (there) me.store(out, p, q);
                }
                left -= kBwdAhead * me.rows;
            }
        });
    }
    if (!a.half[0].part && !a.half[1].part) return;
    // the warp's groups, then the CTA's warps, in order
    float* sums = reinterpret_cast<float*>(rot_smem);  // [warps, dim], over the tables
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (!a.half[k].part) continue;
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float x[2], lo, hi;
                tc::split(sum[k][0][n].v[e / 2], lo, hi);
                x[0] = e % 2 ? hi : lo;
                tc::split(sum[k][1][n].v[e / 2], lo, hi);
                x[1] = e % 2 ? hi : lo;
                for (int o = 16; o >= a.lanes; o >>= 1)
                    x[0] += __shfl_xor_sync(kFullMask, x[0], o), x[1] += __shfl_xor_sync(kFullMask, x[1], o);
                if (me.group == 0 && me.mine[n]) {
                    const int i = Me::place(me.at[n], e, 0), j = Me::place(me.at[n], e, 1);
                    sums[(threadIdx.x >> 5) * a.dim + i] = x[0];
                    if (j >= 0) sums[(threadIdx.x >> 5) * a.dim + j] = x[1];
                }
            }
        __syncthreads();
        for (int i = threadIdx.x; i < a.dim; i += kRotThreads) {
            float x = 0.f;
            for (int w = 0; w < kRotWarps; ++w) x += sums[w * a.dim + i];
            a.half[k].part[static_cast<int64_t>(blockIdx.x) * a.dim + i] = x;
        }
    }
}

// Adds the CTAs' sums of 32 values: warp w takes every 32nd row, then the warps are added in order.
__global__ void __launch_bounds__(1024) rotary_sums_kernel(const float* q_part, const float* k_part, int64_t rows, int32_t dim, void* v_qw, void* v_kw, int32_t param_dtype) {
    __shared__ float sums[32][33];
    const bool k = blockIdx.y;
    const float* part = k ? k_part : q_part;
    void* to = k ? v_kw : v_qw;
    if (!to) return;
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
constexpr int kRotMostPerSm = 8;
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

// Units of work: a token with all its heads, so that its sines are taken once; where there are fewer tokens
// than half the warps that fit, one turn of a warp's groups.
template <typename K>
int rot_divide(RotArgs& a, int64_t tokens, K kernel, size_t smem) {
    int per_sm = 0;
    cuda_check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kRotThreads, smem), "qk_norm_rotary");
    const int64_t most = static_cast<int64_t>(sm_count()) * std::min(std::max(per_sm, 1), kRotMostPerSm);
    const int rows = 32 / a.lanes;
    for (RotHalf& h : a.half) h.turns = (h.heads + rows - 1) / rows;
    const int turns = a.half[0].turns + a.half[1].turns;
    a.chunk = tokens * 2 >= most * kRotWarps ? turns : 1;
    a.chunks = (turns + a.chunk - 1) / a.chunk;
    a.units = tokens * a.chunks;
    return static_cast<int>(std::min(most, (a.units + kRotWarps - 1) / kRotWarps));
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
    by_layout(in, v, [&](auto t, auto n, auto nb, auto slots) {
        constexpr int V = decltype(n)::value, NV = decltype(slots)::value;
        constexpr bool NB = decltype(nb)::value;
        const auto kernel = rotary_fwd_kernel<decltype(t), V, NB, NV>;
        const size_t smem = Rot<decltype(t), V, NB, NV>::smem_bytes(a);
        const int blocks = rot_divide(a, tokens, kernel, smem);
        SX_LAUNCH(kernel, blocks, kRotThreads, smem, s, a);
    });
}

size_t qk_norm_rotary_bwd_workspace(const SxRotaryInputs& in) {
    return in.norm ? static_cast<size_t>(sm_count()) * kRotMostPerSm * 2 * in.head_dim * 4 : 0;
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
    by_layout(in, v, [&](auto t, auto n, auto nb, auto slots) {
        constexpr int V = decltype(n)::value, NV = decltype(slots)::value;
        constexpr bool NB = decltype(nb)::value;
        const auto kernel = rotary_bwd_kernel<decltype(t), V, NB, NV>;
        const size_t smem = std::max<size_t>(Rot<decltype(t), V, NB, NV>::smem_bytes(a), static_cast<size_t>(kRotWarps) * in.head_dim * 4);
        const int blocks = rot_divide(a, tokens, kernel, smem);
        float* part = static_cast<float*>(ws);
        if (g.v_q_weight) a.half[0].part = part;
        if (g.v_k_weight) a.half[1].part = part + static_cast<int64_t>(blocks) * in.head_dim;
        SX_LAUNCH(kernel, blocks, kRotThreads, smem, s, a);
        if (g.v_q_weight || g.v_k_weight)
            SX_LAUNCH(rotary_sums_kernel, dim3(blocks_for(in.head_dim, 32), 2), 1024, 0, s, a.half[0].part, a.half[1].part, blocks,
                      in.head_dim, g.v_q_weight, g.v_k_weight, in.param_dtype);
    });
}

}  // namespace sx

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
// in the same way. The token's rows come to shared memory by bulk copies, while other warps work on theirs,
// and leave from their place there by bulk copies: the loops then have no addresses of memory and no
// registers for rows on their way. Rows that such copies do not reach (16 bytes) are read and written value by
// value.
// Angles: position x frequency in turns, the frequency / 2 pi and the product as two 64-bit numbers each, whole turns
// taken off both and then the nearest quarter; what is left is at most an eighth, which 32 bits have to 2^-28 of a
// turn. N turns are off by N 2^-104 of one; from 2^80 on the angle is 0.
#include <algorithm>
#include <cmath>

#include "sx_internal.h"
#include "sx_network.h"
#include "sx_tcgen05.cuh"

namespace sx {

__device__ uint32_t g_rotary_status;

uint32_t rotary_status() {
    uint32_t st = 0;
    const uint32_t zero = 0;
    cuda_check(cudaDeviceSynchronize(), "rotary_status");
    cuda_check(cudaMemcpyFromSymbol(&st, g_rotary_status, sizeof(st)), "rotary_status");
    if (st) cuda_check(cudaMemcpyToSymbol(g_rotary_status, &zero, sizeof(zero)), "rotary_status");
    return st;
}

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
    int32_t stage;          // bytes of a unit's rows of one kind in shared memory
    int32_t pos_dtype, param_dtype, axes, dim, pairs, slots, lanes;  // slots: V pairs each; lanes: of a row's group
    int32_t mode, norm;
    int32_t axis_dims[4];
    float eps, inv_dim;
    double turns[2][kRotMostPairs];  // frequency / 2 pi, and what that lacks
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

// V values in pairs that one instruction works on.
template <int V>
struct Values {
    static constexpr int N = (V + 1) / 2;
    tc::Two v[N];
};

// A unit's rows of queries or keys: heads from `head` on, `n` of them, row `at` of the unit's first.
struct RotRun {
    int head, n, at;
};
__device__ __forceinline__ RotRun rot_run(const RotArgs& a, int rows, int chunk, int k) {
    const int begin = chunk * a.chunk, end = min(begin + a.chunk, a.half[0].turns + a.half[1].turns), q = a.half[0].turns;
    const int from = k ? max(begin, q) - q : begin, to = k ? end - q : min(end, q);
    return {from * rows, max(min(to * rows, a.half[k].heads) - from * rows, 0), k ? (max(begin, q) - begin) * rows : 0};
}

constexpr int kTable = 2 * kRotMostPairs;  // floats of a table: V first entries and V seconds of up to 128 / V slots

struct RotShared {
    alignas(16) float weights[2][kTable];       // of queries and keys
    alignas(16) float angles[kRotWarps][kTable];  // cosines and sines of each warp's token
    double turns[2][kRotMostPairs];
    uint64_t full[kRotWarps];  // barriers of the stages
    uint8_t axis[kRotMostPairs];
    uint32_t failed;
};

// The thread's part of a kernel.
template <typename T, int V, bool NB, int NV>
struct Rot {
    static constexpr int W = V < 4 ? V : 4;                   // values of a table access
    static constexpr int kPiece = kRotMostPairs / V * W;      // floats from an access' entries to the slots' next ones
    static constexpr int N = Values<V>::N;
    const RotArgs& a;
    RotShared& sh;
    float* table;
    int lane, group, in_group, rows;  // rows: groups of a warp
    int first[NV], second[NV];        // where the slots are in a head; 0 where the slot is not the thread's own
    bool mine[NV], pair[NV], turned[NV];

    __device__ Rot(const RotArgs& a, RotShared& sh) : a(a), sh(sh), table(sh.angles[threadIdx.x >> 5]), lane(threadIdx.x & 31) {
        for (int i = threadIdx.x; i < a.pairs; i += kRotThreads) sh.turns[0][i] = a.turns[0][i], sh.turns[1][i] = a.turns[1][i], sh.axis[i] = a.axis[i];
        for (int i = threadIdx.x; i < 2 * a.slots * V; i += kRotThreads) {
            const int k = i >= a.slots * V, at = i - k * a.slots * V;
            const Slot s = slot_at<V>(a, at / V);
            const int one = place(s.first, s.second, at % V, 0), two = place(s.first, s.second, at % V, 1);
            *entry(sh.weights[k], at, 0) = rot_param(a.half[k].weight, a.param_dtype, one);
            *entry(sh.weights[k], at, V) = two < 0 ? 0.f : rot_param(a.half[k].weight, a.param_dtype, two);
        }
        group = lane / a.lanes;
        in_group = lane % a.lanes;
        rows = 32 / a.lanes;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int slot = in_group + n * a.lanes;
            mine[n] = slot < a.slots;
            turned[n] = slot * V < a.pairs;
            const Slot s = mine[n] ? slot_at<V>(a, slot) : Slot{0, 0};
            pair[n] = V > 1 || s.second >= 0;
            first[n] = s.first, second[n] = pair[n] ? s.second : 0;
        }
        for (int i = lane; i < a.slots * V; i += 32) *entry(table, i, 0) = 1.f, *entry(table, i, V) = 0.f;  // not rotated
        __syncthreads();
    }
    static __device__ float* entry(float* t, int pair, int skip) {
        const int slot = pair / V, e = pair % V + skip;
        return t + e / W * kPiece + slot * W + e % W;
    }
    // The entries of the thread's slot n: V of them from `skip`.
    __device__ __forceinline__ Values<V> entries(const float* t, int n, int skip) const {
        const int slot = mine[n] ? in_group + n * a.lanes : 0;
        const float* from = t + slot * W;
        Values<V> r;
#pragma unroll
        for (int e = 0; e < V; e += W) {
            const auto x = *reinterpret_cast<const Pack<float, W>*>(from + (skip + e) / W * kPiece);
            if constexpr (W == 1) {
                r.v[0] = tc::two(x.v[0], 0.f);
            } else {
#pragma unroll
                for (int k = 0; k < W; k += 2) r.v[(e + k) / 2] = tc::two(x.v[k], x.v[k + 1]);
            }
        }
        return r;
    }
    // A unit of work, and what of it are queries' and keys' rows.
    struct Unit {
        int64_t batch, token;
        int chunk;
        RotRun run[2];
    };
    __device__ Unit first_unit(int64_t unit) const {
        const int64_t t = unit / a.chunks, b = t / a.tokens;
        Unit u{b, t - b * a.tokens, static_cast<int>(unit - t * a.chunks), {}};
        u.run[0] = rot_run(a, rows, u.chunk, 0), u.run[1] = rot_run(a, rows, u.chunk, 1);
        return u;
    }
    __device__ void next_unit(Unit& u, int step) const {  // `step` units on
        if (a.chunks > 1) {
            const uint32_t c = static_cast<uint32_t>(u.chunk + step), t = c / static_cast<uint32_t>(a.chunks);
            u.chunk = static_cast<int>(c - t * a.chunks);
            u.token += t;
            u.run[0] = rot_run(a, rows, u.chunk, 0), u.run[1] = rot_run(a, rows, u.chunk, 1);
        } else {
            u.token += step;
        }
        if (u.token >= a.tokens) {
            const uint32_t t = static_cast<uint32_t>(u.token), n = static_cast<uint32_t>(a.tokens), b = t / n;  // both below 2^31
            u.token = t - b * n;
            u.batch += b;
        }
    }
    // Lane i's position along axis i.
    __device__ double position(const Unit& t) const {
        if (lane >= a.axes) return 0.;
        const int64_t i = t.batch * a.pos_batch + t.token * a.pos_token + lane * a.pos_axis;
        if (a.pos_dtype == SXCUDA_POS_F32) return static_cast<const float*>(a.positions)[i];
        if (a.pos_dtype == SXCUDA_POS_I32) return static_cast<const int32_t*>(a.positions)[i];
        return static_cast<double>(static_cast<const int64_t*>(a.positions)[i]);
    }
    __device__ void angles(double mine_position) const {
        __syncwarp();
        for (int i = lane; i - lane < a.pairs; i += 32) {
            const int j = i < a.pairs ? i : 0;
            const double at = __shfl_sync(kFullMask, mine_position, sh.axis[j]), turn = sh.turns[0][j];
            const double all = at * turn, rest = fma(at, sh.turns[1][j], fma(at, turn, -all));
            // of a position that is not finite NaN is left
            const double t = fabs(all) < 0x1p80 ? (all - rint(all)) + (rest - rint(rest)) : at - at;
            // t in quarters, rounded to a whole number by the sum: its low bits say which quarter
            const double magic = 6755399441055744., up = fma(4., t, magic);
            const int q = __double2loint(up);
            const float2 cs = eighth(static_cast<float>(fma(-0.25, up - magic, t)));
            const float c = q & 1 ? cs.y : cs.x, s = q & 1 ? cs.x : cs.y;
            if (i < a.pairs) {
                *entry(table, i, 0) = __uint_as_float(__float_as_uint(c) ^ static_cast<uint32_t>(q + 1 & 2) << 30);
                *entry(table, i, V) = __uint_as_float(__float_as_uint(s) ^ static_cast<uint32_t>(q & 2) << 30);
            }
        }
        __syncwarp();
    }
    // Cosine and sine of r turns, |r| <= 1/8, by their series to the 10th and 9th power (1.1e-10 and 2e-9 are left).
    static __device__ __forceinline__ float2 eighth(float r) {
        const float x = 6.2831853071795865f * r, z = x * x;
        float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
        c = fmaf(z, c, -1.3888889e-3f);
        c = fmaf(z, c, 4.1666667e-2f);
        c = fmaf(z, c, -0.5f);
        float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
        s = fmaf(z, s, 8.3333333e-3f);
        s = fmaf(z, s, -1.6666667e-1f);
        return {fmaf(z, c, 1.f), fmaf(x * z, s, x)};
    }
    // The place in the head of the first (second) value of a slot's pair e; -1: there is none.
    static __device__ int place(int first, int second, int e, int which) {
        if constexpr (NB) {
            const int i = 2 * e + which;
            return i < V ? first + i : second < 0 ? -1 : second + i - V;
        } else {
            return which ? (second < 0 ? -1 : second + e) : first + e;
        }
    }
    // A row's values, first ones and partners. A slot that is not the thread's own has others' values, which its sums
    // leave out.
    __device__ __forceinline__ void load(const T* row, Values<V> (&p)[NV], Values<V> (&q)[NV]) const {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const auto x = *reinterpret_cast<const Pack<T, V>*>(row + first[n]), y = *reinterpret_cast<const Pack<T, V>*>(row + second[n]);
            if constexpr (V == 1) {
                p[n].v[0] = tc::two(to_f32(x.v[0]), 0.f);
                q[n].v[0] = tc::two(pair[n] ? to_f32(y.v[0]) : 0.f, 0.f);
            } else {
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    if constexpr (NB) {  // pair e is the values 2 e and 2 e + 1
                        const float2 one = two_of(2 * e < V ? x : y, 2 * e % V), other = two_of(2 * e + 2 < V ? x : y, (2 * e + 2) % V);
                        p[n].v[e / 2] = tc::two(one.x, other.x), q[n].v[e / 2] = tc::two(one.y, other.y);
                    } else {
                        const float2 one = two_of(x, e), other = two_of(y, e);
                        p[n].v[e / 2] = tc::two(one.x, one.y), q[n].v[e / 2] = tc::two(other.x, other.y);
                    }
                }
            }
        }
    }
    __device__ __forceinline__ void store(T* row, const Values<V> (&p)[NV], const Values<V> (&q)[NV]) const {
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
                    if constexpr (NB) {
                        two_to(2 * e < V ? x : y, 2 * e % V, a0, b0);
                        two_to(2 * e + 2 < V ? x : y, (2 * e + 2) % V, a1, b1);
                    } else {
                        two_to(x, e, a0, a1);
                        two_to(y, e, b0, b1);
                    }
                }
            }
            *reinterpret_cast<Pack<T, V>*>(row + first[n]) = x;
            if (pair[n]) *reinterpret_cast<Pack<T, V>*>(row + second[n]) = y;
        }
    }
    static __device__ __forceinline__ float2 two_of(const Pack<T, V>& x, int i) {
        if constexpr (std::is_same_v<T, __half>) return __half22float2(reinterpret_cast<const __half2*>(x.v)[i / 2]);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(x.v)[i / 2]);
        else return {x.v[i], x.v[i + 1]};
    }
    static __device__ __forceinline__ void two_to(Pack<T, V>& x, int i, float lo, float hi) {
        if constexpr (std::is_same_v<T, __half>) reinterpret_cast<__half2*>(x.v)[i / 2] = __floats2half2_rn(lo, hi);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) reinterpret_cast<__nv_bfloat162*>(x.v)[i / 2] = __floats2bfloat162_rn(lo, hi);
        else x.v[i] = lo, x.v[i + 1] = hi;
    }
    static __device__ float both(tc::Two x) {
        float lo, hi;
        tc::split(x, lo, hi);
        return lo + hi;
    }
    __device__ float group_sum(float x) const {
#pragma unroll
        for (int o = 16; o; o >>= 1)
            if (a.lanes > o) x += __shfl_xor_sync(kFullMask, x, o);
        return x;
    }
    __device__ float rstd(const Values<V> (&p)[NV], const Values<V> (&q)[NV]) const {
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            tc::Two ss = tc::two(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < N; ++e) ss = tc::fma2(p[n].v[e], p[n].v[e], tc::fma2(q[n].v[e], q[n].v[e], ss));
            sum += mine[n] ? both(ss) : 0.f;
        }
        return rsqrtf(fmaf(group_sum(sum), a.inv_dim, a.eps));  // within 2 units of the last place
    }

    // What a token's rows of queries or of keys are multiplied by: weight times cosine and sine, for a pair
    // (x1, x2) -> (x1 a - x2 b, x1 c + x2 d).
    struct Turn {
        Values<V> a[NV], b[NV], c[NV], d[NV];  // b with its sign turned
    };
    __device__ __forceinline__ void turn_of(int k, Turn& t) const {
        const tc::Two minus = tc::two(-1.f, -1.f);
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const Values<V> cosine = entries(table, n, 0), sine = entries(table, n, V);
            const Values<V> w0 = entries(sh.weights[k], n, 0), w1 = entries(sh.weights[k], n, V);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                t.a[n].v[e] = tc::mul2(w0.v[e], cosine.v[e]), t.c[n].v[e] = tc::mul2(w0.v[e], sine.v[e]);
                t.b[n].v[e] = tc::mul2(tc::mul2(w1.v[e], sine.v[e]), minus), t.d[n].v[e] = tc::mul2(w1.v[e], cosine.v[e]);
            }
        }
    }
    // A row of the group's, forward: from `x` to `out` where there is one. REST: the head has values that are not rotated,
    // which are left out of the turn: times a sine of zero an infinite one would be NaN in a value that has no part in
    // it. That costs 1 to 4% (4 x 8192 tokens, 16 (4) heads x 128, 96 of them rotated 64 -> 66 us, backward 105 -> 106), which
    // heads that are rotated as a whole do not pay: a kernel each.
    template <bool REST>
    __device__ __forceinline__ void forward(const T* x, T* out, const Turn& t, bool there) const {
        Values<V> p[NV], q[NV];
        load(x, p, q);
        if (a.norm) {
            const float r = rstd(p, q);
            const tc::Two rr = tc::two(r, r);
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int e = 0; e < N; ++e) p[n].v[e] = tc::mul2(p[n].v[e], rr), q[n].v[e] = tc::mul2(q[n].v[e], rr);
        }
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const tc::Two x1 = p[n].v[e], x2 = q[n].v[e];
                const tc::Two other = tc::mul2(x2, t.b[n].v[e]);
                if (REST) p[n].v[e] = tc::mul2(x1, t.a[n].v[e]);
                q[n].v[e] = tc::mul2(x2, t.d[n].v[e]);
                if (!REST || turned[n]) p[n].v[e] = tc::fma2(x1, t.a[n].v[e], other), q[n].v[e] = tc::fma2(x1, t.c[n].v[e], q[n].v[e]);
            }
        if (there) store(out, p, q);
    }
    // The same backward, from the gradient `g` (and x, with norm) to `out`; adds to the weight's sums.
    template <bool REST>
    __device__ __forceinline__ void backward(const T* x, const T* g, T* out, int k, bool there, Values<V> (&sum)[2][NV]) const {
        const tc::Two minus = tc::two(-1.f, -1.f);
        Values<V> p[NV], q[NV];
        load(g, p, q);
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const Values<V> c = entries(table, n, 0), s = entries(table, n, V);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const tc::Two g1 = p[n].v[e], g2 = q[n].v[e];
                const tc::Two u1 = tc::fma2(g1, c.v[e], tc::mul2(g2, s.v[e])), u2 = tc::fma2(g2, c.v[e], tc::mul2(tc::mul2(g1, minus), s.v[e]));
                if (!REST || turned[n]) p[n].v[e] = u1, q[n].v[e] = u2;
            }
        }
        if (a.norm) {
            Values<V> x0[NV], x1[NV];
            load(x, x0, x1);
            const float r = rstd(x0, x1);
            const tc::Two rr = tc::two(r, r);
            float dots = 0.f;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                tc::Two dot = tc::two(0.f, 0.f);
                const Values<V> w0 = entries(sh.weights[k], n, 0), w1 = entries(sh.weights[k], n, V);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    x0[n].v[e] = tc::mul2(x0[n].v[e], rr), x1[n].v[e] = tc::mul2(x1[n].v[e], rr);
                    if (there) {  // what a group without a row has read is nothing
                        sum[0][n].v[e] = tc::fma2(p[n].v[e], x0[n].v[e], sum[0][n].v[e]);
                        sum[1][n].v[e] = tc::fma2(q[n].v[e], x1[n].v[e], sum[1][n].v[e]);
                    }
                    p[n].v[e] = tc::mul2(p[n].v[e], w0.v[e]), q[n].v[e] = tc::mul2(q[n].v[e], w1.v[e]);
                    dot = tc::fma2(p[n].v[e], x0[n].v[e], tc::fma2(q[n].v[e], x1[n].v[e], dot));
                }
                dots += mine[n] ? both(dot) : 0.f;
            }
            const float m = -group_sum(dots) * a.inv_dim;
            const tc::Two mm = tc::two(m, m);
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    p[n].v[e] = tc::mul2(tc::fma2(x0[n].v[e], mm, p[n].v[e]), rr);
                    q[n].v[e] = tc::mul2(tc::fma2(x1[n].v[e], mm, q[n].v[e]), rr);
                }
        }
        if (there) store(out, p, q);
    }
    // The CTA's sums for the weights' gradients: its warps' groups, then its warps, in order.
    __device__ void leave(const Values<V> (&sum)[2][2][NV]) const {
        float* sums = sh.angles[0];  // [warps, dim], over the tables
        static_assert(sizeof(sh.angles) >= kRotWarps * 256 * 4);
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
                    if (group == 0 && mine[n]) {
                        const int i = place(first[n], second[n], e, 0), j = place(first[n], second[n], e, 1);
                        sums[(threadIdx.x >> 5) * a.dim + i] = x[0];
                        if (pair[n]) sums[(threadIdx.x >> 5) * a.dim + j] = x[1];
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
};

template <int V, int NV>
__device__ __forceinline__ void no_sums(Values<V> (&sum)[2][2][NV]) {
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i)
#pragma unroll
        for (int e = 0; e < Values<V>::N; ++e) sum[i / NV / 2][i / NV % 2][i % NV].v[e] = tc::two(0.f, 0.f);
}

// CTAs an SM holds by their registers.
template <int V, bool BACK>
constexpr int kRotPerSm = V > 2 ? (BACK ? 4 : 6) : V == 2 ? (BACK ? 4 : 6) : (BACK ? 2 : 4);
constexpr int kRotMostPerSm = 7;

// Rows value by value.
template <typename T, bool BACK>
__global__ void __launch_bounds__(kRotThreads, kRotPerSm<1, BACK>) rotary_plain_kernel(const __grid_constant__ RotArgs a) {
    __shared__ RotShared sh;
    const Rot<T, 1, false, 4> me(a, sh);
    Values<1> sum[2][2][4];
    no_sums(sum);
    const int step = static_cast<int>(gridDim.x) * kRotWarps;
    int64_t unit = static_cast<int64_t>(blockIdx.x) * kRotWarps + (threadIdx.x >> 5);
    auto token = me.first_unit(unit);
    for (; unit < a.units; unit += step, me.next_unit(token, step)) {
        me.angles(me.position(token));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const RotHalf& h = a.half[k];
            const RotRun run = token.run[k];
            typename Rot<T, 1, false, 4>::Turn turn;
            if (!BACK && run.n) me.turn_of(k, turn);
            for (int i = 0; i < run.n; i += me.rows) {
                const bool there = i + me.group < run.n;
                const int64_t head = run.head + (there ? i + me.group : i);
                const auto row = [&](const void* p, int64_t batch, int64_t tokens, int64_t heads) {
                    return static_cast<const T*>(p) + token.batch * batch + token.token * tokens + head * heads;
                };
                const T* x = row(h.x, h.x_batch, h.x_token, h.x_head);
                T* out = const_cast<T*>(row(h.out, h.out_batch, h.out_token, h.out_head));
                if constexpr (BACK) me.template backward<true>(x, row(h.g, h.g_batch, h.g_token, h.g_head), out, k, there, sum[k]);
                else me.template forward<true>(x, out, turn, there);
            }
        }
    }
    if constexpr (BACK) me.leave(sum);
}

// Rows by bulk copies: each warp has a stage for a unit's rows (backward: of the gradient, then of x). While it
// fills, other warps work: more warps with a stage each were faster than fewer with two (68 and 72 us for
// 4 x 8192 tokens, 16 (4) heads x 128; backward of 8 x 4096, 16 heads x 64: 93 and 97 us). The forward has a
// token's weights times sines in registers (66 us; the same read for every row from shared memory 68 us).
// bf16: forward 67 us (5.1 TB/s), backward 95 us (4.3 TB/s; latency: 128 registers leave 16 warps an SM, which issue in 55%
// of the cycles with no pipe full).
__device__ __forceinline__ void bulk_store(void* to, uint32_t from, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(from), "r"(bytes) : "memory");
}

template <typename T, int V, bool NB, int NV, bool REST, bool BACK>
__global__ void __launch_bounds__(kRotThreads, kRotPerSm<V, BACK>) rotary_kernel(const __grid_constant__ RotArgs a) {
    __shared__ RotShared sh;
    extern __shared__ __align__(128) uint8_t stages[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t bar = tc::smem_addr(&sh.full[warp]);
    if (lane == 0) {
        tc::bar_init(bar, 1);
        tc::bar_init_fence();
    }
    if (threadIdx.x == 0) sh.failed = 0;
    const Rot<T, V, NB, NV> me(a, sh);
    volatile uint32_t* failed = &sh.failed;
    const int bytes = a.dim * static_cast<int>(sizeof(T)), stage = a.stage * (BACK ? 2 : 1);
    uint8_t* mine = stages + static_cast<size_t>(warp) * stage;
    const uint32_t mine_at = tc::smem_addr(mine);
    Values<V> sum[2][2][NV];
    no_sums(sum);
    // Where a head's rows lie side by side, lane 0 has the queries' copies and lane 1 the keys'; else a lane has a
    // head's. Each lane's own half, as the first case needs it:
    const RotHalf& own = a.half[lane & 1];
    const bool joined = a.half[0].x_head == a.dim && a.half[0].out_head == a.dim && (!BACK || a.half[0].g_head == a.dim) &&
                        (a.half[1].heads == 0 || (a.half[1].x_head == a.dim && a.half[1].out_head == a.dim && (!BACK || a.half[1].g_head == a.dim)));
    const T* own_x = static_cast<const T*>(own.x);
    const T* own_g = static_cast<const T*>(own.g);
    T* own_out = static_cast<T*>(own.out);
    const int64_t x_batch = own.x_batch, x_token = own.x_token, g_batch = own.g_batch, g_token = own.g_token, out_batch = own.out_batch,
                  out_token = own.out_token;
    const auto rows_of = [](const auto& unit, auto* p, int64_t batch, int64_t tokens, int64_t head) {
        return p + unit.batch * batch + unit.token * tokens + head;
    };
    const auto ask = [&](const typename Rot<T, V, NB, NV>::Unit& unit) {
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // each lane's own: the stage's last rows have left
        __syncwarp();
        if (lane == 0) tc::bar_expect(bar, (unit.run[0].n + unit.run[1].n) * bytes * (BACK && a.norm ? 2 : 1));
        __syncwarp();
        if (joined) {
            const RotRun run = lane ? unit.run[1] : unit.run[0];
            if (lane < 2 && run.n) {
                if (BACK) tc::bulk_load(mine_at + run.at * bytes, rows_of(unit, own_g, g_batch, g_token, run.head * a.dim), run.n * bytes, bar);
                if (!BACK || a.norm)
                    tc::bulk_load(mine_at + (BACK ? a.stage : 0) + run.at * bytes, rows_of(unit, own_x, x_batch, x_token, run.head * a.dim), run.n * bytes, bar);
            }
            return;
        }
        for (int k = 0; k < 2; ++k) {
            const RotHalf& h = a.half[k];
            const RotRun run = unit.run[k];
            for (int i = lane; i < run.n; i += 32) {
                const int64_t head = run.head + i;
                if (BACK) tc::bulk_load(mine_at + (run.at + i) * bytes, rows_of(unit, static_cast<const T*>(h.g), h.g_batch, h.g_token, head * h.g_head), bytes, bar);
                if (!BACK || a.norm)
                    tc::bulk_load(mine_at + (BACK ? a.stage : 0) + (run.at + i) * bytes,
                                  rows_of(unit, static_cast<const T*>(h.x), h.x_batch, h.x_token, head * h.x_head), bytes, bar);
            }
        }
    };
    const auto send = [&](const typename Rot<T, V, NB, NV>::Unit& unit) {
        tc::fence_smem_to_async();
        __syncwarp();
        if (joined) {
            const RotRun run = lane ? unit.run[1] : unit.run[0];
            if (lane < 2 && run.n) bulk_store(rows_of(unit, own_out, out_batch, out_token, run.head * a.dim), mine_at + run.at * bytes, run.n * bytes);
        } else {
            for (int k = 0; k < 2; ++k) {
                const RotHalf& h = a.half[k];
                const RotRun run = unit.run[k];
                for (int i = lane; i < run.n; i += 32)
                    bulk_store(rows_of(unit, static_cast<T*>(h.out), h.out_batch, h.out_token, (run.head + i) * h.out_head), mine_at + (run.at + i) * bytes, bytes);
            }
        }
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    };
    const int step = static_cast<int>(gridDim.x) * kRotWarps;
    int64_t unit = static_cast<int64_t>(blockIdx.x) * kRotWarps + warp;
    bool ok = true;
    auto here = me.first_unit(unit), next = here;
    double position = 0.;
    if (unit < a.units) {
        ask(here);
        position = me.position(here);
    }
    uint32_t parity = 0;
    for (; unit < a.units; unit += step, parity ^= 1) {
        me.angles(position);
        if (unit + step < a.units) {
            me.next_unit(next, step);
            position = me.position(next);
        }
        ok = tc::bar_wait(bar, parity, failed);
        if (!ok) break;
        T* rows = reinterpret_cast<T*>(mine);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const RotRun run = here.run[k];
            T* row = rows + (run.at + me.group) * a.dim;
            typename Rot<T, V, NB, NV>::Turn turn;
            if (!BACK && run.n) me.turn_of(k, turn);
            for (int i = 0; i < run.n; i += me.rows, row += me.rows * a.dim) {
                const bool there = i + me.group < run.n;
                if constexpr (BACK) me.template backward<REST>(row + a.stage / static_cast<int>(sizeof(T)), row, row, k, there, sum[k]);
                else me.template forward<REST>(row, row, turn, there);
            }
        }
        send(here);
        here = next;
        if (unit + step < a.units) ask(here);
    }
    if (!ok) {  // nothing may land in this CTA's memory after it has gone
        tc::bar_drain(bar, parity);
        if (lane == 0) atomicOr(&g_rotary_status, 1u);
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    if constexpr (BACK) me.leave(sum);
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
bool view_fits(const SxAttentionView& x, int64_t size, int64_t bytes) {
    const auto fits = [&](int64_t n) { return n * size % bytes == 0; };
    return reinterpret_cast<uintptr_t>(x.data) % bytes == 0 && fits(x.batch_stride) && fits(x.token_stride) && fits(x.head_stride);
}

// Rows that bulk copies reach.
bool bulk_fits(const SxRotaryInputs& in, const SxAttentionView& x) {
    return in.head_dim * dtype_bytes(in.dtype) % 16 == 0 && view_fits(x, dtype_bytes(in.dtype), 16);
}

int rotated_values(const SxRotaryInputs& in) {
    int n = 0;
    for (int i = 0; i < in.axes; ++i) n += in.axis_dims[i];
    return n;
}

// The most pairs a thread can take at once: runs of pairs, of their partners and of what is not rotated are
// multiples of it.
int most_pairs(const SxRotaryInputs& in) {
    const int pairs = rotated_values(in) / 2, rest = in.head_dim - 2 * pairs;
    const auto holds = [&](int n) {
        if (rest % 2 || rest / 2 % n || pairs % n) return false;
        if (in.pairs == SXCUDA_PAIRS_AXIS)
            for (int i = 0; i < in.axes; ++i)
                if (in.axis_dims[i] / 2 % n) return false;
        return true;
    };
    int v = in.dtype == SXCUDA_F32 ? 4 : 8;
    while (v > 1 && !holds(v)) v /= 2;
    return v;
}

RotArgs rot_args(const SxRotaryInputs& in, int v) {
    RotArgs a{};
    const double tau = 6.283185307179586476925286766559, tau_rest = 2.4492935982947064e-16;  // 2 pi is their sum
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
            const double f = in.freqs[a.pairs], turn = f / tau;
            a.turns[0][a.pairs] = turn, a.turns[1][a.pairs] = (std::fma(-turn, tau, f) - turn * tau_rest) / tau;
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

// Launches f's kernel. Units of work: a token with all its heads, so that its sines are taken once, as far as a
// stage holds them; where there are fewer tokens than half the warps that fit, one turn of a warp's groups.
constexpr int kRotStage = 8192;
template <typename K>
int rot_launch(RotArgs& a, int64_t tokens, K kernel, int per_sm, int row_bytes, int kinds, cudaStream_t s, float* part, bool q_part, bool k_part) {
    const int rows = 32 / a.lanes;
    for (RotHalf& h : a.half) h.turns = (h.heads + rows - 1) / rows;
    const int turns = a.half[0].turns + a.half[1].turns;
    const int fits = kinds ? std::min(std::max(kRotStage / (rows * row_bytes), 1), turns) : turns;
    int64_t smem = 0;
    const auto divide = [&](int chunk) {
        a.chunk = chunk;
        a.chunks = (turns + chunk - 1) / chunk;
        a.units = tokens * a.chunks;
        a.stage = (chunk * rows * row_bytes + 127) / 128 * 128;
        smem = static_cast<int64_t>(kRotWarps) * kinds * a.stage;
    };
    divide((turns + (turns + fits - 1) / fits - 1) / ((turns + fits - 1) / fits));
    if (smem > 16384) smem_limit_once(reinterpret_cast<const void*>(kernel), 2 * kRotWarps * kRotStage, "qk_norm_rotary");
    // what registers and shared memory leave room for
    const int held = static_cast<int>(std::min<int64_t>(per_sm, (227 << 10) / (smem + sizeof(RotShared) + 1024)));
    const int64_t most = static_cast<int64_t>(sm_count()) * held;
    if (a.units * 2 < most * kRotWarps) divide(1);
    const int blocks = static_cast<int>(std::min(most, (a.units + kRotWarps - 1) / kRotWarps));
    if (q_part) a.half[0].part = part;
    if (k_part) a.half[1].part = part + static_cast<int64_t>(blocks) * a.dim;
    SX_LAUNCH(kernel, blocks, kRotThreads, smem, s, a);
    return blocks;
}

// Calls f(element, pairs a thread, neighbours, slots a thread, values that are not rotated).
template <typename F>
void by_layout(const SxRotaryInputs& in, int v, F&& f) {
    by_dtype(in.dtype, [&](auto t) {
        using T = decltype(t);
        const auto rest = [&](auto n, auto nb, auto slots) {
            if (rotated_values(in) < in.head_dim) f(t, n, nb, slots, std::true_type{});
            else f(t, n, nb, slots, std::false_type{});
        };
        const auto order = [&](auto n, auto slots) {
            if (in.pairs == SXCUDA_PAIRS_NEIGHBOURS) rest(n, std::true_type{}, slots);
            else rest(n, std::false_type{}, slots);
        };
        // up to 256 values are 16, 32, 64 and 128 slots for 32 lanes
        if constexpr (sizeof(T) == 2)
            if (v == 8) return order(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
        if (v == 4) return order(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
        if (v == 2) return order(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
        rest(std::integral_constant<int, 1>{}, std::false_type{}, std::integral_constant<int, 4>{});  // no order within one
    });
}

}  // namespace

void launch_qk_norm_rotary_fwd(const SxRotaryInputs& in, const SxAttentionView& q_out, const SxAttentionView& k_out, cudaStream_t s) {
    const int64_t tokens = in.batch * in.tokens;
    if (tokens == 0) return;
    const bool bulk = bulk_fits(in, in.q) && bulk_fits(in, q_out) && (!in.k_heads || (bulk_fits(in, in.k) && bulk_fits(in, k_out)));
    const int v = bulk ? most_pairs(in) : 1, row = static_cast<int>(in.head_dim * dtype_bytes(in.dtype));
    RotArgs a = rot_args(in, v);
    const auto set = [](RotHalf& h, const SxAttentionView& x) {
        h.out = x.data, h.out_batch = x.batch_stride, h.out_token = x.token_stride, h.out_head = x.head_stride;
    };
    set(a.half[0], q_out);
    if (in.k_heads) set(a.half[1], k_out);
    by_layout(in, v, [&](auto t, auto n, auto nb, auto slots, auto rest) {
        using T = decltype(t);
        if (bulk) rot_launch(a, tokens, rotary_kernel<T, decltype(n)::value, decltype(nb)::value, decltype(slots)::value, decltype(rest)::value, false>, kRotPerSm<decltype(n)::value, false>, row, 1, s, nullptr, false, false);
        else if constexpr (decltype(n)::value == 1) rot_launch(a, tokens, rotary_plain_kernel<T, false>, kRotPerSm<1, false>, row, 0, s, nullptr, false, false);
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
    const bool bulk = bulk_fits(in, at.q) && bulk_fits(in, g.v_q_out) && bulk_fits(in, g.v_q) &&
                      (!in.k_heads || (bulk_fits(in, at.k) && bulk_fits(in, g.v_k_out) && bulk_fits(in, g.v_k)));
    const int v = bulk ? most_pairs(in) : 1, row = static_cast<int>(in.head_dim * dtype_bytes(in.dtype));
    RotArgs a = rot_args(at, v);
    const auto set = [](RotHalf& h, const SxAttentionView& x, const SxAttentionView& y) {
        h.g = x.data, h.g_batch = x.batch_stride, h.g_token = x.token_stride, h.g_head = x.head_stride;
        h.out = y.data, h.out_batch = y.batch_stride, h.out_token = y.token_stride, h.out_head = y.head_stride;
    };
    set(a.half[0], g.v_q_out, g.v_q);
    if (in.k_heads) set(a.half[1], g.v_k_out, g.v_k);
    by_layout(in, v, [&](auto t, auto n, auto nb, auto slots, auto rest) {
        using T = decltype(t);
        float* part = static_cast<float*>(ws);
        int blocks = 0;
        if (bulk)
            blocks = rot_launch(a, tokens, rotary_kernel<T, decltype(n)::value, decltype(nb)::value, decltype(slots)::value, decltype(rest)::value, true>, kRotPerSm<decltype(n)::value, true>, row, 2, s, part,
                                g.v_q_weight, g.v_k_weight);
        else if constexpr (decltype(n)::value == 1)
            blocks = rot_launch(a, tokens, rotary_plain_kernel<T, true>, kRotPerSm<1, true>, row, 0, s, part, g.v_q_weight, g.v_k_weight);
        if (g.v_q_weight || g.v_k_weight)
            SX_LAUNCH(rotary_sums_kernel, dim3(blocks_for(in.head_dim, 32), 2), 1024, 0, s, a.half[0].part, a.half[1].part, blocks,
                      in.head_dim, g.v_q_weight, g.v_k_weight, in.param_dtype);
    });
}

}  // namespace sx

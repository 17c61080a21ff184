// attention_tc.cu — attention on the tensor cores: 16-bit inputs, head dimensions that are multiples
// of 8 up to 128 (padded by TMA's zero fill to 64 or 128), rows that TMA can copy.
//
// What bounds the kernels, per 128 x 128 tile of scores and SM (cycles; D = 128 / 64):
//   products          1024 / 512 forward (two), 3584 / 1792 backward (seven: s and g v^T twice)
//   exponentials      1024 forward, 2048 backward at 16 a cycle; a share of them is moved to the
//                     multiply-add pipes by a polynomial
//   shared memory     a product of two operands there reads 128 bytes a cycle, all there is; p and ds
//                     are therefore operands in tensor memory, and TMA's writes come on top
// With 128 columns the products and shared memory bound the forward, with 64 the exponentials and the
// path through them (score, maximum, probability and back, some 2000 cycles of latency per tile, which
// two tiles in turn hide in part). Measured, bf16: forward, causal, 16 heads (4 key-value) x 8192 x 128:
// 216 us in short runs, 1272 TFLOP/s of the needed products, 0.77 of the measured rate of large matrix
// products (1657); in a steady run, under the power limit, 254 us, 1082 TFLOP/s, 0.77 of the rate that
// those products sustain (1414). x 64: 191 us. Backward, causal, 2 x 16 (4) x 4096 x 128: 389 us, steady
// 457 us (884 and 752 TFLOP/s counting the five products that the gradient needs); 8 x 16 x 1024 x 64: 191
// us, steady 195 (450 and 441).
// Kept out, measured: one CTA per SM that takes tiles by ticket (short sequences 5% faster, long ones
// 7-13% slower: the loops of both kinds of tile then share too few registers); two warps that issue the
// forward's products (64 columns 5% faster, 128 20% slower); sixteen softmax warps (12% slower).
#include <algorithm>

#include "sx_attention.h"
#include "sx_tcgen05.cuh"

namespace sx {

__device__ uint32_t g_attention_status;

uint32_t attention_status() {
    uint32_t st = 0;
    const uint32_t zero = 0;
    cuda_check(cudaDeviceSynchronize(), "attention_status");
    cuda_check(cudaMemcpyFromSymbol(&st, g_attention_status, sizeof(st)), "attention_status");
    if (st) cuda_check(cudaMemcpyToSymbol(g_attention_status, &zero, sizeof(zero)), "attention_status");
    return st;
}

namespace {

constexpr int kRows = 128;            // rows of every tile: queries or keys
constexpr int kPanel = kRows * 128;   // bytes of a tile's 64 columns
// Tiles of the ring: what shared memory holds beside a CTA's own two at 128 columns, enough at 64.
template <int D>
constexpr int kRing = D == 64 ? 8 : 5;
constexpr int kSmemMost = 232448;

struct TcMaps {
    CUtensorMap q, k, v, g;
};

// A place in the ring that goes round with the tiles, in turn: the slot and the parity of its phase. The
// warps that load and issue are one each, and what they compute between two instructions of theirs is
// time that the tensor cores may wait: they count on instead of dividing.
template <int N>
struct Cursor {
    int slot = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
        if (++slot == N) slot = 0, parity ^= 1;
    }
};

// Rows from `first` of a tile in shared memory become zeros (the padding behind a batch entry's
// length may hold NaN, which a probability of zero would not remove).
template <int D>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int first, int lane) {
    const int n = (kRows - first) * 8;  // 16-byte pieces of a panel's rows
#pragma unroll
    for (int p = 0; p < D / 64; ++p)
        for (int i = lane; i < n; i += 32)
            *reinterpret_cast<uint4*>(tile + p * kPanel + first * 128 + i * 16) = uint4{0, 0, 0, 0};
    tc::fence_smem_to_async();
    __syncwarp();
}

template <int D>
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap* map, int row, int head, int batch, uint32_t bar,
                                          int rows = kRows) {
    tc::bar_expect(bar, D / 64 * rows * 128);
#pragma unroll
    for (int p = 0; p < D / 64; ++p) tc::tma_load(dst + p * kPanel, map, p * 64, row, head, batch, bar);
}

// Products over a whole tile. rows_rows: A and B both with rows along K = D (A B^T). tmem_rows: A in
// tensor memory (128 lanes x 128 values of K, two a column), B's rows along N = D (A B).
template <typename T, int D>
__device__ __forceinline__ void rows_rows(uint32_t one, uint32_t d, uint32_t a, uint32_t b) {
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
        const uint32_t at = (k / 4) * kPanel + (k % 4) * 32;
        tc::mma_ss(one, d, tc::operand(a + at, 16), tc::operand(b + at, 16), tc::shape<T>(kRows, false), k > 0);
    }
}
template <typename T, int D, int STEPS>  // over 64 values of K
__device__ __forceinline__ void tmem_rows(uint32_t one, uint32_t d, uint32_t a, uint32_t b, bool add) {
#pragma unroll
    for (int k = 0; k < STEPS; ++k)
        tc::mma_ts(one, d, a + k * 8, tc::operand(b + k * 2048, kPanel), tc::shape<T>(D, true), add || k > 0);
}
template <typename T, int D, int HALF>  // over 128, the second half HALF columns behind the first
__device__ __forceinline__ void tmem_rows2(uint32_t one, uint32_t d, uint32_t a, uint32_t b, bool add) {
    tmem_rows<T, D, 4>(one, d, a, b, add);
    tmem_rows<T, D, 4>(one, d, a + HALF, b + 64 * 128, true);
}

// A thread's row of a finished D-column sum, times `f`, to memory; zeros where `live` is false.
template <typename T, int D>
__device__ __forceinline__ void store_row(T* out, uint32_t at, float f, int dim, bool written, bool live, bool any) {
    const bool wide = reinterpret_cast<uintptr_t>(out) % 32 == 0;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (any) {
            tc::tmem_load32(o, at + c * 32);
            tc::wait_ld(o);
        }
        uint32_t x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
            x[i] = live ? tc::pack2<T>(__uint_as_float(o[2 * i]) * f, __uint_as_float(o[2 * i + 1]) * f) : 0u;
#pragma unroll
        for (int i = 0; i < 32; i += 16) {
            uint32_t(&y)[8] = *reinterpret_cast<uint32_t(*)[8]>(x + i / 2);
            if (!written) continue;
            if (wide && c * 32 + i + 8 < dim) {
                tc::store32(out + c * 32 + i, y);
            } else {
                if (c * 32 + i < dim) *reinterpret_cast<uint4*>(out + c * 32 + i) = uint4{y[0], y[1], y[2], y[3]};
                if (c * 32 + i + 8 < dim) *reinterpret_cast<uint4*>(out + c * 32 + i + 8) = uint4{y[4], y[5], y[6], y[7]};
            }
        }
        __syncwarp();
    }
}

// The same in 32 bits.
template <int D>
__device__ __forceinline__ void store_part(float* out, uint32_t at, float f, int dim, bool written, bool any) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (any) {
            tc::tmem_load32(o, at + c * 32);
            tc::wait_ld(o);
        }
#pragma unroll
        for (int i = 0; i < 32; i += 4)
            if (written && c * 32 + i < dim)
                *reinterpret_cast<float4*>(out + c * 32 + i) = float4{__uint_as_float(o[i]) * f, __uint_as_float(o[i + 1]) * f,
                                                                       __uint_as_float(o[i + 2]) * f, __uint_as_float(o[i + 3]) * f};
        __syncwarp();
    }
}

// Joins the parts of a query that CTAs with different keys made: out = sum_s 2^(lse_s - lse) out_s. A
// warp per query; parts that saw no key, or none with a score above -inf, are not read. A part that is
// NaN makes the query NaN, and so do scores that are all -inf.
template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a) {
    const int64_t rows = a.batch * a.heads * a.q_len, at = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (at >= rows) return;
    const int lane = threadIdx.x & 31;
    float top = -INFINITY;
    for (int s = lane; s < a.splits; s += 32) top = tc::max_nan(top, a.part_lse2[s * rows + at]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = tc::max_nan(top, __shfl_xor_sync(kFullMask, top, o));
    float total = isnan(top) ? top : 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (top > -INFINITY)
        for (int s = 0; s < a.splits; ++s) {
            const float x = exp2f(a.part_lse2[s * rows + at] - top);
            if (x == 0.f) continue;
            total += x;
            if (lane * 4 < a.dim) {
                const float4 o = *reinterpret_cast<const float4*>(a.part_out + (s * rows + at) * a.dim + lane * 4);
                acc[0] = fmaf(x, o.x, acc[0]);
                acc[1] = fmaf(x, o.y, acc[1]);
                acc[2] = fmaf(x, o.z, acc[2]);
                acc[3] = fmaf(x, o.w, acc[3]);
            }
        }
    const int64_t i = at % a.q_len, bh = at / a.q_len;
    const bool any = attn_sees_any(attn_head(a, bh % a.heads, bh / a.heads), i);
    if (total == 0.f) total = NAN;
    const float f = any ? 1.f / total : 0.f;
    T* out = static_cast<T*>(a.out.data) + bh / a.heads * a.out.batch_stride + bh % a.heads * a.out.head_stride + i * a.out.token_stride;
    if (lane * 4 < a.dim) {
        uint2 x{tc::pack2<T>(acc[0] * f, acc[1] * f), tc::pack2<T>(acc[2] * f, acc[3] * f)};
        *reinterpret_cast<uint2*>(out + lane * 4) = x;
    }
    if (lane == 0) a.lse[at] = any ? (top + log2f(total)) * kLn2 : -INFINITY;
}

// The forward. A CTA owns two tiles of 128 queries of one head; warps 0-3 and 4-7 make their
// probabilities (a thread per query), warp 8 loads, warp 9 issues the products. While one tile's
// warps work on its scores the tensor cores compute for the other: S = Q K^T into tensor memory, the
// probabilities back there in 16 bits, O += P V from there. With 64 columns of O tensor memory has
// room for P beside S, and the next S is computed while the probabilities of this one are made; with
// 128 P lies over S.
constexpr int kFwdThreads = 384;  // warps 10 and 11 only give up their registers
// Of 16 pairs of exponentials, those on the multiply-add pipes.
template <int D>
constexpr int kPoly = D == 64 ? 2 : 4;
template <int D>
struct FwdSmem {
    static constexpr int kTileBytes = D / 64 * kPanel;
    static constexpr int kQ = 0, kRing = 2 * kTileBytes, kSlots = sx::kRing<D>, kBars = kRing + kSlots * kTileBytes;
    static constexpr int kBytes = kBars + 256;
};

template <typename T, int D>
__global__ void __launch_bounds__(kFwdThreads, 1) attn_fwd_tc_kernel(const AttnArgs a, const __grid_constant__ TcMaps maps) {
    using S = FwdSmem<D>;
    constexpr int kSlots = S::kSlots;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = tc::smem_addr(smem);
    const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    volatile uint32_t* failed = reinterpret_cast<uint32_t*>(bars + 30);
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(bars + 31);
    const uint32_t bar0 = base + S::kBars;
    const auto kv_full = [&](int s) { return bar0 + 8 * s; };
    const auto kv_free = [&](int s) { return bar0 + 8 * (kSlots + s); };
    const auto q_full = [&](int t) { return bar0 + 8 * (2 * kSlots + t); };
    const auto s_full = [&](int t) { return bar0 + 8 * (2 * kSlots + 2 + t); };
    const auto p_full = [&](int t, int half) { return bar0 + 8 * (2 * kSlots + 4 + 2 * t + half); };
    const auto o_full = [&](int t) { return bar0 + 8 * (2 * kSlots + 8 + t); };  // apart: of every tile, else of the last
    const auto s_free = [&](int t) { return bar0 + 8 * (2 * kSlots + 10 + t); };
    const uint32_t drained = bar0 + 8 * (2 * kSlots + 12);
    constexpr bool kApart = D == 64;  // P beside S
    constexpr uint32_t kO = 2 * kRows, kP = kApart ? kO + 2 * D : 0, kPStep = kApart ? 64 : kRows;

    // the last queries see the most keys when causal: they start first
    const int split = static_cast<int>(blockIdx.x % a.splits);
    const int64_t block = blockIdx.x / a.splits, heads = (a.packed ? a.kv_heads : a.heads) * a.batch;
    const int64_t pairs = a.packed ? 1 : (a.q_len + 2 * kRows - 1) / (2 * kRows), bh = block % heads;
    const AttnHead w = attn_head(a, a.packed ? bh % a.kv_heads * a.group : bh % a.heads, a.packed ? bh / a.kv_heads : bh / a.heads);
    const int q0 = static_cast<int>((pairs - 1 - block / heads) * 2 * kRows);
    const int kv_len = static_cast<int>(w.kv_len), hk = static_cast<int>(w.h) / a.group;
    // key tiles of each query tile: j0 and on, as many as n
    int n[2], j0 = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int first = q0 + t * kRows;
        n[t] = first >= w.q_len || (a.packed && t) ? 0 : static_cast<int>((attn_keys_end(w, first + kRows) + kRows - 1) / kRows);
    }
    if (a.splits > 1) {
        const int each = (max(n[0], n[1]) + a.splits - 1) / a.splits;
        j0 = split * each;
        for (int t = 0; t < 2; ++t) n[t] = max(min(n[t] - j0, each), 0);
    }
    const int most = max(n[0], n[1]);

    // Warp 8 asks for the first tiles before anything else is ready.
    int loaded = 0;  // tiles of the ring that warp 8 has asked for
    Cursor<kSlots> load_at;
    const auto load_kv = [&] {
        load_rows<D>(base + S::kRing + load_at.slot * S::kTileBytes, loaded & 1 ? &maps.v : &maps.k, (j0 + loaded / 2) * kRows, hk,
                     static_cast<int>(w.b), kv_full(load_at.slot));
    };
    if (warp == 8 && lane == 0) {
        tc::prefetch_map(&maps.q);
        tc::prefetch_map(&maps.k);
        tc::prefetch_map(&maps.v);
        *failed = 0;
        for (int s = 0; s < kSlots; ++s) tc::bar_init(kv_full(s), 1), tc::bar_init(kv_free(s), 1);
        for (int t = 0; t < 2; ++t) {
            tc::bar_init(q_full(t), 1);
            tc::bar_init(s_full(t), 1);
            tc::bar_init(p_full(t, 0), 4);
            tc::bar_init(p_full(t, 1), 4);
            tc::bar_init(o_full(t), 1);
            tc::bar_init(s_free(t), 4);
        }
        tc::bar_init(drained, 1);
        tc::bar_init_fence();
        for (int t = 0; t < 2; ++t)
            if (n[t])
                load_rows<D>(base + S::kQ + t * S::kTileBytes, &maps.q, q0 + t * kRows, static_cast<int>(w.h), static_cast<int>(w.b), q_full(t),
                             a.packed ? static_cast<int>(a.q_len) * a.group : kRows);
    }
    if (warp == 8)
        for (; loaded < min(2 * most, kSlots); ++loaded, load_at.next())
            if (lane == 0) load_kv();
    if (warp == 9) tc::tmem_alloc(tc::smem_addr(tmem_at), 512);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = __shfl_sync(kFullMask, *tmem_at, 0);

    // 384 x 168 registers at the launch = 256 x 216 + 128 x 72
    if (warp >= 8) {
        tc::fewer_registers<72>();
        if (warp == 8) {  // loads: K0 V0 K1 V1 ... around the ring
            for (; loaded < 2 * most; ++loaded, load_at.next()) {
                if (!tc::bar_wait(kv_free(load_at.slot), load_at.parity ^ 1, failed)) break;
                if (lane == 0) load_kv();
                __syncwarp();
            }
        } else if (warp == 9) {  // products
            const uint32_t one = tc::elect();
            const auto scores = [&](int t, int slot) {
                rows_rows<T, D>(one, tmem + t * kRows, base + S::kQ + t * S::kTileBytes, base + S::kRing + slot * S::kTileBytes);
                tc::commit(one, s_full(t));
            };
            Cursor<kSlots> at;
            const bool ragged = kv_len % kRows && kv_len < a.kv_len;
            bool ok = most == 0 || tc::bar_wait(kv_full(0), 0, failed);
            at.next();
            for (int t = 0; ok && t < 2; ++t)
                if (n[t]) {
                    ok = tc::bar_wait(q_full(t), 0, failed);
                    if (ok) scores(t, 0);
                }
            if (ok && most) tc::commit(one, kv_free(0));
            for (int j = 0; ok && j < most; ++j) {
                const int vs = at.slot;
                ok = tc::bar_wait(kv_full(vs), at.parity, failed);
                if (!ok) break;
                at.next();
                const int ks = at.slot;
                if (ragged && (j0 + j + 1) * kRows > kv_len)
                    zero_rows<D>(smem + S::kRing + vs * S::kTileBytes, kv_len - (j0 + j) * kRows, lane);
                if (j + 1 < most) ok = tc::bar_wait(kv_full(ks), at.parity, failed);
                at.next();
                for (int t = 0; ok && t < 2; ++t) {
                    if (j >= n[t]) continue;
                    if (kApart && j + 1 < n[t]) {
                        ok = tc::bar_wait(s_free(t), j & 1, failed);
                        if (!ok) break;
                        tc::fence_after();
                        scores(t, ks);
                    }
                    for (int half = 0; ok && half < 2; ++half) {  // the first 64 keys while the others' p are made
                        ok = tc::bar_wait(p_full(t, half), j & 1, failed);
                        if (!ok) break;
                        tc::fence_after();
                        tmem_rows<T, D, 4>(one, tmem + kO + t * D, tmem + kP + t * kPStep + half * 32,
                                           base + S::kRing + vs * S::kTileBytes + half * 64 * 128, j > 0 || half > 0);
                    }
                    if (!ok) break;
                    if (kApart || j + 1 == n[t]) tc::commit(one, o_full(t));
                    if (!kApart && j + 1 < n[t]) scores(t, ks);
                }
                if (ok) {
                    tc::commit(one, kv_free(vs));
                    if (j + 1 < most) tc::commit(one, kv_free(ks));
                }
            }
        }
    } else {  // softmax: a thread per query
        tc::more_registers<216>();
        const int t = warp >> 2, mine = n[t];
        // the row's query and head (packed: the heads of a group one after the other)
        int row = q0 + t * kRows + (warp & 3) * 32 + lane, h = static_cast<int>(w.h);
        bool mine_to_write = row < a.q_len;
        if (a.packed) {
            const int q_len = static_cast<int>(a.q_len);
            mine_to_write = row < q_len * a.group;
            h += mine_to_write ? row / q_len : 0;
            row %= q_len;
        }
        // rows of no query see nothing: what lies in them (the tile's rest may be anything) must not
        // make the warp move its sums to another maximum
        const bool asked = mine_to_write && row < w.q_len;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + t * kRows, o_at = tmem + lanes + kO + t * D, p_at = tmem + lanes + kP + t * kPStep;
        // m: the base-2 exponent the sums are relative to. In float16, which keeps 11 bits only above
        // 2^-14, probabilities are held times 2^6 (at most 2^14 then); the division by their sum undoes it.
        constexpr float kUp = std::is_same_v<T, __half> ? 6.f : 0.f;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < mine; ++j) {
            ok = tc::bar_wait(s_full(t), j & 1, failed);
            if (!ok) break;
            tc::fence_after();
            uint32_t r[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tc::tmem_load32(r[c], s_at + c * 32);
            tc::wait_ld(r[0], r[1], r[2], r[3]);
            if (kApart) {
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::bar_arrive(s_free(t));
            }
            // keys of this tile that the query sees: those below `end`
            const int64_t last = asked ? static_cast<int64_t>(row) + w.ahead + 1 : 0;
            const int end = static_cast<int>((last < kv_len ? last : kv_len) - static_cast<int64_t>(j0 + j) * kRows);
            if (__any_sync(kFullMask, end < kRows)) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (c * 32 + i >= end) r[c][i] = 0xff800000u;
            }
            // A score that is NaN makes the maximum NaN, and by it the whole row: beside masked scores it
            // would else leave -inf, which stands for a row that has seen no key.
            float top[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                top[c] = tc::max_nan(__uint_as_float(r[c][0]), __uint_as_float(r[c][1]));
#pragma unroll
                for (int i = 2; i < 32; i += 2) top[c] = tc::max_nan(top[c], __uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1]));
            }
            const float seen = tc::max_nan(tc::max_nan(top[0], top[1]), tc::max_nan(top[2], top[3])) * a.scale_log2;
            // The sums move to a new maximum only when it is 2^8 above the old one: 32 bits hold that,
            // and the output's rows are then hardly ever read back and scaled.
            if (j == 0) {
                m = seen;
            } else if (__any_sync(kFullMask, !(seen <= m + 8.f))) {
                if (kApart) {  // the sums are at rest once the last tile's product is complete
                    ok = tc::bar_wait(o_full(t), (j - 1) & 1, failed);
                    if (!ok) break;
                    tc::fence_after();
                }
                const float to = tc::max_nan(m, seen);
                const float f = to == -INFINITY ? 1.f : tc::exp2_approx(m - to);
                l *= f;
                m = to;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tc::tmem_load32(o, o_at + c * 32);
                    tc::wait_ld(o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    tc::tmem_store32(o_at + c * 32, o);
                }
            }
            const float less = m == -INFINITY ? 0.f : kUp - m;
            const tc::Two times = tc::two(a.scale_log2, a.scale_log2), plus = tc::two(less, less);
            tc::Two sum[2] = {tc::two(0.f, 0.f), tc::two(0.f, 0.f)};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t p[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const int e = c * 64 + i * 2;
                    const tc::Two x = tc::fma2(tc::two(__uint_as_float(r[e >> 5][e & 31]), __uint_as_float(r[e >> 5][(e & 31) + 1])), times, plus);
                    float lo, hi;
                    if (i % 16 < kPoly<D>) {
                        tc::exp2_poly(x, lo, hi);
                    } else {
                        tc::split(x, lo, hi);
                        lo = tc::exp2_approx(lo);
                        hi = tc::exp2_approx(hi);
                    }
                    sum[i & 1] = tc::add2(sum[i & 1], tc::two(lo, hi));
                    p[i] = tc::pack2<T>(lo, hi);
                }
                if (kApart && c == 0 && j > 0) {  // the last tile's p have been read
                    ok = tc::bar_wait(o_full(t), (j - 1) & 1, failed);
                    if (!ok) break;
                    tc::fence_after();
                }
                tc::tmem_store32(p_at + c * 32, p);
                tc::wait_st();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::bar_arrive(p_full(t, c));
            }
            if (!ok) break;
            float lo, hi;
            tc::split(tc::add2(sum[0], sum[1]), lo, hi);
            l += lo + hi;
        }
        if (ok && mine) ok = tc::bar_wait(o_full(t), kApart ? (mine - 1) & 1 : 0, failed);
        if (ok) {
            tc::fence_after();
            const int64_t at = (w.b * a.heads + h) * a.q_len + row;
            if (a.splits > 1) {
                const int64_t to = split * (a.batch * a.heads * a.q_len) + at;
                const bool live = asked && m != -INFINITY;
                const float f = live ? 1.f / l : 0.f;
                store_part<D>(a.part_out + to * a.dim, o_at, f, a.dim, mine_to_write && live, mine > 0);
                if (mine_to_write) a.part_lse2[to] = live ? m - kUp + log2f(l) : -INFINITY;
            } else {
                // seen by the mask: where every score is -inf the sum is zero and the row NaN
                const bool live = asked && attn_sees_any(w, row);
                if (l == 0.f) l = NAN;
                const float f = live ? 1.f / l : 0.f;
                T* out = static_cast<T*>(a.out.data) + w.b * a.out.batch_stride + h * a.out.head_stride + row * a.out.token_stride;
                store_row<T, D>(out, o_at, f, a.dim, mine_to_write, live, mine > 0);
                if (mine_to_write) a.lse[at] = live ? (m - kUp + log2f(l)) * kLn2 : -INFINITY;
            }
        }
        tc::fence_before();
    }
    __syncthreads();
    if (*failed) {  // nothing may land in this CTA's memory after it has gone
        if (warp == 8) {
            for (int t = 0; t < 2; ++t)
                if (n[t]) tc::bar_drain(q_full(t), 0);
            for (int i = max(0, loaded - kSlots); i < loaded; ++i) tc::bar_drain(kv_full(i % kSlots), (i / kSlots) & 1);
        } else if (warp == 9) {
            tc::commit(tc::elect(), drained);
            tc::bar_drain(drained, 0);
        }
        __syncthreads();
        if (threadIdx.x == 0) atomicOr(&g_attention_status, 1u);
    }
    if (warp == 9) tc::tmem_free(tmem, 512);
}

// The backward. Both kinds of CTA run 256 threads over a 128 x 128 tile of scores, a thread per row,
// each warpgroup on 64 of the columns; p and ds go back to tensor memory in 16 bits, over the scores
// and over the products they came from, and are the A operands of the second products from there.
//
// A key-value CTA owns 128 keys (rows: keys, columns: queries) and passes over the queries of every
// head that shares them: S = K Q^T, W = V G^T, v_v += P^T G, v_k += dS^T Q. While the warpgroups
// turn S into P the tensor cores compute v_k of the tile before and W; while they turn W into dS,
// v_v and the next S.
//
// A query CTA owns 128 queries (rows: queries, columns: keys): S = Q K^T, W = G V^T, v_q += dS K, with
// the next S a tile ahead.
constexpr int kBwdThreads = 352;
template <int D>
struct BwdSmem {
    static constexpr int kTileBytes = D / 64 * kPanel;
    static constexpr int kOwn = 0, kRing = 2 * kTileBytes, kSlots = sx::kRing<D>, kStats = kRing + kSlots * kTileBytes;
    static constexpr int kBars = kStats + 2 * 2 * kRows * 4;  // lse and delta of two query tiles
    static constexpr int kBytes = kBars + 256;
};

template <int kSlots>
struct BwdBars {
    uint32_t at;
    __device__ uint32_t full(int s) const { return at + 8 * s; }
    __device__ uint32_t free(int s) const { return at + 8 * (kSlots + s); }
    __device__ uint32_t own() const { return at + 8 * (2 * kSlots); }
    __device__ uint32_t s_full(int k) const { return at + 8 * (2 * kSlots + 1 + k); }
    __device__ uint32_t w_full() const { return at + 8 * (2 * kSlots + 3); }
    __device__ uint32_t p_full(int c) const { return at + 8 * (2 * kSlots + 4 + c); }
    __device__ uint32_t ds_full() const { return at + 8 * (2 * kSlots + 6); }
    __device__ uint32_t out_full() const { return at + 8 * (2 * kSlots + 7); }
    __device__ uint32_t stat_full(int k) const { return at + 8 * (2 * kSlots + 8 + k); }
    __device__ uint32_t stat_free(int k) const { return at + 8 * (2 * kSlots + 10 + k); }
    __device__ uint32_t drained() const { return at + 8 * (2 * kSlots + 12); }
    static constexpr int kFailed = 2 * kSlots + 13, kTmem = kFailed + 1;  // words of 8 bytes behind the barriers
};
static_assert((BwdBars<8>::kTmem + 1) * 8 <= 256, "barriers");

template <int kSlots>
__device__ __forceinline__ void bwd_init(const BwdBars<kSlots>& b, volatile uint32_t* failed) {
    *failed = 0;
    for (int s = 0; s < kSlots; ++s) tc::bar_init(b.full(s), 1), tc::bar_init(b.free(s), 1);
    tc::bar_init(b.own(), 1);
    tc::bar_init(b.w_full(), 1);
    for (int c = 0; c < 2; ++c) tc::bar_init(b.p_full(c), 8);
    tc::bar_init(b.ds_full(), 8);
    tc::bar_init(b.out_full(), 1);
    for (int k = 0; k < 2; ++k) tc::bar_init(b.s_full(k), 1), tc::bar_init(b.stat_full(k), 1), tc::bar_init(b.stat_free(k), 8);
    tc::bar_init(b.drained(), 1);
    tc::bar_init_fence();
}

template <typename T>
__device__ __forceinline__ T* row_of(const SxAttentionView& v, int64_t b, int64_t h, int64_t row) {
    return static_cast<T*>(v.data) + b * v.batch_stride + h * v.head_stride + row * v.token_stride;
}

// Tensor memory for the CTA, and everything set up seen by everyone: its address.
__device__ __forceinline__ uint32_t bwd_start(uint32_t* tmem_at, int warp) {
    if (warp == 9) tc::tmem_alloc(tc::smem_addr(tmem_at), 512);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    return __shfl_sync(kFullMask, *tmem_at, 0);
}

// What the loading warp has asked for: tiles of the ring, the CTA's own tiles, lse and delta tiles.
struct Loaded {
    int ring = 0;
    bool own = false;
    int stats = 0;
};

// float16 keeps 11 bits only above 2^-14: p and ds are held times powers of two, so that what a
// gradient is summed from does not vanish before the sum. p is at most 1; for ds, out being a mean of rows
// of v, |p (g v - delta)| <= 2 max|g| max|v| with the rows' norms, which `ds` times takes to at most 2^14.
// What ds holds is then off by at most 2^-25 / `ds`, 2^-38 of that bound, where its own 11 bits end. The
// maxima are those of the heads that share a key head (whose gradient is one sum), so that no other head's
// or batch entry's magnitudes take bits away.
struct HalfScale {
    float p = 1.f, ds = 1.f;
};
template <typename T>
__device__ __forceinline__ HalfScale half_scale(const AttnArgs& a, int64_t b, int64_t hk) {
    HalfScale h;
    if constexpr (std::is_same_v<T, __half>) {
        const uint32_t* largest = a.largest + 2 * (b * a.kv_heads + hk);
        const float bound = 2.f * sqrtf(__uint_as_float(largest[0])) * sqrtf(__uint_as_float(largest[1]));
        h.p = 1.f / exp2f(kHalfShift);
        if (bound > 0x1p-80f && bound < 0x1p80f) h.ds = exp2f(14.f - ceilf(log2f(bound)));
    }
    return h;
}

__device__ __forceinline__ tc::Two pair(const uint32_t (&r)[32], int i) { return tc::two(__uint_as_float(r[i]), __uint_as_float(r[i + 1])); }
__device__ __forceinline__ void set_pair(uint32_t (&r)[32], int i, tc::Two x) {
    float lo, hi;
    tc::split(x, lo, hi);
    r[i] = __float_as_uint(lo);
    r[i + 1] = __float_as_uint(hi);
}
// Of 16 pairs of exponentials of the backward, those on the multiply-add pipes. Measured, 8 x 16 x 1024 x 64
// and causal 2 x 16 (4) x 4096 x 128 bf16: 3 of them 190.4 and 449.6 us, 4 194.8 and 451.4, 5 191.8 and
// 451.3.
constexpr int kPolyBwd = 3;
__device__ __forceinline__ void exp_pair(uint32_t (&r)[32], int i, tc::Two x) {
    float lo, hi;
    if (i / 2 % 16 * kPolyBwd % 16 < kPolyBwd) {
        tc::exp2_poly(x, lo, hi);
    } else {
        tc::split(x, lo, hi);
        lo = tc::exp2_approx(lo);
        hi = tc::exp2_approx(hi);
    }
    r[i] = __float_as_uint(lo);
    r[i + 1] = __float_as_uint(hi);
}
template <typename T>
__device__ __forceinline__ tc::Two scaled(tc::Two x, tc::Two by) {
    if constexpr (std::is_same_v<T, __half>) return tc::mul2(x, by);
    return x;
}
// Columns outside lo..hi become zeros (a key or query that is not seen; what was there may be NaN).
__device__ __forceinline__ void keep_columns(uint32_t (&r)[32], int lo, int hi) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (i < lo || i >= hi) r[i] = 0u;
}

template <typename T, int D>
__device__ __forceinline__ Loaded bwd_kv_tile(const AttnArgs& a, const TcMaps& maps, int64_t block, uint8_t* smem,
                                            const BwdBars<kRing<D>>& bars, volatile uint32_t* failed, uint32_t* tmem_at) {
    using S = BwdSmem<D>;
    constexpr int kSlots = S::kSlots;
    const uint32_t base = tc::smem_addr(smem);
    const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    // the first keys are seen by the most queries when causal: they start first
    const int64_t heads = static_cast<int64_t>(a.kv_heads) * a.batch;
    const int hk = static_cast<int>(block % heads % a.kv_heads), batch = static_cast<int>(block % heads / a.kv_heads);
    const int k0 = static_cast<int>(block / heads) * kRows;
    const AttnHead w = attn_head(a, hk * a.group, batch);
    const int q_len = static_cast<int>(w.q_len);
    const int64_t begin = attn_queries_begin(w, k0);
    const int first = static_cast<int>(begin / kRows);
    const int tiles = k0 >= w.kv_len || begin >= q_len ? 0 : (q_len + kRows - 1) / kRows - first;
    const int total = tiles * a.group;
    const auto slot = [&](int s) { return base + S::kRing + s * S::kTileBytes; };
    // with 64 columns of the sums there is room for the next S beside this one
    constexpr bool kAhead = D == 64;
    constexpr uint32_t kW = kAhead ? 2 * kRows : kRows, kVV = kW + kRows, kVK = kVV + D;
    const auto s_col = [](int i) { return kAhead ? static_cast<uint32_t>(i & 1) * kRows : 0u; };
    const auto s_bar = [&](int i) { return bars.s_full(kAhead ? i & 1 : 0); };
    const auto s_par = [](int i) { return static_cast<uint32_t>(kAhead ? i >> 1 : i) & 1; };

    int it = 0, load_tile = 0, load_h = hk * a.group;
    Cursor<kSlots> load_at;
    const auto load_next = [&] {
        if (lane == 0)
            load_rows<D>(slot(load_at.slot), it & 1 ? &maps.g : &maps.q, (first + load_tile) * kRows, load_h, batch, bars.full(load_at.slot));
        if (it & 1 && ++load_tile == tiles) load_tile = 0, ++load_h;
        ++it;
        load_at.next();
        __syncwarp();
    };
    if (warp == 8) {  // the first tiles are asked for before anything else is ready
        if (lane == 0) {
            tc::prefetch_map(&maps.q);
            tc::prefetch_map(&maps.g);
            bwd_init(bars, failed);
            if (total) {
                tc::bar_expect(bars.own(), 2 * S::kTileBytes);
                for (int p = 0; p < D / 64; ++p) {
                    tc::tma_load(base + S::kOwn + p * kPanel, &maps.k, p * 64, k0, hk, batch, bars.own());
                    tc::tma_load(base + S::kOwn + S::kTileBytes + p * kPanel, &maps.v, p * 64, k0, hk, batch, bars.own());
                }
            }
        }
        while (it < min(2 * total, kSlots)) load_next();
    }
    const uint32_t tmem = bwd_start(tmem_at, warp);

    if (warp == 8) {  // loads: Q0 G0 Q1 G1 ... around the ring
        while (it < 2 * total) {
            if (!tc::bar_wait(bars.free(load_at.slot), load_at.parity ^ 1, failed)) break;
            load_next();
        }
        return {it, total > 0, 0};
    } else if (warp == 10) {  // loads of lse and delta, two tiles ahead (a warp of their own: in line with
                              // the others they held the next queries up until a tile's end)
        int i = 0, tile = 0;
        int64_t at = (static_cast<int64_t>(batch) * a.heads + hk * a.group) * a.q_pad + first * kRows;
        for (; i < total; ++i) {
            if (i >= 2 && !tc::bar_wait(bars.stat_free(i & 1), (i / 2 - 1) & 1, failed)) break;
            if (lane == 0) {
                const uint32_t to = base + S::kStats + (i & 1) * 2 * kRows * 4;
                tc::bar_expect(bars.stat_full(i & 1), 2 * kRows * 4);
                tc::bulk_load(to, a.minus_lse2 + at, kRows * 4, bars.stat_full(i & 1));
                tc::bulk_load(to + kRows * 4, a.minus_delta + at, kRows * 4, bars.stat_full(i & 1));
            }
            at += kRows;
            if (++tile == tiles) tile = 0, at += a.q_pad - tiles * kRows;
            __syncwarp();
        }
        return {0, false, i};
    } else if (warp == 9) {  // products
        const uint32_t one = tc::elect();
        Cursor<kSlots> at;
        int to_end = tiles;  // tiles to the end of a head's queries, where padding is zeroed
        const bool ragged = q_len % kRows && q_len < a.q_len;
        uint32_t queries = 0, grads = 0;  // slots of the tile that is worked on
        const auto arrived = [&] {
            if (!tc::bar_wait(bars.full(at.slot), at.parity, failed)) return false;
            if (ragged && to_end == 1) zero_rows<D>(smem + S::kRing + at.slot * S::kTileBytes, q_len % kRows, lane);
            return true;
        };
        const auto scores = [&](int i) {
            if (!arrived()) return false;
            rows_rows<T, D>(one, tmem + s_col(i), base + S::kOwn, slot(at.slot));
            tc::commit(one, s_bar(i));
            at.next();
            return true;
        };
        const auto weights = [&] {
            if (!arrived()) return false;
            rows_rows<T, D>(one, tmem + kW, base + S::kOwn + S::kTileBytes, slot(at.slot));
            tc::commit(one, bars.w_full());
            at.next();
            if (--to_end == 0) to_end = tiles;
            return true;
        };
        bool ok = total == 0 || (tc::bar_wait(bars.own(), 0, failed) && scores(0) && weights());
        grads = 1;
        for (int i = 0; ok && i < total; ++i) {
            const uint32_t q_next = at.slot;
            if (kAhead && i + 1 < total) ok = scores(i + 1);
            for (int c = 0; ok && c < 2; ++c) {  // half of the queries while the others' p are made
                ok = tc::bar_wait(bars.p_full(c), i & 1, failed);
                if (!ok) break;
                tc::fence_after();
                const uint32_t p = tmem + s_col(i) + c * 16, g = slot(grads) + c * 32 * 128;
                tmem_rows<T, D, 2>(one, tmem + kVV, p, g, i > 0 || c > 0);
                tmem_rows<T, D, 2>(one, tmem + kVV, p + 64, g + 64 * 128, true);
            }
            if (!ok) break;
            tc::commit(one, bars.free(grads));
            if (!kAhead && i + 1 < total) ok = scores(i + 1);
            if (!ok) break;
            ok = tc::bar_wait(bars.ds_full(), i & 1, failed);
            if (!ok) break;
            tc::fence_after();
            tmem_rows2<T, D, 64>(one, tmem + kVK, tmem + kW, slot(queries), i > 0);
            tc::commit(one, i + 1 < total ? bars.free(queries) : bars.out_full());
            queries = q_next;
            grads = at.slot;
            if (i + 1 < total) ok = weights();
        }
    } else {
        const int half = warp >> 2;
        const int64_t key = k0 + (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t w_at = tmem + lanes + half * 64 + kW;
        const HalfScale scale = half_scale<T>(a, batch, hk);
        const tc::Two times = tc::two(a.scale_log2, a.scale_log2), ds_scale = tc::two(scale.p * scale.ds, scale.p * scale.ds);
        bool ok = true;
        int tile = 0;
        for (int i = 0; i < total; ++i) {
            const int64_t q0 = static_cast<int64_t>(first + tile) * kRows + half * 64;
            if (++tile == tiles) tile = 0;
            ok = tc::bar_wait(s_bar(i), s_par(i), failed) && tc::bar_wait(bars.stat_full(i & 1), (i / 2) & 1, failed);
            if (!ok) break;
            tc::fence_after();
            const uint32_t s_at = tmem + lanes + half * 64 + s_col(i);
            const ulonglong2* lse = reinterpret_cast<const ulonglong2*>(smem + S::kStats + (i & 1) * 2 * kRows * 4) + half * 16;
            const ulonglong2* delta = lse + kRows / 4;
            uint32_t r[2][32];
            tc::tmem_load32(r[0], s_at);
            tc::tmem_load32(r[1], s_at + 32);
            tc::wait_ld(r[0], r[1]);
            // the queries of this half that see the key: columns lo..hi
            const int lo = static_cast<int>(key < w.kv_len ? max(key - w.ahead - q0, static_cast<int64_t>(0)) : 64);
            const int hi = static_cast<int>(min(w.q_len - q0, static_cast<int64_t>(64)));
            const bool cut = __any_sync(kFullMask, lo > 0 || hi < 64);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const ulonglong2 x = lse[c * 8 + e / 4];
                    exp_pair(r[c], e, tc::fma2(pair(r[c], e), times, tc::Two{x.x}));
                    exp_pair(r[c], e + 2, tc::fma2(pair(r[c], e + 2), times, tc::Two{x.y}));
                }
                if (cut) keep_columns(r[c], lo - c * 32, hi - c * 32);
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) p[e] = tc::pack2<T>(__uint_as_float(r[c][2 * e]), __uint_as_float(r[c][2 * e + 1]));
                tc::tmem_store16(s_at + c * 16, p);
                tc::wait_st();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::bar_arrive(bars.p_full(c));
            }
            ok = tc::bar_wait(bars.w_full(), i & 1, failed);
            if (!ok) break;
            tc::fence_after();
            uint32_t g[2][32];
            tc::tmem_load32(g[0], w_at);
            tc::tmem_load32(g[1], w_at + 32);
            tc::wait_ld(g[0], g[1]);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const ulonglong2 x = delta[c * 8 + e / 4];
                    set_pair(g[c], e, scaled<T>(tc::mul2(pair(r[c], e), tc::add2(pair(g[c], e), tc::Two{x.x})), ds_scale));
                    set_pair(g[c], e + 2, scaled<T>(tc::mul2(pair(r[c], e + 2), tc::add2(pair(g[c], e + 2), tc::Two{x.y})), ds_scale));
                }
                if (cut) keep_columns(g[c], lo - c * 32, hi - c * 32);
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) p[e] = tc::pack2<T>(__uint_as_float(g[c][2 * e]), __uint_as_float(g[c][2 * e + 1]));
                tc::tmem_store16(w_at + c * 16, p);
            }
            tc::wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) {
                tc::bar_arrive(bars.ds_full());
                tc::bar_arrive(bars.stat_free(i & 1));
            }
        }
        if (ok && total) ok = tc::bar_wait(bars.out_full(), 0, failed);
        if (ok) {
            tc::fence_after();
            const bool written = key < a.kv_len, live = total && key < w.kv_len;
            if (half == 0) store_row<T, D>(row_of<T>(a.v_v, batch, hk, key), tmem + lanes + kVV, scale.p, a.dim, written, live, total > 0);
            else store_row<T, D>(row_of<T>(a.v_k, batch, hk, key), tmem + lanes + kVK, a.scale / scale.ds, a.dim, written, live, total > 0);
        }
    }
    return {};
}

template <typename T, int D>
__device__ __forceinline__ Loaded bwd_q_tile(const AttnArgs& a, const TcMaps& maps, int64_t block, uint8_t* smem,
                                           const BwdBars<kRing<D>>& bars, volatile uint32_t* failed, uint32_t* tmem_at) {
    using S = BwdSmem<D>;
    constexpr int kSlots = S::kSlots;
    const uint32_t base = tc::smem_addr(smem);
    const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int64_t heads = static_cast<int64_t>(a.heads) * a.batch, tiles = (a.q_len + kRows - 1) / kRows;
    const int h = static_cast<int>(block % heads % a.heads), batch = static_cast<int>(block % heads / a.heads);
    const int q0 = static_cast<int>(tiles - 1 - block / heads) * kRows, hk = h / a.group;
    const AttnHead w = attn_head(a, h, batch);
    const int kv_len = static_cast<int>(w.kv_len);
    const int n = q0 >= w.q_len ? 0 : static_cast<int>((attn_keys_end(w, q0 + kRows) + kRows - 1) / kRows);
    const auto slot = [&](int s) { return base + S::kRing + s * S::kTileBytes; };
    constexpr uint32_t kW = 2 * kRows, kVQ = 3 * kRows;

    int it = 0;
    Cursor<kSlots> load_at;
    const auto load_next = [&] {
        if (lane == 0) load_rows<D>(slot(load_at.slot), it & 1 ? &maps.v : &maps.k, it / 2 * kRows, hk, batch, bars.full(load_at.slot));
        ++it;
        load_at.next();
        __syncwarp();
    };
    if (warp == 8) {  // the first tiles are asked for before anything else is ready
        if (lane == 0) {
            tc::prefetch_map(&maps.k);
            tc::prefetch_map(&maps.v);
            bwd_init(bars, failed);
            if (n) {
                tc::bar_expect(bars.own(), 2 * S::kTileBytes);
                for (int p = 0; p < D / 64; ++p) {
                    tc::tma_load(base + S::kOwn + p * kPanel, &maps.q, p * 64, q0, h, batch, bars.own());
                    tc::tma_load(base + S::kOwn + S::kTileBytes + p * kPanel, &maps.g, p * 64, q0, h, batch, bars.own());
                }
            }
        }
        while (it < min(2 * n, kSlots)) load_next();
    }
    const uint32_t tmem = bwd_start(tmem_at, warp);

    if (warp == 8) {  // loads: K0 V0 K1 V1 ... around the ring
        while (it < 2 * n) {
            if (!tc::bar_wait(bars.free(load_at.slot), load_at.parity ^ 1, failed)) break;
            load_next();
        }
        return {it, n > 0, 0};
    } else if (warp == 9) {  // products
        const uint32_t one = tc::elect();
        Cursor<kSlots> at;  // the tiles are taken in the order K0 V0 K1 V1 ...
        const bool ragged = kv_len % kRows && kv_len < a.kv_len;
        uint32_t keys = 0, keys_next = 0;
        const auto scores = [&](int j) {
            if (!tc::bar_wait(bars.full(at.slot), at.parity, failed)) return false;
            if (ragged && (j + 1) * kRows > kv_len) zero_rows<D>(smem + S::kRing + at.slot * S::kTileBytes, kv_len - j * kRows, lane);
            rows_rows<T, D>(one, tmem + (j & 1) * kRows, base + S::kOwn, slot(at.slot));
            tc::commit(one, bars.s_full(j & 1));
            keys_next = at.slot;
            at.next();
            return true;
        };
        const auto weights = [&] {
            if (!tc::bar_wait(bars.full(at.slot), at.parity, failed)) return false;
            rows_rows<T, D>(one, tmem + kW, base + S::kOwn + S::kTileBytes, slot(at.slot));
            tc::commit(one, bars.w_full());
            tc::commit(one, bars.free(at.slot));
            at.next();
            return true;
        };
        bool ok = n == 0 || (tc::bar_wait(bars.own(), 0, failed) && scores(0) && weights());
        for (int j = 0; ok && j < n; ++j) {
            keys = keys_next;
            if (j + 1 < n) ok = scores(j + 1);
            if (ok) ok = tc::bar_wait(bars.ds_full(), j & 1, failed);
            if (!ok) break;
            tc::fence_after();
            tmem_rows2<T, D, 64>(one, tmem + kVQ, tmem + kW, slot(keys), j > 0);
            tc::commit(one, j + 1 < n ? bars.free(keys) : bars.out_full());
            if (j + 1 < n) ok = weights();
        }
    } else if (warp < 8) {
        const int half = warp >> 2;
        const int64_t row = q0 + (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + half * 64, w_at = s_at + kW;
        const int64_t at = (static_cast<int64_t>(batch) * a.heads + h) * a.q_pad + row;  // q_pad holds whole tiles
        const tc::Two lse = tc::two(a.minus_lse2[at], a.minus_lse2[at]), delta = tc::two(a.minus_delta[at], a.minus_delta[at]);
        const HalfScale scale = half_scale<T>(a, batch, hk);
        const tc::Two times = tc::two(a.scale_log2, a.scale_log2), ds_scale = tc::two(scale.p * scale.ds, scale.p * scale.ds);
        bool ok = true;
        for (int j = 0; j < n; ++j) {
            ok = tc::bar_wait(bars.s_full(j & 1), (j >> 1) & 1, failed);
            if (!ok) break;
            tc::fence_after();
            uint32_t r[2][32];
            tc::tmem_load32(r[0], s_at + (j & 1) * kRows);
            tc::tmem_load32(r[1], s_at + (j & 1) * kRows + 32);
            tc::wait_ld(r[0], r[1]);
            const int64_t last = row < w.q_len ? row + w.ahead + 1 : 0;
            const int end = static_cast<int>((last < kv_len ? last : kv_len) - static_cast<int64_t>(j) * kRows - half * 64);
            const bool cut = __any_sync(kFullMask, end < 64);
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 32; e += 2) exp_pair(r[c], e, tc::fma2(pair(r[c], e), times, lse));
            ok = tc::bar_wait(bars.w_full(), j & 1, failed);
            if (!ok) break;
            tc::fence_after();
            uint32_t g[2][32];
            tc::tmem_load32(g[0], w_at);
            tc::tmem_load32(g[1], w_at + 32);
            tc::wait_ld(g[0], g[1]);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int e = 0; e < 32; e += 2)
                    set_pair(g[c], e, scaled<T>(tc::mul2(pair(r[c], e), tc::add2(pair(g[c], e), delta)), ds_scale));
                if (cut) keep_columns(g[c], 0, end - c * 32);
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) p[e] = tc::pack2<T>(__uint_as_float(g[c][2 * e]), __uint_as_float(g[c][2 * e + 1]));
                tc::tmem_store16(w_at + c * 16, p);
            }
            tc::wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::bar_arrive(bars.ds_full());
        }
        if (ok && n) ok = tc::bar_wait(bars.out_full(), 0, failed);
        if (ok) {
            tc::fence_after();
            // each warpgroup writes half of the row's columns
            T* out = row_of<T>(a.v_q, batch, h, row) + half * (D / 2);
            store_row<T, D / 2>(out, tmem + lanes + kVQ + half * (D / 2), a.scale / scale.ds, a.dim - half * (D / 2), row < a.q_len,
                                n && row < w.q_len, n > 0);
        }
    }
    return {};
}

// One launch holds both kinds of CTA: the query CTAs fill the SMs that the key-value CTAs' last wave
// leaves idle.
template <typename T, int D>
__global__ void __launch_bounds__(kBwdThreads, 1) attn_bwd_tc_kernel(const AttnArgs a, const __grid_constant__ TcMaps maps, int64_t kv_blocks) {
    using S = BwdSmem<D>;
    constexpr int kSlots = S::kSlots;
    extern __shared__ __align__(1024) uint8_t smem[];
    const BwdBars<S::kSlots> bars{tc::smem_addr(smem) + S::kBars};
    uint64_t* words = reinterpret_cast<uint64_t*>(smem + S::kBars);
    volatile uint32_t* failed = reinterpret_cast<uint32_t*>(words + bars.kFailed);
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(words + bars.kTmem);
    const int warp = __shfl_sync(kFullMask, static_cast<int>(threadIdx.x >> 5), 0);
    const Loaded asked = blockIdx.x < kv_blocks ? bwd_kv_tile<T, D>(a, maps, blockIdx.x, smem, bars, failed, tmem_at)
                                                : bwd_q_tile<T, D>(a, maps, blockIdx.x - kv_blocks, smem, bars, failed, tmem_at);
    tc::fence_before();
    __syncthreads();
    if (*failed) {  // nothing may land in this CTA's memory after it has gone
        if (warp == 8 || warp == 10) {
            if (asked.own) tc::bar_drain(bars.own(), 0);
            for (int i = max(0, asked.ring - kSlots); i < asked.ring; ++i) tc::bar_drain(bars.full(i % kSlots), (i / kSlots) & 1);
            for (int i = max(0, asked.stats - 2); i < asked.stats; ++i) tc::bar_drain(bars.stat_full(i & 1), (i / 2) & 1);
        } else if (warp == 9) {
            tc::commit(tc::elect(), bars.drained());
            tc::bar_drain(bars.drained(), 0);
        }
        __syncthreads();
        if (threadIdx.x == 0) atomicOr(&g_attention_status, 1u);
    }
    if (warp == 9) tc::tmem_free(__shfl_sync(kFullMask, *tmem_at, 0), 512);
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
        if (!p || found != cudaDriverEntryPointSuccess) throw RuntimeError("attention: the driver has no cuTensorMapEncodeTiled");
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// Boxes of 128 tokens x 64 values of one head; what lies beyond the tensor reads as zero.
CUtensorMap make_map(const AttnArgs& a, const SxAttentionView& v, int64_t tokens, int64_t heads, int box_tokens = kRows, int box_heads = 1) {
    CUtensorMap m;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.dim), static_cast<cuuint64_t>(tokens),
                                static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(a.batch)};
    // an axis of one entry may have any stride: the row's own length stands for it
    const auto bytes = [&](int64_t n, int64_t stride) { return static_cast<cuuint64_t>(2 * (n > 1 ? stride : a.dim)); };
    const cuuint64_t strides[3] = {bytes(tokens, v.token_stride), bytes(heads, v.head_stride), bytes(a.batch, v.batch_stride)};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_tokens), static_cast<cuuint32_t>(box_heads), 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = encode_fn()(&m, a.dtype == SXCUDA_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                   4, v.data, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw RuntimeError("attention: cuTensorMapEncodeTiled failed with " + std::to_string(static_cast<int>(r)));
    return m;
}

// Rows that 16-byte copies reach, and strides a tensor map takes.
bool copies(const AttnArgs& a, const SxAttentionView& v, int64_t tokens, int64_t heads) {
    const auto fits = [](int64_t n, int64_t stride) { return n <= 1 || (stride > 0 && stride % 8 == 0 && stride < (1ll << 38)); };
    return reinterpret_cast<uintptr_t>(v.data) % 16 == 0 && fits(tokens, v.token_stride) && fits(heads, v.head_stride) &&
           fits(a.batch, v.batch_stride);
}

template <typename F>
void by_type_dim(const AttnArgs& a, F&& f) {
    const auto dim = [&](auto t) {
        if (a.dim <= 64) f(t, std::integral_constant<int, 64>{});
        else f(t, std::integral_constant<int, 128>{});
    };
    if (a.dtype == SXCUDA_F16) dim(__half{});
    else dim(__nv_bfloat16{});
}

}  // namespace

// A scale that is not above zero would turn the row maximum around; no key or query leaves nothing to map.
bool attention_tc_takes(const AttnArgs& a) {
    return a.dtype != SXCUDA_F32 && a.dim % 8 == 0 && a.scale > 0.f && a.q_len > 0 && a.kv_len > 0 &&
           copies(a, a.q, a.q_len, a.heads) && copies(a, a.k, a.kv_len, a.kv_heads) && copies(a, a.v, a.kv_len, a.kv_heads);
}
bool attention_tc_takes_view(const AttnArgs& a, const SxAttentionView& v, int64_t tokens, int64_t heads) {
    return copies(a, v, tokens, heads);
}

// The queries of the heads that share a key-value head make one tile where they fit in it: the keys are
// then read once for all of them. Where there are at most half as many CTAs as SMs the keys are split over
// several (two tiles of them at least) and their parts joined. Measured, bf16 x 128, whole and in two, three
// parts (us): 74 CTAs of one query on 8192 keys 118.8, 75.8, 98.3, of 200 queries 131.1, 94.1, 123.0 (on
// 1024 keys 26.6, 36.9, 49.2: there the join costs more than it gains); 80 CTAs of one query 118.8, 129.1,
// 98.3; 120 CTAs 122.9, 133.1, 137.3.
AttnPlan attention_fwd_plan(const AttnArgs& a) {
    AttnPlan p;
    p.packed = a.group > 1 && a.q_len * a.group <= kRows;
    p.blocks = p.packed ? a.kv_heads * a.batch : (a.q_len + 2 * kRows - 1) / (2 * kRows) * a.heads * a.batch;
    const int64_t tiles = (a.kv_len + kRows - 1) / kRows, sms = sm_count();
    if (p.blocks > 0 && p.blocks * 2 <= sms) p.splits = static_cast<int32_t>(std::max<int64_t>(std::min(sms / p.blocks, tiles / 2), 1));
    return p;
}

void launch_attention_fwd_tc(const AttnArgs& args, cudaStream_t s) {
    AttnArgs a = args;
    const AttnPlan plan = attention_fwd_plan(a);
    a.packed = plan.packed;
    a.splits = plan.splits;
    by_type_dim(a, [&](auto t, auto d) {
        constexpr int D = decltype(d)::value;
        const auto kernel = attn_fwd_tc_kernel<decltype(t), D>;
        constexpr int smem = FwdSmem<D>::kBytes;
        static_assert(smem <= kSmemMost, "shared memory");
        smem_limit_once(reinterpret_cast<const void*>(kernel), smem, "attention_fwd");
        TcMaps maps;
        maps.q = plan.packed ? make_map(a, a.q, a.q_len, a.heads, static_cast<int>(a.q_len), a.group) : make_map(a, a.q, a.q_len, a.heads);
        maps.k = make_map(a, a.k, a.kv_len, a.kv_heads);
        maps.v = make_map(a, a.v, a.kv_len, a.kv_heads);
        const int64_t grid = plan.blocks * plan.splits;
        if (grid > INT32_MAX) throw_invalid("attention_fwd", "too many query tiles");
        SX_LAUNCH(kernel, static_cast<unsigned>(grid), kFwdThreads, smem, s, a, maps);
        if (plan.splits > 1) {
            const auto join = attn_join_kernel<decltype(t)>;
            SX_LAUNCH(join, blocks_for(a.batch * a.heads * a.q_len, 8), 256, 0, s, a);
        }
    });
}

void launch_attention_bwd_tc(const AttnArgs& a, cudaStream_t s) {
    by_type_dim(a, [&](auto t, auto d) {
        constexpr int D = decltype(d)::value;
        const auto kernel = attn_bwd_tc_kernel<decltype(t), D>;
        constexpr int smem = BwdSmem<D>::kBytes;
        static_assert(smem <= kSmemMost, "shared memory");
        smem_limit_once(reinterpret_cast<const void*>(kernel), smem, "attention_bwd");
        TcMaps maps;
        maps.q = make_map(a, a.q, a.q_len, a.heads);
        maps.k = make_map(a, a.k, a.kv_len, a.kv_heads);
        maps.v = make_map(a, a.v, a.kv_len, a.kv_heads);
        maps.g = make_map(a, a.g, a.q_len, a.heads);
        const int64_t kv_blocks = (a.kv_len + kRows - 1) / kRows * a.kv_heads * a.batch;
        const int64_t grid = kv_blocks + (a.q_len + kRows - 1) / kRows * a.heads * a.batch;
        if (grid > INT32_MAX) throw_invalid("attention_bwd", "too many tiles");
        SX_LAUNCH(kernel, static_cast<unsigned>(grid), kBwdThreads, smem, s, a, maps, kv_blocks);
    });
}

}  // namespace sx

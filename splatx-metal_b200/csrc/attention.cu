// attention.cu — softmax attention, forward and backward, for any element type, head dimension up
// to 128 and strides, on the CUDA cores in 32 bits. 16-bit inputs whose rows can be copied in
// 16-byte pieces take the tensor-core kernels (attention_tc.cu).
//
// With s = scale q k^T, masked:  p = exp(s - lse), out = p v, lse = log sum exp(s), and for the
// gradient g of out:  delta = sum(g out), v_v = p^T g, ds = p (g v^T - delta),
// v_q = scale ds k, v_k = scale ds^T q. No matrix of scores is stored: the forward keeps a running
// maximum and sum per query while it passes over the keys, the backward recomputes p from lse.
// The backward is two kernels: one owns a tile of keys and passes over the queries (and over the
// query heads that share the key-value head), one owns a tile of queries and passes over the keys.
// That computes s and g v^T twice, and needs neither atomics nor partial sums in memory, so results
// do not change between calls. These kernels are bound by the multiply-adds and the shared-memory
// reads that feed them (four rows and four columns a thread): causal 16 heads (4 key-value) x 8192 x 128
// in 32 bits takes the forward 12.0 ms, 23 TFLOP/s (bf16 on the tensor cores 0.22 ms).
#include "sx_attention.h"

namespace sx {

namespace {

constexpr int kT = 64;        // queries and keys of a tile
constexpr int kThreads = 256;  // 16 x 16, four rows and four columns of a tile each
constexpr int kLd = kT + 4;    // padded row of a score tile

__device__ __forceinline__ int tx() { return threadIdx.x & 15; }
__device__ __forceinline__ int ty() { return threadIdx.x >> 4; }
__device__ __forceinline__ float sum16(float x) {
#pragma unroll
    for (int o = 8; o; o >>= 1) x += __shfl_xor_sync(kFullMask, x, o);
    return x;
}
__device__ __forceinline__ float max16(float x) {
#pragma unroll
    for (int o = 8; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(kFullMask, x, o));
    return x;
}

// kT rows from row `r0` of a head into shared memory [kT][D + 4]; zeros beyond the length and the
// head dimension.
template <typename T, int D>
__device__ __forceinline__ void load_tile(float* s, const SxAttentionView& a, int64_t b, int64_t h, int64_t r0,
                                          int64_t len, int dim) {
    const T* p = static_cast<const T*>(a.data) + b * a.batch_stride + h * a.head_stride;
    for (int i = threadIdx.x; i < kT * D; i += kThreads) {
        const int r = i / D, c = i % D;
        s[r * (D + 4) + c] = r0 + r < len && c < dim ? to_f32(p[(r0 + r) * a.token_stride + c]) : 0.f;
    }
}

// s[4 rows of ty][4 columns of tx] of A B^T, both [kT][D + 4].
template <int D>
__device__ __forceinline__ void dot_tile(float (&s)[4][4], const float* A, const float* B) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int c = 0; c < D; c += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(A + (ty() * 4 + i) * (D + 4) + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(B + (tx() + 16 * j) * (D + 4) + c);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                s[i][j] = fmaf(x[i].x, y[j].x, fmaf(x[i].y, y[j].y, fmaf(x[i].z, y[j].z, fmaf(x[i].w, y[j].w, s[i][j]))));
    }
}

// acc[4 rows of ty][D / 16 columns: 4 tx + 64 k] += P V with P [kT][kLd] (row, key), V [kT][D + 4].
template <int D>
__device__ __forceinline__ void add_product(float (&acc)[4][D / 16], const float* P, const float* V) {
#pragma unroll 4
    for (int k = 0; k < kT; ++k) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = P[(ty() * 4 + i) * kLd + k];
#pragma unroll
        for (int n = 0; n < D / 64; ++n) {
            const float4 v = *reinterpret_cast<const float4*>(V + k * (D + 4) + tx() * 4 + n * 64);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[i][n * 4 + 0] = fmaf(p[i], v.x, acc[i][n * 4 + 0]);
                acc[i][n * 4 + 1] = fmaf(p[i], v.y, acc[i][n * 4 + 1]);
                acc[i][n * 4 + 2] = fmaf(p[i], v.z, acc[i][n * 4 + 2]);
                acc[i][n * 4 + 3] = fmaf(p[i], v.w, acc[i][n * 4 + 3]);
            }
        }
    }
}

template <typename T, int D>
__device__ __forceinline__ void store_rows(const float (&acc)[4][D / 16], const float (&f)[4], const SxAttentionView& a,
                                           int64_t b, int64_t h, int64_t r0, int64_t rows, int dim) {
    T* p = static_cast<T*>(a.data) + b * a.batch_stride + h * a.head_stride;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + ty() * 4 + i;
        if (r >= rows) continue;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
            const int c = (n >> 2) * 64 + tx() * 4 + (n & 3);
            if (c < dim) p[r * a.token_stride + c] = from_f32<T>(acc[i][n] * f[i]);
        }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attn_fwd_kernel(const AttnArgs a) {
    extern __shared__ float smem[];
    float* Q = smem;
    float* K = Q + kT * (D + 4);
    float* V = K + kT * (D + 4);
    float* P = V + kT * (D + 4);
    const AttnHead w = attn_head(a, blockIdx.y, blockIdx.z);
    const int64_t q0 = static_cast<int64_t>(blockIdx.x) * kT;
    const int64_t hk = w.h / a.group;
    float acc[4][D / 16] = {}, m[4], l[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = -INFINITY;
    load_tile<T, D>(Q, a.q, w.b, w.h, q0, w.q_len, a.dim);
    const int64_t k_end = attn_keys_end(w, q0 + kT);
    for (int64_t k0 = 0; k0 < k_end; k0 += kT) {
        __syncthreads();
        load_tile<T, D>(K, a.k, w.b, hk, k0, w.kv_len, a.dim);
        load_tile<T, D>(V, a.v, w.b, hk, k0, w.kv_len, a.dim);
        __syncthreads();
        float s[4][4];
        dot_tile<D>(s, Q, K);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t row = q0 + ty() * 4 + i;
            float top = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = attn_sees(w, row, k0 + tx() + 16 * j) ? s[i][j] * a.scale_log2 : -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
            top = max16(top);
            const float base = top == -INFINITY ? 0.f : top;  // a row that has seen no key yet
            const float old = exp2f(m[i] - base);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(s[i][j] - base);
                sum += p;
                P[(ty() * 4 + i) * kLd + tx() + 16 * j] = p;
            }
            l[i] = fmaf(l[i], old, sum16(sum));
            m[i] = top;
#pragma unroll
            for (int n = 0; n < D / 16; ++n) acc[i][n] *= old;
        }
        __syncthreads();
        add_product<D>(acc, P, V);
    }
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = q0 + ty() * 4 + i;
        // a row without keys is one by its mask: a sum that is NaN or zero (every score -inf) is none
        const bool any = attn_sees_any(w, row);
        if (l[i] == 0.f) l[i] = NAN;
        f[i] = any ? 1.f / l[i] : 0.f;
        if (tx() == 0 && row < a.q_len)
            a.lse[(w.b * a.heads + w.h) * a.q_len + row] = any ? (m[i] + log2f(l[i])) * kLn2 : -INFINITY;
    }
    store_rows<T, D>(acc, f, a.out, w.b, w.h, q0, a.q_len, a.dim);
}

// Minus delta = sum(g out) per query, and minus lse in base 2 with -inf for a query that sees no key
// (exp2 then gives 0): what the scores' tiles add. Both arrays have rows of a.q_pad: the tensor-core kernels read whole tiles of them. L
// lanes share a query, each reading V values at a time. Bound by the reads of out and its gradient.
template <typename T, int V, int L>
__global__ void __launch_bounds__(256) attn_delta_kernel(const AttnArgs a) {
    constexpr int kQueries = 256 / L;
    const int per_head = static_cast<int>(a.q_pad / kQueries);
    const int64_t bh = blockIdx.x / per_head, row = static_cast<int64_t>(blockIdx.x % per_head) * kQueries + threadIdx.x / L;
    const AttnHead w = attn_head(a, bh % a.heads, bh / a.heads);
    float s = 0.f, lse = -INFINITY;
    if (row < w.q_len) {
        const T* o = static_cast<const T*>(a.out.data) + w.b * a.out.batch_stride + w.h * a.out.head_stride + row * a.out.token_stride;
        const T* g = static_cast<const T*>(a.g.data) + w.b * a.g.batch_stride + w.h * a.g.head_stride + row * a.g.token_stride;
        for (int c = threadIdx.x % L * V; c < a.dim; c += L * V) {
            const Pack<T, V> x = *reinterpret_cast<const Pack<T, V>*>(o + c), y = *reinterpret_cast<const Pack<T, V>*>(g + c);
#pragma unroll
            for (int e = 0; e < V; ++e) s = fmaf(to_f32(x.v[e]), to_f32(y.v[e]), s);
        }
        const float x = a.lse[bh * a.q_len + row];
        if (x != -INFINITY) lse = fmaf(x, -kLog2e, a.p_shift);
    }
#pragma unroll
    for (int off = L / 2; off; off >>= 1) s += __shfl_xor_sync(kFullMask, s, off);
    if (threadIdx.x % L == 0) {
        a.minus_delta[bh * a.q_pad + row] = -s;
        a.minus_lse2[bh * a.q_pad + row] = lse;
    }
}

// The largest squared norms of the rows of the output's gradient and of v below the lengths, per batch
// entry and key head, as the bits of a float, which order like unsigned numbers (so the atomics' order does
// not matter). A CTA per 64 rows of a head, 16 lanes a row: the first `g_blocks` for the gradient, the
// others for v.
template <typename T>
__global__ void __launch_bounds__(256) attn_largest_kernel(const AttnArgs a, uint32_t g_blocks) {
    const bool is_g = blockIdx.x < g_blocks;
    const SxAttentionView& v = is_g ? a.g : a.v;
    const uint32_t block = is_g ? blockIdx.x : blockIdx.x - g_blocks;
    const int64_t len = is_g ? a.q_len : a.kv_len;
    const int heads = is_g ? a.heads : a.kv_heads, per_head = static_cast<int>((len + 63) / 64);
    const int64_t bh = block / per_head, b = bh / heads, r0 = static_cast<int64_t>(block % per_head) * 64 + threadIdx.x / 16;
    const int64_t end = attn_length(is_g ? a.q_lens : a.kv_lens, b, len);
    const int c = threadIdx.x % 16 * 8;
    const T* p = static_cast<const T*>(v.data) + b * v.batch_stride + bh % heads * v.head_stride + c;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + i * 16;
        float s = 0.f;
        if (r < end && c < a.dim) {
            const Pack<T, 8> x = *reinterpret_cast<const Pack<T, 8>*>(p + r * v.token_stride);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(to_f32(x.v[e]), to_f32(x.v[e]), s);
        }
        top = fmaxf(top, sum16(s));
    }
    top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 16));
    if (threadIdx.x % 32 == 0 && top > 0.f) {
        const int64_t hk = is_g ? bh % heads / a.group : bh % heads;
        atomicMax(a.largest + 2 * (b * a.kv_heads + hk) + !is_g, __float_as_uint(top));
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attn_bwd_kv_kernel(const AttnArgs a) {
    extern __shared__ float smem[];
    float* K = smem;
    float* V = K + kT * (D + 4);
    float* Q = V + kT * (D + 4);
    float* G = Q + kT * (D + 4);
    float* P = G + kT * (D + 4);
    float* S = P + kT * kLd;
    const int64_t k0 = static_cast<int64_t>(blockIdx.x) * kT, hk = blockIdx.y;
    float dk[4][D / 16] = {}, dv[4][D / 16] = {};
    {
        const AttnHead w = attn_head(a, hk * a.group, blockIdx.z);
        load_tile<T, D>(K, a.k, w.b, hk, k0, w.kv_len, a.dim);
        load_tile<T, D>(V, a.v, w.b, hk, k0, w.kv_len, a.dim);
    }
    for (int64_t h = hk * a.group; h < (hk + 1) * a.group; ++h) {
        const AttnHead w = attn_head(a, h, blockIdx.z);
        const float* lse = a.minus_lse2 + (w.b * a.heads + h) * a.q_pad;
        const float* delta = a.minus_delta + (w.b * a.heads + h) * a.q_pad;
        if (k0 >= w.kv_len) break;
        for (int64_t q0 = attn_queries_begin(w, k0) / kT * kT; q0 < w.q_len; q0 += kT) {
            __syncthreads();
            load_tile<T, D>(Q, a.q, w.b, h, q0, w.q_len, a.dim);
            load_tile<T, D>(G, a.g, w.b, h, q0, w.q_len, a.dim);
            __syncthreads();
            float s[4][4], dp[4][4];
            dot_tile<D>(s, K, Q);
            dot_tile<D>(dp, V, G);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t row = q0 + tx() + 16 * j;
                const float x = row < w.q_len ? lse[row] : -INFINITY, d = row < w.q_len ? delta[row] : 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t key = k0 + ty() * 4 + i;
                    const bool seen = attn_sees(w, row, key);
                    const float p = seen ? exp2f(fmaf(s[i][j], a.scale_log2, x)) : 0.f;
                    P[(ty() * 4 + i) * kLd + tx() + 16 * j] = p;
                    S[(ty() * 4 + i) * kLd + tx() + 16 * j] = seen ? p * (dp[i][j] + d) : 0.f;
                }
            }
            __syncthreads();
            add_product<D>(dv, P, G);
            add_product<D>(dk, S, Q);
        }
    }
    const float one[4] = {1.f, 1.f, 1.f, 1.f}, sc[4] = {a.scale, a.scale, a.scale, a.scale};
    store_rows<T, D>(dv, one, a.v_v, blockIdx.z, hk, k0, a.kv_len, a.dim);
    store_rows<T, D>(dk, sc, a.v_k, blockIdx.z, hk, k0, a.kv_len, a.dim);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attn_bwd_q_kernel(const AttnArgs a) {
    extern __shared__ float smem[];
    float* Q = smem;
    float* G = Q + kT * (D + 4);
    float* K = G + kT * (D + 4);
    float* V = K + kT * (D + 4);
    float* S = V + kT * (D + 4);
    const AttnHead w = attn_head(a, blockIdx.y, blockIdx.z);
    const int64_t q0 = static_cast<int64_t>(blockIdx.x) * kT, hk = w.h / a.group;
    float dq[4][D / 16] = {}, x[4], d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = q0 + ty() * 4 + i, at = (w.b * a.heads + w.h) * a.q_pad + row;
        x[i] = row < w.q_len ? a.minus_lse2[at] : -INFINITY;
        d[i] = row < w.q_len ? a.minus_delta[at] : 0.f;
    }
    load_tile<T, D>(Q, a.q, w.b, w.h, q0, w.q_len, a.dim);
    load_tile<T, D>(G, a.g, w.b, w.h, q0, w.q_len, a.dim);
    const int64_t k_end = attn_keys_end(w, q0 + kT);
    for (int64_t k0 = 0; k0 < k_end; k0 += kT) {
        __syncthreads();
        load_tile<T, D>(K, a.k, w.b, hk, k0, w.kv_len, a.dim);
        load_tile<T, D>(V, a.v, w.b, hk, k0, w.kv_len, a.dim);
        __syncthreads();
        float s[4][4], dp[4][4];
        dot_tile<D>(s, Q, K);
        dot_tile<D>(dp, G, V);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool seen = attn_sees(w, q0 + ty() * 4 + i, k0 + tx() + 16 * j);
                const float p = seen ? exp2f(fmaf(s[i][j], a.scale_log2, x[i])) : 0.f;
                S[(ty() * 4 + i) * kLd + tx() + 16 * j] = seen ? p * (dp[i][j] + d[i]) : 0.f;
            }
        __syncthreads();
        add_product<D>(dq, S, K);
    }
    const float sc[4] = {a.scale, a.scale, a.scale, a.scale};
    store_rows<T, D>(dq, sc, a.v_q, w.b, w.h, q0, a.q_len, a.dim);
}

int tile_bytes(int D, int tiles, int scores) {
    return (tiles * kT * (D + 4) + scores * kT * kLd) * static_cast<int>(sizeof(float));
}

template <typename F>
void by_dim(int dim, F&& f) {
    if (dim <= 64) f(std::integral_constant<int, 64>{});
    else f(std::integral_constant<int, 128>{});
}

dim3 tiles_of(const AttnArgs& a, int64_t len, int64_t heads) {
    return dim3(static_cast<unsigned>((len + kT - 1) / kT), static_cast<unsigned>(heads), static_cast<unsigned>(a.batch));
}

}  // namespace

AttnArgs attn_args(const SxAttentionInputs& in) {
    AttnArgs a{};
    a.q = in.q;
    a.k = in.k;
    a.v = in.v;
    a.q_lens = in.q_lens;
    a.kv_lens = in.kv_lens;
    a.batch = in.batch;
    a.q_len = in.q_len;
    a.kv_len = in.kv_len;
    a.q_pad = (in.q_len + 127) / 128 * 128;
    a.heads = in.q_heads;
    a.kv_heads = in.kv_heads;
    a.group = in.kv_heads ? in.q_heads / in.kv_heads : 1;
    a.dim = in.head_dim;
    a.dtype = in.dtype;
    a.causal = in.causal != 0;
    a.scale = in.scale;
    a.scale_log2 = static_cast<float>(static_cast<double>(in.scale) * 1.4426950408889634);
    return a;
}

size_t attention_fwd_workspace(const SxAttentionInputs& in) {
    const AttnArgs a = attn_args(in);
    if (!attention_tc_takes(a)) return 0;
    const AttnPlan p = attention_fwd_plan(a);
    return p.splits > 1 ? static_cast<size_t>(p.splits * a.batch * a.heads * a.q_len) * (a.dim + 1) * sizeof(float) : 0;
}

void launch_attention_fwd(const SxAttentionInputs& in, const SxAttentionView& out, float* lse, void* ws, cudaStream_t s) {
    AttnArgs a = attn_args(in);
    a.out = out;
    a.lse = lse;
    a.part_out = static_cast<float*>(ws);
    a.part_lse2 = a.part_out + attention_fwd_workspace(in) / (a.dim + 1) / sizeof(float) * a.dim;
    if (a.batch == 0 || a.q_len == 0) return;
    if (attention_tc_takes(a) && attention_tc_takes_view(a, a.out, a.q_len, a.heads)) {
        launch_attention_fwd_tc(a, s);
        return;
    }
    by_dtype(a.dtype, [&](auto t) {
        by_dim(a.dim, [&](auto d) {
            constexpr int D = decltype(d)::value;
            const auto kernel = attn_fwd_kernel<decltype(t), D>;
            const int smem = tile_bytes(D, 3, 1);
            smem_limit_once(reinterpret_cast<const void*>(kernel), smem, "attention_fwd");
            SX_LAUNCH(kernel, tiles_of(a, a.q_len, a.heads), kThreads, smem, s, a);
        });
    });
}

size_t attention_bwd_workspace(const SxAttentionInputs& in) {
    const AttnArgs a = attn_args(in);
    return static_cast<size_t>(2 * a.batch * (a.heads * a.q_pad + a.kv_heads) + 4) * sizeof(float);
}

void launch_attention_bwd(const SxAttentionInputs& in, const SxAttentionGradsIn& g, const SxAttentionGrads& out,
                          void* ws, cudaStream_t s) {
    AttnArgs a = attn_args(in);
    a.out = g.out;
    a.g = g.v_out;
    a.v_q = out.v_q;
    a.v_k = out.v_k;
    a.v_v = out.v_v;
    a.lse = const_cast<float*>(g.lse);
    a.minus_lse2 = static_cast<float*>(ws);
    a.minus_delta = a.minus_lse2 + a.batch * a.heads * a.q_pad;
    if (a.batch == 0) return;
    const bool tensor = attention_tc_takes(a) && attention_tc_takes_view(a, a.g, a.q_len, a.heads) &&
                        attention_tc_takes_view(a, a.v_q, a.q_len, a.heads) &&
                        attention_tc_takes_view(a, a.v_k, a.kv_len, a.kv_heads) &&
                        attention_tc_takes_view(a, a.v_v, a.kv_len, a.kv_heads);
    const bool half = tensor && a.dtype == SXCUDA_F16;
    if (half) {
        a.p_shift = kHalfShift;
        a.largest = reinterpret_cast<uint32_t*>(a.minus_delta + a.batch * a.heads * a.q_pad);
        cuda_check(cudaMemsetAsync(a.largest, 0, 2 * a.batch * a.kv_heads * sizeof(uint32_t), s), "attention_bwd");
        const unsigned g_blocks = blocks_for(a.q_len, 64) * a.heads * static_cast<unsigned>(a.batch);
        const unsigned v_blocks = blocks_for(a.kv_len, 64) * a.kv_heads * static_cast<unsigned>(a.batch);
        const auto kernel = attn_largest_kernel<__half>;
        SX_LAUNCH(kernel, g_blocks + v_blocks, 256, 0, s, a, g_blocks);
    }
    by_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        if (a.q_len) {
            const auto run = [&](auto kernel, int lanes) {
                SX_LAUNCH(kernel, static_cast<unsigned>(a.q_pad / (256 / lanes) * a.batch * a.heads), 256, 0, s, a);
            };
            if constexpr (sizeof(T) == 2) {
                if (tensor && attention_tc_takes_view(a, a.out, a.q_len, a.heads)) {
                    if (a.dim <= 64) run(attn_delta_kernel<T, 8, 8>, 8);
                    else run(attn_delta_kernel<T, 8, 16>, 16);
                } else {
                    run(attn_delta_kernel<T, 1, 32>, 32);
                }
            } else {
                run(attn_delta_kernel<T, 1, 32>, 32);
            }
        }
        if (tensor) return;
        by_dim(a.dim, [&](auto d) {
            constexpr int D = decltype(d)::value;
            if (a.kv_len) {
                const auto kernel = attn_bwd_kv_kernel<T, D>;
                const int smem = tile_bytes(D, 4, 2);
                smem_limit_once(reinterpret_cast<const void*>(kernel), smem, "attention_bwd");
                SX_LAUNCH(kernel, tiles_of(a, a.kv_len, a.kv_heads), kThreads, smem, s, a);
            }
            if (a.q_len) {
                const auto kernel = attn_bwd_q_kernel<T, D>;
                const int smem = tile_bytes(D, 4, 1);
                smem_limit_once(reinterpret_cast<const void*>(kernel), smem, "attention_bwd");
                SX_LAUNCH(kernel, tiles_of(a, a.q_len, a.heads), kThreads, smem, s, a);
            }
        });
    });
    if (tensor) launch_attention_bwd_tc(a, s);
}

}  // namespace sx

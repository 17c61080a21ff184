// sx_attention.h — what the attention kernels share: their arguments and the mask.
#pragma once

#include <cmath>
#include <type_traits>

#include "sx_internal.h"
#include "sx_network.h"

namespace sx {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 2^14 times a probability is the most of them that float16 holds with room for rounding.
constexpr float kHalfShift = 14.f;

struct AttnArgs {
    SxAttentionView q, k, v, out, g, v_q, v_k, v_v;
    const int32_t* q_lens;
    const int32_t* kv_lens;
    float* lse;    // [batch, heads, q_len]
    float* minus_lse2;   // [batch, heads, q_pad]: minus the log-sums in base 2, -inf where nothing is seen
    float* minus_delta;  // [batch, heads, q_pad]
    // float16 on the tensor cores: probabilities are held times 2^p_shift, and ds times a power of two
    // taken from the largest squared norms of the rows of the output's gradient and of v: [batch,
    // kv_heads, 2], the bits of a float each.
    float p_shift;
    uint32_t* largest;
    int64_t batch, q_len, kv_len, q_pad;
    int32_t heads, kv_heads, group, dim, dtype;
    bool causal;
    float scale, scale_log2;
    // the tensor-core forward: heads of a group in one tile; parts of the keys per query, and what the
    // CTAs of a part leave: [splits, batch, heads, q_len, dim] and the same without dim
    bool packed;
    int32_t splits;
    float* part_out;
    float* part_lse2;
};
AttnArgs attn_args(const SxAttentionInputs& in);
struct AttnPlan {
    bool packed = false;
    int32_t splits = 1;
    int64_t blocks = 0;
};
AttnPlan attention_fwd_plan(const AttnArgs& a);

// The tensor-core kernels (attention_tc.cu): whether they take q, k and v, or another view of the
// call, and their launch.
bool attention_tc_takes(const AttnArgs& a);
bool attention_tc_takes_view(const AttnArgs& a, const SxAttentionView& v, int64_t tokens, int64_t heads);
void launch_attention_fwd_tc(const AttnArgs& a, cudaStream_t s);
void launch_attention_bwd_tc(const AttnArgs& a, cudaStream_t s);

// One query head of one batch entry, with its lengths. Query i sees the keys j < kv_len with
// j <= i + ahead.
struct AttnHead {
    int64_t b, h, q_len, kv_len, ahead;
};

__device__ __forceinline__ int64_t attn_length(const int32_t* lens, int64_t b, int64_t most) {
    if (!lens) return most;
    const int64_t n = lens[b];
    return n < 0 ? 0 : n > most ? most : n;
}

__device__ __forceinline__ AttnHead attn_head(const AttnArgs& a, int64_t h, int64_t b) {
    AttnHead w{b, h, attn_length(a.q_lens, b, a.q_len), attn_length(a.kv_lens, b, a.kv_len), 0};
    w.ahead = a.causal ? w.kv_len - w.q_len : w.kv_len;
    return w;
}
__device__ __forceinline__ bool attn_sees(const AttnHead& w, int64_t i, int64_t j) {
    return i < w.q_len && j < w.kv_len && j <= i + w.ahead;
}
__device__ __forceinline__ bool attn_sees_any(const AttnHead& w, int64_t i) { return attn_sees(w, i, 0); }
// The end of the keys that any query before `i_end` sees.
__device__ __forceinline__ int64_t attn_keys_end(const AttnHead& w, int64_t i_end) {
    const int64_t last = (i_end < w.q_len ? i_end : w.q_len) - 1;
    const int64_t end = last + w.ahead + 1 < w.kv_len ? last + w.ahead + 1 : w.kv_len;
    return last < 0 || end < 0 ? 0 : end;
}
// The first query that sees key j or a later one.
__device__ __forceinline__ int64_t attn_queries_begin(const AttnHead& w, int64_t j) {
    return j > w.ahead ? j - w.ahead : 0;
}

}  // namespace sx

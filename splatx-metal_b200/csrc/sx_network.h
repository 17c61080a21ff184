// sx_network.h — launchers of the network operators (layer norm, AdamW over many tensors,
// attention, linear layers, norm and rotation of queries and keys) and the element-type helpers they share. Every launcher enqueues on `stream` and
// throws sx::RuntimeError on a launch failure; arguments are validated by the C entry points.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/splatx_cuda.h"
#include "sx_common.cuh"

namespace sx {

inline int64_t dtype_bytes(int32_t dtype) { return dtype == SXCUDA_F32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N consecutive values as one aligned access (N * sizeof(T) = 2..16 bytes).
template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
    T v[N];
};

inline int sm_count() {
    static std::atomic<int> known[64];  // of each device, once asked for
    int dev = 0, n = 0;
    cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
    if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    cuda_check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "SM count");
    if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

// Calls f with a value of the element type that a dtype names.
template <typename F>
void by_dtype(int32_t dtype, F&& f) {
    if (dtype == SXCUDA_F32) f(float{});
    else if (dtype == SXCUDA_F16) f(__half{});
    else f(__nv_bfloat16{});
}

void launch_layer_norm_fwd(const SxLayerNormInputs& in, void* y, int64_t y_stride, float* mean,
                           float* rstd, cudaStream_t s);
size_t layer_norm_bwd_workspace(const SxLayerNormInputs& in);
void launch_layer_norm_bwd(const SxLayerNormInputs& in, const SxLayerNormGradsIn& g,
                           const SxLayerNormGrads& out, void* ws, cudaStream_t s);

void launch_adamw(const SxAdamwTensor* t, int64_t n, const SxAdamwConfig& cfg, cudaStream_t s);

// The attention kernels' status word of the current device, read and cleared (synchronises).
uint32_t attention_status();
size_t attention_fwd_workspace(const SxAttentionInputs& in);
void launch_attention_fwd(const SxAttentionInputs& in, const SxAttentionView& out, float* lse,
                          void* ws, cudaStream_t s);
size_t attention_bwd_workspace(const SxAttentionInputs& in);
void launch_attention_bwd(const SxAttentionInputs& in, const SxAttentionGradsIn& g,
                          const SxAttentionGrads& out, void* ws, cudaStream_t s);

// The status words of the linear and rotation kernels of the current device, read and cleared (synchronises).
uint32_t linear_status();
uint32_t rotary_status();
size_t linear_fwd_workspace(const SxLinearInputs& in);
void launch_linear_fwd(const SxLinearInputs& in, const SxLinearOutputs& out, void* ws, cudaStream_t s);
size_t linear_bwd_workspace(const SxLinearInputs& in, const SxLinearGradsIn& g, const SxLinearGrads& out);
void launch_linear_bwd(const SxLinearInputs& in, const SxLinearGradsIn& g, const SxLinearGrads& out, void* ws,
                       cudaStream_t s);

void launch_qk_norm_rotary_fwd(const SxRotaryInputs& in, const SxAttentionView& q_out, const SxAttentionView& k_out,
                               cudaStream_t s);
size_t qk_norm_rotary_bwd_workspace(const SxRotaryInputs& in);
void launch_qk_norm_rotary_bwd(const SxRotaryInputs& in, const SxRotaryGrads& g, void* ws, cudaStream_t s);

}  // namespace sx

// sx_network.h — launchers of the network operators (layer norm, AdamW over many tensors,
// attention) and the element-type helpers they share. Every launcher enqueues on `stream` and
// throws sx::RuntimeError on a launch failure; arguments are validated by the C entry points.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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
    int dev = 0, n = 0;
    cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
    cuda_check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "SM count");
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

}  // namespace sx

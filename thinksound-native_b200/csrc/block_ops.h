// block_ops.h — the transformer-block operators of include/tsn.h (block norm, rotary positions with
// several axes, differential attention) behind their C entry points.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "runtime.h"

namespace tsn {

int block_norm(DeviceCtx & c, const tsn_block_norm_args & a);
int rope_plan(uint32_t D, uint32_t axes, const uint32_t * pairs, const double * theta, const double * scale, int layout,
              tsn_rope_plan_t * out);
int rope_axes(DeviceCtx & c, const tsn_rope_plan_t & p, const tsn_rope_args & a);
cudaError_t configure_diff_attn();   // once per device, before the first launch
int diff_attn(DeviceCtx & c, const tsn_diff_attn_args & a);

inline bool known_type(int t) { return t == TSN_F32 || t == TSN_F16 || t == TSN_BF16; }
inline size_t type_size(int t) { return t == TSN_F32 ? 4 : 2; }

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

} // namespace tsn

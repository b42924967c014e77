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

// Pairs of f32 through the two-wide FP32 instructions, each lane rounded once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n fma.rn.f32x2 z, x, y, z;\n"
        " mov.b64 {%0, %1}, z;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// Two 16-bit values of one word, the first in its low half, to and from f32.
template <class T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*(const __half2 *) &w); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t *) &h;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t *) &h;
}

// N consecutive elements (16 or 32 bytes, 16-byte aligned) as they lie in memory.
template <class T, int N> struct Words { uint4 w[sizeof(T) * N / 16]; };
template <class T, int N> __device__ __forceinline__ Words<T, N> load_words(const T * p) {
    Words<T, N> r;
#pragma unroll
    for (int i = 0; i < (int) (sizeof(T) * N / 16); ++i) r.w[i] = ((const uint4 *) p)[i];
    return r;
}
template <class T, int N> __device__ __forceinline__ void store_words(T * p, const float * v) {
    uint32_t x[sizeof(T) * N / 4];
#pragma unroll
    for (int i = 0; i < (int) (sizeof(T) * N / 4); ++i) {
        if constexpr (sizeof(T) == 4) x[i] = __float_as_uint(v[i]);
        else x[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
#pragma unroll
    for (int i = 0; i < (int) (sizeof(T) * N / 16); ++i) ((uint4 *) p)[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
}
template <class T, int N> __device__ __forceinline__ void to_floats(const Words<T, N> & r, float * v) {
    const uint32_t * x = (const uint32_t *) r.w;
#pragma unroll
    for (int i = 0; i < (int) (sizeof(T) * N / 4); ++i) {
        if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(x[i]);
        else { const float2 f = unpack2<T>(x[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    }
}

} // namespace tsn

// attn_ops.cuh — device pieces that the attention operators share: exponentials, roundings, masks of 32 keys, mma.sync.
#pragma once
#include "block_ops.h"
#include "ptx.cuh"

namespace tsn {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t r, float & a, float & b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t f2_neg(uint64_t a) { return a ^ 0x8000000080000000ull; }
__device__ __forceinline__ uint64_t fadd2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// (2^x, 2^y) on the FMA pipe, x and y clamped to -126 or more: 2^i p(f), i the nearest whole number, f = x - i in [-1/2, 1/2],
// p the polynomial of least relative error there (Remez exchange): 7.5e-5 at degree 3, 2.6e-6 at degree 4, each below
// an eighth of half a unit of the 16-bit type that the result is rounded to. Adding 1.5 * 2^23 rounds to i and leaves
// it in the low bits. NaN becomes 0x7f7fffff, which rounds to infinity in either 16-bit type. ZERO: what was clamped becomes 0 (p(0) < 1, so 2^-126 p(0) is subnormal).
template <bool BF16, bool ZERO>
__device__ __forceinline__ uint64_t ex2_fma(uint64_t xy) {
    float x, y;
    f2_unpack(xy, x, y);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-126.0f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(y) : "f"(-126.0f));
    const uint64_t v = f2_pack(x, y), magic = f2_pack(12582912.0f, 12582912.0f), r = fadd2(v, magic);
    const uint64_t f = fadd2(v, fadd2(magic, f2_neg(r)));
    auto two = [](float c) { return f2_pack(c, c); };
    uint64_t q;
    if (BF16) {
        q = ffma2(two(0.0551716685f), f, two(0.242611125f));
        q = ffma2(q, f, two(0.693260968f));
        q = ffma2(q, f, two(0.999928057f));
    } else {
        q = ffma2(two(0.00957010221f), f, two(0.0559178591f));
        q = ffma2(q, f, two(0.240247443f));
        q = ffma2(q, f, two(0.693121791f));
        q = ffma2(q, f, two(0.999999285f));
    }
    float a, b, i, j;
    f2_unpack(q, a, b);
    f2_unpack(r, i, j);
    uint64_t e = f2_pack(__uint_as_float(__float_as_uint(a) + (__float_as_uint(i) << 23)), __uint_as_float(__float_as_uint(b) + (__float_as_uint(j) << 23)));
    if (ZERO) asm("mul.rn.ftz.f32x2 %0, %0, %1;" : "+l"(e) : "l"(two(1.0f)));
    return e;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    uint32_t r;
    if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
// a and b += the two 16-bit values of a word, in f32
template <bool BF16>
__device__ __forceinline__ void add_rounded(float & a, float & b, uint32_t two) {
    if (BF16) asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n add.rn.f32.bf16 %0, l, %0;\n add.rn.f32.bf16 %1, h, %1;\n}" : "+f"(a), "+f"(b) : "r"(two));
    else asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n add.rn.f32.f16 %0, l, %0;\n add.rn.f32.f16 %1, h, %1;\n}" : "+f"(a), "+f"(b) : "r"(two));
}
// the low n bits of a word, n of any sign and size
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
// of two 16-bit values, the non-finite ones set to zero
template <bool BF16>
__device__ __forceinline__ uint32_t finite_only(uint32_t v) {
    const uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
    if ((v & e) == e) v &= 0xffff0000u;
    if ((v & (e << 16)) == (e << 16)) v &= 0x0000ffffu;
    return v;
}

// 32 scores s of a row become 2^(c s + neg): P as 16-bit pairs, and the sum of these rounded values, so that what rounding
// takes from a key's share in the product it takes from the divisor too. Every fourth pair takes the FMA pipe.
template <bool BF16, bool MASKED>
__device__ __forceinline__ void exponentials(const uint32_t * s, uint32_t * pk, float c, float ref, float (&sum)[4]) {
    const float neg = ref == -INFINITY ? 0.0f : -ref;
    const uint64_t c2 = f2_pack(c, c), neg2 = f2_pack(neg, neg);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const uint64_t v = ffma2(f2_pack(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), c2, neg2);
        float y, z;
        if (e % 4 == 3) {
            f2_unpack(ex2_fma<BF16, MASKED>(v), y, z);
        } else {
            f2_unpack(v, y, z);
            y = ex2(y);
            z = ex2(z);
        }
        pk[e] = pack16<BF16>(y, z);
        add_rounded<BF16>(sum[2 * (e & 1)], sum[2 * (e & 1) + 1], pk[e]);
    }
}
__device__ __forceinline__ float greatest(const uint32_t * s) {   // of 32
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < 32; e += 2) mx[(e >> 1) & 1] = fmaxf(mx[(e >> 1) & 1], fmaxf(__uint_as_float(s[e]), __uint_as_float(s[e + 1])));
    return fmaxf(mx[0], mx[1]);
}
__device__ __forceinline__ void hide(uint32_t * s, uint32_t vis) {   // scores of the keys that the row does not see
    if (__any_sync(~0u, vis != ~0u))
#pragma unroll
        for (int e = 0; e < 32; ++e)
            if (!((vis >> e) & 1u)) s[e] = 0xff800000u;   // -inf
}

// E (2 or 4) words of shared or, past the L1 cache, global memory
template <int E, bool GLOBAL>
__device__ __forceinline__ void read_words(const float * at, float * v) {
    if (E == 4) {
        const float4 x = GLOBAL ? __ldcg((const float4 *) at) : *(const float4 *) at;
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
        const float2 x = GLOBAL ? __ldcg((const float2 *) at) : *(const float2 *) at;
        v[0] = x.x; v[1] = x.y;
    }
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the 8 x 8 matrix of 16-bit elements that the warp holds, transposed
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

} // namespace tsn

// diff_attn.cu — differential attention (tsn_diff_attn).
//
// One pass over the keys with the running maximum and sum of both softmax maps: the unnormalised sums
// O_m = sum_j 2^(s_mj - max_m) v_j are rescaled when a maximum grows, and o = O_1 / l_1 - lambda O_2 / l_2.
// One warp per query row on the CUDA cores.
#include "block_ops.h"

namespace tsn {

namespace {

template <class T, int D>   // D = 2 d, the width of a head
__global__ void diff_attn_kernel(const __grid_constant__ tsn_diff_attn_args a) {
    constexpr int E = D / 32, d = D / 2;
    const int lane = threadIdx.x & 31;
    const long long row = (long long) blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= (long long) a.B * a.Sq * a.H) return;
    const int h = (int) (row % a.H);
    const long long b = row / a.H / a.Sq, i = row / a.H % a.Sq;
    const int hk = h / (int) (a.H / a.Hk);
    const int n = a.key_len ? max(0, min(a.key_len[b], (int) a.Sk)) : (int) a.Sk;
    const long long last = a.causal ? min((long long) n - 1, i + n - (long long) a.Sq) : n - 1;
    // lane l holds elements E l .. E l + E - 1: the first half of the warp has map 1, the second map 2
    const T * q = (const T *) a.q.p + b * a.q.sb + i * a.q.ss + h * a.q.sh + E * lane;
    float qv[E], o1[E] = {}, o2[E] = {};
    const float c = a.scale * 1.44269504088896341f;
    for (int e = 0; e < E; ++e) qv[e] = to_f32(q[e]);
    float m = -INFINITY, l = 0.0f;   // this half's map
    bool bad = false;
    for (long long j = 0; j <= last; ++j) {
        if (a.key_mask && !a.key_mask[b * a.mask_sb + j]) continue;
        const T * k = (const T *) a.k.p + b * a.k.sb + j * a.k.ss + hk * a.k.sh + E * lane;
        const T * v = (const T *) a.v.p + b * a.v.sb + j * a.v.ss + hk * a.v.sh + E * lane;
        float s = 0.0f;
        for (int e = 0; e < E; ++e) s = fmaf(qv[e], to_f32(k[e]), s);
        for (int x = 8; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= c;
        const float mn = fmaxf(m, s);
        const float ref = mn == -INFINITY ? 0.0f : mn;
        const float f = exp2f(m - ref), p = to_f32(from_f32<T>(exp2f(s - ref)));
        m = mn;
        l = l * f + p;
        const float f1 = __shfl_sync(0xffffffffu, f, 0), f2 = __shfl_sync(0xffffffffu, f, 16);
        const float p1 = __shfl_sync(0xffffffffu, p, 0), p2 = __shfl_sync(0xffffffffu, p, 16);
        for (int e = 0; e < E; ++e) {
            const float vv = to_f32(v[e]);
            bad |= !(fabsf(vv) < INFINITY);
            o1[e] = fmaf(p1, vv, o1[e] * f1);
            o2[e] = fmaf(p2, vv, o2[e] * f2);
        }
    }
    bad = __any_sync(0xffffffffu, bad);
    const float l1 = __shfl_sync(0xffffffffu, l, 0), l2 = __shfl_sync(0xffffffffu, l, 16);
    float z1 = 0.0f, z2 = 0.0f;
    for (int e = lane; e < d; e += 32) {
        z1 += a.lq1[h * a.lam_sh + e] * a.lk1[h * a.lam_sh + e];
        z2 += a.lq2[h * a.lam_sh + e] * a.lk2[h * a.lam_sh + e];
    }
    for (int x = 16; x; x >>= 1) { z1 += __shfl_xor_sync(0xffffffffu, z1, x); z2 += __shfl_xor_sync(0xffffffffu, z2, x); }
    const float lam = expf(z1) - expf(z2) + a.lambda_init;
    const float w1 = l1 == 0.0f ? 0.0f : 1.0f / l1, w2 = l2 == 0.0f ? 0.0f : lam / l2;
    float ss = 0.0f;
    for (int e = 0; e < E; ++e) {
        o1[e] = bad ? NAN : o1[e] * w1 - o2[e] * w2;
        ss += o1[e] * o1[e];
    }
    for (int x = 16; x; x >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, x);
    const float g = rsqrtf(ss / (float) D + a.eps) * (1.0f - a.lambda_init);
    T * out = (T *) a.out.p + b * a.out.sb + i * a.out.ss + h * a.out.sh + E * lane;
    for (int e = 0; e < E; ++e) out[e] = from_f32<T>(o1[e] * g * (a.norm_w ? a.norm_w[E * lane + e] : 1.0f));
}

template <class T>
cudaError_t launch(const tsn_diff_attn_args & a, cudaStream_t s) {
    const long long rows = (long long) a.B * a.Sq * a.H;
    if (a.d == 32) diff_attn_kernel<T, 64><<<(unsigned) ((rows + 3) / 4), 128, 0, s>>>(a);
    else diff_attn_kernel<T, 128><<<(unsigned) ((rows + 3) / 4), 128, 0, s>>>(a);
    return cudaGetLastError();
}

} // namespace

int diff_attn(DeviceCtx & c, const tsn_diff_attn_args & in) {
    tsn_diff_attn_args a = in;
    if (a.type != TSN_F16 && a.type != TSN_BF16) return fail(TSN_ERR_ARG, "tsn_diff_attn: type must be TSN_F16 or TSN_BF16");
    if (a.d != 32 && a.d != 64) return fail(TSN_ERR_ARG, "tsn_diff_attn: d must be 32 or 64");
    if (a.H == 0 || a.Hk == 0 || a.H % a.Hk || a.H / a.Hk > 128)
        return fail(TSN_ERR_ARG, "tsn_diff_attn: H must be a multiple of Hk, at most 128 times it");
    if (a.Sq > (1u << 30) || a.Sk > (1u << 30) || a.B > 65535 || a.H > 65535)
        return fail(TSN_ERR_ARG, "tsn_diff_attn: at most 2^30 queries or keys, 65535 sequences or heads");
    if (!(a.scale >= 0.0f) || !(a.eps >= 0.0f)) return fail(TSN_ERR_ARG, "tsn_diff_attn: negative scale or eps");
    if (a.B == 0 || a.Sq == 0) return TSN_OK;
    if ((long long) a.B * a.Sq * a.H > 0x7fffffffLL * 4) return fail(TSN_ERR_ARG, "tsn_diff_attn: too many query rows");
    if (!a.q.p || !a.out.p || (a.Sk && (!a.k.p || !a.v.p)) || !a.lq1 || !a.lk1 || !a.lq2 || !a.lk2)
        return fail(TSN_ERR_ARG, "tsn_diff_attn: null operand");
    auto aligned = [&](const tsn_heads & t, uint32_t S, uint32_t H) {   // a stride that is never taken does not count
        return ((uintptr_t) t.p & 15) == 0 && (a.B == 1 || t.sb % 8 == 0) && (S <= 1 || t.ss % 8 == 0) && (H == 1 || t.sh % 8 == 0);
    };
    if (!aligned(a.q, a.Sq, a.H) || !aligned(a.out, a.Sq, a.H) || (a.Sk && (!aligned(a.k, a.Sk, a.Hk) || !aligned(a.v, a.Sk, a.Hk))))
        return fail(TSN_ERR_ARG, "tsn_diff_attn: base addresses and strides must be multiples of 16 bytes");
    if ((a.B > 1 && !a.out.sb) || (a.Sq > 1 && !a.out.ss) || (a.H > 1 && !a.out.sh))
        return fail(TSN_ERR_ARG, "tsn_diff_attn: a result with a stride of 0");
    if (a.scale == 0.0f) a.scale = a.d == 32 ? 0.17677669529663687f : 0.125f;
    cudaError_t e = a.type == TSN_F16 ? launch<__half>(a, c.stream) : launch<__nv_bfloat16>(a, c.stream);
    if (e != cudaSuccess) return fail(TSN_ERR_CUDA, std::string("tsn_diff_attn: ") + cudaGetErrorString(e));
    return TSN_OK;
}

} // namespace tsn

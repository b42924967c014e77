// paged_attn.cu — attention of new tokens over a paged key/value cache (tsn_paged_attn), and over the pages that a token has
// chosen (the second kernel of tsn_sparse_attn).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - ref),  ref the running maximum, in one pass over the keys.
// A warp takes one query head: each lane holds D / 32 elements of q and o.
#include <cmath>

#include "attn_ops.cuh"
#include "kernels.h"
#include "paged.h"

namespace tsn {

cudaError_t configure_page_select();

namespace {

constexpr float LOG2E = 1.44269504088896341f;

struct Args {
    tsn_paged c;
    uint32_t H, window, picks;
    int causal, page_log2;
    float scale;   // times log2(e)
    tsn_rows q, out;
    const int * chosen;   // null: every page
};

template <class T, int D>
__global__ void __launch_bounds__(128) paged_attn_warp(const __grid_constant__ Args p) {
    constexpr int E = D / 32;
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long item = (long long) blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= (long long) p.c.N * p.H) return;
    const int row = (int) (item / p.H), h = (int) (item % p.H), hk = h / (int) (p.H / p.c.Hk);
    const int b = seq_of_row(p.c, row);
    if (b < 0) return;
    const int place = place_of_row(p.c, b, row), page = 1 << p.page_log2;
    const int all = (int) min((long long) max(0, p.c.len[b]), (long long) p.c.M << p.page_log2);
    int lo = 0, hi = all;
    if (p.causal) hi = (int) min((long long) hi, (long long) place + 1);
    if (p.window) lo = (int) max(0ll, (long long) place - (long long) p.window + 1);
    const T * qp = (const T *) p.q.p + row * p.q.sb + h * p.q.st + lane * E;
    float q[E], o[E] = {}, l = 0.0f, ref = -INFINITY;
    for (int e = 0; e < E; ++e) q[e] = to_f32(qp[e]) * p.scale;
    const int * chosen = p.chosen ? p.chosen + ((long long) row * p.c.Hk + hk) * p.picks : nullptr;
    const int pages = chosen ? (int) p.picks : (hi + page - 1) >> p.page_log2;
    for (int x = chosen ? 0 : lo >> p.page_log2; x < pages; ++x) {
        const int index = chosen ? chosen[x] : x;
        if (index < 0) break;
        const int id = page_of(p.c, b, index);
        if (id < 0) continue;
        const T * kp = (const T *) p.c.k.p + id * p.c.k.sb + hk * p.c.k.sh + lane * E, * vp = (const T *) p.c.v.p + id * p.c.v.sb + hk * p.c.v.sh + lane * E;
        for (int t = max(0, lo - index * page); t < page && index * page + t < hi; ++t) {
            float s = 0.0f;
            for (int e = 0; e < E; ++e) s = fmaf(q[e], to_f32(kp[t * p.c.k.ss + e]), s);
            for (int x2 = 16; x2; x2 >>= 1) s += __shfl_xor_sync(~0u, s, x2);
            if (s > ref) {
                const float f = ex2(ref - s);
                ref = s;
                l *= f;
                for (int e = 0; e < E; ++e) o[e] *= f;
            }
            const float w = ex2(s - (ref == -INFINITY ? 0.0f : ref));
            l += w;
            for (int e = 0; e < E; ++e) o[e] = fmaf(w, to_f32(vp[t * p.c.v.ss + e]), o[e]);
        }
    }
    T * out = (T *) p.out.p + row * p.out.sb + h * p.out.st + lane * E;
    for (int e = 0; e < E; ++e) out[e] = from_f32<T>(l == 0.0f ? 0.0f : o[e] / l);
}

cudaError_t launch(const Args & p, cudaStream_t s) {
    const dim3 grid((unsigned) (((long long) p.c.N * p.H + 3) / 4));
    const bool bf = p.c.type == TSN_BF16;
    cudaError_t e;
    if (p.c.D == 64) e = bf ? launch_cl(paged_attn_warp<__nv_bfloat16, 64>, grid, dim3(128), 0, s, dim3(1), p) : launch_cl(paged_attn_warp<__half, 64>, grid, dim3(128), 0, s, dim3(1), p);
    else e = bf ? launch_cl(paged_attn_warp<__nv_bfloat16, 128>, grid, dim3(128), 0, s, dim3(1), p) : launch_cl(paged_attn_warp<__half, 128>, grid, dim3(128), 0, s, dim3(1), p);
    if (e != cudaSuccess) cudaGetLastError();
    return e;
}

} // namespace

cudaError_t configure_paged() { return configure_page_select(); }

int paged_attn(DeviceCtx & c, const tsn_paged_attn_args & a) {
    if (a.c.N == 0 || a.c.B == 0) return TSN_OK;
    Args p{a.c, a.H, a.window, 0, a.causal, log2_of(a.c.page), (a.scale == 0.0f ? 1.0f / std::sqrt((float) a.c.D) : a.scale) * LOG2E, a.q, a.out, nullptr};
    const cudaError_t e = launch(p, c.stream);
    return e == cudaSuccess ? TSN_OK : fail(TSN_ERR_CUDA, std::string("tsn_paged_attn: ") + cudaGetErrorString(e));
}

int sparse_attn(DeviceCtx & c, const tsn_sparse_attn_args & a) {
    if (a.c.N == 0 || a.c.B == 0) return TSN_OK;
    cudaError_t e = launch_page_select(a, c.stream);
    Args p{a.c, a.H, 0, a.picks, 1, log2_of(a.c.page), (a.scale == 0.0f ? 1.0f / std::sqrt((float) a.c.D) : a.scale) * LOG2E, a.q, a.out, a.chosen};
    if (e == cudaSuccess) e = launch(p, c.stream);
    else cudaGetLastError();
    return e == cudaSuccess ? TSN_OK : fail(TSN_ERR_CUDA, std::string("tsn_sparse_attn: ") + cudaGetErrorString(e));
}

} // namespace tsn

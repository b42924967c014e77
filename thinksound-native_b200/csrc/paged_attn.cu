// paged_attn.cu — attention of new tokens over a paged key/value cache (tsn_paged_attn), and over the pages that a token has
// chosen (the second kernel of tsn_sparse_attn).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - ref),  ref the running maximum, in one pass over the keys.
// A warp takes one query head: each lane holds D / 32 elements of q and o.
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "paged_attn.h"
#include "split_ws.h"

namespace tsn {

cudaError_t configure_page_select();

namespace {

template <class T, int D>
__global__ void __launch_bounds__(128) paged_attn_warp(const __grid_constant__ PagedArgs p) {
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

cudaError_t launch(const PagedArgs & p, cudaStream_t s) {
    const dim3 grid((unsigned) (((long long) p.c.N * p.H + 3) / 4));
    const bool bf = p.c.type == TSN_BF16;
    if (p.c.D == 64) return bf ? launch_cl(paged_attn_warp<__nv_bfloat16, 64>, grid, dim3(128), 0, s, dim3(1), p) : launch_cl(paged_attn_warp<__half, 64>, grid, dim3(128), 0, s, dim3(1), p);
    return bf ? launch_cl(paged_attn_warp<__nv_bfloat16, 128>, grid, dim3(128), 0, s, dim3(1), p) : launch_cl(paged_attn_warp<__half, 128>, grid, dim3(128), 0, s, dim3(1), p);
}

PagedArgs args_of(const DeviceCtx & c, const tsn_paged & cache, uint32_t H, float scale) {
    PagedArgs p{};
    p.c = cache;
    if (p.c.P == 0) p.c.M = 0;   // no page: no key
    p.H = (int) H;
    p.G = (int) (H / cache.Hk);
    p.page_log2 = log2_of(cache.page);
    p.scale = (scale == 0.0f ? 1.0f / std::sqrt((float) cache.D) : scale) * PAGED_LOG2E;
    p.err = c.d_err;
    return p;
}

// Rows of a kv head up to which groups of 8 or 16 are taken
constexpr uint64_t FEW = 32;

// The few-rows kernel with what it needs of the workspace.
int few_rows(DeviceCtx & c, const char * name, PagedArgs & p, uint32_t most) {
    size_t groups = 0, bytes = 0;
    SplitUse use;
    plan_paged_rows(p, most, &groups, &bytes);
    if (groups) {
        if (const int rc = split_begin(c, name, groups, bytes, use)) return rc;
        p.count = use.count;
        p.part = use.part;
    }
    cudaError_t e = launch_paged_rows(p, most, c.stream);
    if (e == cudaSuccess && groups) e = split_end(c, use);
    if (e == cudaSuccess) return TSN_OK;
    cudaGetLastError();
    return fail(TSN_ERR_CUDA, std::string(name) + ": " + cudaGetErrorString(e));
}

} // namespace

// {D, page, Hk, P} views with {64, tokens, 1, 1} boxes. A dimension of one element has a stride that is never taken: any valid one
// stands in. Without pages nothing is loaded, but the map of some page has to be valid.
bool make_page_maps(const tsn_paged & c, uint32_t tokens, CUtensorMap * tk, CUtensorMap * tv) {
    const PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
    if (!enc) return false;
    if (c.P == 0) return true;
    bool ok = true;
    for (int i = 0; i < 2; ++i) {
        const tsn_heads & t = i ? c.v : c.k;
        const cuuint64_t row = c.D * 2;
        const cuuint64_t dims[4] = {c.D, c.page, c.Hk, c.P};
        const cuuint64_t strides[3] = {(cuuint64_t) t.ss * 2, c.Hk > 1 ? (cuuint64_t) t.sh * 2 : row, c.P > 1 ? (cuuint64_t) t.sb * 2 : row};
        const cuuint32_t box[4] = {64, tokens, 1, 1}, es[4] = {1, 1, 1, 1};
        ok = ok && enc(i ? tv : tk, c.type == TSN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, t.p, dims, strides, box, es,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    return ok;
}

cudaError_t configure_paged() {
    cudaError_t e = configure_page_select();
    if (e == cudaSuccess) e = configure_paged_rows();
    return e;
}

int paged_attn(DeviceCtx & c, const tsn_paged_attn_args & a) {
    if (a.c.N == 0 || a.c.B == 0) return TSN_OK;
    PagedArgs p = args_of(c, a.c, a.H, a.scale);
    p.q = a.q;
    p.out = a.out;
    p.causal = a.causal != 0;
    p.window = (int) a.window;
    const uint32_t most = !a.c.q_start ? 1 : a.most ? std::min(a.most, a.c.N) : a.c.N;
    if ((uint64_t) most * p.G <= FEW) return few_rows(c, "tsn_paged_attn", p, most);
    const cudaError_t e = launch(p, c.stream);
    if (e == cudaSuccess) return TSN_OK;
    cudaGetLastError();
    return fail(TSN_ERR_CUDA, std::string("tsn_paged_attn: ") + cudaGetErrorString(e));
}

int sparse_attn(DeviceCtx & c, const tsn_sparse_attn_args & a) {
    if (a.c.N == 0 || a.c.B == 0) return TSN_OK;
    PagedArgs p = args_of(c, a.c, a.H, a.scale);
    p.q = a.q;
    p.out = a.out;
    p.causal = 1;
    p.picks = (int) a.picks;
    p.chosen = a.chosen;
    if ((uint64_t) a.c.N * a.c.Hk * ((p.G + 7) / 8) > 0x7fffffffu) return fail(TSN_ERR_ARG, "tsn_sparse_attn: too many query rows");
    const cudaError_t e = launch_page_select(a, c.stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(TSN_ERR_CUDA, std::string("tsn_sparse_attn: ") + cudaGetErrorString(e));
    }
    return few_rows(c, "tsn_sparse_attn", p, 1);
}

} // namespace tsn

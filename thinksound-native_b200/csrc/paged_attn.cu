// paged_attn.cu — attention of new tokens over a paged key/value cache (tsn_paged_attn), and over the pages that a token has
// chosen (the second kernel of tsn_sparse_attn).
// The kernels are in paged_rows.cu (few query rows of a kv head) and paged_tiles.cu; here is which of them runs.
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "paged_attn.h"
#include "split_ws.h"

namespace tsn {

cudaError_t configure_page_select();

namespace {

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
    if (e == cudaSuccess) e = configure_paged_tiles();
    return e;
}

namespace {
PagedArgs args_of(const DeviceCtx & c, const tsn_paged_attn_args & a, uint32_t & most) {
    PagedArgs p = args_of(c, a.c, a.H, a.scale);
    p.q = a.q;
    p.out = a.out;
    p.causal = a.causal != 0;
    p.window = (int) a.window;
    most = !a.c.q_start ? 1 : a.most ? std::min(a.most, a.c.N) : a.c.N;
    return p;
}
} // namespace

// The few-rows kernel whatever the rows are; what it reports is for the caller to fetch.
int selftest_paged_timeout(DeviceCtx & c, const tsn_paged_attn_args & a, uint32_t block) {
    if (a.c.N == 0 || a.c.B == 0) return TSN_OK;
    uint32_t most;
    PagedArgs p = args_of(c, a, most);
    p.give_up = (int) block + 1;
    return few_rows(c, "tsn_selftest_paged_timeout", p, most);
}

int paged_attn(DeviceCtx & c, const tsn_paged_attn_args & a) {
    if (a.c.N == 0 || a.c.B == 0) return TSN_OK;
    uint32_t most;
    PagedArgs p = args_of(c, a, most);
    // Up to eight rows of a kv head go to the kernel for few; beyond, the one that the estimates of both prefer: groups of rows read
    // the keys anew, but go to every SM where a tile's keys have eight at most. us by groups / by tiles, heads of 128, bf16:
    // 16 tokens x 4 heads, 8 kv heads over 8192 keys 37/24; 16 streams of 4 tokens over 4096 56/60, of 8 tokens 95/61; 64 streams of 4
    // over 1000 57/78, of 8 164/79; one kv head over 32 768 keys, 64 rows 29/60, 128 rows 35/61.
    if ((uint64_t) most * p.G <= 8 || paged_rows_cost(p, most) < plan_paged_tiles(p, most)) return few_rows(c, "tsn_paged_attn", p, most);
    const cudaError_t e = launch_paged_tiles(p, c.stream);
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

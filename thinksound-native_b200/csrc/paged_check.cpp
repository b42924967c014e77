// paged_check.cpp — the refusals of the paged cache's operators (include/tsn.h). Host only: an argument that is refused is
// refused before any device work.
#include <cmath>
#include <initializer_list>

#include "paged.h"

namespace tsn {

namespace {

int refuse(const char * name, const char * why) { return fail(TSN_ERR_ARG, std::string(name) + ": " + why); }

// strides that are taken are positive multiples of 16 bytes (8 elements), below 2^39 elements
bool stride_ok(uint32_t extent, int64_t s, int align) { return extent <= 1 || (s > 0 && s % align == 0 && s < (1ll << 39)); }

int check_cache(const char * name, const tsn_paged & c) {
    if (c.type != TSN_F16 && c.type != TSN_BF16) return refuse(name, "type must be TSN_F16 or TSN_BF16");
    if (c.page < 16 || c.page > 1024 || (c.page & (c.page - 1))) return refuse(name, "page must be a power of two, 16..1024");
    if (c.B > 65535 || c.Hk < 1 || c.Hk > 65535) return refuse(name, "at most 65535 sequences, 1 to 65535 heads");
    if (c.N > (1u << 30) || c.P > 0x7fffffffu || (uint64_t) c.M * c.page > (1u << 30))
        return refuse(name, "at most 2^30 new tokens and places of a sequence, 2^31 - 1 pages");
    if (c.N == 0 || c.B == 0) return c.N && !c.q_start ? refuse(name, "without q_start, N must be B") : TSN_OK;
    if (!c.q_start && c.N != c.B) return refuse(name, "without q_start, N must be B");
    if (!c.len || (c.M && !c.table) || (c.P && (!c.k.p || !c.v.p))) return refuse(name, "null cache, table or len");
    if ((((uintptr_t) c.len | (uintptr_t) c.table | (uintptr_t) c.q_start) & 3)) return refuse(name, "an address that is no multiple of its element's size");
    if (c.B > 1 && c.M && c.table_sb < 0) return refuse(name, "a negative stride of the table");
    for (const tsn_heads * t : {&c.k, &c.v})
        if (((uintptr_t) t->p & 15) || !stride_ok(c.P, t->sb, 8) || !stride_ok(c.page, t->ss, 8) || !stride_ok(c.Hk, t->sh, 8))
            return refuse(name, "base addresses and strides of k and v must be multiples of 16 bytes, strides positive");
    return TSN_OK;
}

// [extent, heads, D] rows of inputs (a stride of 0 repeats) or results
int check_rows(const char * name, const tsn_rows & r, uint32_t extent, uint32_t heads, int size, bool result) {
    if (!r.p) return refuse(name, "null operand");
    const int align = 16 / size;
    auto ok = [&](uint32_t n, int64_t s) { return n <= 1 || (s % align == 0 && (!result || s != 0)); };
    if (((uintptr_t) r.p & 15) || !ok(extent, r.sb) || !ok(heads, r.st))
        return refuse(name, "addresses and strides must be multiples of 16 bytes, a result's not 0");
    return TSN_OK;
}

int check_heads(const char * name, const tsn_paged & c, uint32_t H, float scale) {
    if (c.D != 64 && c.D != 128) return refuse(name, "D must be 64 or 128");
    if (H == 0 || H > 65535 || H % c.Hk || H / c.Hk > 128) return refuse(name, "H must be a multiple of Hk, at most 128 times it");
    if (!(scale >= 0.0f) || !std::isfinite(scale)) return refuse(name, "scale must be finite, not negative");
    if ((uint64_t) c.N * (H / c.Hk) > (1u << 30)) return refuse(name, "more than 2^30 query rows of a kv head");
    return TSN_OK;
}

} // namespace

int check_cache_append(const tsn_rope_plan_t * plan, const tsn_cache_append_args * a) {
    const char * const name = "tsn_cache_append";
    if (!plan || !a) return fail(TSN_ERR_ARG, "null argument");
    const tsn_rope_plan_t & p = *plan;
    if (p.D < 2 || p.D > 2 * TSN_ROPE_MAX_PAIRS || p.D % 2 || p.P > p.D / 2 || p.axes < 1 || p.axes > TSN_ROPE_MAX_AXES ||
        (p.layout != TSN_ROPE_INTERLEAVED && p.layout != TSN_ROPE_HALF))
        return refuse(name, "not a plan of tsn_rope_plan");
    for (uint32_t j = 0; j < p.P; ++j)
        if (p.axis[j] >= p.axes) return refuse(name, "not a plan of tsn_rope_plan");
    if (int rc = check_cache(name, a->c)) return rc;
    if (a->c.D != p.D || p.D % 8) return refuse(name, "D must be the plan's, a multiple of 8");
    if (a->xtype != a->c.type && a->xtype != TSN_F32) return refuse(name, "xtype must be the cache's type or TSN_F32");
    if (!(a->eps >= 0.0f)) return refuse(name, "negative eps");
    if (a->c.N == 0 || a->c.B == 0) return TSN_OK;
    const int size = (int) type_size(a->xtype);
    const bool queries = a->q.p && a->Hq;
    if (a->Hq > 65535) return refuse(name, "at most 65535 heads");
    int rc = check_rows(name, a->k, a->c.N, a->c.Hk, size, false);
    if (!rc) rc = check_rows(name, a->v, a->c.N, a->c.Hk, size, false);
    if (!rc && queries) rc = check_rows(name, a->q, a->c.N, a->Hq, size, false);
    if (!rc && queries) rc = check_rows(name, a->q_out, a->c.N, a->Hq, 2, true);
    if (!rc && a->means.p) rc = check_rows(name, a->means, a->c.P, a->c.Hk, 2, true);
    if (rc) return rc;
    if (!a->pos && p.P && p.axes != 1) return refuse(name, "null positions of a plan with several axes");
    if (((uintptr_t) a->pos | (uintptr_t) a->q_norm | (uintptr_t) a->k_norm) & 3) return refuse(name, "an address that is no multiple of its element's size");
    return TSN_OK;
}

int check_paged_attn(const tsn_paged_attn_args * a) {
    const char * const name = "tsn_paged_attn";
    if (!a) return fail(TSN_ERR_ARG, "null argument");
    if (int rc = check_cache(name, a->c)) return rc;
    if (int rc = check_heads(name, a->c, a->H, a->scale)) return rc;
    if (a->window > (1u << 30)) return refuse(name, "a window of more than 2^30 tokens");
    if (a->window && !a->causal) return refuse(name, "a window without causal");
    if (a->c.N == 0 || a->c.B == 0) return TSN_OK;
    int rc = check_rows(name, a->q, a->c.N, a->H, 2, false);
    if (!rc) rc = check_rows(name, a->out, a->c.N, a->H, 2, true);
    return rc;
}

int check_sparse_attn(const tsn_sparse_attn_args * a) {
    const char * const name = "tsn_sparse_attn";
    if (!a) return fail(TSN_ERR_ARG, "null argument");
    if (int rc = check_cache(name, a->c)) return rc;
    if (int rc = check_heads(name, a->c, a->H, a->scale)) return rc;
    if (a->last < 1 || a->picks > 1024 || (uint64_t) a->first + a->last > a->picks) return refuse(name, "first + last, last at least 1, must be at most picks, which is at most 1024");
    if (a->c.M > 16384) return refuse(name, "at most 16384 pages of a sequence");
    if (a->c.N == 0 || a->c.B == 0) return TSN_OK;
    int rc = check_rows(name, a->q, a->c.N, a->H, 2, false);
    if (!rc) rc = check_rows(name, a->out, a->c.N, a->H, 2, true);
    if (!rc && a->c.P) rc = check_rows(name, a->means, a->c.P, a->c.Hk, 2, false);
    if (rc) return rc;
    if (!a->chosen || ((uintptr_t) a->chosen & 3)) return refuse(name, "null or unaligned chosen");
    return TSN_OK;
}

} // namespace tsn

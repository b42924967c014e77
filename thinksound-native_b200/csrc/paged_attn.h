// paged_attn.h — what the kernels of attention over the paged cache share: a call's arguments and a warp's view of its batch.
#pragma once
#include <cuda.h>

#include "attn_ops.cuh"
#include "paged.h"

namespace tsn {

constexpr int SMS = 148;
constexpr float PAGED_LOG2E = 1.44269504088896341f;

struct PagedArgs {
    tsn_paged c;
    tsn_rows q, out;
    const int * chosen;   // the pages of each row and kv head, or null: all
    int H, G, picks;      // G: query heads of a kv head
    int causal, window, page_log2;
    float scale;          // times log2(e)
    // split keys
    int whole, parts;     // whole: no unit is split; parts of a unit where the pages are chosen
    float * part;
    unsigned int * count;
    int * err;
    int give_up;          // a test of the failure path: the block (from 1) whose first unit's waits count as run out
};

// A probability is 2^(x - ref + ABOVE), x the score in log2 units and ref the reference of its row: the greatest x so far or up to
// LAZY below it. bf16 has the exponents of f32. In f16 numbers from 2^-14 on have all bits and those below 2^-25 are zero, so its
// range above 1 is used up to 2^15: keys up to 2^21 below the greatest keep their bits, and each one further below is off by up to 2^-32
// of the greatest one's share. (With ABOVE 0 the share of 131 072 equal keys 16 nats below one other was off by 6 %. With LAZY 4 and
// ABOVE 11 the tiles take 1 to 4 % more time, with 2 and 13 7 to 15 %.)
template <bool BF16>
struct Reference {
    static constexpr float LAZY = 8.0f, ABOVE = BF16 ? 0.0f : 7.0f;
};

// {D, page, Hk, P} views of keys and values with {64, tokens, 1, 1} boxes
bool make_page_maps(const tsn_paged & c, uint32_t tokens, CUtensorMap * tk, CUtensorMap * tv);

// Keys that a row at a place sees: lo .. hi - 1; n: the sequence's cached keys.
__device__ __forceinline__ int seen_to(const PagedArgs & p, int place, int n) {
    return p.causal ? max(0, min(n, place + (place < 0x7fffffff))) : n;
}
__device__ __forceinline__ int seen_from(const PagedArgs & p, int place) {
    return p.window ? (int) max(0ll, (long long) place - p.window + 1) : 0;
}
__device__ __forceinline__ int cached(const PagedArgs & p, int len) {
    return (int) min((long long) max(0, len), (long long) p.c.M << p.page_log2);
}
// the place of the first of n new tokens
__device__ __forceinline__ int first_place(int len, int n) { return (int) max(-0x40000000ll, (long long) len - n); }

// The values of keys from .. until - 1 that are not finite, added to E columns of a row: where rows see different keys of a
// tile, the product took zeros in their place. They are added whatever the keys' probabilities: the column is not finite either way, as
// it is where the product takes them (p times infinity, or NaN where p is 0). Rare, one key after another.
template <bool BF16, int E>
__device__ __noinline__ void add_not_finite(const PagedArgs & p, int b, int hk, int from, int until, int col, float * o) {
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    for (int j = from; j < until; ++j) {
        const int id = page_of(p.c, b, j >> p.page_log2);
        if (id < 0) continue;
        const T * v = (const T *) p.c.v.p + id * p.c.v.sb + (long long) (j & ((1 << p.page_log2) - 1)) * p.c.v.ss + hk * p.c.v.sh + col;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float x = to_f32(v[e]);
            if (!isfinite(x)) o[e] += x;
        }
    }
}

cudaError_t configure_paged_rows();
// A few query rows of a kv head at a time (most: new tokens of a sequence). The plan sets how keys are split, and says how many counters
// and bytes of the workspace that takes; the launch comes after these are there.
void plan_paged_rows(PagedArgs & p, uint32_t most, size_t * groups, size_t * bytes);
cudaError_t launch_paged_rows(const PagedArgs & p, uint32_t most, cudaStream_t s);
// About what it takes, in microseconds: groups of rows read the keys anew, which come at 1.4 ns a slab of 16.
double paged_rows_cost(const PagedArgs & p, uint32_t most);

cudaError_t configure_paged_tiles();
// 256 query rows of a kv head at a time. The plan sets the parts of the keys and returns about what the call takes, in microseconds.
double plan_paged_tiles(PagedArgs & p, uint32_t most);
cudaError_t launch_paged_tiles(const PagedArgs & p, cudaStream_t s);

} // namespace tsn

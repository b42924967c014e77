// paged.h — the operators of the paged key/value cache (include/tsn.h): checks of their arguments, which need no device, and
// what their kernels share of a batch.
#pragma once
#include "block_ops.h"

namespace tsn {

// TSN_OK, or the refusal: before any device work
int check_cache_append(const tsn_rope_plan_t * plan, const tsn_cache_append_args * a);
int check_paged_attn(const tsn_paged_attn_args * a);
int check_sparse_attn(const tsn_sparse_attn_args * a);
// of checked arguments
int cache_append(DeviceCtx & c, const tsn_rope_plan_t & plan, const tsn_cache_append_args & a);
int paged_attn(DeviceCtx & c, const tsn_paged_attn_args & a);
int sparse_attn(DeviceCtx & c, const tsn_sparse_attn_args & a);
int selftest_paged_timeout(DeviceCtx & c, const tsn_paged_attn_args & a, uint32_t block);
cudaError_t launch_page_select(const tsn_sparse_attn_args & a, cudaStream_t s);
cudaError_t configure_paged();   // once per device, before the first launch

// A page's tokens are a power of two, given to kernels as its exponent.
inline int log2_of(uint32_t x) {
    int n = 0;
    while ((1u << n) < x) ++n;
    return n;
}

// Row at which the new tokens of sequence b start (b up to B), within 0..N whatever q_start holds.
__device__ __forceinline__ int seq_start(const tsn_paged & c, int b) {
    return c.q_start ? max(0, min(c.q_start[b], (int) c.N)) : b;
}

// The sequence of a row, by a whole warp; -1: none. A step leaves a 32nd of the sequences.
__device__ __forceinline__ int seq_of_row(const tsn_paged & c, int row) {
    if (!c.q_start) return row < (int) c.N ? row : -1;
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = (int) c.B;   // the last of the numbers 0..B-1 whose start is not above the row lies in lo..hi-1
    while (true) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const unsigned below = __ballot_sync(~0u, at < hi && c.q_start[at] <= row);
        if (!below) return -1;
        const int k = 31 - __clz(below);
        lo += k * step;
        hi = min(hi, lo + step);
        if (step <= 1) break;
    }
    return row < c.q_start[lo + 1] ? lo : -1;
}

// The same by a single thread.
__device__ __forceinline__ int seq_of_row_alone(const tsn_paged & c, int row) {
    if (!c.q_start) return row < (int) c.N ? row : -1;
    if (c.q_start[0] > row) return -1;
    int lo = 0, hi = (int) c.B;   // the last start that is not above the row lies in lo .. hi - 1
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (c.q_start[mid] <= row) lo = mid;
        else hi = mid;
    }
    return row < c.q_start[lo + 1] ? lo : -1;
}

// The place of a row of sequence b among its tokens: len - n + i, kept within 32 bits.
__device__ __forceinline__ int place_of_row(const tsn_paged & c, int b, int row) {
    const long long p = (long long) c.len[b] - seq_start(c, b + 1) + row;
    return (int) max(-0x40000000ll, min(p, 0x7fffffffll));
}

// The page of a place, or -1: no page
__device__ __forceinline__ int page_of(const tsn_paged & c, int b, int index) {
    if (index < 0 || index >= (int) c.M) return -1;
    const int id = c.table[b * c.table_sb + index];
    return id >= 0 && id < (int) c.P ? id : -1;
}

} // namespace tsn

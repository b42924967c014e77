// paged_tiles.cu — attention over the paged cache for many query rows of a kv head, on the tcgen05 tensor cores.
//
//   o = sum_j p_j v_j / l,  l = sum_j p_j,  p_j = 2^(c q.k_j - ref + ABOVE)
// in one pass over the keys; ref follows the row's running maximum and moves, with o and l rescaled, when that has grown by more than
// LAZY (struct Reference). P is rounded to 16 bits, as the tensor cores take it; scores, maxima, sums and o are f32, and l is the sum of the rounded ones, so
// that rounding cancels where values are alike, and a NaN, which the FMA pipe's exponential only has after rounding (as an
// infinity), reaches l. That takes a mixed add a value instead of a packed one for two: 795 -> 803 us for the 4096 tokens below, 702 -> 768 with 64-wide heads.
// A unit is 256 query rows of a sequence and kv head, (token, head of the group), as two tiles of 128, so that heads of a group share
// the keys; a CTA takes a unit or, where there are few, a part of its keys, the parts of a cluster adding up their sums. 384 threads:
//   warps 0-3, 4-7  softmax of a tile, one row a thread: S from TMEM, mask, maximum, exponentials, P over S's columns
//   warp 8          TMA: 128 keys, then their values, through one ring of stages; a tile may lie in several pages, a lane a box
//   warps 9, 10     issue a tile's products: P_j V, then Q K_j+1 (so that S_j+1 being there means that O holds tile j)
//   warp 11         where some keys are not seen by all rows: makes the tiles' V rows fit for the product
// While one tile's products run, the other's exponentials do. TMEM: S of both tiles (2 x 128 columns) and O (2 x D).
// Values behind keys that are not there may be NaN, and 0 * NaN is NaN: those rows of V are cleared. Where rows differ in what they
// see, values that are not finite are cleared too and added again to the rows that do see them.
// Every wait is bounded; barriers of a whole block or cluster are on paths that all threads take.
// What bounds it: 256 rows x 128 keys of 128 elements are 2048 cycles of the tensor cores (both products at 64 cycles an instruction of
// 128 x 128 x 16, measured alone) and 1790 of the SFU (16 exponentials a cycle, one pair of eight on the FMA pipe). A tile's way is
// 170 cycles for S to arrive, 280 for the maximum, 1220 for the exponentials, 150 to hand P over, then its products: the two tiles'
// ways interleave at about 3800 cycles. 4096 tokens over 16 384 keys (32 heads over 8, bf16) take 810 us, 1.19
// PFLOP/s, in short runs and 940 to 950 in long ones, where the power limit holds the clock; 64-wide heads 768 us (0.63).
// Tried and worse, when the kernel took 816 us: products under a branch that the compiler takes for divergent (100 cycles an instruction; 1245 us), both tiles'
// products by one warp (880), side by side without turns (980), turns for the second half of P only (910), every fourth pair on
// the FMA pipe (976) or none (845), exponentials before the maximum, done again where it moves (1370), spinning instead of suspended
// waits (+1 to 3 %), registers moved to the softmax warps (+2 %).
#include "kernels.h"
#include "paged_attn.h"

#include <algorithm>
#include <atomic>

namespace tsn {

namespace {

constexpr int ROWS = 256, KEYS = 128, THREADS = 384;

template <int D>
struct Lay {
    static constexpr int ATOMS = D / 64, BOX = KEYS * 128, TILE = KEYS * D * 2;   // boxes of 128 rows x 64 elements
    static constexpr int STAGES = D == 128 ? 5 : 10, DEEP = 16;                   // DEEP: above the tiles on their way
    static constexpr int OFF_RING = 2 * TILE, OFF_BAR = OFF_RING + STAGES * TILE, TOTAL = OFF_BAR + 640;   // Q's two tiles first
    static constexpr int SUM_ROW = D + 4;
    static constexpr int EVERY = 8;   // one pair of exponentials of so many takes the FMA pipe
    static constexpr uint32_t TM_O = 2 * KEYS, TM = 512;
    static_assert(TOTAL + 64 <= 227 * 1024, "one CTA's shared memory");
    static_assert(ROWS * SUM_ROW * 4 <= STAGES * TILE, "the rows' sums fit in the ring");
    static_assert(TM_O + 2 * D <= TM, "tensor memory");
    static_assert((12 + 3 * STAGES) * 8 + (2 + DEEP + 4 * STAGES) * 4 <= 640, "barriers");
};

__device__ __forceinline__ void bar_n(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

template <int D, bool BF16>
__global__ void __launch_bounds__(THREADS, 1)
paged_tiles_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ PagedArgs p) {
    using L = Lay<D>;
    constexpr int CH = D / 8, STAGES = L::STAGES;   // CH: 16-byte pieces of a head
    constexpr float LAZY = Reference<BF16>::LAZY, ABOVE = Reference<BF16>::ABOVE;
    extern __shared__ __align__(1024) uint8_t smem[];
    // sequence, its first row, kv head, first query row, query rows, length, new tokens, tokens of rows 127 and the last; (token, head) of the rows
    __shared__ int unit_of[9];
    __shared__ uint16_t row_of[ROWS];
    // the warp's number as the compiler knows it to be one for all lanes: products issued under a branch that it takes for divergent
    // cost 100 cycles and more each
    const int tid = threadIdx.x, warp = __shfl_sync(~0u, tid >> 5, 0), lane = tid & 31;
    const bool fits = (smem_u32(smem) & 1023) == 0;   // the swizzled tiles need 1024-byte alignment
    if (!fits && tid == 0 && p.err) atomicCAS(p.err, 0, DEV_BAD_ARGS);
    uint64_t * bar = (uint64_t *) (smem + L::OFF_BAR);
    // v_ready counts the tiles that pass through warp 11: a stage holds keys one time and values another
    uint64_t * q_full = bar, * s_full = bar + 2, * p_full = bar + 4, * o_full = bar + 6, * p_half = bar + 8, * turn = bar + 10, * full = bar + 12, * empty = full + STAGES, * v_ready = empty + STAGES;
    uint32_t * words = (uint32_t *) (v_ready + STAGES);   // TMEM address, abort flag, slabs with pages [DEEP tiles], keys of a tile that are not finite [STAGES tiles][4]
    volatile int * abort_flag = (volatile int *) (words + 1);
    volatile uint32_t * paged = words + 2, * not_finite = paged + L::DEEP;

    if (tid == 0) {
        for (int t = 0; t < 2; ++t) { mbar_init(&q_full[t], 4); mbar_init(&s_full[t], 1); mbar_init(&p_full[t], 4); mbar_init(&o_full[t], 1); mbar_init(&p_half[t], 4); mbar_init(&turn[t], 1); }
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 2); mbar_init(&v_ready[s], 1); }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 8 && lane == 0 && p.c.P) { tma_prefetch(&tk); tma_prefetch(&tv); }
    pdl_wait();   // from here on memory that earlier work may have written or may still read
    // Tensor memory after the wait and before the trigger: of two kernels on one SM, neither can hold what the other waits for.
    if (warp == 9) tmem_alloc(words, L::TM);

    // this CTA's unit: units of a sequence are (group of rows, kv head), the last rows, which see most, first
    const unsigned split = blockIdx.x % p.parts;
    if (warp == 0) {
        const long long gid = blockIdx.x / p.parts;
        long long before = 0;
        if (lane == 0) unit_of[0] = -1;
        __syncwarp();
        for (int b0 = 0; b0 < (int) p.c.B && before <= gid; b0 += 32) {
            const int b = b0 + lane;
            int start = 0, n = 0, len = 0;
            if (b < (int) p.c.B) {
                start = seq_start(p.c, b);
                n = max(0, seq_start(p.c, b + 1) - start);
                len = p.c.len[b];
            }
            const long long groups = ((long long) n * p.G + ROWS - 1) / ROWS, mine = groups * p.c.Hk;
            long long upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long v = __shfl_up_sync(~0u, upto, o);
                if (lane >= o) upto += v;
            }
            const long long at = before + upto - mine;
            if (at <= gid && gid < at + mine) {
                const unsigned u = (unsigned) (gid - at);
                const int first = ((int) groups - 1 - (int) (u / p.c.Hk)) * ROWS, last = n * p.G - 1;
                unit_of[0] = b;
                unit_of[1] = start;
                unit_of[2] = (int) (u % p.c.Hk);
                unit_of[3] = first;
                unit_of[4] = min(ROWS, last + 1 - first);
                unit_of[5] = len;
                unit_of[6] = n;
                unit_of[7] = min(last, first + 127) / p.G;
                unit_of[8] = last < first + ROWS ? last / p.G : (first + ROWS - 1) / p.G;
            }
            before += __shfl_sync(~0u, upto, 31);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(~0u, words[0], 0), TM_O = tmem + L::TM_O;
    const int b = unit_of[0];
    if (b < 0) {   // more CTAs than units, the whole cluster of them
        __syncthreads();
        if (warp == 9) tmem_dealloc(tmem, L::TM);
        return;
    }
    const int row0 = unit_of[1], hk = unit_of[2], r0 = unit_of[3], R = unit_of[4], len = unit_of[5], n = cached(p, len);
    const int place0 = first_place(len, unit_of[6]), token0 = r0 / p.G;
    // rows 0 .. 255 are (token, head of the group); a row at a place sees keys seen_from .. seen_to - 1
    auto hi_at = [&](int token) { return seen_to(p, place0 + token, n); };
    auto lo_at = [&](int token) { return min(seen_from(p, place0 + token), n); };
    const int token127 = unit_of[7], token_last = unit_of[8], token128 = R > 128 ? (r0 + 128) / p.G : token_last;
    // tiles of keys that some row sees, this part of them
    const int least = hi_at(token0), latest = lo_at(token_last);   // before least and from latest on every row sees
    const int tile0 = lo_at(token0) / KEYS, all_tiles = max(0, (hi_at(token_last) + KEYS - 1) / KEYS - tile0);
    const int per = (all_tiles + p.parts - 1) / p.parts;
    const int t0 = tile0 + min(all_tiles, (int) split * per), nt = fits ? tile0 + min(all_tiles, ((int) split + 1) * per) - t0 : 0;
    auto mixed = [&](int base) { return least < min(n, base + KEYS) || base < latest; };   // rows see different keys of the tile
    auto unfit = [&](int base) { return base + KEYS > n || mixed(base); };                 // its values pass through warp 11
    // the part's tiles that tile t of the rows sees: ja .. jb - 1
    auto from_of = [&](int t) { return 128 * t < R ? min(nt, max(0, lo_at(t ? token128 : token0) / KEYS - t0)) : 0; };
    auto until_of = [&](int t) { return 128 * t < R ? max(from_of(t), min(nt, (hi_at(t ? token_last : token127) + KEYS - 1) / KEYS - t0)) : 0; };

    if (warp >= 8) {
        if (warp == 8) {
            // Pages of a tile: a lane each of its boxes' rows, read one tile ahead
            const int box = min(KEYS, 1 << p.page_log2), pieces = KEYS / box;
            const int piece = lane % pieces, atom = lane / pieces;
            auto page_at = [&](int j) {
                const int key = (t0 + j) * KEYS + piece * box;
                return key < n ? page_of(p.c, b, key >> p.page_log2) : (int) p.c.P;   // what is behind the end counts as there, but is not loaded
            };
            int next = nt > 0 ? page_at(0) : 0;
            bool go = true;
            for (int j = 0; j < nt && go; ++j) {
                const int id = next;
                if (j + 1 < nt) next = page_at(j + 1);
                const uint32_t gone = __ballot_sync(~0u, lane < pieces && id < 0);
                uint32_t slabs = 0xffu;
                if (gone)
                    for (int x = 0; x < pieces; ++x)
                        if ((gone >> x) & 1u) slabs &= ~(((1u << (box / 16)) - 1u) << (x * (box / 16)));
                const int slot = ((t0 + j) * KEYS + piece * box) & ((1 << p.page_log2) - 1), page = id < 0 ? (int) p.c.P : id;   // past the last page: zeros
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    const int i = 2 * j + kv, s = i % STAGES;
                    if (i >= STAGES && !mbar_wait_soon(&empty[s], (i / STAGES - 1) & 1, abort_flag, p.err, DEV_TIMEOUT_EMPTY)) go = false;
                    go = __all_sync(~0u, go);
                    if (!go) break;
                    if (lane == 0) {
                        if (kv == 0) paged[j % L::DEEP] = slabs;
                        mbar_expect_tx(&full[s], L::TILE);
                    }
                    __syncwarp();
                    if (atom < L::ATOMS)
                        tma_load_4d(smem + L::OFF_RING + s * L::TILE + atom * L::BOX + piece * box * 128, kv ? &tv : &tk, &full[s], 64 * atom, slot, hk, page);
                }
            }
        } else if (warp == 11) {
            int seen = 0;
            for (int j = 0; j < nt; ++j) {
                const int base = (t0 + j) * KEYS, i = 2 * j + 1, s = i % STAGES;
                // every use of a stage in turn: a parity tells a use only from the one before
                if (!mbar_wait_soon(&full[(i - 1) % STAGES], ((i - 1) / STAGES) & 1, abort_flag, p.err, DEV_TIMEOUT_FULL) ||
                    !mbar_wait_soon(&full[s], (i / STAGES) & 1, abort_flag, p.err, DEV_TIMEOUT_FULL)) break;
                __syncwarp();
                if (!unfit(base)) continue;
                uint8_t * v = smem + L::OFF_RING + s * L::TILE;
                const bool mix = mixed(base);
                // rows of keys that are not there, a lane a key
                for (int key = max(0, n - base) + lane; key < KEYS; key += 32)
#pragma unroll
                    for (int y = 0; y < CH; ++y) *(uint4 *) (v + key * 128 + (y >> 3) * L::BOX + (y & 7) * 16) = make_uint4(0, 0, 0, 0);
                __syncwarp();
                uint32_t bad[4] = {0, 0, 0, 0};
                if (mix) {
                    // Mostly all are finite, and one look finds that out: with an exponent of ones, one more at the exponent's
                    // lowest bit carries into the sign's place.
                    constexpr uint32_t ONE = BF16 ? 0x00800080u : 0x04000400u;
                    uint32_t any = 0;
#pragma unroll 16
                    for (int y = lane; y < L::TILE / 16; y += 32) {
                        const uint4 o = *(const uint4 *) (v + y * 16);
                        any |= ((o.x & 0x7fff7fffu) + ONE) | ((o.y & 0x7fff7fffu) + ONE) | ((o.z & 0x7fff7fffu) + ONE) | ((o.w & 0x7fff7fffu) + ONE);
                    }
                    if (__any_sync(~0u, any & 0x80008000u)) {
                        constexpr int AT_ONCE = 32 / CH;   // rows of one step
                        const int sub = lane / CH, ch = lane % CH;
#pragma unroll 1
                        for (int y = 0; y < KEYS; y += AT_ONCE) {
                            const int key = y + sub;
                            uint4 * at = (uint4 *) (v + (ch >> 3) * L::BOX + key * 128 + (ch & 7) * 16);   // whichever piece lies there
                            const uint4 o = *at;
                            const uint4 f = make_uint4(finite_only<BF16>(o.x), finite_only<BF16>(o.y), finite_only<BF16>(o.z), finite_only<BF16>(o.w));
                            const bool found = o.x != f.x || o.y != f.y || o.z != f.z || o.w != f.w;
                            if (found) *at = f;
#pragma unroll
                            for (int w = 0; w < 4; ++w)
                                if (found && key >> 5 == w) bad[w] |= 1u << (key & 31);
                        }
#pragma unroll
                        for (int w = 0; w < 4; ++w) bad[w] = __reduce_or_sync(~0u, bad[w]);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    for (int w = 0; w < 4; ++w) not_finite[4 * (seen % STAGES) + w] = bad[w];
                    mbar_arrive(&v_ready[seen % STAGES]);
                }
                ++seen;
            }
        } else {
            // In steps j = -1 .. nt - 1: P_j V, then Q K_j+1 of this warp's tile of rows, by turns where both tiles have some: side
            // by side, both would end late, and both tiles' exponentials would run at the same time (980 us for 816).
            const auto one = [](int x) { return __shfl_sync(~0u, x, 0); };   // as warp
            const int t = warp - 9, tiles = one(nt), ja = one(from_of(t)), jb = one(until_of(t)), other_a = one(from_of(1 - t)), other_b = one(until_of(1 - t));
            const uint32_t lead = elect_lane(), id_s = umma_idesc_f16(KEYS, BF16), id_pv = umma_idesc_f16(D, BF16, 1);
            const uint64_t qd = umma_desc_sw128(smem + t * L::TILE), kd = umma_desc_sw128(smem + L::OFF_RING), vd = umma_desc_sw128_mn(smem + L::OFF_RING, L::BOX);
            const uint32_t ts = tmem + KEYS * t, to = TM_O + D * t;
            auto wait = [&](uint64_t * at, int parity, int code) { return __all_sync(~0u, mbar_wait_soon(at, (uint32_t) parity, abort_flag, p.err, code)) != 0; };
            bool go = true;
            int turns = 0, fits_seen = 0;
            for (int j = -1; j < tiles && go; ++j) {
                const int iv = 2 * j + 1, ik = 2 * j + 2, sv = iv % STAGES, sk = ik % STAGES;   // the stages of V_j and K_j+1
                const bool pv = j >= ja && j < jb, qk = j + 1 >= ja && j + 1 < jb;
                const bool by_turns = (pv || qk) && j + 1 >= other_a && j < other_b && other_a < other_b;
                if (j >= 0) {
                    go = wait(&full[sv], (iv / STAGES) & 1, DEV_TIMEOUT_FULL);
                    if (one(unfit((t0 + j) * KEYS))) {
                        go = go && wait(&v_ready[fits_seen % STAGES], (fits_seen / STAGES) & 1, DEV_TIMEOUT_FULL);
                        ++fits_seen;
                    }
                }
                if (j + 1 < tiles) go = go && wait(&full[sk], (ik / STAGES) & 1, DEV_TIMEOUT_FULL);
                if (qk && j + 1 == ja) go = go && wait(&q_full[t], 0, DEV_TIMEOUT_FULL);
                const uint64_t v = vd + (uint64_t) (sv * (L::TILE >> 4)), k = kd + (uint64_t) (sk * (L::TILE >> 4));
                if (pv && go) go = wait(&p_half[t], (j - ja) & 1, DEV_TIMEOUT_TMEM);
                if (by_turns && go) {
                    if (t || turns) go = wait(&turn[t], (turns - 1 + t) & 1, DEV_TIMEOUT_TMEM);
                    ++turns;
                }
                if (pv && go) {
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < KEYS / 32; ++kk) umma_f16_ts_if(lead, to, ts + 8 * kk, v + 128 * kk, id_pv, j > ja || kk > 0);
                    go = wait(&p_full[t], (j - ja) & 1, DEV_TIMEOUT_TMEM);
                }
                if (!go) break;
                if (pv) {
                    tc_fence_after();
#pragma unroll
                    for (int kk = KEYS / 32; kk < KEYS / 16; ++kk) umma_f16_ts_if(lead, to, ts + 8 * kk, v + 128 * kk, id_pv, 1);
                    umma_commit_if(lead, &empty[sv]);
                    if (j + 1 == jb) umma_commit_if(lead, &o_full[t]);
                } else if (j >= 0 && lead) {
                    mbar_arrive(&empty[sv]);   // a stage that this tile does not use
                }
                if (qk) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        umma_f16_if(lead, ts, qd + (kk / 4) * (L::BOX >> 4) + 2 * (kk % 4), k + (kk / 4) * (L::BOX >> 4) + 2 * (kk % 4), id_s, kk != 0);
                    umma_commit_if(lead, &s_full[t]);
                    umma_commit_if(lead, &empty[sk]);
                } else if (j + 1 < tiles && lead) {
                    mbar_arrive(&empty[sk]);
                }
                if (by_turns && lead) mbar_arrive(&turn[1 - t]);
            }
        }
        __syncwarp();
        pdl_trigger();
        if (p.parts > 1) {
            cluster_sync_all();
            cluster_sync_all();
        }
    } else {
        const int t = warp >> 2, row = tid & 127, ja = from_of(t), jb = until_of(t), mine = 128 * t + row;   // row of the unit
        const uint32_t lane0 = (uint32_t) ((warp & 3) * 32) << 16, ts = tmem + KEYS * t + lane0, to = TM_O + D * t + lane0;
        const bool there = mine < R;
        const int token = (r0 + mine) / p.G;
        row_of[mine] = (uint16_t) ((token - token0) << 7 | (r0 + mine - token * p.G));   // at most 256 tokens, 128 heads
        bar_n(1 + t, 128);
        auto address = [&](const tsn_rows & x, int r) {   // of row r of the unit
            const int u = row_of[r];
            return (uint16_t *) x.p + (long long) (row0 + token0 + (u >> 7)) * x.sb + (long long) (hk * p.G + (u & 127)) * x.st;
        };
        uint8_t * qs = smem + t * L::TILE;
        if (ja < jb) {   // Q into its swizzled boxes, rows past the last one as zeros
            uint4 q[CH];
            const int ch = row % CH;
#pragma unroll
            for (int y = 0; y < CH; ++y) {
                const int r = row / CH + 128 / CH * y;
                q[y] = make_uint4(0, 0, 0, 0);
                if (128 * t + r < R) q[y] = *(const uint4 *) (address(p.q, 128 * t + r) + ch * 8);
            }
#pragma unroll
            for (int y = 0; y < CH; ++y) {
                const int r = row / CH + 128 / CH * y;
                *(uint4 *) (qs + (ch >> 3) * L::BOX + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = q[y];
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[t]);
        }
        const int hi = there ? hi_at(token) : n, lo = there ? lo_at(token) : 0;
        const int rows_end = min(R, 128 * t + 128);
        const int sure_hi = ja < jb ? hi_at(t ? token128 : token0) : 0, sure_lo = ja < jb ? lo_at(t ? token_last : token127) : 0;   // every row of the tile sees keys sure_lo .. sure_hi - 1
        float l = 0.0f, raw = -INFINITY;   // raw: the score that the reference is of
        bool ok = true, poison = false;
        int fits_seen = 0;   // tiles of the part whose values passed through warp 11
        for (int j = 0; j < ja; ++j) fits_seen += unfit((t0 + j) * KEYS);
        // Tile j: all its scores into registers, the maximum, then the exponentials; P replaces S half by half, and the first half's
        // product may start while the second half's exponentials run.
        auto tile = [&](int j) {
            const int base = (t0 + j) * KEYS;
            uint32_t x[128];
#pragma unroll
            for (int w = 0; w < 4; ++w) tmem_request32(ts + 32 * w, x + 32 * w);
            const uint32_t slabs = paged[j % L::DEEP];
            const bool masked = base < sure_lo || base + KEYS > sure_hi || slabs != 0xffu;
            uint32_t vis[4] = {~0u, ~0u, ~0u, ~0u};
            if (masked)
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    vis[w] = low_bits(hi - base - 32 * w) & ~low_bits(lo - base - 32 * w) & ((slabs >> (2 * w) & 1u ? 0xffffu : 0u) | (slabs >> (2 * w) & 2u ? 0xffff0000u : 0u));
#pragma unroll
            for (int w = 0; w < 4; ++w) tmem_landed32(x + 32 * w);
            if (masked)
#pragma unroll
                for (int w = 0; w < 4; ++w) hide(x + 32 * w, vis[w]);
            float mx[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) mx[w] = greatest(x + 32 * w);
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            const bool move = (top - raw) * p.scale > LAZY;
            if (__any_sync(~0u, move)) {
                // a row moves its reference by itself, so its result does not depend on its neighbours
                const float f = move ? ex2(__fmul_ru(raw, p.scale) - __fmul_ru(top, p.scale)) : 1.0f;
                if (move) { raw = top; l *= f; }
                if (j > ja) {   // O holds the tiles before: their products were issued before these scores'
#pragma unroll 1
                    for (int y = 0; y < D; y += 16) {
                        float o[16];
                        tmem_ld16(to + y, o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] *= f;
                        tmem_st16(to + y, (const uint32_t *) o);
                    }
                }
            }
            // c s - ref in one rounding: ref is c raw rounded up and ABOVE - ref down, so that no probability exceeds 2^15 however large
            // the scores are. The greatest one falls below 2^ABOVE by the steps of numbers this size: from 2^26 on, where neighbouring f32
            // scores are 4 log2 units and more apart, c becomes a power of two, whose products are exact. (With c raw rounded to nearest
            // rows of scores of 2^36 were NaN or zero. Scores scaled and subtracted one after the other where a row needs it: 7 % more time.)
            const float high = __fmul_ru(raw, p.scale);
            const bool far = fabsf(high) >= 0x1p26f && raw != -INFINITY;
            const float c = far ? __uint_as_float(__float_as_uint(p.scale) & 0x7f800000u) : p.scale;
            const float neg = raw == -INFINITY ? 0.0f : __fadd_rd(ABOVE, far ? -(raw * c) : -high);
            const uint64_t neg2 = f2_pack(neg, neg), c2 = f2_pack(c, c);
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t pk[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const uint64_t v = ffma2(f2_pack(__uint_as_float(x[64 * h + 2 * e]), __uint_as_float(x[64 * h + 2 * e + 1])), c2, neg2);
                    float y, z;
                    if (e % L::EVERY == L::EVERY - 1) {
                        f2_unpack(ex2_fma<BF16, true>(v), y, z);
                    } else {
                        f2_unpack(v, y, z);
                        y = ex2(y);
                        z = ex2(z);
                    }
                    pk[e] = pack16<BF16>(y, z);
                    add_rounded<BF16>(sum[2 * (e & 1)], sum[2 * (e & 1) + 1], pk[e]);
                }
                tmem_st32(ts + 32 * h, pk);
                if (h == 0) {
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_half[t]);
                }
            }
            l += (sum[0] + sum[2]) + (sum[1] + sum[3]);
            if (unfit(base)) {
                if (mixed(base)) {
                    if (!mbar_wait_soon(&v_ready[fits_seen % STAGES], (fits_seen / STAGES) & 1, abort_flag, p.err, DEV_TIMEOUT_FULL)) ok = false;
#pragma unroll
                    for (int w = 0; w < 4; ++w) poison |= (not_finite[4 * (fits_seen % STAGES) + w] & vis[w]) != 0;
                }
                ++fits_seen;
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[t]);
        };
        for (int j = ja; j < jb && ok; ++j) {
            if (!mbar_wait_soon(&s_full[t], (j - ja) & 1, abort_flag, p.err, DEV_TIMEOUT_TMEM)) { ok = false; break; }
            __syncwarp();
            tc_fence_after();
            tile(j);
        }
        if (ok && ja < jb) ok = mbar_wait_soon(&o_full[t], 0, abort_flag, p.err, DEV_TIMEOUT_TMEM);
        __syncwarp();
        tc_fence_after();
        pdl_trigger();
        // ------------------------------------------------------------ results
        auto piece = [&](int x, float * o) {   // 32 columns of O
            if (ja < jb) {
                tmem_ld32(to + x, o);
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0.0f;
            }
            if (poison && there) {
                float sums[32];   // a copy, as it goes through memory
#pragma unroll
                for (int e = 0; e < 32; ++e) sums[e] = o[e];
                for (int j = ja; j < jb; ++j)
                    if (mixed((t0 + j) * KEYS))
                        add_not_finite<BF16, 32>(p, b, hk, max(lo, (t0 + j) * KEYS), min(hi, (t0 + j + 1) * KEYS), x, sums);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = sums[e];
            }
        };
        if (p.parts > 1) {
            bar_n(3, 256);   // both tiles are done with the ring
            float * sums = (float *) (smem + L::OFF_RING);
            {
                float * dst = sums + mine * L::SUM_ROW;
#pragma unroll 1
                for (int x = 0; x < D; x += 32) {
                    float o[32];
                    piece(x, o);
#pragma unroll
                    for (int e = 0; e < 32; e += 4) *(float4 *) (dst + x + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
                dst[D] = __fmul_ru(raw, p.scale);   // the reference
                dst[D + 1] = l;
            }
            cluster_sync_all();
            // this CTA's share of the rows: first each part's factors, 2^(ref - greatest) / l, in Q's place, then the parts' sums, a
            // row by D / 4 lanes, four steps of rows at once
            const int share = (R + p.parts - 1) / p.parts, from = (int) split * share, here = max(0, min(R - from, share));
            const uint32_t at0 = smem_u32(sums + from * L::SUM_ROW);
            float * fac = (float *) smem;   // [row][8 parts]
            if (tid < here) {
                float ref_of[8], top = -INFINITY, sum = 0.0f;
                float4 st[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < p.parts) {
                        st[i] = dsmem_ld4(dsmem_map(at0 + (tid * L::SUM_ROW + D) * 4, (uint32_t) i));
                        top = fmaxf(top, st[i].x);
                    }
                const float low = top == -INFINITY ? 0.0f : top;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < p.parts) {
                        ref_of[i] = ex2(st[i].x - low);
                        sum += ref_of[i] * st[i].y;
                    }
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < p.parts) fac[tid * 8 + i] = sum == 0.0f ? -1.0f : ref_of[i] * inv;   // -1: no key has a share, and no sum of values counts
            }
            bar_n(3, 256);
            constexpr int LANES = D / 4, STEP = 8 * (32 / LANES), AT_ONCE = 4;   // lanes of a row; rows of a step of all warps
            const int col = (lane % LANES) * 4;
            for (int y0 = warp * (32 / LANES) + lane / LANES; y0 < here; y0 += STEP * AT_ONCE) {
                float o[AT_ONCE][4] = {};
                for (int i = 0; i < p.parts; ++i)
#pragma unroll
                    for (int y = 0; y < AT_ONCE; ++y) {
                        const int r = y0 + y * STEP;
                        if (r < here) {
                            const float4 v = dsmem_ld4(dsmem_map(at0 + (r * L::SUM_ROW + col) * 4, (uint32_t) i));
                            const float f = fac[r * 8 + i];
                            o[y][0] = fmaf(f, v.x, o[y][0]); o[y][1] = fmaf(f, v.y, o[y][1]);
                            o[y][2] = fmaf(f, v.z, o[y][2]); o[y][3] = fmaf(f, v.w, o[y][3]);
                        }
                    }
#pragma unroll
                for (int y = 0; y < AT_ONCE; ++y) {
                    const int r = y0 + y * STEP;
                    if (r < here && !*abort_flag)
                        *(uint2 *) (address(p.out, from + r) + col) = fac[r * 8] < 0.0f ? make_uint2(0u, 0u) : make_uint2(pack16<BF16>(o[y][0], o[y][1]), pack16<BF16>(o[y][2], o[y][3]));
                }
            }
            cluster_sync_all();   // nobody leaves while its sums are read
        } else {
            // through Q's place, so that whole rows are written
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
            for (int x = 0; x < D; x += 32) {
                float o[32];
                piece(x, o);
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = l == 0.0f ? 0u : pack16<BF16>(o[e + 2 * k] * inv, o[e + 2 * k + 1] * inv);
                    const int ch = (x + e) / 8;
                    *(uint4 *) (qs + row * (D * 2) + ((ch ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            bar_n(1 + t, 128);
            if (!*abort_flag && fits)
                for (int i = row; i < (rows_end - 128 * t) * CH; i += 128) {
                    const int r = i / CH, ch = i % CH;
                    *(uint4 *) (address(p.out, 128 * t + r) + ch * 8) = *(const uint4 *) (qs + r * (D * 2) + ((ch ^ (r & 7)) << 4));
                }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, L::TM);
    }
    if (*abort_flag && tid == 0) {
        // let copies that were issued but never consumed land before the CTA's shared memory is reused
        const uint64_t t1 = global_ns();
        while (global_ns() - t1 < 20000ull) {}
    }
}

// clusters of 1 to 8 CTAs that run at once (one CTA per SM; a cluster lies within a GPC)
std::atomic<int> g_clusters[9];

template <int D, bool BF16>
cudaError_t launch(const PagedArgs & p, unsigned grid, cudaStream_t s) {
    CUtensorMap tk{}, tv{};
    if (!make_page_maps(p.c, (uint32_t) std::min(KEYS, 1 << p.page_log2), &tk, &tv)) return cudaErrorInvalidValue;
    return launch_cl(paged_tiles_kernel<D, BF16>, dim3(grid), dim3(THREADS), Lay<D>::TOTAL, s, dim3((unsigned) p.parts), tk, tv, p);
}

} // namespace

cudaError_t configure_paged_tiles() {
    cudaError_t e = cudaSuccess;
    auto set = [&](auto * k, int bytes) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    };
    set(paged_tiles_kernel<64, false>, Lay<64>::TOTAL);
    set(paged_tiles_kernel<64, true>, Lay<64>::TOTAL);
    set(paged_tiles_kernel<128, false>, Lay<128>::TOTAL);
    set(paged_tiles_kernel<128, true>, Lay<128>::TOTAL);
    g_clusters[1] = SMS;
    for (unsigned n = 2; n <= 8 && e == cudaSuccess; ++n) {
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim = {n, 1, 1};
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(n * SMS);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = Lay<128>::TOTAL;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        int count = 0;
        e = cudaOccupancyMaxActiveClusters(&count, paged_tiles_kernel<128, true>, &cfg);
        g_clusters[n] = count;
    }
    return e;
}

namespace {
// units at most: a sequence has a last one that is not full
long long units_of(const PagedArgs & p) { return std::min<long long>(p.c.N, (long long) p.c.N * p.G / ROWS + p.c.B) * p.c.Hk; }
}

double plan_paged_tiles(PagedArgs & p, uint32_t most) {
    const long long units = std::min(units_of(p), (long long) p.c.B * (((long long) most * p.G + ROWS - 1) / ROWS) * p.c.Hk);
    // As many parts of a cluster as take the least time, in microseconds: start and end of a CTA 5, a tile of 128-wide heads 2 and of
    // 64-wide ones 1.7; with parts 4 to add them up and 5 for each wave of clusters; g_clusters[size] run at a time. Four
    // key tiles a part at least, eight parts at most (the largest portable cluster). The keys are what the tables have room for: lengths
    // are on the device. us in 1, 2, 4 and 8 parts: 64 tokens x 4 heads of 128 over 32 768 keys, 8 kv heads 448, 234, 125, 80; 4 x 517
    // tokens x 3 heads of 64 with a window of 2000, 8 kv heads, 76, 85, 128, 235 (the others measured when these were 78 and 69).
    long long keys = (long long) p.c.M << p.page_log2;
    if (p.window) keys = std::min<long long>(keys, (long long) p.window + ROWS);
    const long long tiles = (keys + KEYS - 1) / KEYS;
    double least = 0.0;
    for (int parts = 1; parts <= 8 && (parts == 1 || parts * 4 <= tiles); ++parts) {
        const long long room = std::max(1, g_clusters[parts].load(std::memory_order_relaxed));
        const double cost = (double) ((units + room - 1) / room) * (5.0 + (parts > 1 ? 5.0 : 0.0) + (double) ((tiles + parts - 1) / parts) * (p.c.D == 64 ? 1.7 : 2.0)) + (parts > 1 ? 4.0 : 0.0);
        if (parts == 1 || cost < least) { least = cost; p.parts = parts; }
    }
    return least;
}

cudaError_t launch_paged_tiles(const PagedArgs & p, cudaStream_t s) {
    const long long units = units_of(p);
    if (units * p.parts > 0x7fffffffLL) return cudaErrorInvalidValue;
    const unsigned grid = (unsigned) (units * p.parts);
    const bool bf = p.c.type == TSN_BF16;
    if (p.c.D == 64) return bf ? launch<64, true>(p, grid, s) : launch<64, false>(p, grid, s);
    return bf ? launch<128, true>(p, grid, s) : launch<128, false>(p, grid, s);
}

} // namespace tsn

// paged_rows.cu — attention over the paged cache for a few query rows of a kv head: single tokens, drafts, picked pages.
//
//   o = sum_j p_j v_j / l,  l = sum_j p_j,  p_j = 2^(c q.k_j - ref + ABOVE);  ref follows the row's running maximum and moves when that has
//   grown by more than LAZY (struct Reference), with o and l rescaled. P is rounded to 16 bits, as the tensor cores take it; l is the sum of the rounded ones.
// Bound by reading K and V. mma.sync takes 8 rows (NT times) with the keys, and for the product with V the columns, on its 16-row
// side: S^T = K Q^T, O^T = V^T P^T; P^T is S^T's layout transposed in registers. Each warp streams 16-key slabs of its own by TMA,
// a page holding whole slabs, through a ring of its own; the warps' sums meet in shared memory.
// A unit is a kv head with up to 8 NT rows of a sequence, and its slabs. Lengths are on the device, so the device deals
// them out: all units' slabs in a row, an equal share for each CTA; one of eight warps or two or three of four fill an SM. A share may begin and end
// inside a unit; the CTA that is the last of a unit to arrive adds up its parts, in their order. Units of few slabs are not cut:
// a trip through the workspace costs more.
// 16 tokens over caches of 16 384 to 32 768 keys (32 heads over 8 of 128, bf16) take 260 us: 1.64 GB, 6.3 TB/s, 0.96 of the
// measured copy; 24 x 4 tokens over up to 8191 112 us (5.5 TB/s; 16 rows take twice the products and the registers of a second CTA);
// two tokens over 704 keys 8.1 us, from the launch through lengths, pages and keys to the warps' sums one after another.
// Where pages are chosen, a CTA takes a unit (a token's rows of a kv head) or a part of it; lists of many tokens come from L2, at 8 to 12 TB/s.
#include "kernels.h"
#include "paged_attn.h"

#include <algorithm>

namespace tsn {

namespace {

constexpr int SLAB = 16;   // keys of a slab
// Slabs of a share at least, slabs up to which a unit is not cut, parts of a unit at most (fewer slabs a part otherwise). One token, 8 kv
// heads of 128, 2 x 1000 keys: with units of up to 32 slabs whole 15.7 us, 64: 12.1.
constexpr int LEAST = 16, SHORT = 64, MOST_PARTS = 64;
static_assert(LEAST <= SHORT, "what a unit counts as without its slabs is never cut");
// Units up to which eight warps share one, a CTA an SM; above, two or three CTAs of four warps an SM, of which one loads while
// another adds up its unit's sums. us by eight / by four (two CTAs): 16 units of 704 keys 8.0/10.5, 8 of 1000 12.1/16.5, one of 32 768 15.7/21.7, 192 of
// 8191 142/148, but 256 of 1000 29.4/27.1, 1024 of 300 45.5/38.2.
constexpr long long FEW_UNITS = 200;

template <int D, int NT, int W, bool LIST>
struct RowLay {
    // CTAs of an SM: three with two slabs a ring start and end beside one another where two with three do so less (400 tokens x 4
    // kv heads, 16 pages of 64: 71 and 97 us; 64 tokens over 1500 keys, 8 kv heads of 64, 46.8 and 55.5), but 16 rows without
    // picked pages do not fit in the registers of three (4 tokens over 1000 keys, 64 streams: 94.8 and 57.4). With picked pages they do, one
    // word of 128-wide heads spilled.
    static constexpr int CTAS = W == 8 ? 1 : LIST || NT == 1 ? 3 : 2;
    static constexpr int BOX = SLAB * 128, HALF = SLAB * D * 2, STAGE = 2 * HALF, RING = (CTAS == 3 ? 2 : 3) * (128 / D);   // a slab's keys, then its values
    static constexpr int ROWS = 8 * NT, ROW = D + 4;   // words of a row's sums: o, ref, l
    static constexpr int OFF_BAR = W * RING * STAGE, TOTAL = OFF_BAR + W * RING * 8 + 64;
    static_assert(ROWS * ROW * 4 <= RING * STAGE, "a warp's sums fit in its ring");
    static_assert(CTAS * (TOTAL + 2048) <= 228 * 1024, "they fit");
};
constexpr int part_words(int D, int rows) { return rows * (D + 4); }

// Sequence b of the batch: its rows and slabs. Every group of its rows takes the same slabs. A unit is dealt out as `weight` slabs: LEAST
// of them at least, as even one of a single slab waits for its pages, keys and sums in turn, longer than 16 slabs stream (16 units of 16
// and of 60 keys, 16 rows of 128: 8.3 and 8.8 us; 91 and 26.7 where a CTA took as many as hold LEAST slabs).
struct Seq {
    int start, n, place, len, from, slabs, weight;   // first row, new tokens, the first one's place, cached keys; slabs from .. from + slabs - 1
    long long units;
};
template <int ROWS>
__device__ __forceinline__ Seq sequence(const PagedArgs & p, int b) {
    Seq s;
    s.start = seq_start(p.c, b);
    s.n = max(0, seq_start(p.c, b + 1) - s.start);
    const int len = p.c.len[b];
    s.len = cached(p, len);
    s.place = first_place(len, s.n);
    s.from = min(seen_from(p, s.place), s.len) / SLAB;
    s.slabs = (s.len + SLAB - 1) / SLAB - s.from;
    s.units = ((long long) s.n * p.G + ROWS - 1) / ROWS * p.c.Hk;
    s.weight = max(s.slabs, LEAST);
    return s;
}

template <int D, bool BF16, int NT, bool LIST, int W>
__global__ void __launch_bounds__(32 * W, RowLay<D, NT, W, LIST>::CTAS)
paged_rows_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ PagedArgs p) {
    using L = RowLay<D, NT, W, LIST>;
    constexpr int E = D / 32, RING = L::RING, ROWS = L::ROWS;
    constexpr float LAZY = Reference<BF16>::LAZY, ABOVE = Reference<BF16>::ABOVE;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ int first_seq, first_off;
    __shared__ long long first_unit, share_from, share_to, share_per;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (smem_u32(smem) & 1023) {
        if (tid == 0 && p.err) atomicCAS(p.err, 0, DEV_BAD_ARGS);
        return;
    }
    uint64_t * full = (uint64_t *) (smem + L::OFF_BAR) + warp * RING;
    volatile int * flags = (volatile int *) (smem + L::OFF_BAR + W * RING * 8);   // abort, last to arrive, rows to mend
    if (lane == 0) {
        if (p.c.P) { tma_prefetch(&tk); tma_prefetch(&tv); }
        for (int s = 0; s < RING; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
    }
    if (tid == 0) flags[0] = flags[2] = 0;
    pdl_wait();

    // ---------------------------------------------------------------- this CTA's share
    if (!LIST && warp == 0) {
        constexpr int AT_ONCE = 4;
        long long total = 0;
        int longest = 0;
        for (int b0 = 0; b0 < (int) p.c.B; b0 += 32 * AT_ONCE) {
#pragma unroll
            for (int y = 0; y < AT_ONCE; ++y) {
                const int b = b0 + 32 * y + lane;
                if (b < (int) p.c.B) {
                    const Seq s = sequence<ROWS>(p, b);
                    total += s.units * s.weight;
                    if (s.units) longest = max(longest, s.weight);
                }
            }
        }
#pragma unroll
        for (int x = 16; x; x >>= 1) total += __shfl_xor_sync(~0u, total, x);
        longest = __reduce_max_sync(~0u, longest);
        const long long per = max(max((total + gridDim.x - 1) / gridDim.x, (long long) LEAST), (long long) (longest + MOST_PARTS - 1) / MOST_PARTS);
        const long long x0 = min(total, per * blockIdx.x), x1 = min(total, x0 + per);
        if (lane == 0) {
            share_from = share_to = total;
            share_per = per;
            first_seq = first_off = 0;
            first_unit = 0;
        }
        __syncwarp();
        // the sequences that the share's ends lie in; an end inside a unit that is not cut moves to the unit's start
        long long before = 0;
        for (int b0 = 0; b0 < (int) p.c.B && before <= x1; b0 += 32) {
            const int b = b0 + lane;
            Seq s{};
            if (b < (int) p.c.B) s = sequence<ROWS>(p, b);
            const long long mine = s.units * s.weight;
            long long upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long v = __shfl_up_sync(~0u, upto, o);
                if (lane >= o) upto += v;
            }
            const long long at = before + upto - mine;
            auto cut = [&](long long x) {   // x as an end of the share, at <= x < at + mine
                const long long u = (x - at) / s.weight;
                return p.whole || s.weight <= SHORT ? at + u * s.weight : x;
            };
            if (mine && at <= x0 && x0 < at + mine) {
                const long long x = cut(x0), u = (x - at) / s.weight;
                share_from = x;
                first_seq = b;
                first_unit = u;
                first_off = (int) (x - at - u * s.weight);
            }
            if (mine && at <= x1 && x1 < at + mine) share_to = cut(x1);
            before += __shfl_sync(~0u, upto, 31);
        }
    }
    __syncthreads();

    const int g0 = lane >> 2, c0 = (lane & 3) * 2;   // scores: keys g0 (+ 8) by rows c0, c0 + 1
    // addresses of ldmatrix: K rows (key), two groups of 8 keys by two of 8 elements; V rows (key), two groups of 8 columns by two
    // of 8 keys
    const int krow = (lane & 7) + (((lane >> 3) & 1) << 3), kch = lane >> 4;
    const int vrow = (lane & 7) + ((lane >> 4) << 3), vch = (lane >> 3) & 1;
    uint8_t * ring = smem + warp * RING * L::STAGE;
    unsigned turn = 0;   // slabs that this warp has taken: stage turn % RING, parity turn / RING

    int b = LIST ? 0 : first_seq, off = LIST ? 0 : first_off;
    long long unit = LIST ? 0 : first_unit, at = LIST ? 0 : share_from;
    const long long to = LIST ? 1 : share_to;
    Seq s{};
    if (!LIST && at < to) s = sequence<ROWS>(p, b);
    while (at < to) {
        // ------------------------------------------------------------ the unit, and this CTA's slabs of it
        int hk, first, R, place0, s0, s1, n, row0, part = 0, parts = 1, owner = (int) blockIdx.x;
        if (LIST) {
            const int groups = (p.G + ROWS - 1) / ROWS;
            const unsigned u = blockIdx.x / p.parts;
            part = (int) (blockIdx.x % p.parts);
            parts = p.parts;
            owner = (int) (u * p.parts);
            first = (int) (u % groups) * ROWS;
            hk = (int) (u / groups % p.c.Hk);
            row0 = (int) (u / groups / p.c.Hk);
            R = min(ROWS, p.G - first);
            b = seq_of_row(p.c, row0);
            if (b < 0) return;   // a row of no sequence
            const int len = p.c.len[b];
            place0 = place_of_row(p.c, b, row0);
            n = min(cached(p, len), place0 + 1);
            const int own = place0 < 0 ? -1 : place0 >> p.page_log2, pages = own >= (int) p.c.M ? 0 : min(own + 1, p.picks);
            const int slabs = pages ? ((pages - 1) << (p.page_log2 - 4)) + ((place0 & ((1 << p.page_log2) - 1)) >> 4) + 1 : 0;
            const int chunk = (slabs + parts - 1) / parts;
            s0 = min(slabs, part * chunk);
            s1 = min(slabs, s0 + chunk);
        } else {
            hk = (int) (unit % p.c.Hk);
            first = (int) (unit / p.c.Hk) * ROWS;
            R = (int) min((long long) ROWS, (long long) s.n * p.G - first);
            row0 = s.start;
            n = s.len;
            place0 = s.place;
            const int take = (int) min((long long) (s.weight - off), to - at);
            s0 = s.from + off;
            s1 = s.from + min(off + take, s.slabs);
            const long long begin = at - off;   // of the unit
            if (take < s.weight) {
                owner = (int) (begin / share_per);
                part = (int) blockIdx.x - owner;
                parts = (int) ((begin + s.weight - 1) / share_per) - owner + 1;
            }
            at += take;
            off = 0;
        }
        const int * chosen = LIST ? p.chosen + ((long long) row0 * p.c.Hk + hk) * p.picks : nullptr;
        auto page_index = [&](int slab) { return LIST ? chosen[slab >> (p.page_log2 - 4)] : slab >> (p.page_log2 - 4); };
        // rows r: token (first + r) / G, head (first + r) % G; rows past the last one see all. Keys lo .. hi - 1
        auto place_of = [&](int r) { return LIST ? place0 : place0 + (first + r) / p.G; };
        auto hi_of = [&](int r) { return r < R ? seen_to(p, place_of(r), n) : n; };
        auto lo_of = [&](int r) { return r < R ? seen_from(p, place_of(r)) : 0; };
        const int least = hi_of(0), latest = lo_of(R - 1);   // before least and from latest on every row sees
        // After a wait that gave up nothing is loaded any more, but the share is walked to its end: every part arrives, so that the
        // counters are zero after the call whatever became of it.
        const int mine = !flags[0] && s1 - s0 > warp ? (s1 - s0 - warp + W - 1) / W : 0;

        // pages of the warp's slabs, 32 at once, and which of them are none
        auto load_ids = [&](int i) {
            const int k = i + lane;
            return k < mine ? page_of(p.c, b, page_index(s0 + warp + k * W)) : -1;
        };
        auto load_base = [&](int i) {   // list: the first key of each slab
            const int k = i + lane, slab = s0 + warp + k * W;
            return k < mine ? (page_index(slab) << p.page_log2) + ((slab << 4) & ((1 << p.page_log2) - 1)) : 0;
        };
        int ids = load_ids(0), next_ids = mine > 32 ? load_ids(32) : -1;
        uint32_t even = __ballot_sync(~0u, ids >= 0), odd = 0u;
        auto request = [&](int i) {   // slab i of this warp, by all lanes
            if (i && (i & 31) == 0) {
                ids = next_ids;
                const uint32_t are = __ballot_sync(~0u, ids >= 0);
                if (i & 32) odd = are;
                else even = are;
                next_ids = i + 32 < mine ? load_ids(i + 32) : -1;
            }
            const int id = __shfl_sync(~0u, ids, i & 31);
            if (lane == 0) {
                const unsigned st = (turn + i) % RING;
                uint8_t * dst = ring + st * L::STAGE;
                const int slot = ((s0 + warp + i * W) << 4) & ((1 << p.page_log2) - 1), page = id < 0 ? (int) p.c.P : id;   // past the last page: zeros
                mbar_expect_tx(&full[st], L::STAGE);
#pragma unroll
                for (int x = 0; x < D / 64; ++x) {
                    tma_load_4d(dst + x * L::BOX, &tk, &full[st], 64 * x, slot, hk, page);
                    tma_load_4d(dst + L::HALF + x * L::BOX, &tv, &full[st], 64 * x, slot, hk, page);
                }
            }
        };
        for (int i = 0; i < RING && i < mine; ++i) request(i);
        const bool give_up = p.give_up == (int) blockIdx.x + 1;
        if (give_up && tid == 0) {
            flags[0] = 1;
            if (p.err) atomicCAS(p.err, 0, DEV_TIMEOUT_FULL);
        }

        // Q^T as B operands: row g0 of each eight, rows past the last one as zeros
        uint32_t qb[NT][D / 16][2];
        int hi[NT][2], lo[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = 8 * t + g0, u = first + r;
            const uint16_t * q = (const uint16_t *) p.q.p + (LIST ? row0 : row0 + u / p.G) * p.q.sb + (long long) (hk * p.G + (LIST ? u : u % p.G)) * p.q.st;
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) qb[t][k][h] = r < R ? *(const uint32_t *) (q + 16 * k + 8 * h + c0) : 0u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                hi[t][h] = hi_of(8 * t + c0 + h);
                lo[t][h] = lo_of(8 * t + c0 + h);
            }
        }
        float o[NT][D / 16][4], l[NT][2], ref[NT][2];   // O^T: columns 16 x + g0 (+ 8) by rows c0, c0 + 1
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            l[t][0] = l[t][1] = 0.0f;
            ref[t][0] = ref[t][1] = -INFINITY;
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[t][x][k] = 0.0f;
        }
        uint32_t to_mend = 0;   // rows that see a value which is not finite, among those with rows that do not
        int bases = LIST ? load_base(0) : 0;
        for (int i = 0; i < mine && !give_up; ++i) {
            if (LIST && i && (i & 31) == 0) bases = load_base(i);
            const int base = LIST ? __shfl_sync(~0u, bases, i & 31) : (s0 + warp + i * W) * SLAB;
            const unsigned st = (turn + i) % RING;
            const uint32_t there = ((i & 32 ? odd : even) >> (i & 31)) & 1u ? low_bits(n - base) & 0xffffu : 0u;   // the keys that exist
            if (!mbar_wait_soon(&full[st], ((turn + i) / RING) & 1, flags, p.err, DEV_TIMEOUT_FULL)) break;
            __syncwarp();
            const uint32_t kt = smem_u32(ring + st * L::STAGE), vt = kt + L::HALF;
            float sc[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < 4; ++k) sc[t][k] = 0.0f;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const int col = 16 * k;
                uint32_t f[4];
                ldmatrix4<false>(f, kt + (col / 64) * L::BOX + krow * 128 + ((((col % 64) / 8 + kch) ^ (krow & 7)) << 4));
#pragma unroll
                for (int t = 0; t < NT; ++t) mma16816<BF16>(sc[t], f, qb[t][k][0], qb[t][k][1]);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < 4; ++k) sc[t][k] = __fmul_rn(sc[t][k], p.scale);   // rounded by itself, so that the greatest one less itself is zero however large
            const bool gone = there != 0xffffu, mixed = least < min(n, base + SLAB) || base < latest;
            uint32_t vis[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) vis[t][h] = there & low_bits(hi[t][h] - base) & ~low_bits(lo[t][h] - base);
            if (gone || mixed) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (!((vis[t][k & 1] >> (g0 + 8 * (k >> 1))) & 1u)) sc[t][k] = -INFINITY;
            }
            bool move = false;
            float top[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[t][h] = fmaxf(sc[t][h], sc[t][2 + h]);
                    move |= top[t][h] - ref[t][h] > LAZY;
                }
            if (__any_sync(~0u, move)) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float m = top[t][h];
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, x));
                        if (m - ref[t][h] > LAZY) {   // a row moves its reference by itself
                            const float f = ex2(ref[t][h] - m);
                            ref[t][h] = m;
                            l[t][h] *= f;
#pragma unroll
                            for (int x = 0; x < D / 16; ++x) { o[t][x][h] *= f; o[t][x][2 + h] *= f; }
                        }
                    }
            }
            uint32_t pb[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float r0 = ref[t][0] == -INFINITY ? 0.0f : ref[t][0], r1 = ref[t][1] == -INFINITY ? 0.0f : ref[t][1];
                const uint32_t p0 = pack16<BF16>(ex2(sc[t][0] - r0 + ABOVE), ex2(sc[t][1] - r1 + ABOVE));
                const uint32_t p1 = pack16<BF16>(ex2(sc[t][2] - r0 + ABOVE), ex2(sc[t][3] - r1 + ABOVE));
                add_rounded<BF16>(l[t][0], l[t][1], p0);   // the sums are of what the product takes
                add_rounded<BF16>(l[t][0], l[t][1], p1);
                pb[t][0] = movmatrix(p0);
                pb[t][1] = movmatrix(p1);
            }
            if (!gone && !mixed) {
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    uint32_t f[4];
                    ldmatrix4<true>(f, vt + (x / 4) * L::BOX + vrow * 128 + (((2 * (x % 4) + vch) ^ (vrow & 7)) << 4));
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma16816<BF16>(o[t][x], f, pb[t][0], pb[t][1]);
                }
            } else {
                // values behind keys that are not there count as zero; where rows differ, so do those that are not finite, and
                // rows that see one are marked
                const auto word = [](uint32_t two) { return (two & 1u ? 0xffffu : 0u) | (two & 2u ? 0xffff0000u : 0u); };
                const uint32_t keep[2] = {word(there >> c0), word(there >> (c0 + 8))};
                uint32_t bad = 0;
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    uint32_t f[4];
                    ldmatrix4<true>(f, vt + (x / 4) * L::BOX + vrow * 128 + (((2 * (x % 4) + vch) ^ (vrow & 7)) << 4));
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        f[y] &= keep[y >> 1];
                        if (mixed) {
                            const uint32_t g = finite_only<BF16>(f[y]), diff = f[y] ^ g;
                            if (diff & 0xffffu) bad |= 1u << (c0 + 8 * (y >> 1));
                            if (diff >> 16) bad |= 2u << (c0 + 8 * (y >> 1));
                            f[y] = g;
                        }
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma16816<BF16>(o[t][x], f, pb[t][0], pb[t][1]);
                }
                bad = __reduce_or_sync(~0u, bad);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (bad & vis[t][h]) to_mend |= 1u << (8 * t + c0 + h);
            }
            __syncwarp();   // every lane has its operands: the stage may be loaded again
            if (i + RING < mine) request(i + RING);
        }
        turn += (unsigned) mine;
        if (at >= to || LIST) pdl_trigger();   // from here on little memory is read: the next kernel's blocks would have taken bandwidth before
        // the warp's sums in its ring, then warp w adds up rows w, w + W, ... of all warps
        float * sums = (float *) ring;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float m = l[t][h];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) m += __shfl_xor_sync(~0u, m, x);
                float * dst = sums + (8 * t + c0 + h) * L::ROW;
                // the reference is the same in the lanes of a row: it moves by all their maxima
                if (g0 == 0) {
                    dst[D] = ref[t][h];
                    dst[D + 1] = m;
                }
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    dst[16 * x + g0] = o[t][x][h];
                    dst[16 * x + g0 + 8] = o[t][x][2 + h];
                }
            }
        to_mend = __reduce_or_sync(~0u, to_mend);
        if (lane == 0 && to_mend) atomicOr((int *) &flags[2], (int) to_mend);
        __syncthreads();
        const uint32_t mend = (uint32_t) flags[2];
        float * const space = p.part ? p.part + (size_t) owner * 2 * part_words(D, ROWS) : nullptr;
        auto slot = [&](int i) { return space + (size_t) (i == 0 ? 1 : 2 * i) * part_words(D, ROWS); };   // the owner's second, the others' first
        auto result = [&](int r, const float * v, float sum) {
            const int u = first + r;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            uint32_t x[E / 2];
#pragma unroll
            for (int e = 0; e < E; e += 2) x[e / 2] = sum == 0.0f ? 0u : pack16<BF16>(v[e] * inv, v[e + 1] * inv);
            uint16_t * out = (uint16_t *) p.out.p + (LIST ? row0 : row0 + u / p.G) * p.out.sb + (long long) (hk * p.G + (LIST ? u : u % p.G)) * p.out.st + E * lane;
            if constexpr (E == 4) *(uint2 *) out = make_uint2(x[0], x[1]);
            else *(uint32_t *) out = x[0];
        };
        for (int r = warp; r < R && !flags[0]; r += W) {
            float v[E] = {}, f[W], top = -INFINITY, sum = 0.0f;
            auto set = [&](int i) { return (const float *) (smem + i * RING * L::STAGE) + r * L::ROW; };
#pragma unroll
            for (int i = 0; i < W; ++i) top = fmaxf(top, f[i] = set(i)[D]);
            const float low = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                f[i] = ex2(f[i] - low);
                sum = fmaf(f[i], set(i)[D + 1], sum);
                float w[E];
                read_words<E, false>(set(i) + E * lane, w);
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = fmaf(f[i], w[e], v[e]);
            }
            if (!LIST && (mend >> r) & 1u) {
                const int from = max(lo_of(r), s0 * SLAB), until = min(hi_of(r), s1 * SLAB), bottom = (latest + SLAB - 1) / SLAB * SLAB, upper = least / SLAB * SLAB;
                add_not_finite<BF16, E>(p, b, hk, from, min(until, bottom), E * lane, v);
                add_not_finite<BF16, E>(p, b, hk, max(from, max(bottom, upper)), until, E * lane, v);
            }
            if (parts == 1) {
                result(r, v, sum);
            } else {
                float * dst = slot(part) + r * L::ROW;
                if constexpr (E == 4) *(float4 *) (dst + E * lane) = make_float4(v[0], v[1], v[2], v[3]);
                else *(float2 *) (dst + E * lane) = make_float2(v[0], v[1]);
                if (lane == 0) { dst[D] = top; dst[D + 1] = sum; }
            }
        }
        if (parts > 1) {
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const bool last = atomicAdd(&p.count[owner], 1u) + 1u == (unsigned) parts;
                if (last) p.count[owner] = 0;   // for the next call
                __threadfence();
                flags[1] = last;
            }
            __syncthreads();
            if (flags[1]) {
                // A row by one warp, or with fewer rows than warps by several, which take every `share`-th part and meet in shared memory.
                const int share = R >= W ? 1 : W / R;
                float * meet = (float *) smem;   // [warps][D]
                for (int x = warp; x < (R * share + W - 1) / W * W && !flags[0]; x += W) {
                    const int r = x / share, mine_of = x % share;
                    float v[E] = {}, top = -INFINITY, sum = 0.0f;
                    if (r < R) {
                        auto set = [&](int i) { return (const float *) slot(i) + r * L::ROW; };
                        constexpr int N32 = (MOST_PARTS + 1 + 31) / 32;   // a share that begins inside a slab's part adds one
                        float refs[N32], ls[N32];
#pragma unroll
                        for (int y = 0; y < N32; ++y) {
                            const int i = 32 * y + lane;
                            refs[y] = i < parts ? __ldcg(set(i) + D) : -INFINITY;
                            ls[y] = i < parts ? __ldcg(set(i) + D + 1) : 0.0f;
                            top = fmaxf(top, refs[y]);
                        }
#pragma unroll
                        for (int y = 16; y; y >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, y));
                        const float low = top == -INFINITY ? 0.0f : top;
#pragma unroll
                        for (int y = 0; y < N32; ++y) {
                            refs[y] = ex2(refs[y] - low);
                            sum += refs[y] * ls[y];
                        }
#pragma unroll
                        for (int y = 16; y; y >>= 1) sum += __shfl_xor_sync(~0u, sum, y);
                        constexpr int AT_ONCE = 8;
                        for (int i0 = mine_of; i0 < parts; i0 += share * AT_ONCE) {
                            float w[AT_ONCE][4];
#pragma unroll
                            for (int k = 0; k < AT_ONCE; ++k)
                                if (i0 + k * share < parts) read_words<E, true>(set(i0 + k * share) + E * lane, w[k]);
#pragma unroll
                            for (int k = 0; k < AT_ONCE; ++k) {
                                const int i = i0 + k * share;
                                float f = 0.0f;
#pragma unroll
                                for (int y = 0; y < N32; ++y) {
                                    const float g = __shfl_sync(~0u, refs[y], i & 31);
                                    if (i >> 5 == y) f = g;
                                }
                                if (i < parts)
#pragma unroll
                                    for (int e = 0; e < E; ++e) v[e] = fmaf(f, w[k][e], v[e]);
                            }
                        }
                    }
                    if (share > 1) {
#pragma unroll
                        for (int e = 0; e < E; ++e) meet[warp * D + E * lane + e] = v[e];
                        __syncthreads();
                        if (r < R && mine_of == 0)
                            for (int y = 1; y < share; ++y)
#pragma unroll
                                for (int e = 0; e < E; ++e) v[e] += meet[(warp + y) * D + E * lane + e];
                    }
                    if (r < R && mine_of == 0) result(r, v, sum);
                }
            }
        }
        if (LIST) break;
        if (at < to) {
            __syncthreads();   // the rings are free again
            if (tid == 0) flags[2] = 0;
            fence_proxy_async_smem();   // the sums were written where the next copies land
            if (++unit == s.units) {
                unit = 0;
                do {
                    if (++b >= (int) p.c.B) return;   // (not reached while lengths and starts stay what they were)
                    s = sequence<ROWS>(p, b);
                } while (s.units == 0);
            }
            __syncthreads();
        }
    }
    if (flags[0] && tid == 0) {
        // let copies that were issued but never consumed land before the CTA's shared memory is reused
        const uint64_t t1 = global_ns();
        while (global_ns() - t1 < 20000ull) {}
    }
}

template <int D, bool BF16, int NT, bool LIST, int W>
cudaError_t launch(const PagedArgs & p, unsigned grid, cudaStream_t s) {
    CUtensorMap tk{}, tv{};
    if (!make_page_maps(p.c, SLAB, &tk, &tv)) return cudaErrorInvalidValue;
    return launch_cl(paged_rows_kernel<D, BF16, NT, LIST, W>, dim3(grid), dim3(32 * W), RowLay<D, NT, W, LIST>::TOTAL, s, dim3(1), tk, tv, p);
}
template <int D, bool BF16, int NT>
cudaError_t launch(const PagedArgs & p, int warps, unsigned grid, cudaStream_t s) {
    if (p.chosen) return warps == 8 ? launch<D, BF16, NT, true, 8>(p, grid, s) : launch<D, BF16, NT, true, 4>(p, grid, s);
    return warps == 8 ? launch<D, BF16, NT, false, 8>(p, grid, s) : launch<D, BF16, NT, false, 4>(p, grid, s);
}
template <int D, bool BF16>
cudaError_t launch(const PagedArgs & p, int nt, int warps, unsigned grid, cudaStream_t s) {
    return nt == 1 ? launch<D, BF16, 1>(p, warps, grid, s) : launch<D, BF16, 2>(p, warps, grid, s);
}

// How a call's rows are grouped: eights of a group, units (about), warps and CTAs.
struct Plan {
    int nt, warps;
    long long units;
    unsigned ctas;
};
Plan plan_of(const PagedArgs & p, uint32_t most) {
    Plan r;
    r.nt = (long long) p.G * (p.chosen ? 1 : most) > 8 ? 2 : 1;
    const int rows = 8 * r.nt;
    if (p.chosen || !p.c.q_start) r.units = (long long) p.c.N * ((p.G + rows - 1) / rows) * p.c.Hk;
    else r.units = std::min((long long) p.c.B * (((long long) most * p.G + rows - 1) / rows), (long long) p.c.N * p.G / rows + p.c.B) * p.c.Hk;
    r.warps = r.units <= FEW_UNITS ? 8 : 4;
    // As many as run at once; picked pages with 16 rows, of which three would, are cut into parts for two.
    r.ctas = r.warps == 8 ? SMS : r.nt == 1 ? 3 * SMS : 2 * SMS;
    return r;
}

} // namespace

double paged_rows_cost(const PagedArgs & p, uint32_t most) {
    long long keys = (long long) p.c.M << p.page_log2;
    if (p.window) keys = std::min(keys, (long long) p.window + most);
    return 10.0 + 1.4e-3 * (double) plan_of(p, most).units * (double) ((keys + SLAB - 1) / SLAB);
}

void plan_paged_rows(PagedArgs & p, uint32_t most, size_t * groups, size_t * bytes) {
    const Plan r = plan_of(p, most);
    p.whole = 1;
    p.parts = 1;
    *groups = *bytes = 0;
    unsigned ctas = r.ctas;
    if (p.chosen) {
        const long long slabs = ((long long) p.picks << p.page_log2) / SLAB;
        p.parts = (int) std::max(1ll, std::min({r.ctas / r.units, slabs / LEAST, (long long) MOST_PARTS}));
        if (slabs <= SHORT) p.parts = 1;
        ctas = (unsigned) (r.units * p.parts);
        p.whole = p.parts == 1;
    } else {
        p.whole = (((long long) p.c.M << p.page_log2) + SLAB - 1) / SLAB <= SHORT;
    }
    if (!p.whole) {
        *groups = ctas;
        *bytes = (size_t) ctas * 2 * part_words((int) p.c.D, 8 * r.nt) * 4;
    }
}

cudaError_t launch_paged_rows(const PagedArgs & p, uint32_t most, cudaStream_t s) {
    const Plan r = plan_of(p, most);
    const unsigned grid = p.chosen ? (unsigned) (r.units * p.parts) : r.ctas;
    const bool bf = p.c.type == TSN_BF16;
    if (p.c.D == 64) return bf ? launch<64, true>(p, r.nt, r.warps, grid, s) : launch<64, false>(p, r.nt, r.warps, grid, s);
    return bf ? launch<128, true>(p, r.nt, r.warps, grid, s) : launch<128, false>(p, r.nt, r.warps, grid, s);
}

cudaError_t configure_paged_rows() {
    cudaError_t e = cudaSuccess;
    auto set = [&](auto * k, int bytes) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    };
#define SET(D, B, NT, W) \
    set(paged_rows_kernel<D, B, NT, false, W>, RowLay<D, NT, W, false>::TOTAL); \
    set(paged_rows_kernel<D, B, NT, true, W>, RowLay<D, NT, W, true>::TOTAL);
    SET(64, false, 1, 4) SET(64, false, 2, 4) SET(64, true, 1, 4) SET(64, true, 2, 4)
    SET(128, false, 1, 4) SET(128, false, 2, 4) SET(128, true, 1, 4) SET(128, true, 2, 4)
    SET(64, false, 1, 8) SET(64, false, 2, 8) SET(64, true, 1, 8) SET(64, true, 2, 8)
    SET(128, false, 1, 8) SET(128, false, 2, 8) SET(128, true, 1, 8) SET(128, true, 2, 8)
#undef SET
    return e;
}

} // namespace tsn

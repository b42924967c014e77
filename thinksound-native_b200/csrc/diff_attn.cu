// diff_attn.cu — differential attention (tsn_diff_attn): diff_attn_tc on the tcgen05 tensor cores, and
// diff_attn_rows for at most 32 query rows of a kv head.
//
//   o = O_1 / l_1 - lambda O_2 / l_2,   O_m = sum_j p_mj v_j,  l_m = sum_j p_mj,  p_mj = 2^(c q_m.k_mj - ref_m)
// in one pass over the keys: ref_m follows the running maximum of the row, O_m and l_m are rescaled when it
// moves, which is only when the maximum has grown by more than 2^8 (f32 and both 16-bit types hold that without
// loss). The two maps share every value tile, so K and V are read once for both.
// P is rounded to 16 bits, as the tensor cores take it; scores, maxima, sums and O are f32.
//
// Values behind masked keys may be NaN, and 0 * NaN is NaN. So V rows of masked keys count as zero, and where
// causal rows differ in what they see, non-finite values of a V row become zero and each row that sees such a
// key is marked: its result is NaN.
// Every wait is bounded; barriers of a whole block or cluster are on paths that all threads take.
#include "block_ops.h"
#include "kernels.h"
#include "ptx.cuh"

#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <mutex>

namespace tsn {

namespace {

constexpr int ROWS = 128, KEYS = 64;
constexpr int THREADS = 384;
constexpr float LOG2E = 1.44269504088896341f;
constexpr float LAZY = 8.0f;   // log2 units that a maximum may grow before O is rescaled

struct Args {
    tsn_diff_attn_args a;
    float c;                    // scale * log2(e)
    int G;                      // query heads per kv head
    int R;                      // Sq * G rows of one kv head
    int splits, kv_b;           // parts of the keys; 0: every batch reads the same keys
    int chunk;                  // few rows: slabs of a part
    float * part;
    unsigned int * count;
    int * err;
};

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

// A row's sums as they are added up over warps, CTAs or parts of the keys: O [2 maps][D], then ref and l of both maps.
constexpr int row_words(int D) { return 2 * D + 4; }

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

// Adds up `count` (1 to 64) sets of a row's sums, one warp: rd(i, k) is word k of set i, rdv(i, k, v) D / 32 words from k
// on. Returns O (this lane's D / 32 columns), ref and l. The order is that of the sets. Eight sets are read at once.
template <int D, class Rd, class RdV>
__device__ __forceinline__ void add_up(int count, int lane, float (&sum)[2][D / 32], float (&top)[2], float (&l)[2], Rd rd, RdV rdv) {
    constexpr int E = D / 32;
    const bool one = lane < count, two = lane + 32 < count;
    float w[2][2];   // the factors of sets lane and lane + 32
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const float r1 = one ? rd(lane, 2 * D + m) : -INFINITY, r2 = two ? rd(lane + 32, 2 * D + m) : -INFINITY;
        const float l1 = one ? rd(lane, 2 * D + 2 + m) : 0.0f, l2 = two ? rd(lane + 32, 2 * D + 2 + m) : 0.0f;
        top[m] = fmaxf(r1, r2);
#pragma unroll
        for (int x = 16; x; x >>= 1) top[m] = fmaxf(top[m], __shfl_xor_sync(~0u, top[m], x));
        const float ref = top[m] == -INFINITY ? 0.0f : top[m];
        w[m][0] = ex2(r1 - ref);
        w[m][1] = ex2(r2 - ref);
        l[m] = w[m][0] * l1 + w[m][1] * l2;
#pragma unroll
        for (int x = 16; x; x >>= 1) l[m] += __shfl_xor_sync(~0u, l[m], x);
#pragma unroll
        for (int e = 0; e < E; ++e) sum[m][e] = 0.0f;
    }
#pragma unroll 1
    for (int i = 0; i < count; i += 8) {
        float v[2][8][4];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + k < count) rdv(i + k, m * D + E * lane, v[m][k]);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float f = __shfl_sync(~0u, i < 32 ? w[m][0] : w[m][1], (i + k) & 31);
                if (i + k < count)
#pragma unroll
                    for (int e = 0; e < E; ++e) sum[m][e] = fmaf(f, v[m][k][e], sum[m][e]);
            }
    }
}

// The norm's factor of a row from its sum of squares and both maps' sums: NaN where o is not finite. A row that sees no
// key has no sums; its o is zero and stays so, also with an eps of 0 (0 * 1 / sqrt(0) would be NaN).
template <int D>
__device__ __forceinline__ float norm_factor(float ss, float eps, float l1, float l2) {
    if (l1 == 0.0f && l2 == 0.0f) return 0.0f;
    return ss < INFINITY ? rsqrtf(ss * (1.0f / D) + eps) : NAN;
}

// The result of one row from its sums, one warp: lam lambda of its head, nw the norm's weights.
template <int D, bool BF16>
__device__ __forceinline__ void write_row(const Args & p, int b, int hk, int i, int g, float lam, const float * nw, int lane,
                                          const float (&sum)[2][D / 32], const float (&l)[2]) {
    constexpr int E = D / 32;
    const tsn_diff_attn_args & a = p.a;
    const float w1 = l[0] == 0.0f ? 0.0f : 1.0f / l[0], w2 = l[1] == 0.0f ? 0.0f : lam / l[1];
    float ss = 0.0f, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] = sum[0][e] * w1 - sum[1][e] * w2;
        ss += v[e] * v[e];
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) ss += __shfl_xor_sync(~0u, ss, x);
    const float f = norm_factor<D>(ss, a.eps, l[0], l[1]);
    uint32_t x[E / 2];
#pragma unroll
    for (int e = 0; e < E; e += 2) x[e / 2] = pack16<BF16>(v[e] * f * nw[E * lane + e], v[e + 1] * f * nw[E * lane + e + 1]);
    uint16_t * out = (uint16_t *) a.out.p + b * a.out.sb + (long long) i * a.out.ss + (long long) (hk * p.G + g) * a.out.sh + E * lane;
    if constexpr (E == 4) *(uint2 *) out = make_uint2(x[0], x[1]);
    else *(uint32_t *) out = x[0];
}

// ================================================================ tensor cores
// diff_attn_tc: one CTA per 128 query rows of one kv head (rows are (token, query head of the group), so a group's
// heads share the K and V tiles) and, where there are few rows, per part of the keys; a cluster holds the parts.
// 384 threads:
//   warp 8      TMA: streams 64-key K and V tiles through a ring of stages
//   warps 9-10  one for each map m issue O_m += P_m V (M 128, N 2 d, K 64; P_m from TMEM) of tile j and then
//               S_m = Q_m K_m^T (M 128, N 64, K d) of tile j + BUF. (One thread for both maps, under a branch of its
//               own, took 1100 cycles for a map's eight products, commits and waits: twice what they run.)
//   warp 11     where some keys are masked: makes the tiles' V rows fit for the product (see above)
//   warps 0-3   map 1, warps 4-7 map 2: one row per thread. S_m from TMEM, mask, maximum, exponentials, P_m over
//               S_m's columns; O_m stays in TMEM
// TMEM at d = 64: S in two buffers per map (4 x 64 columns), so that a map's next scores are there when its
// softmax is done, and O_1, O_2 (128 each): all 512 columns.
// What bounds it: 2 exponentials for 12 d operations. At d = 64 a 128 x 64 tile pair takes 1024 cycles of the SFU
// (16 exponentials a cycle), 768 with every fourth pair on the FMA pipe, and 896 of the tensor cores (the products with
// N 64 wait for shared memory). 8125 tokens of 16 heads take 890 to 930 us, 0.87 to 0.91 PFLOP/s, about 1650 cycles a
// tile pair at the 1.65 GHz that the power limit leaves: both maps' warps tend to compute, and to wait for TMEM, at the same time.
// The sums of the rounded probabilities are one mixed add a value; with the unrounded ones, two to a packed add, it
// was 870. Measured before that, and left: 32-key tiles on 16 softmax warps (1050 us), turns of the maps for the SFU (975 to 1080), 128-key
// tiles with one buffer (1287), the next tile's scores requested a half tile ahead (960).
// Parts of the keys: each CTA leaves its rows' sums in its shared memory and, after a cluster barrier, adds up its
// share of the rows over the cluster, in the order of the parts.
template <int D>
struct Lay {
    static constexpr int BUF = 2;
    static constexpr int Q = ROWS * D * 2, BOX = KEYS * 128, TILE = KEYS * D * 2;   // boxes of 64 keys x 64 elements
    static constexpr int STAGES = 6;
    static constexpr int OFF_K = Q, OFF_V = OFF_K + STAGES * TILE, OFF_LAM = OFF_V + STAGES * TILE;
    static constexpr int OFF_W = OFF_LAM + 128 * 4, OFF_BAR = OFF_W + 128 * 4, TOTAL = OFF_BAR + 320;
    static constexpr uint32_t TM_O = 2 * BUF * KEYS, TM = 512;
    static_assert(TOTAL <= 227 * 1024, "one CTA's shared memory");
    static_assert(ROWS * row_words(D) * 4 <= 2 * STAGES * TILE, "the rows' sums fit in the ring");
    static_assert(TM_O + 2 * D <= TM, "tensor memory");
    static_assert(ROWS * (8 * 8 + 8) <= Q, "the parts' factors and the rows' sums fit in Q's place");
};

template <int D, bool BF16>
__global__ void __launch_bounds__(THREADS, 1)
diff_attn_tc(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ Args p) {
    using L = Lay<D>;
    constexpr int d = D / 2, ATOMS = D / 64, CH = D / 8, BUF = L::BUF;   // CH: 16-byte pieces of a head
    constexpr int QBOX = ROWS * 128;
    extern __shared__ __align__(1024) uint8_t smem[];
    const tsn_diff_attn_args & a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool fits = (smem_u32(smem) & 1023) == 0;   // the swizzled tiles need 1024-byte alignment
    if (!fits && tid == 0 && p.err) atomicCAS(p.err, 0, DEV_BAD_ARGS);
    float * lam = (float *) (smem + L::OFF_LAM), * nw = (float *) (smem + L::OFF_W);
    uint64_t * bar = (uint64_t *) (smem + L::OFF_BAR);
    uint64_t * q_full = bar, * full = bar + 1, * empty = full + L::STAGES, * s_full = empty + L::STAGES, * p_full = s_full + 2 * BUF,
             * o_full = p_full + 2 * BUF, * v_ready = o_full + 2 * BUF;
    uint32_t * words = (uint32_t *) (v_ready + L::STAGES);   // TMEM address, abort flag, keys of each stage with non-finite values [2]
    volatile int * abort_flag = (volatile int *) (words + 1);
    static_assert((1 + 3 * L::STAGES + 6 * BUF) * 8 + (2 + 2 * L::STAGES) * 4 <= 320, "barriers");

    if (tid == 0) {
        mbar_init(q_full, 8);
        for (int s = 0; s < L::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 2); mbar_init(&v_ready[s], 1); }
        for (int x = 0; x < 2 * BUF; ++x) { mbar_init(&s_full[x], 1); mbar_init(&p_full[x], 4); mbar_init(&o_full[x], 1); }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 8 && lane == 0 && a.Sk > 0) { tma_prefetch(&tk); tma_prefetch(&tv); }
    pdl_wait();   // from here on memory that earlier work may have written or may still read
    // Tensor memory after the wait and before the trigger: of two kernels on one SM, neither can hold what the other waits for.
    if (warp == 9) tmem_alloc(words, L::TM);

    // this CTA's rows, keys and part of them; long rows of a causal call come first
    const unsigned gid = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
    const int hk = (int) (gid % a.Hk), b = (int) (gid / a.Hk % a.B);
    const int r0 = (int) ((p.R + ROWS - 1) / ROWS - 1 - gid / a.Hk / a.B) * ROWS, rows = min(ROWS, p.R - r0);
    const int i0 = r0 / p.G, rem0 = r0 % p.G;   // row t: token i0 + (rem0 + t) / G, head (rem0 + t) % G
    const int n = a.key_len ? max(0, min(a.key_len[b], (int) a.Sk)) : (int) a.Sk;
    auto limit = [&](int t) {   // keys before which row t sees
        if (!a.causal) return n;
        return max(0, min(n, i0 + (rem0 + t) / p.G + n - (int) a.Sq + 1));   // at most 2^30 each
    };
    const int most = limit(rows - 1), least = limit(0);
    const int all_tiles = (most + KEYS - 1) / KEYS, per = (all_tiles + p.splits - 1) / p.splits;
    const int t0 = min(all_tiles, (int) split * per), nt = fits ? min(all_tiles, t0 + per) - t0 : 0;
    const uint8_t * mask = a.key_mask ? a.key_mask + b * a.mask_sb : nullptr;
    auto mixed = [&](int base) { return a.causal && least < min(n, base + KEYS); };   // rows see different keys of the tile
    const bool mend = nt > 0 && (mask || (t0 + nt) * KEYS > n || mixed((t0 + nt - 1) * KEYS));

    uint4 q[ROWS * CH / 256];   // Q, on its way while the barriers and tensor memory are set up
    if (warp < 8) {
#pragma unroll
        for (int y = 0; y < ROWS * CH / 256; ++y) {
            const int r = (tid + 256 * y) / CH, ch = tid % CH, u = rem0 + r;
            q[y] = make_uint4(0, 0, 0, 0);
            if (r < rows)
                q[y] = *(const uint4 *) ((const uint16_t *) a.q.p + b * a.q.sb + (long long) (i0 + u / p.G) * a.q.ss +
                                         (long long) (hk * p.G + u % p.G) * a.q.sh + ch * 8);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(~0u, words[0], 0), TM_O = tmem + L::TM_O;

    // the row of a softmax thread
    const int m = warp >> 2, t = tid & 127;
    const uint32_t lane0 = (uint32_t) ((warp & 3) * 32) << 16;
    float l = 0.0f, ref = -INFINITY;
    bool ok = true;

    if (warp >= 8) {
        if (warp == 8) {
            if (lane == 0) {
                for (int j = 0; j < nt; ++j) {
                    const int s = j % L::STAGES;
                    if (j >= L::STAGES && !mbar_wait_soon(&empty[s], (j / L::STAGES - 1) & 1, abort_flag, p.err, DEV_TIMEOUT_EMPTY)) break;
                    mbar_expect_tx(&full[s], 2 * L::TILE);
                    for (int x = 0; x < ATOMS; ++x) {
                        tma_load_4d(smem + L::OFF_K + s * L::TILE + x * L::BOX, &tk, &full[s], 64 * x, (t0 + j) * KEYS, hk, b * p.kv_b);
                        tma_load_4d(smem + L::OFF_V + s * L::TILE + x * L::BOX, &tv, &full[s], 64 * x, (t0 + j) * KEYS, hk, b * p.kv_b);
                    }
                }
            }
        } else if (warp == 11) {
            uint32_t mb[2] = {};   // whether the keys of the next tile are seen
            auto fetch = [&](int j) {
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const int key = (t0 + j) * KEYS + 32 * w + lane;
                    mb[w] = key < n && (!mask || mask[key] != 0);
                }
            };
            if (mend) fetch(0);
            for (int j = 0; j < nt && mend; ++j) {
                const int base = (t0 + j) * KEYS, s = j % L::STAGES;
                uint32_t gone[2], bad[2] = {0, 0};
#pragma unroll
                for (int w = 0; w < 2; ++w) gone[w] = ~__ballot_sync(~0u, mb[w] != 0);
                if (j + 1 < nt) fetch(j + 1);
                if (!mbar_wait_soon(&full[s], (j / L::STAGES) & 1, abort_flag, p.err, DEV_TIMEOUT_FULL)) break;
                __syncwarp();
                constexpr int AT_ONCE = 32 / CH;   // rows of one step
                const int sub = lane / CH, ch = lane % CH;
                auto at = [&](int key) {
                    return (uint4 *) (smem + L::OFF_V + s * L::TILE + (ch >> 3) * L::BOX + key * 128 + (((ch & 7) ^ (key & 7)) << 4));
                };
                // rows of masked keys, a lane a key: no chain from key to key, and in banks of their own (85.6 us for 2048 tokens of
                // 8 heads and two arms with an eighth of the keys masked, 97.4 with two keys after two)
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    if ((gone[w] >> lane) & 1u) {
                        uint8_t * row = smem + L::OFF_V + s * L::TILE + (32 * w + lane) * 128;
#pragma unroll
                        for (int y = 0; y < CH; ++y) *(uint4 *) (row + (y >> 3) * L::BOX + (((y & 7) ^ (lane & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                __syncwarp();
                // non-finite values, where some rows see the key and others do not
                if (mixed(base))
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
#pragma unroll 4
                        for (int y = 0; y < 32; y += AT_ONCE) {
                            const int key = 32 * w + y + sub;
                            const uint4 o = *at(key);
                            const uint4 f = make_uint4(finite_only<BF16>(o.x), finite_only<BF16>(o.y), finite_only<BF16>(o.z), finite_only<BF16>(o.w));
                            if (o.x != f.x || o.y != f.y || o.z != f.z || o.w != f.w) {
                                *at(key) = f;
                                bad[w] |= 1u << (key & 31);
                            }
                        }
                        bad[w] = __reduce_or_sync(~0u, bad[w]);
                    }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    words[2 + 2 * s] = bad[0];
                    words[3 + 2 * s] = bad[1];
                    mbar_arrive(&v_ready[s]);
                }
            }
        } else if (warp >= 9) {
            const int mm = warp - 9;
            const uint32_t lead = elect_lane(), id_s = umma_idesc_f16(KEYS, BF16), id_pv = umma_idesc_f16(D, BF16, 1);
            // map 2's halves of Q and K: the second box at d = 64, the second half of each 128-byte row at d = 32
            const uint64_t qd = umma_desc_sw128(smem + mm * (D == 128 ? QBOX : 64));
            const uint64_t kd = umma_desc_sw128(smem + L::OFF_K + mm * (D == 128 ? L::BOX : 64)), vd = umma_desc_sw128_mn(smem + L::OFF_V, L::BOX);
            const uint32_t to = TM_O + D * mm, ts = tmem + KEYS * BUF * mm;
            auto qk = [&](int j) {
                const int s = j % L::STAGES, x = j % BUF;
                if (!mbar_wait_soon(&full[s], (j / L::STAGES) & 1, abort_flag, p.err, DEV_TIMEOUT_FULL)) return false;
                const uint64_t k = kd + (uint64_t) (s * (L::TILE >> 4));
#pragma unroll
                for (int kk = 0; kk < d / 16; ++kk) umma_f16_if(lead, ts + KEYS * x, qd + 2 * kk, k + 2 * kk, id_s, kk != 0);
                umma_commit_if(lead, &s_full[mm * BUF + x]);
                return true;
            };
            bool go = nt > 0 && mbar_wait_soon(q_full, 0, abort_flag, p.err, DEV_TIMEOUT_FULL);
            for (int j = 0; j < BUF && j < nt && go; ++j) go = qk(j);
            for (int j = 0; j < nt && go; ++j) {
                const int s = j % L::STAGES, x = j % BUF;
                if (!mbar_wait_soon(&p_full[mm * BUF + x], (j / BUF) & 1, abort_flag, p.err, DEV_TIMEOUT_TMEM)) break;
                if (mend && !mbar_wait_soon(&v_ready[s], (j / L::STAGES) & 1, abort_flag, p.err, DEV_TIMEOUT_FULL)) break;
                tc_fence_after();
                const uint64_t v = vd + (uint64_t) (s * (L::TILE >> 4));
#pragma unroll
                for (int kk = 0; kk < KEYS / 16; ++kk)
                    umma_f16_ts_if(lead, to, ts + KEYS * x + 32 + 8 * kk, v + 128 * kk, id_pv, j > 0 || kk > 0);
                umma_commit_if(lead, &empty[s]);
                if (j + BUF < nt) go = qk(j + BUF);
                else umma_commit_if(lead, &o_full[mm * BUF + nt - 1 - j]);   // the last BUF tiles, [0] the last
            }
        }
        // the barriers of the other warps' results
        __syncwarp();
        pdl_trigger();
        if (p.splits > 1) {
            __syncthreads();
            cluster_sync_all();
            __syncthreads();
            cluster_sync_all();
        } else {
            for (int i = 0; i < 4; ++i) __syncthreads();
        }
    } else {
        if (fits) {
            // Q into its swizzled boxes, rows past the last one as zeros; lambda of each head of the group; weights
#pragma unroll
            for (int y = 0; y < ROWS * CH / 256; ++y) {
                const int r = (tid + 256 * y) / CH, ch = tid % CH;
                *(uint4 *) (smem + (ch >> 3) * QBOX + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = q[y];
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            for (int g = warp; g < p.G; g += 8) {
                const long long h = (long long) (hk * p.G + g) * a.lam_sh;
                float z1 = 0.0f, z2 = 0.0f;
                for (int e = lane; e < d; e += 32) { z1 += a.lq1[h + e] * a.lk1[h + e]; z2 += a.lq2[h + e] * a.lk2[h + e]; }
#pragma unroll
                for (int x = 16; x; x >>= 1) { z1 += __shfl_xor_sync(~0u, z1, x); z2 += __shfl_xor_sync(~0u, z2, x); }
                if (lane == 0) lam[g] = expf(z1) - expf(z2) + a.lambda_init;
            }
            if (tid < D) nw[tid] = (a.norm_w ? a.norm_w[tid] : 1.0f) * (1.0f - a.lambda_init);

            const uint32_t to = TM_O + D * m + lane0;
            const int lim = t < rows ? limit(t) : n;   // keys before which this row sees
            bool poison = false;
            uint32_t mb[2] = {};   // mask bytes of the next tile
            auto fetch_mask = [&](int j) {
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const int key = (t0 + j) * KEYS + 32 * w + lane;
                    mb[w] = key < n ? mask[key] : 0u;
                }
            };
            auto arrived = [&](int j) {   // tile j's scores
                const bool go = mbar_wait_soon(&s_full[m * BUF + j % BUF], (j / BUF) & 1, abort_flag, p.err, DEV_TIMEOUT_TMEM);
                __syncwarp();
                tc_fence_after();
                return go;
            };
            // A tile is taken in two halves of 32 keys, so that a half's scores come from TMEM while the other half's
            // exponentials run. P replaces the second half's scores; the first half's stay until the tile is done.
            uint32_t s1[32], vis[2] = {~0u, ~0u};
            float sum[4];
            // the first half of tile j, whose scores are there, and the maximum over both
            auto first_half = [&](auto masked, int j) {
                constexpr bool MASKED = decltype(masked)::value;
                const uint32_t at = tmem + KEYS * (m * BUF + j % BUF) + lane0;
                uint32_t s0[32], pk[16];
                tmem_request32(at, s0);
                if (MASKED) {
                    const int base = (t0 + j) * KEYS;
#pragma unroll
                    for (int w = 0; w < 2; ++w)
                        vis[w] = (mask ? __ballot_sync(~0u, mb[w] != 0) : low_bits(n - base - 32 * w)) & low_bits(lim - base - 32 * w);
                    if (mask && j + 1 < nt) fetch_mask(j + 1);
                }
                tmem_landed32(s0);
                tmem_request32(at + 32, s1);
                if (MASKED) hide(s0, vis[0]);
                // against the reference of the tiles before; the few tiles whose maximum is too far above it are done again
                sum[0] = sum[1] = sum[2] = sum[3] = 0.0f;
                exponentials<BF16, MASKED>(s0, pk, p.c, ref, sum);
                const float top0 = greatest(s0);
                tmem_landed32(s1);
                if (MASKED) hide(s1, vis[1]);
                const float top = fmaxf(top0, greatest(s1)) * p.c;
                const bool move = top > ref + LAZY;
                if (__any_sync(~0u, move)) {
                    // a row moves its reference by itself, so its result does not depend on its neighbours
                    const float f = move ? ex2(ref - top) : 1.0f;
                    if (move) { ref = top; l *= f; }
                    if (j > 0) {
                        // O is complete up to tile j - 1: the scores issued after that product are there, or its own commit
                        const int i = j - 1 + BUF;
                        uint64_t * done = i < nt ? &s_full[m * BUF + i % BUF] : &o_full[m * BUF + nt - j];
                        if (!mbar_wait_soon(done, i < nt ? (i / BUF) & 1 : 0, abort_flag, p.err, DEV_TIMEOUT_TMEM)) ok = false;
                        __syncwarp();
                        tc_fence_after();
#pragma unroll 1
                        for (int y = 0; y < D && ok; y += 16) {
                            float o[16];
                            tmem_ld16(to + y, o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] *= f;
                            tmem_st16(to + y, (const uint32_t *) o);
                        }
                    }
                    tmem_request32(at, s0);
                    tmem_landed32(s0);
                    if (MASKED) hide(s0, vis[0]);
                    sum[0] = sum[1] = sum[2] = sum[3] = 0.0f;
                    exponentials<BF16, MASKED>(s0, pk, p.c, ref, sum);
                }
                tmem_st16(at + 32, pk);
            };
            auto tiles = [&](auto masked, int from, int until) {
                constexpr bool MASKED = decltype(masked)::value;
                for (int j = from; j < until && ok; ++j) {
                    if (!arrived(j)) { ok = false; break; }
                    first_half(masked, j);
                    const int x = m * BUF + j % BUF;
                    uint32_t pk[16];
                    exponentials<BF16, MASKED>(s1, pk, p.c, ref, sum);
                    tmem_st16(tmem + KEYS * x + lane0 + 48, pk);
                    l += (sum[0] + sum[2]) + (sum[1] + sum[3]);
                    tmem_st_wait();
                    if (MASKED && m == 0 && mixed((t0 + j) * KEYS)) {
                        if (!mbar_wait_soon(&v_ready[j % L::STAGES], (j / L::STAGES) & 1, abort_flag, p.err, DEV_TIMEOUT_FULL)) ok = false;
                        const volatile uint32_t * bad = words + 2 + 2 * (j % L::STAGES);
                        poison |= (bad[0] & vis[0]) != 0 || (bad[1] & vis[1]) != 0;
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[x]);
                }
            };
            if (nt > 0) {
                if (mask) fetch_mask(0);
                const int clear = mask ? 0 : min(nt, max(0, least / KEYS - t0));   // tiles that every row sees whole
                tiles(std::false_type(), 0, clear);
                tiles(std::true_type(), clear, nt);
            }
            // no score above -inf: the FMA pipe's exponentials gave its keys 2^-126 each
            if (ref == -INFINITY && l < INFINITY) l = 0.0f;
            if (poison) l = NAN;
            if (ok && nt > 0) ok = mbar_wait_soon(&o_full[m * BUF], 0, abort_flag, p.err, DEV_TIMEOUT_TMEM);
            __syncwarp();
            tc_fence_after();
        }
        pdl_trigger();
        // ------------------------------------------------------------ results
        if (p.splits > 1) {
            // this part's sums in place of K and V: [row][row_words], a row 16 bytes past a multiple of all banks
            __syncthreads();   // both maps are done with the ring
            float * sums = (float *) (smem + L::OFF_K);
            if (fits) {
                float * to = sums + t * row_words(D);
#pragma unroll
                for (int x = 0; x < D; x += 32) {
                    float v[32];
                    if (nt > 0) {
                        tmem_ld32(TM_O + D * m + lane0 + x, v);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = 0.0f;
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 4) *(float4 *) (to + m * D + x + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                }
                to[2 * D + m] = ref;
                to[2 * D + 2 + m] = l;
            }
            cluster_sync_all();
            // this CTA's share of the rows: first each part's factors, 2^(ref - greatest) / l and that times -lambda, in Q's
            // place, then the parts' sums, a row by D / 4 lanes, four steps of rows at once
            const int share = (rows + p.splits - 1) / p.splits, from = (int) split * share, here = max(0, min(rows - from, share));
            const uint32_t at0 = smem_u32(sums) + from * row_words(D) * 4;
            float2 * fac = (float2 *) smem, * rl = fac + ROWS * 8;   // [row][8 parts]; [row] sums of both maps
            if (tid < here) {
                float4 st[8];   // ref and l of both maps
                float2 top = make_float2(-INFINITY, -INFINITY), sum = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < p.splits) {
                        st[i] = dsmem_ld4(dsmem_map(at0 + (tid * row_words(D) + 2 * D) * 4, (uint32_t) i));
                        top = make_float2(fmaxf(top.x, st[i].x), fmaxf(top.y, st[i].y));
                    }
                if (top.x == -INFINITY) top.x = 0.0f;
                if (top.y == -INFINITY) top.y = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < p.splits) {
                        st[i].x = ex2(st[i].x - top.x);
                        st[i].y = ex2(st[i].y - top.y);
                        sum.x += st[i].x * st[i].z;
                        sum.y += st[i].y * st[i].w;
                    }
                const float w1 = sum.x == 0.0f ? 0.0f : 1.0f / sum.x, w2 = sum.y == 0.0f ? 0.0f : -lam[(rem0 + from + tid) % p.G] / sum.y;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < p.splits) fac[tid * 8 + i] = make_float2(st[i].x * w1, st[i].y * w2);
                rl[tid] = sum;
            }
            __syncthreads();
            constexpr int LANES = D / 4, STEP = 8 * (32 / LANES), AT_ONCE = 4;   // of a row; rows of a step of all warps
            const int col = (lane % LANES) * 4;
            for (int y0 = warp * (32 / LANES) + lane / LANES; y0 < (here + STEP - 1) / STEP * STEP; y0 += STEP * AT_ONCE) {
                float o[AT_ONCE][4] = {};
                for (int i = 0; i < p.splits; ++i)
#pragma unroll
                    for (int y = 0; y < AT_ONCE; ++y) {
                        const int r = y0 + y * STEP;
                        if (r < here) {
                            const uint32_t at = dsmem_map(at0 + (r * row_words(D) + col) * 4, (uint32_t) i);
                            const float4 v = dsmem_ld4(at), w = dsmem_ld4(at + D * 4);
                            const float2 f = fac[r * 8 + i];
                            o[y][0] = fmaf(f.x, v.x, fmaf(f.y, w.x, o[y][0])); o[y][1] = fmaf(f.x, v.y, fmaf(f.y, w.y, o[y][1]));
                            o[y][2] = fmaf(f.x, v.z, fmaf(f.y, w.z, o[y][2])); o[y][3] = fmaf(f.x, v.w, fmaf(f.y, w.w, o[y][3]));
                        }
                    }
#pragma unroll
                for (int y = 0; y < AT_ONCE; ++y) {
                    const int r = y0 + y * STEP;
                    float ss = o[y][0] * o[y][0] + o[y][1] * o[y][1] + o[y][2] * o[y][2] + o[y][3] * o[y][3];
#pragma unroll
                    for (int x = LANES / 2; x; x >>= 1) ss += __shfl_xor_sync(~0u, ss, x);
                    if (r >= here || *abort_flag) continue;
                    const float g = norm_factor<D>(ss, a.eps, rl[r].x, rl[r].y);
                    const float4 w = *(const float4 *) (nw + col);
                    const int u = rem0 + from + r;
                    *(uint2 *) ((uint16_t *) a.out.p + b * a.out.sb + (long long) (i0 + u / p.G) * a.out.ss + (long long) (hk * p.G + u % p.G) * a.out.sh + col) =
                        make_uint2(pack16<BF16>(o[y][0] * g * w.x, o[y][1] * g * w.y), pack16<BF16>(o[y][2] * g * w.z, o[y][3] * g * w.w));
                }
            }
            cluster_sync_all();   // nobody leaves while its sums are read
        } else {
            // o = O_1 / l_1 - lambda O_2 / l_2, thread (row t, half m of the columns); RMSNorm over both halves; the result
            // through Q's place, so that whole rows are written. In place of K: row sums [2][128], sums of squares [2][128]
            float * rl = (float *) (smem + L::OFF_K), * rss = rl + 256;
            float o[d], l1, l2;
            tc_fence_before();
            __syncthreads();   // both maps are done with the ring, and their O is there
            tc_fence_after();
            rl[tid] = l;
            __syncthreads();
            {
                l1 = rl[t];
                l2 = rl[128 + t];
                const float w1 = l1 == 0.0f ? 0.0f : 1.0f / l1;
                const float w2 = l2 == 0.0f ? 0.0f : t < rows ? lam[(rem0 + t) % p.G] / l2 : 0.0f;
#pragma unroll
                for (int e = 0; e < d; ++e) o[e] = 0.0f;
                if (nt > 0) {
#pragma unroll
                    for (int x = 0; x < d; x += 32) {
                        float v[32];
                        tmem_ld32(TM_O + lane0 + m * d + x, o + x);
                        tmem_ld32(TM_O + D + lane0 + m * d + x, v);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[x + e] = o[x + e] * w1 - v[e] * w2;
                    }
                }
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < d; ++e) ss += o[e] * o[e];
                rss[tid] = ss;
            }
            __syncthreads();
            {
                const float ss = rss[t] + rss[128 + t];
                const float g = norm_factor<D>(ss, a.eps, l1, l2);
#pragma unroll
                for (int e = 0; e < d; e += 8) {
                    uint32_t x[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        x[k] = pack16<BF16>(o[e + 2 * k] * g * nw[m * d + e + 2 * k], o[e + 2 * k + 1] * g * nw[m * d + e + 2 * k + 1]);
                    const int ch = m * (CH / 2) + e / 8;
                    *(uint4 *) (smem + t * (D * 2) + ((ch ^ (t & 7)) << 4)) = make_uint4(x[0], x[1], x[2], x[3]);
                }
            }
            __syncthreads();
            if (!*abort_flag && fits)
                for (int i = tid; i < rows * CH; i += 256) {
                    const int r = i / CH, ch = i % CH, u = rem0 + r;
                    *(uint4 *) ((uint16_t *) a.out.p + b * a.out.sb + (long long) (i0 + u / p.G) * a.out.ss +
                                (long long) (hk * p.G + u % p.G) * a.out.sh + ch * 8) =
                        *(const uint4 *) (smem + r * (D * 2) + ((ch ^ (r & 7)) << 4));
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

// ================================================================ few rows
// diff_attn_rows: a few rows of a kv head (one token with its group's heads, or a few), bound by reading K and V.
// A 128-row tile would spend its time on rows that do not exist; here mma.sync takes 8 rows, with the keys (and for
// the product with V the columns) on its 16-row side: S^T = K Q^T, O^T = V^T P^T, 24 products for 16 keys of 8 KB.
// P^T is S^T's layout transposed in registers (movmatrix). With the rows on the 16-row side, half of it empty, twice
// the products and exponentials made one token over four caches of 32 768 keys take 97 us.
// Each warp streams its own 16-key slabs (slab w, w + W, ...) by TMA through a ring of its own, so warps never wait
// for one another: scores, online softmax and O of both maps stay in the warp's registers. The warps' sums
// are added up in shared memory at the end, the parts of split keys through the workspace.
// One token over four caches of 20 480 to 32 768 keys (32 heads over 8, bf16) takes 73.5 us: 436 MB, 5.93 TB/s, 0.91 of the
// measured copy; one over two caches of up to 704 keys 9.0 us, most of it the way from the launch to the first keys.
constexpr int SLAB = 16, RING = 3, SOME = 8, W = 8;   // keys of a slab, slabs of a ring, rows of a group, warps
// Rows up to which groups of 8 are taken instead of a tile of 128. bf16, d 64, causal, us by groups / by tiles at 8, 32 and 64
// rows a kv head: one head over 32 768 keys 18.6/59.5, 20.5/60.3, 29.2/61.6 (parts go to more SMs than a cluster has); 8 over
// 4096 13.6/15.5, 15.6/16.6, 21.4/18.1; 2 x 8 over 704 10.3/12.3, 11.1/12.9, 11.3/14.2. Each group reads the keys anew, so
// where there are more groups than SMs tiles are ahead from 24 rows on: 8 x 8 over 512 10.2/13.2, 19.1/13.8, 36.4/15.2;
// 4 x 8 over 8192 31.9/37.1, 54.3/37.9, 133/39.8. The bound takes only the rows into account.
constexpr int FEW = 32;

template <int D>
struct RowLay {
    static constexpr int BOX = SLAB * 128, HALF = SLAB * D * 2, STAGE = 2 * HALF;   // a slab's keys, then its values
    static constexpr int OFF_LAM = W * RING * STAGE, OFF_W = OFF_LAM + 16 * 4, OFF_BAR = OFF_W + D * 4;
    static constexpr int TOTAL = OFF_BAR + W * RING * 8 + 16;
    static constexpr int SUMS = SOME * row_words(D);   // after the last slab, in a warp's ring
    static_assert(W * SUMS * 4 <= W * RING * STAGE, "the warps' sums fit in their rings");
};

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

template <int D, bool BF16>
__global__ void __launch_bounds__(32 * W, 1)
diff_attn_rows(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ Args p) {
    using L = RowLay<D>;
    constexpr int d = D / 2, E = D / 32;
    extern __shared__ __align__(1024) uint8_t smem[];
    const tsn_diff_attn_args & a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (smem_u32(smem) & 1023) {
        if (tid == 0 && p.err) atomicCAS(p.err, 0, DEV_BAD_ARGS);
        return;
    }
    float * lam = (float *) (smem + L::OFF_LAM), * nw = (float *) (smem + L::OFF_W);
    uint64_t * full = (uint64_t *) (smem + L::OFF_BAR) + warp * RING;
    volatile int * flags = (volatile int *) (smem + L::OFF_BAR + W * RING * 8);   // abort, last to arrive

    // All groups of a part lie next to one another: the groups of 8 rows of a kv head read the same keys at about the same
    // time, and the kv heads neighbouring ones (a head's row is 256 bytes, too little for DRAM by itself).
    const int eights = (p.R + SOME - 1) / SOME;
    const unsigned groups = gridDim.x / p.splits, gid = blockIdx.x % groups, split = blockIdx.x / groups;
    const int hk = (int) (gid / eights % a.Hk), b = (int) (gid / eights / a.Hk);
    const int first = (int) (gid % eights) * SOME, R = min(SOME, p.R - first);   // row r: token (first + r) / G, head (first + r) % G
    if (lane == 0) {
        if (a.Sk > 0) { tma_prefetch(&tk); tma_prefetch(&tv); }
        for (int s = 0; s < RING; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
    }
    pdl_wait();
    const int n = a.key_len ? max(0, min(a.key_len[b], (int) a.Sk)) : (int) a.Sk;
    auto limit = [&](int r) {   // keys before which row r sees; rows past the last one see all
        if (!a.causal || r >= R) return n;
        return max(0, min(n, (first + r) / p.G + n - (int) a.Sq + 1));   // at most 2^30 each
    };
    const int least = limit(0);
    // this CTA's slabs, and this warp's
    const int s0 = (int) min((long long) (n + SLAB - 1) / SLAB, (long long) split * p.chunk);
    const int s1 = min((n + SLAB - 1) / SLAB, s0 + p.chunk);
    const int mine = s1 - s0 > warp ? (s1 - s0 - warp + W - 1) / W : 0;

    if (tid == 0) flags[0] = 0;
    __syncwarp();
    uint8_t * ring = smem + warp * RING * L::STAGE;
    auto request = [&](int i) {   // slab i of this warp, one lane
        uint8_t * at = ring + (i % RING) * L::STAGE;
        const int key = (s0 + warp + i * W) * SLAB;
        mbar_expect_tx(&full[i % RING], L::STAGE);
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
            tma_load_4d(at + x * L::BOX, &tk, &full[i % RING], 64 * x, key, hk, b * p.kv_b);
            tma_load_4d(at + L::HALF + x * L::BOX, &tv, &full[i % RING], 64 * x, key, hk, b * p.kv_b);
        }
    };
    if (lane == 0)
        for (int i = 0; i < RING && i < mine; ++i) request(i);

    // lambda of each row's head, the norm's weights
    for (int r = warp; r < R; r += W) {
        const long long h = (long long) (hk * p.G + (first + r) % p.G) * a.lam_sh;
        float z1 = 0.0f, z2 = 0.0f;
        for (int e = lane; e < d; e += 32) { z1 += a.lq1[h + e] * a.lk1[h + e]; z2 += a.lq2[h + e] * a.lk2[h + e]; }
#pragma unroll
        for (int x = 16; x; x >>= 1) { z1 += __shfl_xor_sync(~0u, z1, x); z2 += __shfl_xor_sync(~0u, z2, x); }
        if (lane == 0) lam[r] = expf(z1) - expf(z2) + a.lambda_init;
    }
    for (int e = tid; e < D; e += 32 * W) nw[e] = (a.norm_w ? a.norm_w[e] : 1.0f) * (1.0f - a.lambda_init);

    // Q^T as B operands: row lane / 4, rows past the last one as zeros. Scores: keys lane / 4 (+ 8) by rows c0, c0 + 1.
    const int g0 = lane >> 2, c0 = (lane & 3) * 2;
    uint32_t qb[2][d / 16][2];
    {
        const int u = first + g0;
        const uint16_t * q = (const uint16_t *) a.q.p + b * a.q.sb + (long long) (u / p.G) * a.q.ss + (long long) (hk * p.G + u % p.G) * a.q.sh;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int k = 0; k < d / 16; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) qb[m][k][h] = g0 < R ? *(const uint32_t *) (q + m * d + 16 * k + 8 * h + c0) : 0u;
    }
    const int lim[2] = {limit(c0), limit(c0 + 1)};
    const uint8_t * mask = a.key_mask ? a.key_mask + b * a.mask_sb : nullptr;
    __syncthreads();   // the abort flag, lambda and the weights are set

    float o[2][D / 16][4], l[2][2] = {}, ref[2][2];   // O^T: columns 16 x + lane / 4 (+ 8) by rows c0, c0 + 1
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        ref[m][0] = ref[m][1] = -INFINITY;
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[m][x][k] = 0.0f;
    }
    bool poison[2] = {false, false};
    // addresses of ldmatrix: K rows (key), two groups of 8 keys by two of 8 elements; V rows (key), two groups of 8 columns
    // by two of 8 keys
    const int krow = (lane & 7) + (((lane >> 3) & 1) << 3), kch = lane >> 4;
    const int vrow = (lane & 7) + ((lane >> 4) << 3), vch = (lane >> 3) & 1;
    uint32_t mb = mask && mine > 0 && lane < SLAB && (s0 + warp) * SLAB + lane < n ? mask[(s0 + warp) * SLAB + lane] : 0u;
    for (int i = 0; i < mine; ++i) {
        const int base = (s0 + warp + i * W) * SLAB;
        uint32_t there = low_bits(n - base) & 0xffffu;   // the keys that exist
        if (mask) {
            there = __ballot_sync(~0u, mb != 0);
            const int key = base + W * SLAB + lane;
            mb = lane < SLAB && key < n ? mask[key] : 0u;
        }
        if (!mbar_wait_soon(&full[i % RING], (i / RING) & 1, flags, p.err, DEV_TIMEOUT_FULL)) break;
        __syncwarp();
        const uint32_t kt = smem_u32(ring + (i % RING) * L::STAGE), vt = kt + L::HALF;
        float s[2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int k = 0; k < 4; ++k) s[m][k] = 0.0f;
#pragma unroll
            for (int k = 0; k < d / 16; ++k) {
                const int col = m * d + 16 * k;
                uint32_t f[4];
                ldmatrix4<false>(f, kt + (col / 64) * L::BOX + krow * 128 + ((((col % 64) / 8 + kch) ^ (krow & 7)) << 4));
                mma16816<BF16>(s[m], f, qb[m][k][0], qb[m][k][1]);
            }
        }
        const bool gone = there != 0xffffu, mixed = a.causal && least < min(n, base + SLAB);
        uint32_t vis[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) vis[h] = there & low_bits(lim[h] - base);
        if (gone || mixed) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (!((vis[k & 1] >> (g0 + 8 * (k >> 1))) & 1u)) s[m][k] = -INFINITY;
        }
        bool move = false;
        float top[2][2];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                top[m][h] = fmaxf(s[m][h], s[m][2 + h]) * p.c;
                move |= top[m][h] > ref[m][h] + LAZY;
            }
        if (__any_sync(~0u, move)) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float t = top[m][h];
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) t = fmaxf(t, __shfl_xor_sync(~0u, t, x));
                    if (t > ref[m][h] + LAZY) {   // a row moves its reference by itself
                        const float f = ex2(ref[m][h] - t);
                        ref[m][h] = t;
                        l[m][h] *= f;
#pragma unroll
                        for (int x = 0; x < D / 16; ++x) { o[m][x][h] *= f; o[m][x][2 + h] *= f; }
                    }
                }
        }
        uint32_t pb[2][2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const float n0 = ref[m][0] == -INFINITY ? 0.0f : -ref[m][0], n1 = ref[m][1] == -INFINITY ? 0.0f : -ref[m][1];
            const float e0 = ex2(fmaf(s[m][0], p.c, n0)), e1 = ex2(fmaf(s[m][1], p.c, n1));
            const float e2 = ex2(fmaf(s[m][2], p.c, n0)), e3 = ex2(fmaf(s[m][3], p.c, n1));
            const uint32_t p0 = pack16<BF16>(e0, e1), p1 = pack16<BF16>(e2, e3);
            add_rounded<BF16>(l[m][0], l[m][1], p0);   // the sums are of what the product takes
            add_rounded<BF16>(l[m][0], l[m][1], p1);
            pb[m][0] = movmatrix(p0);
            pb[m][1] = movmatrix(p1);
        }
        if (!gone && !mixed) {
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
                uint32_t f[4];
                ldmatrix4<true>(f, vt + (x / 4) * L::BOX + vrow * 128 + (((2 * (x % 4) + vch) ^ (vrow & 7)) << 4));
#pragma unroll
                for (int m = 0; m < 2; ++m) mma16816<BF16>(o[m][x], f, pb[m][0], pb[m][1]);
            }
        } else {
            // values behind masked keys count as zero; where rows differ, so do non-finite ones, and rows that see one are marked
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
                for (int m = 0; m < 2; ++m) mma16816<BF16>(o[m][x], f, pb[m][0], pb[m][1]);
            }
            bad = __reduce_or_sync(~0u, bad);
            poison[0] |= (bad & vis[0]) != 0;
            poison[1] |= (bad & vis[1]) != 0;
        }
        __syncwarp();   // every lane has its operands: the stage may be loaded again
        if (lane == 0 && i + RING < mine) request(i + RING);
    }

    pdl_trigger();   // from here on little memory is read: the next kernel's blocks would have taken bandwidth before
    // the warp's sums in its ring, then warp w adds up rows w, w + W, ... of all warps
    float * sums = (float *) ring;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float t = l[m][h];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) t += __shfl_xor_sync(~0u, t, x);
            float * to = sums + (c0 + h) * row_words(D);
            if (g0 == 0) {
                to[2 * D + m] = ref[m][h];
                to[2 * D + 2 + m] = poison[h] ? NAN : t;
            }
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
                to[m * D + 16 * x + g0] = o[m][x][h];
                to[m * D + 16 * x + g0 + 8] = o[m][x][2 + h];
            }
        }
    __syncthreads();
    const size_t size = (size_t) R * row_words(D);   // of a part
    float * part = p.part + (size_t) gid * p.splits * (SOME * row_words(D));
    for (int r = warp; r < R && !flags[0]; r += W) {
        float sum[2][E], top[2], rl[2];
        auto at = [&](int i, int k) { return (const float *) (smem + i * RING * L::STAGE) + r * row_words(D) + k; };
        add_up<D>(W, lane, sum, top, rl, [&](int i, int k) { return *at(i, k); },
                  [&](int i, int k, float * v) { read_words<E, false>(at(i, k), v); });
        if (p.splits == 1) {
            write_row<D, BF16>(p, b, hk, (first + r) / p.G, (first + r) % p.G, lam[r], nw, lane, sum, rl);
        } else {
            float * to = part + split * size + r * row_words(D);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                if constexpr (E == 4) *(float4 *) (to + m * D + E * lane) = make_float4(sum[m][0], sum[m][1], sum[m][2], sum[m][3]);
                else *(float2 *) (to + m * D + E * lane) = make_float2(sum[m][0], sum[m][1]);
                if (lane == 0) { to[2 * D + m] = top[m]; to[2 * D + 2 + m] = rl[m]; }
            }
        }
    }
    if (p.splits > 1) {
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            const bool last = atomicAdd(&p.count[gid], 1u) + 1u == (unsigned) p.splits;
            if (last) p.count[gid] = 0;   // for the next call
            __threadfence();
            flags[1] = last;
        }
        __syncthreads();
        if (flags[1])
            for (int r = warp; r < R && !flags[0]; r += W) {
                float sum[2][E], top[2], rl[2];
                auto at = [&](int i, int k) { return part + i * size + r * row_words(D) + k; };
                add_up<D>(p.splits, lane, sum, top, rl, [&](int i, int k) { return __ldcg(at(i, k)); },
                          [&](int i, int k, float * v) { read_words<E, true>(at(i, k), v); });
                write_row<D, BF16>(p, b, hk, (first + r) / p.G, (first + r) % p.G, lam[r], nw, lane, sum, rl);
            }
    }
    if (flags[0] && tid == 0) {
        // let copies that were issued but never consumed land before the CTA's shared memory is reused
        const uint64_t t1 = global_ns();
        while (global_ns() - t1 < 20000ull) {}
    }
}

// ---------------------------------------------------------------- host
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static const PFN_cuTensorMapEncodeTiled_v12000 enc = [] {
        cudaDriverEntryPointQueryResult q{};
        void * fn = nullptr;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return (PFN_cuTensorMapEncodeTiled_v12000) fn;
    }();
    return enc;
}

// {2 d, Sk, Hk, B} view of keys or values with {64, box_keys, 1, 1} boxes. A dimension of one element has a
// stride that is never taken: any valid one stands in.
bool make_kv_map(CUtensorMap * m, const tsn_diff_attn_args & a, const tsn_heads & t, uint32_t B, uint32_t box_keys) {
    const PFN_cuTensorMapEncodeTiled_v12000 enc = encoder();
    if (!enc) return false;
    const cuuint64_t row = 2 * a.d * 2;
    const cuuint64_t dims[4] = {2 * a.d, a.Sk, a.Hk, B};
    const cuuint64_t strides[3] = {a.Sk > 1 ? (cuuint64_t) t.ss * 2 : row, a.Hk > 1 ? (cuuint64_t) t.sh * 2 : row,
                                   B > 1 ? (cuuint64_t) t.sb * 2 : row};
    const cuuint32_t box[4] = {64, box_keys, 1, 1}, es[4] = {1, 1, 1, 1};
    return enc(m, a.type == TSN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, t.p, dims, strides,
               box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr size_t COUNTERS = 4096, WORKSPACE = COUNTERS * 4 + ((size_t) 32 << 20);
constexpr int SMS = 148;

// Host calls that touch no stream of the program, so that they also work while one of them is being captured.
struct Uncaptured {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    Uncaptured() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~Uncaptured() { cudaThreadExchangeStreamCaptureMode(&mode); }
};
cudaError_t zero(void * p, size_t bytes) {   // and waits for it
    Uncaptured u;
    cudaStream_t s = nullptr;
    cudaError_t e = cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking);
    if (e == cudaSuccess) e = cudaMemsetAsync(p, 0, bytes, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (s) cudaStreamDestroy(s);
    return e;
}
cudaError_t allocate(void ** p, size_t bytes) {
    Uncaptured u;
    return cudaMalloc(p, bytes);
}
int failed(cudaError_t e) {
    cudaGetLastError();
    return fail(e == cudaErrorMemoryAllocation ? TSN_ERR_OOM : TSN_ERR_CUDA, std::string("tsn_diff_attn: ") + cudaGetErrorString(e));
}

// The device's workspace, ordered after the last call that used it. Streams are told apart by their id, which no other
// stream of the process ever has: a handle may stand for one stream per thread, or be given out again.
int workspace(DeviceCtx & c, unsigned long long stream) {
    cudaError_t e = cudaSuccess;
    if (!c.split_ws) {
        void * p = nullptr;
        e = allocate(&p, WORKSPACE);
        if (e == cudaSuccess) e = zero(p, COUNTERS * 4);
        if (e == cudaSuccess && !c.split_ev) e = cudaEventCreateWithFlags(&c.split_ev, cudaEventDisableTiming);
        if (e != cudaSuccess) { cudaFree(p); return failed(e); }
        c.split_ws = p;
    }
    if (c.split_used && c.split_stream != stream) e = cudaStreamWaitEvent(c.stream, c.split_ev, 0);
    return e == cudaSuccess ? TSN_OK : failed(e);
}

// Workspaces of captured calls. One belongs to its call's graph, so that replays need no order among themselves or with other
// calls; when the graph and its executables are gone it lies here until another capture, or the device's end, takes it.
struct Block {
    void * p;
    size_t bytes;
    int ordinal;
    Block * next;
};
std::mutex g_idle_mu;
Block * g_idle = nullptr;

void CUDART_CB make_idle(void * block) {   // no CUDA calls in here
    std::lock_guard<std::mutex> lk(g_idle_mu);
    Block * b = (Block *) block;
    b->next = g_idle;
    g_idle = b;
}

int graph_workspace(const DeviceCtx & c, cudaGraph_t graph, size_t bytes, void ** out) {
    size_t size = (size_t) 1 << 18;   // powers of two, so that they fit the calls of later captures
    while (size < bytes) size *= 2;
    Block * b = nullptr;
    {
        std::lock_guard<std::mutex> lk(g_idle_mu);
        for (Block ** at = &g_idle; *at; at = &(*at)->next)
            if ((*at)->ordinal == c.ordinal && (*at)->bytes == size) {
                b = *at;
                *at = b->next;
                break;
            }
    }
    if (!b) {
        b = new Block{nullptr, size, c.ordinal, nullptr};
        const cudaError_t e = allocate(&b->p, size);
        if (e != cudaSuccess) { delete b; return failed(e); }
    }
    cudaUserObject_t object = nullptr;
    cudaError_t e = zero(b->p, size);
    if (e == cudaSuccess) e = cudaUserObjectCreate(&object, b, make_idle, 1, cudaUserObjectNoDestructorSync);
    if (e != cudaSuccess) {
        make_idle(b);
        return failed(e);
    }
    e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
    if (e != cudaSuccess) {
        cudaUserObjectRelease(object, 1);
        return failed(e);
    }
    *out = b->p;
    return TSN_OK;
}

template <int D, bool BF16>
cudaError_t launch_tc(const CUtensorMap & tk, const CUtensorMap & tv, const Args & p, unsigned grid, cudaStream_t s) {
    return launch_cl(diff_attn_tc<D, BF16>, dim3(grid), dim3(THREADS), Lay<D>::TOTAL, s, dim3((unsigned) p.splits), tk, tv, p);
}
template <int D, bool BF16>
cudaError_t launch_rows(const CUtensorMap & tk, const CUtensorMap & tv, const Args & p, unsigned grid, cudaStream_t s) {
    return launch_cl(diff_attn_rows<D, BF16>, dim3(grid), dim3(32 * W), RowLay<D>::TOTAL, s, dim3(1), tk, tv, p);
}

// clusters of 1 to 8 CTAs of diff_attn_tc that run at once (one CTA per SM; a cluster lies within a GPC)
std::atomic<int> g_clusters[9];

} // namespace

cudaError_t configure_diff_attn() {
    cudaError_t e = cudaSuccess;
    auto set = [&](auto * k, int bytes) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    };
    set(diff_attn_rows<64, false>, RowLay<64>::TOTAL);
    set(diff_attn_rows<64, true>, RowLay<64>::TOTAL);
    set(diff_attn_rows<128, false>, RowLay<128>::TOTAL);
    set(diff_attn_rows<128, true>, RowLay<128>::TOTAL);
    set(diff_attn_tc<64, false>, Lay<64>::TOTAL);
    set(diff_attn_tc<64, true>, Lay<64>::TOTAL);
    set(diff_attn_tc<128, false>, Lay<128>::TOTAL);
    set(diff_attn_tc<128, true>, Lay<128>::TOTAL);
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
        e = cudaOccupancyMaxActiveClusters(&count, diff_attn_tc<128, true>, &cfg);
        g_clusters[n] = count;
    }
    return e;
}

void release_diff_attn(int ordinal) {
    Block * gone = nullptr;
    {
        std::lock_guard<std::mutex> lk(g_idle_mu);
        for (Block ** at = &g_idle; *at;) {
            Block * b = *at;
            if (b->ordinal != ordinal) { at = &b->next; continue; }
            *at = b->next;
            b->next = gone;
            gone = b;
        }
    }
    while (gone) {   // without the lock: freeing may wait for a thread of the driver's that is in make_idle
        Block * b = gone;
        gone = b->next;
        cudaFree(b->p);
        delete b;
    }
}

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

    // a batch stride of 0 in both K and V: one batch of keys. In one of them only, the map needs real strides.
    Args p{};
    p.kv_b = a.B > 1 && (a.k.sb || a.v.sb) ? 1 : 0;
    const uint32_t KB = p.kv_b ? a.B : 1;
    auto mappable = [&](const tsn_heads & t) {
        auto fits = [](int64_t s) { return s > 0 && s < (1ll << 39); };
        return (a.Sk <= 1 || fits(t.ss)) && (a.Hk == 1 || fits(t.sh)) && (KB == 1 || fits(t.sb));
    };
    if (a.Sk && (!mappable(a.k) || !mappable(a.v)))
        return fail(TSN_ERR_ARG, "tsn_diff_attn: strides of k and v must be positive (0 only for the batch, in both)");
    p.a = a;
    p.c = a.scale * LOG2E;
    p.G = (int) (a.H / a.Hk);
    if ((long long) a.Sq * p.G > (1ll << 30)) return fail(TSN_ERR_ARG, "tsn_diff_attn: more than 2^30 query rows of a kv head");
    p.R = (int) a.Sq * p.G;
    p.err = c.d_err;
    const bool rows = p.R <= FEW;
    const long long groups = (long long) (rows ? (p.R + SOME - 1) / SOME : (p.R + ROWS - 1) / ROWS) * a.B * a.Hk;   // below 2^60
    if (rows) {
        // As many parts as take the least time, in units of what one CTA takes for a slab (93 ns): the start of a CTA is 30,
        // a trip of the sums through the workspace 30 and a half for each part; past 74 CTAs at once (of 8 KB slabs) they
        // wait for HBM. One token of 32 heads over 8, four caches of 32 768 keys: 87 us with one wave of 128 CTAs (6.2
        // TB/s), 93 to 163 with two to sixteen; 16 heads over 704 keys: 9.6 us in one part or eight, 11.3 in two.
        const long long slabs = ((long long) a.Sk + SLAB - 1) / SLAB, room = (long long) (WORKSPACE - COUNTERS * 4) / (SOME * (4 * a.d + 4) * 4);
        double least = 0.0;
        for (long long parts = 1; parts <= 64 && (parts == 1 || (groups <= (long long) COUNTERS && groups * parts <= room)); ++parts) {
            const long long chunk = std::max(1ll, (slabs + parts - 1) / parts), ctas = groups * parts;
            const double crowd = std::max(1.0, std::min<long long>(ctas, SMS) * (a.d / 64.0) / 74.0);
            const double cost = (double) ((ctas + SMS - 1) / SMS) * (30.0 + chunk * crowd) + (parts > 1 ? 30.0 + 0.5 * parts : 0.0);
            if (parts == 1 || cost < least) {
                least = cost;
                p.chunk = (int) chunk;
                p.splits = (int) std::max(1ll, (slabs + chunk - 1) / chunk);
            }
        }
    } else {
        // As many parts of a cluster as take the least time, in microseconds: start and end of a CTA 7, a tile of a 64-wide map
        // 1 (of a 32-wide one 0.7), adding up the parts 3; clusters of one size run g_clusters[size] at a time. Four key tiles
        // a part at least, eight parts at most (the largest portable cluster).
        const long long tiles = ((long long) a.Sk + KEYS - 1) / KEYS;
        double least = 0.0;
        for (int parts = 1; parts <= 8 && (parts == 1 || parts * 4 <= tiles); ++parts) {
            const long long room = std::max(1, g_clusters[parts].load(std::memory_order_relaxed));
            const double cost = (double) ((groups + room - 1) / room) * (7.0 + (double) ((tiles + parts - 1) / parts) * (a.d == 64 ? 1.0 : 0.7)) + (parts > 1 ? 3.0 : 0.0);
            if (parts == 1 || cost < least) { least = cost; p.splits = parts; }
        }
    }
    if (groups * p.splits > 0x7fffffffLL) return fail(TSN_ERR_ARG, "tsn_diff_attn: too many query rows");
    const bool shared = rows && p.splits > 1;   // through the workspace
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    unsigned long long stream = 0;
    if (shared) {
        cudaGraph_t graph = nullptr;
        cudaError_t e = cudaStreamGetCaptureInfo(c.stream, &capture, nullptr, &graph, nullptr, nullptr);
        if (e == cudaSuccess && capture == cudaStreamCaptureStatusInvalidated) e = cudaErrorStreamCaptureInvalidated;
        if (e == cudaSuccess && capture == cudaStreamCaptureStatusNone) e = cudaStreamGetId(c.stream, &stream);
        if (e != cudaSuccess) return failed(e);
        size_t counters = COUNTERS * 4;
        void * ws = nullptr;
        int rc;
        if (capture == cudaStreamCaptureStatusNone) {
            rc = workspace(c, stream);
            ws = c.split_ws;
        } else {
            counters = ((size_t) groups * 4 + 255) & ~(size_t) 255;
            rc = graph_workspace(c, graph, counters + (size_t) groups * p.splits * (SOME * (4 * a.d + 4) * 4), &ws);
        }
        if (rc) return rc;
        p.count = (unsigned int *) ws;
        p.part = (float *) ((char *) ws + counters);
    }
    CUtensorMap tk{}, tv{};
    if (a.Sk && (!make_kv_map(&tk, a, a.k, KB, rows ? SLAB : KEYS) || !make_kv_map(&tv, a, a.v, KB, rows ? SLAB : KEYS)))
        return fail(TSN_ERR_ARG, "tsn_diff_attn: k or v cannot be described to the tensor memory accelerator");
    const unsigned grid = (unsigned) (groups * p.splits);
    const bool bf = a.type == TSN_BF16;
    cudaError_t e;
    if (rows)
        e = a.d == 32 ? (bf ? launch_rows<64, true>(tk, tv, p, grid, c.stream) : launch_rows<64, false>(tk, tv, p, grid, c.stream))
                      : (bf ? launch_rows<128, true>(tk, tv, p, grid, c.stream) : launch_rows<128, false>(tk, tv, p, grid, c.stream));
    else
        e = a.d == 32 ? (bf ? launch_tc<64, true>(tk, tv, p, grid, c.stream) : launch_tc<64, false>(tk, tv, p, grid, c.stream))
                      : (bf ? launch_tc<128, true>(tk, tv, p, grid, c.stream) : launch_tc<128, false>(tk, tv, p, grid, c.stream));
    if (e != cudaSuccess) cudaGetLastError();
    if (e == cudaSuccess && shared && capture == cudaStreamCaptureStatusNone) {
        e = cudaEventRecord(c.split_ev, c.stream);
        c.split_used = true;
        c.split_stream = stream;
    }
    if (e != cudaSuccess) return fail(TSN_ERR_CUDA, std::string("tsn_diff_attn: ") + cudaGetErrorString(e));
    return TSN_OK;
}

} // namespace tsn

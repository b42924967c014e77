// page_select.cu — which pages a token attends to (the first kernel of tsn_sparse_attn).
//
//   s_x = (sum_g q_g) . mean_x for the pages x before the token's own;  the `picks` best, `first` and `last` ones always
// The picks are whole numbers, and a sum rounded to 32 bits would exchange pages whose scores nearly agree, so scores are
// summed in 64 bits: products of 16-bit values are exact there. A 16-bit value becomes an f64 by shifting its f32 bits
// right by 3 into the high word, which is the value times 2^-896 exactly, subnormals and zero included (a conversion
// instruction has a quarter of the FMAs' rate); q carries a factor of 2^880 against it. Factors that all scores share change no order.
//
// Scores: D / 8 lanes read a mean, a warp eight means a lane at once (four for four tokens) and the next ones ahead; partial sums are exchanged so that each
// lane ends with whole ones. A block takes one token and kv head, or, where there are many tokens, four neighbouring ones,
// which share the reads while they are of one sequence.
// Picks: scores, rounded to f32, which keeps their order but for ties, are counted in bins of equal width between the least and the
// greatest; the bin that the last pick falls into is taken apart again, by their bits, until few scores are left, and these are ranked against one
// another in 64 bits. (Where more agree in 32 bits, the same goes on in 64.) The picks are written in the order of the pages.
// 8 tokens x 8 kv heads over 2048 pages take 20 us (two blocks a token), 400 tokens x 4 over 600 pages 55 us: instructions, about
// half of them FMAs' and conversions', the rest exchanges and the picks' small steps. Reads under branches took 2.4 times
// as long, scores sorted by radix with a 64-bit compare 2 to 3 times.
#include "kernels.h"
#include "paged.h"
#include "ptx.cuh"

#include <cfloat>
#include <type_traits>

namespace tsn {

namespace {

struct Select {
    tsn_sparse_attn_args a;
    int page_log2, G;
    int parts;   // blocks of a cluster that share a token's pages
};

// Two 16-bit values of a word, each times 2^-896: the low words of such f64 are zero.
template <class T>
__device__ __forceinline__ void scaled(uint32_t w, double & a, double & b) {
    int x, y;   // f32 bits
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x = (int) (w << 16);
        y = (int) w;   // what lies below is cut off with the shifted bits
    } else {
        const float2 f = unpack2<T>(w);
        x = __float_as_int(f.x);
        y = __float_as_int(f.y);
    }
    a = __hiloint2double((x >> 3) & (int) 0x8fffffff, 0);
    b = __hiloint2double((y >> 3) & (int) (std::is_same<T, __nv_bfloat16>::value ? 0x8fffe000 : 0x8fffffff), 0);
}

// A group of GT threads (whole warps) of a block, with a barrier of its own.
template <int GT>
struct Group {
    static constexpr int WARPS = GT / 32, BINS = 4 * GT, FEW = 64;   // FEW: scores that are ranked, each against the others
    static constexpr int LOG_BINS = GT == 128 ? 9 : 11;
    static_assert(1 << LOG_BINS == BINS, "bins");
    int id, tid, lane, warp;
    struct Space {
        unsigned int hist[BINS];
        uint64_t lo[WARPS], hi[WARPS];
        double rank_v;
        uint32_t lo32[WARPS], hi32[WARPS];
        int2 red[WARPS];
        unsigned int digit, above, inside, listed, rank_need;
        unsigned short list[FEW];
    } * m;
    __device__ __forceinline__ void sync() const { asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(GT) : "memory"); }
    // the least and the greatest over the group
    __device__ __forceinline__ void range(uint64_t & lo, uint64_t & hi) const {
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            lo = min(lo, (uint64_t) __shfl_xor_sync(~0u, (unsigned long long) lo, o));
            hi = max(hi, (uint64_t) __shfl_xor_sync(~0u, (unsigned long long) hi, o));
        }
        if (lane == 0) { m->lo[warp] = lo; m->hi[warp] = hi; }
        sync();
        for (int w = 0; w < WARPS; ++w) {
            lo = min(lo, m->lo[w]);
            hi = max(hi, m->hi[w]);
        }
    }
    __device__ __forceinline__ void range(uint32_t & lo, uint32_t & hi) const {
        lo = __reduce_min_sync(~0u, lo);
        hi = __reduce_max_sync(~0u, hi);
        if (lane == 0) { m->lo32[warp] = lo; m->hi32[warp] = hi; }
        sync();
        lo = __reduce_min_sync(~0u, m->lo32[lane % WARPS]);
        hi = __reduce_max_sync(~0u, m->hi32[lane % WARPS]);
    }
    // sums of the threads before this one
    __device__ __forceinline__ int2 before(int2 v) const {
        int2 s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(~0u, s.x, o), y = __shfl_up_sync(~0u, s.y, o);
            if (lane >= o) { s.x += x; s.y += y; }
        }
        if (lane == 31) m->red[warp] = s;
        sync();
        int2 t = lane < warp ? m->red[lane % WARPS] : make_int2(0, 0);
        t.x = __reduce_add_sync(~0u, t.x);
        t.y = __reduce_add_sync(~0u, t.y);
        return make_int2(s.x - v.x + t.x, s.y - v.y + t.y);
    }
    // Counts the bins and takes the one that the last pick falls into: bin(j) or -1. Returns it.
    template <class Bin>
    __device__ __forceinline__ int divide(int c, unsigned & need, unsigned & left, Bin bin) const {
        for (int i = tid; i < BINS; i += GT) m->hist[i] = 0;
        sync();
        for (int j = tid; j < c; j += GT) {
            const int x = bin(j);
            if (x >= 0) atomicAdd(&m->hist[x], 1u);
        }
        sync();
        // thread t: bins from the highest down, 4 t ..
        unsigned int h[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += h[i] = m->hist[BINS - 1 - 4 * tid - i];
        unsigned int above = (unsigned) before(make_int2((int) sum, 0)).x;
        if (above < need && need <= above + sum) {
            int i = 0;
            while (above + h[i] < need) above += h[i++];
            m->digit = (unsigned) (BINS - 1 - 4 * tid - i);
            m->above = above;
            m->inside = h[i];
        }
        sync();
        need -= m->above;
        left = m->inside;
        return (int) m->digit;
    }
    static __device__ __forceinline__ uint32_t ordered(float f) {   // bits in the order of the numbers, and back
        const uint32_t x = __float_as_uint(f);
        return x >> 31 ? ~x : x | 0x80000000u;
    }
    static __device__ __forceinline__ uint64_t ordered(double f) {
        const uint64_t x = (uint64_t) __double_as_longlong(f);
        return x >> 63 ? ~x : x | (1ull << 63);
    }
    static __device__ __forceinline__ double number(uint64_t x) { return __longlong_as_double((long long) (x >> 63 ? x & ~(1ull << 63) : ~x)); }
    static __device__ __forceinline__ float number(uint32_t x) { return __uint_as_float(x >> 31 ? x & 0x7fffffffu : ~x); }
    // The `picks` pages of n: `first` ones, those from top on, and the best of the scores s, f of pages first .. top - 1; n > picks.
    __device__ void pick(const double * s, const float * f, int n, int first, int top, int picks, int * chosen) const {
        const int c = top - first;                       // pages that compete
        unsigned int need = (unsigned) (picks - first - (n - top)), left = (unsigned) c;
        double bound = DBL_MAX;                          // picked: scores above it, and the first `equal` of those that are it
        unsigned int equal = 0;
        if (need) {
            uint32_t lo32 = ~0u, hi32 = 0;               // not decided: scores lo .. hi, of them those in bin `digit` (-1: all)
            for (int j = tid; j < c; j += GT) { lo32 = min(lo32, ordered(f[j])); hi32 = max(hi32, ordered(f[j])); }
            range(lo32, hi32);
            // The first round's bins are of equal width in the scores, where that is a number; the others' in the bits, so that each
            // leaves 2^-LOG_BINS of the numbers that are possible: the rounds end.
            const float least = number(lo32), width = (float) BINS / (number(hi32) - least);
            const bool even = width > 0.0f && width < INFINITY;
            bool first_round = true;
            int digit = -1, shift = 0;
            auto bin = [&](int j) {
                const uint32_t k = ordered(f[j]);
                if (k < lo32 || k > hi32) return -1;
                return even && first_round ? min(BINS - 1, (int) ((f[j] - least) * width)) : (int) ((k - lo32) >> shift);
            };
            auto undecided = [&](int j) { return digit < 0 ? ordered(f[j]) >= lo32 && ordered(f[j]) <= hi32 : bin(j) == digit; };
            while (lo32 < hi32 && left > (unsigned) FEW && need < left) {
                if (digit >= 0) {                        // the bin's own range
                    uint32_t lo = ~0u, hi = 0;
                    for (int j = tid; j < c; j += GT)
                        if (undecided(j)) { lo = min(lo, ordered(f[j])); hi = max(hi, ordered(f[j])); }
                    range(lo, hi);
                    lo32 = lo;
                    hi32 = hi;
                    digit = -1;
                    first_round = false;
                    if (lo == hi) break;
                }
                shift = max(0, 32 - __clz(hi32 - lo32) - LOG_BINS);
                digit = divide(c, need, left, bin);
            }
            if (left > (unsigned) FEW) {                 // more than can be ranked: on in 64 bits
                uint64_t lo = ~0ull, hi = 0;
                for (int j = tid; j < c; j += GT)
                    if (undecided(j)) { lo = min(lo, ordered(s[j])); hi = max(hi, ordered(s[j])); }
                range(lo, hi);
                int shift64 = 0;
                auto bin64 = [&](int j) {
                    const uint64_t k = ordered(s[j]);
                    return k < lo || k > hi ? -1 : (int) ((k - lo) >> shift64);
                };
                while (lo < hi && left > (unsigned) FEW && need < left) {
                    shift64 = max(0, 64 - __clzll((long long) (hi - lo)) - LOG_BINS);
                    const int d = divide(c, need, left, bin64);
                    uint64_t lo2 = ~0ull, hi2 = 0;
                    for (int j = tid; j < c; j += GT)
                        if (bin64(j) == d) { lo2 = min(lo2, ordered(s[j])); hi2 = max(hi2, ordered(s[j])); }
                    range(lo2, hi2);
                    lo = lo2;
                    hi = hi2;
                }
                if (left > (unsigned) FEW) {
                    bound = number(lo);
                    equal = need == left ? (unsigned) c : need;   // all of them, or all are the same
                } else {
                    rank(s, c, need, left, bound, equal, [&](int j) { return ordered(s[j]) >= lo && ordered(s[j]) <= hi; });
                }
            } else {
                rank(s, c, need, left, bound, equal, undecided);
            }
        }
        const int per = (n + GT - 1) / GT, j0 = min(n, tid * per), j1 = min(n, j0 + per);
        auto kind = [&](int j) {   // 2: picked, 1: it is the bound, 0: not picked
            if (j < first || j >= top) return 2;
            const double v = s[j - first];
            return v > bound ? 2 : v == bound ? 1 : 0;
        };
        int2 count = make_int2(0, 0);
        for (int j = j0; j < j1; ++j) {
            const int k = kind(j);
            count.x += k == 2;
            count.y += k == 1;
        }
        sync();   // the sums' place may still be read
        int2 at = before(count);
        if (count.x || count.y)
            for (int j = j0; j < j1; ++j) {
                const int k = kind(j);
                if (k == 2 || (k == 1 && at.y < (int) equal)) chosen[at.x + min(at.y, (int) equal)] = j;
                at.x += k == 2;
                at.y += k == 1;
            }
    }
    // Of at most FEW scores, the one with need - 1 before it, in 64 bits and then in the order of the pages.
    template <class In>
    __device__ __forceinline__ void rank(const double * s, int c, unsigned need, unsigned left, double & bound, unsigned & equal, In in) const {
        if (tid == 0) m->listed = 0;
        sync();
        for (int j = tid; j < c; j += GT)
            if (in(j)) m->list[atomicAdd(&m->listed, 1u)] = (unsigned short) j;
        sync();
        if (tid < (int) left) {
            const int mine = m->list[tid];
            const double v = s[mine];
            unsigned int greater = 0, earlier = 0;
            for (int i = 0; i < (int) left; ++i) {
                const int j = m->list[i];
                const double w = s[j];
                greater += w > v;
                earlier += w == v && j < mine;
            }
            if (greater + earlier + 1 == need) {
                m->rank_v = v;
                m->rank_need = need - greater;
            }
        }
        sync();
        bound = m->rank_v;
        equal = m->rank_need;
    }
};

// TOK tokens of a block, GT threads for each in the end.
template <class T, int D, int TOK, int GT>
__global__ void __launch_bounds__(TOK * GT, 1) page_select_kernel(const __grid_constant__ Select p) {
    constexpr int THREADS = TOK * GT, LPH = D / 8, SIDE = 32 / LPH, BATCH = TOK == 1 ? 8 : 4;   // BATCH: means of a lane at once
    constexpr int SUMS = TOK * BATCH, KEPT = SUMS > LPH ? SUMS / LPH : 1, SAME = LPH > SUMS ? LPH / SUMS : 1;   // of a lane; in the end; lanes with the same
    extern __shared__ __align__(16) double scores[];   // [TOK][M], then the same in f32
    __shared__ typename Group<GT>::Space space[TOK];
    __shared__ __align__(16) double qs[TOK][4][LPH][2];   // a lane's four pairs of elements, neighbouring lanes side by side
    __shared__ int seq[TOK], place[TOK];
    const tsn_sparse_attn_args & a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, parts = TOK > 1 ? 1 : p.parts, part = TOK > 1 ? 0 : (int) blockIdx.x % parts,
              row0 = (int) blockIdx.x / parts * TOK, hk = (int) blockIdx.y;
    if (TOK == 1 && parts > 1) cluster_arrive();
    pdl_wait();
    if (warp < TOK) {
        const int row = row0 + warp, b = row < (int) a.c.N ? seq_of_row(a.c, row) : -1, pl = b < 0 ? 0 : place_of_row(a.c, b, row);
        if (lane == 0) {
            seq[warp] = b;
            place[warp] = pl;
        }
    }
    for (int i = tid; i < TOK * D; i += THREADS) {
        const int t = i / D, e = i % D, row = row0 + t;
        double s = 0.0;
        if (row < (int) a.c.N) {
            const T * q = (const T *) a.q.p + row * a.q.sb + (long long) (hk * p.G) * a.q.st + e;
            for (int g = 0; g < p.G; g += 4) {   // four heads' loads at once
                T v[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) v[y] = g + y < p.G ? q[(g + y) * a.q.st] : from_f32<T>(0.0f);
#pragma unroll
                for (int y = 0; y < 4; ++y) s += (double) to_f32(v[y]);
            }
        }
        qs[t][e / 2 % 4][e / 8][e % 2] = s * 0x1p880;
    }
    __syncthreads();
    if (TOK == 1 && parts > 1) cluster_wait();   // the first block runs: scores may be stored into its shared memory
    pdl_trigger();
    const int picks = (int) a.picks, first = (int) a.first;
    float * rounded = (float *) (scores + TOK * a.c.M);
    auto pages_of = [&](int t) {   // the token's own and those before
        const int own = place[t] < 0 ? -1 : place[t] >> p.page_log2;
        return own >= (int) a.c.M ? 0 : own + 1;
    };
    const int sub = lane / LPH, e0 = (lane % LPH) * 8;
    for (int t0 = 0, t1; t0 < TOK; t0 = t1) {   // tokens t0 .. t1 - 1 are of one sequence
        t1 = t0 + 1;
        while (t1 < TOK && seq[t1] == seq[t0]) ++t1;
        const int b = seq[t0];
        if (b < 0) continue;
        // pages that compete for some token: first .. top - 1
        int top = 0;
        for (int t = t0; t < t1; ++t)
            if (pages_of(t) > picks) top = max(top, pages_of(t) - (int) a.last);
        const int m = top - first;
        const int * table = a.c.table + b * a.c.table_sb;
        // lane (sub, l) reads its 8 elements of means j0 + sub * BATCH + y. No page: zeros
        const int STEP = THREADS / 32 * (BATCH * SIDE) * parts;
        const int ahead = first + sub * BATCH + lane % BATCH;
        auto page_at = [&](int j) { return j + ahead < top ? table[j + ahead] : -1; };
        Words<T, 8> r[2][BATCH];
        uint32_t there[2];
        auto fetch = [&](int id, int x) {
            there[x] = __ballot_sync(~0u, id >= 0 && id < (int) a.c.P) >> (sub * LPH);
            const int safe = id >= 0 && id < (int) a.c.P ? id : 0;
#pragma unroll
            for (int y = 0; y < BATCH; ++y)
                r[x][y] = load_words<T, 8>((const T *) a.means.p + (long long) __shfl_sync(~0u, safe, sub * LPH + y) * a.means.sb + hk * a.means.st + e0);
        };
        if (a.c.P == 0) {   // nothing to read: every score is that of zero means
            for (int t = t0; t < t1; ++t)
                for (int j = tid; j < m; j += THREADS) { scores[t * a.c.M + j] = 0.0; rounded[t * a.c.M + j] = 0.0f; }
            continue;
        }
        auto sums = [&](int j0, int x) {
            double s[SUMS];   // token t, mean y at t * BATCH + y
#pragma unroll
            for (int i = 0; i < SUMS; ++i) s[i] = 0.0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                double2 q[TOK];
#pragma unroll
                for (int t = 0; t < TOK; ++t) q[t] = *(const double2 *) qs[t][e][lane % LPH];
#pragma unroll
                for (int y = 0; y < BATCH; ++y) {
                    double u, v;
                    scaled<T>(((const uint32_t *) r[x][y].w)[e], u, v);
#pragma unroll
                    for (int t = 0; t < TOK; ++t) s[t * BATCH + y] = fma(q[t].y, v, fma(q[t].x, u, s[t * BATCH + y]));
                }
            }
            // The lanes' parts of the sums are added up while each lane keeps half of them, then half of these: the lanes' bits, from the
            // highest down, are the sums' that it ends with.
            int n = SUMS;
#pragma unroll
            for (int o = LPH / 2; o; o >>= 1) {
                const bool up = (lane & o) != 0;
                if (n > 1) {
                    n /= 2;
#pragma unroll
                    for (int i = 0; i < SUMS / 2; ++i)
                        if (i < n) {
                            const double give = up ? s[i] : s[i + n], keep = up ? s[i + n] : s[i];
                            s[i] = keep + __shfl_xor_sync(~0u, give, o);
                        }
                } else {
                    s[0] += __shfl_xor_sync(~0u, s[0], o);
                }
            }
#pragma unroll
            for (int k = 0; k < KEPT; ++k) {
                const int i = lane % LPH / SAME * KEPT + k, t = i / BATCH, y = i % BATCH, mine = j0 + first + sub * BATCH + y;
                if (mine < top && lane % SAME == 0 && t >= t0 && t < t1) {
                    // numbers that bins can be made of: NaN and what exceeds 2^1000 (of queries that are not finite) at the ends
                    const double v = (there[x] >> y) & 1u ? fmin(fmax(s[k], -0x1p1000), 0x1p1000) + 0.0 : 0.0;   // -0 becomes 0
                    const float f = fminf(fmaxf((float) v, -FLT_MAX), FLT_MAX);
                    const int at = t * (int) a.c.M + mine - first;
                    if (TOK > 1 || parts == 1) {
                        scores[at] = v;
                        rounded[at] = f;
                    } else {   // the scores of a cluster's blocks meet in the first one
                        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(dsmem_map(smem_u32(scores + at), 0)), "d"(v) : "memory");
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dsmem_map(smem_u32(rounded + at), 0)), "f"(f) : "memory");
                    }
                }
            }
        };
        int j0 = (warp + part * (THREADS / 32)) * (BATCH * SIDE), id = page_at(j0);
        if (j0 < m) fetch(id, 0);
        id = page_at(j0 + STEP);
        while (j0 < m) {
            if (j0 + STEP < m) fetch(id, 1);
            id = page_at(j0 + 2 * STEP);
            sums(j0, 0);
            j0 += STEP;
            if (j0 >= m) break;
            if (j0 + STEP < m) fetch(id, 0);
            id = page_at(j0 + 2 * STEP);
            sums(j0, 1);
            j0 += STEP;
        }
    }
    __syncwarp();
    if (parts > 1) {
        cluster_sync_all();
        if (part) return;
    } else {
        __syncthreads();
    }
    Group<GT> g;
    g.id = TOK == 1 ? 0 : tid / GT;
    g.tid = tid % GT;
    g.lane = lane;
    g.warp = g.tid >> 5;
    g.m = &space[g.id];
    const int n = pages_of(g.id);
    if (seq[g.id] < 0) return;   // a row of no sequence
    int * chosen = a.chosen + ((long long) (row0 + g.id) * a.c.Hk + hk) * picks;
    if (n <= picks)
        for (int j = g.tid; j < picks; j += GT) chosen[j] = j < n ? j : -1;
    else
        g.pick(scores + g.id * a.c.M, rounded + g.id * a.c.M, n, first, n - (int) a.last, picks, chosen);
}

constexpr int MANY = 4;   // tokens of a block where there are many
constexpr int MOST = 16384 * 12;   // bytes of scores

template <class T, int D>
cudaError_t launch(const Select & p, cudaStream_t s) {
    const size_t bytes = (size_t) p.a.c.M * 12;
    // Four tokens a block share the reads; single ones fill the GPU with fewer tokens, and hold the scores of more pages.
    if ((long long) p.a.c.N * p.a.c.Hk >= 2 * MANY * 148 && MANY * bytes <= MOST)
        return launch_cl(page_select_kernel<T, D, MANY, 128>, dim3((p.a.c.N + MANY - 1) / MANY, p.a.c.Hk), dim3(MANY * 128), MANY * bytes, s, dim3(1), p);
    // As many blocks for a token as there are SMs for, up to four, each with 512 pages or more.
    Select one = p;
    while (one.parts < 4 && (long long) p.a.c.N * p.a.c.Hk * one.parts * 2 <= 148 && p.a.c.M >= 1024u * one.parts) one.parts *= 2;
    return launch_cl(page_select_kernel<T, D, 1, 512>, dim3(p.a.c.N * one.parts, p.a.c.Hk), dim3(512), bytes, s, dim3((unsigned) one.parts), one);
}

} // namespace

cudaError_t launch_page_select(const tsn_sparse_attn_args & a, cudaStream_t s) {
    const Select p{a, log2_of(a.c.page), (int) (a.H / a.c.Hk), 1};
    const bool bf = a.c.type == TSN_BF16;
    if (a.c.D == 64) return bf ? launch<__nv_bfloat16, 64>(p, s) : launch<__half, 64>(p, s);
    return bf ? launch<__nv_bfloat16, 128>(p, s) : launch<__half, 128>(p, s);
}

cudaError_t configure_page_select() {
    cudaError_t e = cudaSuccess;
    auto set = [&](auto * k) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST);
    };
    set(page_select_kernel<__half, 64, 1, 512>);
    set(page_select_kernel<__half, 128, 1, 512>);
    set(page_select_kernel<__nv_bfloat16, 64, 1, 512>);
    set(page_select_kernel<__nv_bfloat16, 128, 1, 512>);
    set(page_select_kernel<__half, 64, MANY, 128>);
    set(page_select_kernel<__half, 128, MANY, 128>);
    set(page_select_kernel<__nv_bfloat16, 64, MANY, 128>);
    set(page_select_kernel<__nv_bfloat16, 128, MANY, 128>);
    return e;
}

} // namespace tsn

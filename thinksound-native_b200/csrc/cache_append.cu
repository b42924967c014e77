// cache_append.cu — new tokens into a paged key/value cache, with the heads' norm and the rotary positions (tsn_cache_append).
//
// Bound by HBM: q, k and v are read once, q_out and the pages written once. As in tsn_rope_axes a block takes a few whole
// tokens, computes their cosines and sines once into shared memory (64-bit phases), and its warps run over the heads, 8 elements a
// lane, loads some ahead. What the cache adds is a chain of small reads for each token (its sequence, length and page), a lane
// a token, while the heads' loads are on their way.
// The means of the pages are a second kernel, which reads the touched pages' keys after the first has written them.
// 37 000 tokens x 48 heads of 128, bf16, with means take 215 us (986 MB, 4.6 TB/s, 0.70 of the measured copy), 191 of them the first
// kernel: half reads, half writes, at 130 instructions a warp's 512 bytes and 64 registers; 3136 tokens from f32 12 to 16 us
// (3.5 to 4.7 TB/s), 256 tokens with means 10 to 11 us, 4 tokens 4.9 us (the call).
// Loads two tokens ahead: with four 254 us, with one 232; 8 tokens a block: with 16 218, with 4 227.
#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "paged.h"

namespace tsn {

namespace {

__device__ __forceinline__ float phase(int pos, uint64_t turn) {   // pos * turn modulo one turn, in [-1/2, 1/2) turns
    const uint64_t p = (uint64_t) (long long) pos * turn;
    return (float) (int) (p >> 32) * 0x1p-32f;
}

constexpr int WARPS = 8, MAX_TOK = 8;
enum { NEXT, LANES, SHARED };   // where the other element of a lane's pairs is: with the lane, another lane, shared memory

struct Append {
    tsn_cache_append_args a;
    int page_log2, tok, span;   // tokens of a block, chunks of it
};

// Block (x, y): tokens x * tok .., chunks y * span .. of 32 / LPH heads: the queries', then the keys', then the values'. A warp takes a
// chunk through the block's tokens, so that a token costs its lanes a load, a store and the arithmetic (items that were each
// worked out for themselves took as long as the memory traffic), loads AHEAD tokens before; then its next chunk.
template <class TX, class T, int LPH, int PAIR>
__global__ void __launch_bounds__(32 * WARPS, 4) cache_append_kernel(const __grid_constant__ tsn_rope_plan_t p, const __grid_constant__ Append n) {
    constexpr int SIDE = 32 / LPH, AHEAD = sizeof(TX) == 4 ? 1 : 2;
    constexpr bool SAME = std::is_same<TX, T>::value;
    __shared__ __align__(16) float turn[MAX_TOK * 3 * TSN_ROPE_MAX_PAIRS];   // of a token's pairs: cosines, sines, sines with the other sign
    __shared__ float mate[PAIR == SHARED ? WARPS : 1][32 * 9];               // a lane's 8 elements, one word of padding between lanes
    __shared__ int place[MAX_TOK], spot[MAX_TOK], slot[MAX_TOK];             // spot: the page, -1: none
    pdl_wait();
    const tsn_cache_append_args & a = n.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int D = (int) p.D, P = (int) p.P, Hq = (int) a.Hq, Hk = (int) a.c.Hk, tok = n.tok;
    const long long s0 = (long long) blockIdx.x * tok;
    const int here = (int) min((long long) tok, a.c.N - s0);
    const int sub = lane / LPH, at = (lane & (LPH - 1)) * 8;
    const int q_chunks = (Hq + SIDE - 1) / SIDE, k_chunks = (Hk + SIDE - 1) / SIDE, chunks = q_chunks + 2 * k_chunks;
    const int until = min(chunks, ((int) blockIdx.y + 1) * n.span);
    const float inv_D = 1.0f / (float) D;
    const int row = (P + 3) & ~3;   // a token's pairs in the table, from a 16-byte boundary on

    // the chunk: queries', keys' or values', the lane's head and its elements
    int chunk = (int) blockIdx.y * n.span + warp, what = 0, head = 0;
    bool mine = false;
    const TX * x = nullptr;
    long long dx = 0;
    Words<TX, 8> ring[AHEAD];
    auto begin = [&] {   // with the first tokens' loads
        what = chunk < q_chunks ? 0 : chunk < q_chunks + k_chunks ? 1 : 2;
        head = (chunk - (what == 0 ? 0 : what == 1 ? q_chunks : q_chunks + k_chunks)) * SIDE + sub;
        mine = chunk < until && at < D && head < (what == 0 ? Hq : Hk);
        const tsn_rows & in = what == 0 ? a.q : what == 1 ? a.k : a.v;
        dx = in.sb;
        x = (const TX *) in.p + s0 * dx + head * in.st + at;
#pragma unroll
        for (int y = 0; y < AHEAD; ++y) {
            if (mine && y < here) ring[y] = load_words<TX, 8>(x);
            x += dx;
        }
    };
    begin();   // before the table: the loads are on their way
    if (warp == 0) {   // a lane a token; mostly all are of one sequence
        const int b0 = seq_of_row(a.c, (int) s0), b1 = here > 1 ? seq_of_row(a.c, (int) s0 + here - 1) : b0;
        if (lane < here) {
            const int i = (int) s0 + lane, b = b0 == b1 && b0 >= 0 ? b0 : seq_of_row_alone(a.c, i);   // whole sequences may lie between rows of none
            const int pl = b < 0 ? 0 : place_of_row(a.c, b, i);
            place[lane] = pl;
            spot[lane] = b < 0 ? -2 : page_of(a.c, b, pl >> n.page_log2);   // -2: a row of no sequence
            slot[lane] = pl & ((1 << n.page_log2) - 1);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < here * P; i += 32 * WARPS) {
        const int k = i / P, j = i % P;
        const int pos = a.pos ? a.pos[(s0 + k) * a.pos_ss + p.axis[j]] : place[k];
        float sn, cs;
        sincospif(2.0f * phase(pos, p.turn[j]), &sn, &cs);
        float * t = turn + k * 3 * row + j;
        t[0] = cs;
        t[row] = sn;
        t[2 * row] = -sn;
    }
    __syncthreads();

    // halves: the lane's pairs, whether its elements are the first or the second ones, and the lane that holds the others
    const bool low = at < P, turned = at < 2 * P;
    const int other = PAIR == LANES && turned ? (low ? lane + P / 8 : lane - P / 8) : lane;
    for (; chunk < until; chunk += WARPS) {
        float2 w[4];
        const float * wp = what == 0 ? a.q_norm : what == 1 ? a.k_norm : nullptr;
        if (wp)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = mine ? make_float2(wp[at + 2 * i], wp[at + 2 * i + 1]) : make_float2(0.0f, 0.0f);
        const tsn_heads & to = what == 1 ? a.c.k : a.c.v;
        T * const out = what == 0 ? (T *) a.q_out.p + s0 * a.q_out.sb + head * a.q_out.st + at : (T *) to.p + head * to.sh + at;
        auto target = [&](int k) {   // where token k goes; null: nowhere
            if (what == 0) return spot[k] == -2 ? nullptr : out + k * a.q_out.sb;
            return spot[k] < 0 ? nullptr : out + spot[k] * to.sb + slot[k] * to.ss;
        };
        for (int k0 = 0; k0 < here; k0 += AHEAD)
#pragma unroll
            for (int y = 0; y < AHEAD; ++y) {
                const int k = k0 + y;
                if (k >= here) break;
                const Words<TX, 8> raw = ring[y];
                if (mine && k + AHEAD < here) ring[y] = load_words<TX, 8>(x);
                x += dx;
                if (SAME && what == 2) {   // values go as they are
                    T * const dst = target(k);
                    if (mine && dst) *(uint4 *) dst = raw.w[0];
                    continue;
                }
                float u[8];
                to_floats<TX, 8>(raw, u);
                if (wp) {
                    float2 q = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int i = 0; i < 8; i += 2) q = fma2(make_float2(u[i], u[i + 1]), make_float2(u[i], u[i + 1]), q);
                    float ss = mine ? q.x + q.y : 0.0f;
#pragma unroll
                    for (int o = LPH >> 1; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    const float inv = rsqrtf(fmaf(ss, inv_D, a.eps));
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const float2 r = mul2(make_float2(u[i], u[i + 1]), mul2(w[i / 2], make_float2(inv, inv)));
                        u[i] = r.x;
                        u[i + 1] = r.y;
                    }
                }
                const float * tr = turn + k * 3 * row;
                if (what == 2) {
                } else if (PAIR == NEXT) {
                    const int j = at >> 1;   // the lane's four pairs
                    if (j < P) {
                        const float4 c = *(const float4 *) (tr + j), s = *(const float4 *) (tr + row + j);
                        const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (j + i < P) {
                                const float v = u[2 * i];
                                u[2 * i] = v * cs[i] - u[2 * i + 1] * sn[i];
                                u[2 * i + 1] = v * sn[i] + u[2 * i + 1] * cs[i];
                            }
                    }
                } else if (PAIR == LANES) {
                    float m[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) m[i] = __shfl_sync(0xffffffffu, u[i], other);
                    if (turned) {
                        const float * t = tr + (low ? at : at - P);
                        const float * sines = t + (low ? 2 * row : row);
#pragma unroll
                        for (int i = 0; i < 8; i += 4) {
                            const float4 c = *(const float4 *) (t + i), s = *(const float4 *) (sines + i);
                            const float2 a0 = fma2(make_float2(m[i], m[i + 1]), make_float2(s.x, s.y), mul2(make_float2(u[i], u[i + 1]), make_float2(c.x, c.y)));
                            const float2 a1 = fma2(make_float2(m[i + 2], m[i + 3]), make_float2(s.z, s.w), mul2(make_float2(u[i + 2], u[i + 3]), make_float2(c.z, c.w)));
                            u[i] = a0.x;
                            u[i + 1] = a0.y;
                            u[i + 2] = a1.x;
                            u[i + 3] = a1.y;
                        }
                    }
                } else {
                    float * m = mate[warp];
#pragma unroll
                    for (int i = 0; i < 8; ++i) m[lane * 9 + i] = u[i];
                    __syncwarp();
                    const int base = lane & ~(LPH - 1);   // the head's first lane
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int e = at + i;
                        if (e < 2 * P) {
                            const int o = e < P ? e + P : e - P, j = e < P ? e : e - P;
                            u[i] = fmaf(m[(base + (o >> 3)) * 9 + (o & 7)], tr[(e < P ? 2 * row : row) + j], u[i] * tr[j]);
                        }
                    }
                    __syncwarp();
                }
                T * const dst = target(k);
                if (mine && dst) store_words<T, 8>(dst, u);
            }
        if (chunk + WARPS < until) {
            chunk += WARPS;
            begin();
            chunk -= WARPS;
        }
    }
}

// The mean key of every page that a new token went into: the work of the token that is the page's last, a warp a head. Sums are
// f32, over the keys in the order of lanes, then of the lanes.
template <class T, int LPH>
__global__ void __launch_bounds__(32 * WARPS) cache_means_kernel(const __grid_constant__ Append n) {
    constexpr int SIDE = 32 / LPH, AHEAD = 8;   // keys of a step, steps whose loads run at once
    pdl_wait();
    const tsn_cache_append_args & a = n.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = (int) a.c.D, Hk = (int) a.c.Hk;
    const int sub = lane / LPH, at = (lane & (LPH - 1)) * 8;
    const bool mine = at < D;
    // a lane a token: whether it is its page's last, that page and the slot
    const long long s0 = (long long) blockIdx.x * n.tok;
    int id_of = -1, slot_of = 0;
    if (lane < n.tok && s0 + lane < a.c.N) {
        const int i = (int) s0 + lane, b = seq_of_row_alone(a.c, i);
        if (b >= 0) {
            const int pl = place_of_row(a.c, b, i);
            slot_of = pl & ((1 << n.page_log2) - 1);
            if (slot_of + 1 == (1 << n.page_log2) || i + 1 == seq_start(a.c, b + 1)) id_of = page_of(a.c, b, pl >> n.page_log2);
        }
    }
    for (uint32_t left = __ballot_sync(~0u, id_of >= 0); left; left &= left - 1) {
        const int from = __ffs(left) - 1, id = __shfl_sync(~0u, id_of, from), slot = __shfl_sync(~0u, slot_of, from);
        for (int h = warp; h < Hk; h += WARPS) {
            const T * key = (const T *) a.c.k.p + id * a.c.k.sb + h * a.c.k.sh + at;
            float sum[8] = {};
            for (int t = sub; t <= slot; t += SIDE * AHEAD) {
                Words<T, 8> r[AHEAD];
#pragma unroll
                for (int y = 0; y < AHEAD; ++y)
                    if (mine && t + y * SIDE <= slot) r[y] = load_words<T, 8>(key + (t + y * SIDE) * a.c.k.ss);
#pragma unroll
                for (int y = 0; y < AHEAD; ++y)
                    if (mine && t + y * SIDE <= slot) {
                        float u[8];
                        to_floats<T, 8>(r[y], u);
#pragma unroll
                        for (int e = 0; e < 8; ++e) sum[e] += u[e];
                    }
            }
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
#pragma unroll
                for (int o = LPH; o < 32; o <<= 1) sum[e] += __shfl_xor_sync(~0u, sum[e], o);
                sum[e] /= (float) (slot + 1);
            }
            if (mine && sub == 0) store_words<T, 8>((T *) a.means.p + id * a.means.sb + h * a.means.st + at, sum);
        }
    }
}

template <class TX, class T>
cudaError_t launch(const tsn_rope_plan_t & p, Append & n, cudaStream_t s) {
    const tsn_cache_append_args & a = n.a;
    int lph = 1;
    while (lph * 8 < (int) p.D) lph *= 2;
    const int side = 32 / lph, chunks = (int) ((a.Hq + side - 1) / side + 2 * ((a.c.Hk + side - 1) / side));
    const long long turns = (chunks + WARPS - 1) / WARPS;
    // Tokens of a block share its start; fewer while four blocks per SM take them all, and with few tokens their heads go to several.
    n.span = (long long) a.c.N * turns <= 8 * 148 ? WARPS : chunks;
    n.tok = (int) std::min<long long>(MAX_TOK, ((long long) a.c.N * (n.span == WARPS ? turns : 1) + 4 * 148 - 1) / (4 * 148));
    const dim3 blocks((a.c.N + n.tok - 1) / n.tok, (unsigned) ((chunks + n.span - 1) / n.span));
    const int pair = p.layout == TSN_ROPE_INTERLEAVED ? NEXT : p.P % 8 == 0 ? LANES : SHARED;
    const int mean_tok = (int) std::max(1u, std::min(32u, a.c.N / 1024));
    cudaError_t e = cudaSuccess;
    auto go = [&](auto L) {
        constexpr int LPH = decltype(L)::value;
        if (pair == NEXT) e = launch_cl(cache_append_kernel<TX, T, LPH, NEXT>, blocks, dim3(32 * WARPS), 0, s, dim3(1), p, n);
        else if (pair == LANES) e = launch_cl(cache_append_kernel<TX, T, LPH, LANES>, blocks, dim3(32 * WARPS), 0, s, dim3(1), p, n);
        else e = launch_cl(cache_append_kernel<TX, T, LPH, SHARED>, blocks, dim3(32 * WARPS), 0, s, dim3(1), p, n);
        if (e != cudaSuccess || !a.means.p) return;
        n.tok = mean_tok;
        e = launch_cl(cache_means_kernel<T, LPH>, dim3((a.c.N + mean_tok - 1) / mean_tok), dim3(32 * WARPS), 0, s, dim3(1), n);
    };
    if (lph == 1) go(std::integral_constant<int, 1>());
    else if (lph == 2) go(std::integral_constant<int, 2>());
    else if (lph == 4) go(std::integral_constant<int, 4>());
    else if (lph == 8) go(std::integral_constant<int, 8>());
    else if (lph == 16) go(std::integral_constant<int, 16>());
    else go(std::integral_constant<int, 32>());
    if (e != cudaSuccess) cudaGetLastError();
    return e;
}

} // namespace

int cache_append(DeviceCtx & c, const tsn_rope_plan_t & p, const tsn_cache_append_args & a) {
    if (a.c.N == 0 || a.c.B == 0) return TSN_OK;
    Append n{a, log2_of(a.c.page), 1, 1};
    if (!n.a.q.p) n.a.Hq = 0;
    const bool wide = a.xtype == TSN_F32;
    const cudaError_t e = a.c.type == TSN_F16 ? (wide ? launch<float, __half>(p, n, c.stream) : launch<__half, __half>(p, n, c.stream))
                                              : (wide ? launch<float, __nv_bfloat16>(p, n, c.stream) : launch<__nv_bfloat16, __nv_bfloat16>(p, n, c.stream));
    if (e != cudaSuccess) return fail(TSN_ERR_CUDA, std::string("tsn_cache_append: ") + cudaGetErrorString(e));
    return TSN_OK;
}

} // namespace tsn

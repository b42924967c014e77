// rope_axes.cu — rotary positions with several axes after an optional RMSNorm of each head (tsn_rope_axes).
//
// Pair j of a head turns by pos[axis j] * turn[j] turns, turn[j] a 64-bit fraction of a turn per position:
// the product of the two wraps at whole turns in 64-bit integer arithmetic, so the angle is as exact at
// position 10^6 as at 0 (a 32-bit product of position and frequency is off by 10^6 * 2^-24 rad there).
// Bound by HBM: every head is read and written once. A block takes a few whole tokens: it computes the tokens'
// cosines and sines once for all their heads into shared memory (in 64-bit phases and sincospi, which
// would cost more than the memory traffic if each head did it), then its warps run over the heads, 8 elements a
// lane, with several heads of a token side by side in a warp and their RMSNorm by shuffles.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "block_ops.h"
#include "kernels.h"

namespace tsn {

namespace {

// pos * turn modulo one turn, in [-1/2, 1/2) turns
__device__ __forceinline__ float phase(int pos, uint64_t turn) {
    const uint64_t p = (uint64_t) (long long) pos * turn;
    return (float) (int) (p >> 32) * 0x1p-32f;
}

// The address of a head row: heads 0 .. Hq - 1 are the queries', the following the keys'.
template <class T>
struct Row {
    const T * x;
    T * y;
};
template <class T>
__device__ __forceinline__ Row<T> row_of(const tsn_rope_args & a, int Hq, long long b, long long s, int head) {
    const bool is_q = head < Hq;
    const tsn_heads & i = is_q ? a.q : a.k, & o = is_q ? a.q_out : a.k_out;
    const int h = is_q ? head : head - Hq;
    return {(const T *) i.p + b * i.sb + s * i.ss + h * i.sh, (T *) o.p + b * o.sb + s * o.ss + h * o.sh};
}

__device__ __forceinline__ float2 turn_of(const tsn_rope_plan_t & p, const tsn_rope_args & a, long long b, long long s, int j) {
    float sn, cs;
    sincospif(2.0f * phase(a.pos[b * a.pos_sb + s * a.pos_ss + p.axis[j]], p.turn[j]), &sn, &cs);
    return make_float2(cs, sn);
}

constexpr int WARPS = 8, MAX_TOK = 8;

// How a lane finds the other element of its pairs.
enum { NEXT, LANES, SHARED };   // interleaved: its own; halves: another lane's (P a multiple of 8), or shared memory

// Heads whose rows start at 16-byte boundaries, D a multiple of 8. LPH: lanes of a head, the power of two from
// D / 8 up. Block (x, b, z): tokens x * tok .. of sequence b, chunks 8 z .. of 32 / LPH heads. A warp takes one chunk,
// queries' or keys', through the block's tokens, so that a token costs its lanes a load, a store and the
// arithmetic; with fewer chunks than warps, several warps share a chunk's tokens.
// Loads run one round ahead of the arithmetic: 32 500 tokens x 64 heads of 64, bf16, written head-major, take 101 us
// (5.2 TB/s, 0.80 of the measured copy) with two tokens a round at four blocks per SM; 110 with one, 108 with four at
// fewer blocks, 113 without the round ahead. With 16 tokens a block 104, with 32 113. (With other inputs from call to call
// 108.) Four blocks leave a thread 64 registers: the 16-bit forms spill 8 to 44 bytes, with SHARED up to 124.
template <class T, int LPH, int PAIR>
__global__ void __launch_bounds__(32 * WARPS, 4) rope_rows8(const __grid_constant__ tsn_rope_plan_t p, const __grid_constant__ tsn_rope_args a, int tok) {
    constexpr int SIDE = 32 / LPH, AHEAD = sizeof(T) == 4 ? 1 : 2;   // tokens of a round: 16 or 32 bytes a lane each
    __shared__ __align__(16) float2 turn[MAX_TOK * TSN_ROPE_MAX_PAIRS + 8];
    __shared__ float mate[PAIR == SHARED ? WARPS : 1][32 * 9];   // a lane's 8 elements, one word of padding between lanes
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int D = (int) p.D, P = (int) p.P, Hq = a.q.p ? (int) a.Hq : 0, Hk = a.k.p ? (int) a.Hk : 0;
    const long long b = blockIdx.y, s0 = (long long) blockIdx.x * tok;
    const int n = (int) min((long long) tok, a.S - s0);
    const int sub = lane / LPH, at = (lane & (LPH - 1)) * 8;
    const int q_chunks = (Hq + SIDE - 1) / SIDE, chunks = q_chunks + (Hk + SIDE - 1) / SIDE;
    const int sharing = chunks < WARPS ? WARPS / chunks : 1;   // warps of a chunk
    const float inv_D = 1.0f / (float) D;
    const int row = (P + 1) & ~1;   // a token's pairs in the table, from a 16-byte boundary on

    const int chunk = sharing > 1 ? (warp < sharing * chunks ? warp % chunks : chunks) : (int) blockIdx.z * WARPS + warp;
    const bool is_q = chunk < q_chunks;
    const tsn_heads & hi = is_q ? a.q : a.k, & ho = is_q ? a.q_out : a.k_out;
    const float * wp = is_q ? a.q_norm : a.k_norm;
    const int head = (is_q ? chunk : chunk - q_chunks) * SIDE + sub, from = sharing > 1 ? warp / chunks : 0;
    const bool mine = chunk < chunks && at < D && head < (is_q ? Hq : Hk);
    const T * x = (const T *) hi.p + b * hi.sb + (s0 + from) * hi.ss + head * hi.sh + at;
    T * y = (T *) ho.p + b * ho.sb + (s0 + from) * ho.ss + head * ho.sh + at;
    const long long dx = sharing * hi.ss, dy = sharing * ho.ss;
    Words<T, 8> raw[AHEAD], next[AHEAD];
    auto fetch = [&](int k0) {
#pragma unroll
        for (int c = 0; c < AHEAD; ++c)
            if (mine && k0 + c * sharing < n) next[c] = load_words<T, 8>(x + c * dx);
        x += AHEAD * dx;
    };
    fetch(from);   // before the table: the loads are on their way
    float2 w[4];
    if (wp)
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = mine ? make_float2(wp[at + 2 * i], wp[at + 2 * i + 1]) : make_float2(0.0f, 0.0f);
    for (int i = threadIdx.x; i < n * P; i += 32 * WARPS) turn[i / P * row + i % P] = turn_of(p, a, b, s0 + i / P, i % P);
    __syncthreads();
    if (chunk >= chunks) return;

    for (int k0 = from; k0 < n; k0 += AHEAD * sharing) {
#pragma unroll
        for (int c = 0; c < AHEAD; ++c) raw[c] = next[c];
        fetch(k0 + AHEAD * sharing);
#pragma unroll
        for (int c = 0; c < AHEAD; ++c) {
            const int k = k0 + c * sharing;
            if (k >= n) break;
            float u[8];
            to_floats<T, 8>(raw[c], u);
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
            const float2 * tr = turn + k * row;
            if (PAIR == NEXT) {
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const int j = (at + i) >> 1;
                    const float4 cs = *(const float4 *) (tr + (j < row ? j : 0));
                    const float2 v = make_float2(u[i], u[i + 2]);
                    if (j < P) {
                        u[i] = v.x * cs.x - u[i + 1] * cs.y;
                        u[i + 1] = v.x * cs.y + u[i + 1] * cs.x;
                    }
                    if (j + 1 < P) {
                        u[i + 2] = v.y * cs.z - u[i + 3] * cs.w;
                        u[i + 3] = v.y * cs.w + u[i + 3] * cs.z;
                    }
                }
            } else if (PAIR == LANES) {
                const bool low = at < P, turned = at < 2 * P;
                const int other = turned ? (low ? lane + P / 8 : lane - P / 8) : lane;
                const float4 * cs = (const float4 *) (tr + (turned ? (low ? at : at - P) : 0));
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float4 c2 = cs[i / 2];
                    const float m0 = __shfl_sync(0xffffffffu, u[i], other), m1 = __shfl_sync(0xffffffffu, u[i + 1], other);
                    if (turned) {
                        u[i] = fmaf(u[i], c2.x, low ? -m0 * c2.y : m0 * c2.y);
                        u[i + 1] = fmaf(u[i + 1], c2.z, low ? -m1 * c2.w : m1 * c2.w);
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
                        const int o = e < P ? e + P : e - P;
                        const float v = m[(base + (o >> 3)) * 9 + (o & 7)];
                        const float2 cs = tr[e < P ? e : e - P];
                        u[i] = fmaf(u[i], cs.x, e < P ? -v * cs.y : v * cs.y);
                    }
                }
                __syncwarp();
            }
            if (mine) store_words<T, 8>(y + c * dy, u);
        }
        y += AHEAD * dy;
    }
}

// Any D, strides and alignment: one warp per head row.
template <class T>
__global__ void __launch_bounds__(32 * WARPS) rope_rows1(const __grid_constant__ tsn_rope_plan_t p, const __grid_constant__ tsn_rope_args a) {
    __shared__ float buf[WARPS][2 * TSN_ROPE_MAX_PAIRS];
    pdl_wait();
    const int lane = threadIdx.x & 31, D = (int) p.D, P = (int) p.P, Hq = a.q.p ? (int) a.Hq : 0, H = Hq + (a.k.p ? (int) a.Hk : 0);
    const long long item = (long long) blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (item >= (long long) a.B * a.S * H) return;
    const int head = (int) (item % H);
    const long long t = item / H, b = t / a.S, s = t % a.S;
    const Row<T> r = row_of<T>(a, Hq, b, s, head);
    const float * w = head < Hq ? a.q_norm : a.k_norm;
    float * u = buf[threadIdx.x >> 5];
    float ss = 0.0f;
    for (int e = lane; e < D; e += 32) {
        const float v = to_f32(r.x[e]);
        u[e] = v;
        ss = fmaf(v, v, ss);
    }
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    __syncwarp();
    const float inv = rsqrtf(ss / (float) D + a.eps);
    auto normed = [&](int e) { return w ? u[e] * (inv * w[e]) : u[e]; };
    for (int j = lane; j < P; j += 32) {
        const float2 cs = turn_of(p, a, b, s, j);
        const int e0 = p.layout == TSN_ROPE_HALF ? j : 2 * j, e1 = p.layout == TSN_ROPE_HALF ? j + P : 2 * j + 1;
        const float p0 = normed(e0), p1 = normed(e1);
        r.y[e0] = from_f32<T>(p0 * cs.x - p1 * cs.y);
        r.y[e1] = from_f32<T>(p0 * cs.y + p1 * cs.x);
    }
    for (int e = 2 * P + lane; e < D; e += 32) r.y[e] = from_f32<T>(normed(e));
}

template <class T>
cudaError_t launch(const tsn_rope_plan_t & p, const tsn_rope_args & a, cudaStream_t s) {
    auto rows16 = [&](const tsn_heads & h, uint32_t H) {
        return !h.p || !H || ((((uintptr_t) h.p) | (uintptr_t) (a.B > 1 ? h.sb : 0) * sizeof(T) | (uintptr_t) (a.S > 1 ? h.ss : 0) * sizeof(T) |
                               (uintptr_t) (H > 1 ? h.sh : 0) * sizeof(T)) & 15) == 0;
    };
    const long long tokens = (long long) a.B * a.S;
    const int H = (int) ((a.q.p ? a.Hq : 0) + (a.k.p ? a.Hk : 0));
    cudaError_t e = cudaSuccess;
    if (p.D % 8 == 0 && a.B <= 65535 && rows16(a.q, a.Hq) && rows16(a.k, a.Hk) && (!a.q.p || rows16(a.q_out, a.Hq)) && (!a.k.p || rows16(a.k_out, a.Hk))) {
        int lph = 1;
        while (lph * 8 < (int) p.D) lph *= 2;
        // Tokens of a block: 8 share its start; fewer while four blocks per SM take them all (not a few more, which would
        // be a second wave).
        const int side = 32 / lph, chunks = (int) ((a.q.p ? a.Hq : 0) + side - 1) / side + (int) ((a.k.p ? a.Hk : 0) + side - 1) / side;
        const long long turns = (chunks + WARPS - 1) / WARPS;
        const int tok = (int) std::min<long long>(MAX_TOK, (tokens * turns + 4 * 148 - 1) / (4 * 148));
        const dim3 blocks((a.S + tok - 1) / tok, a.B, (unsigned) turns);
        const int pair = p.layout == TSN_ROPE_INTERLEAVED ? NEXT : p.P % 8 == 0 ? LANES : SHARED;
        auto go = [&](auto L) {
            constexpr int LPH = decltype(L)::value;
            if (pair == NEXT) e = launch_cl(rope_rows8<T, LPH, NEXT>, blocks, dim3(32 * WARPS), 0, s, dim3(1), p, a, tok);
            else if (pair == LANES) e = launch_cl(rope_rows8<T, LPH, LANES>, blocks, dim3(32 * WARPS), 0, s, dim3(1), p, a, tok);
            else e = launch_cl(rope_rows8<T, LPH, SHARED>, blocks, dim3(32 * WARPS), 0, s, dim3(1), p, a, tok);
        };
        if (lph == 1) go(std::integral_constant<int, 1>());
        else if (lph == 2) go(std::integral_constant<int, 2>());
        else if (lph == 4) go(std::integral_constant<int, 4>());
        else if (lph == 8) go(std::integral_constant<int, 8>());
        else if (lph == 16) go(std::integral_constant<int, 16>());
        else go(std::integral_constant<int, 32>());
    } else {
        e = launch_cl(rope_rows1<T>, dim3((unsigned) ((tokens * H + WARPS - 1) / WARPS)), dim3(32 * WARPS), 0, s, dim3(1), p, a);
    }
    if (e != cudaSuccess) cudaGetLastError();
    return e;
}

} // namespace

int rope_plan(uint32_t D, uint32_t axes, const uint32_t * pairs, const double * theta, const double * scale, int layout,
              tsn_rope_plan_t * out) {
    if (!pairs || !theta || !scale || !out) return fail(TSN_ERR_ARG, "tsn_rope_plan: null argument");
    if (D < 2 || D > 2 * TSN_ROPE_MAX_PAIRS || D % 2) return fail(TSN_ERR_ARG, "tsn_rope_plan: D must be even, 2..256");
    if (axes < 1 || axes > TSN_ROPE_MAX_AXES) return fail(TSN_ERR_ARG, "tsn_rope_plan: 1 to 4 axes");
    if (layout != TSN_ROPE_INTERLEAVED && layout != TSN_ROPE_HALF) return fail(TSN_ERR_ARG, "tsn_rope_plan: unknown layout");
    tsn_rope_plan_t p{};
    p.D = D; p.axes = axes; p.layout = layout;
    for (uint32_t x = 0; x < axes; ++x) {
        if (!(theta[x] > 0.0) || !std::isfinite(theta[x]) || !std::isfinite(scale[x]))
            return fail(TSN_ERR_ARG, "tsn_rope_plan: theta must be positive and scale finite");
        if (pairs[x] > D / 2 || p.P + pairs[x] > D / 2) return fail(TSN_ERR_ARG, "tsn_rope_plan: more pairs than D / 2");
        for (uint32_t i = 0; i < pairs[x]; ++i, ++p.P) {
            const double turns = scale[x] * std::pow(theta[x], -(double) i / pairs[x]) / (2.0 * 3.14159265358979323846);
            if (!std::isfinite(turns)) return fail(TSN_ERR_ARG, "tsn_rope_plan: theta and scale give turns that are not finite");
            const double part = turns - std::floor(turns);   // whole turns per position turn nothing
            p.turn[p.P] = part >= 1.0 ? 0 : (uint64_t) std::ldexp(part, 64);
            p.axis[p.P] = (uint8_t) x;
        }
    }
    *out = p;
    return TSN_OK;
}

int rope_axes(DeviceCtx & c, const tsn_rope_plan_t & p, const tsn_rope_args & a) {
    if (!known_type(a.type)) return fail(TSN_ERR_ARG, "tsn_rope_axes: unknown type");
    if (p.D < 2 || p.D > 2 * TSN_ROPE_MAX_PAIRS || p.D % 2 || p.P > p.D / 2 || p.axes < 1 || p.axes > TSN_ROPE_MAX_AXES)
        return fail(TSN_ERR_ARG, "tsn_rope_axes: not a plan of tsn_rope_plan");
    for (uint32_t j = 0; j < p.P; ++j)
        if (p.axis[j] >= p.axes) return fail(TSN_ERR_ARG, "tsn_rope_axes: not a plan of tsn_rope_plan");
    const long long heads = (a.q.p ? (long long) a.Hq : 0) + (a.k.p ? (long long) a.Hk : 0);
    const long long tokens = (long long) a.B * a.S;
    if (tokens == 0 || heads == 0) return TSN_OK;
    if (heads > 65536 || tokens > 0x7fffffffLL || tokens > (0x7fffffffLL * WARPS) / heads) return fail(TSN_ERR_ARG, "tsn_rope_axes: too many rows");
    if ((a.q.p && a.Hq && !a.q_out.p) || (a.k.p && a.Hk && !a.k_out.p) || (p.P && !a.pos))
        return fail(TSN_ERR_ARG, "tsn_rope_axes: null result or positions");
    auto distinct = [&](const tsn_heads & o, uint32_t H) {
        return (a.B == 1 || o.sb) && (a.S == 1 || o.ss) && (H == 1 || o.sh);
    };
    if ((a.q.p && a.Hq && !distinct(a.q_out, a.Hq)) || (a.k.p && a.Hk && !distinct(a.k_out, a.Hk)))
        return fail(TSN_ERR_ARG, "tsn_rope_axes: a result with a stride of 0");
    const uintptr_t addresses = (uintptr_t) a.q.p | (uintptr_t) a.k.p | (uintptr_t) (a.q.p ? a.q_out.p : nullptr) | (uintptr_t) (a.k.p ? a.k_out.p : nullptr);
    if ((addresses & (type_size(a.type) - 1)) || (((uintptr_t) a.pos | (uintptr_t) a.q_norm | (uintptr_t) a.k_norm) & 3))
        return fail(TSN_ERR_ARG, "tsn_rope_axes: an address that is no multiple of its element's size");
    cudaError_t e = a.type == TSN_F32   ? launch<float>(p, a, c.stream)
                    : a.type == TSN_F16 ? launch<__half>(p, a, c.stream)
                                        : launch<__nv_bfloat16>(p, a, c.stream);
    if (e != cudaSuccess) return fail(TSN_ERR_CUDA, std::string("tsn_rope_axes: ") + cudaGetErrorString(e));
    return TSN_OK;
}

} // namespace tsn

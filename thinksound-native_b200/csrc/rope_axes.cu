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

#include "block_ops.h"

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

constexpr int WARPS = 8, MAX_TOK = 4;

// Heads whose rows start at 16-byte boundaries, D a multiple of 8. lph: lanes of a head, the power of two from
// D / 8 up; tok: tokens of a block. A warp's item is a chunk of 32 / lph heads of one token, queries' or keys'.
template <class T, bool HALF>
__global__ void __launch_bounds__(32 * WARPS) rope_rows8(const __grid_constant__ tsn_rope_plan_t p, const __grid_constant__ tsn_rope_args a,
                                                         int lph, int tok) {
    __shared__ float2 turn[MAX_TOK * TSN_ROPE_MAX_PAIRS];
    __shared__ __align__(16) float weight[2][2 * TSN_ROPE_MAX_PAIRS];
    __shared__ T * start[MAX_TOK][4];                  // a token's first head: q, k, q_out, k_out
    __shared__ float mate[HALF ? WARPS : 1][32 * 9];   // a lane's 8 elements, one word of padding between lanes
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int D = (int) p.D, P = (int) p.P, Hq = a.q.p ? (int) a.Hq : 0, Hk = a.k.p ? (int) a.Hk : 0;
    const unsigned first = blockIdx.x * (unsigned) tok;
    const int n = (int) min((unsigned) tok, a.B * a.S - first);
    const int side = 32 / lph, sub = lane / lph, at = (lane & (lph - 1)) * 8;
    const int q_chunks = (Hq + side - 1) / side, chunks = q_chunks + (Hk + side - 1) / side;
    const bool in = at < D;
    const float inv_D = 1.0f / (float) D;

    if (threadIdx.x < 4 * n) {
        const unsigned t = first + (threadIdx.x >> 2), b = t / a.S, s = t % a.S;
        const tsn_heads & h = (threadIdx.x & 3) == 0 ? a.q : (threadIdx.x & 3) == 1 ? a.k : (threadIdx.x & 3) == 2 ? a.q_out : a.k_out;
        start[threadIdx.x >> 2][threadIdx.x & 3] = (T *) h.p + b * h.sb + s * h.ss;
    }
    for (int i = threadIdx.x; i < n * P; i += 32 * WARPS) {
        const unsigned t = first + i / P;
        turn[i] = turn_of(p, a, t / a.S, t % a.S, i % P);
    }
    for (int i = threadIdx.x; i < D; i += 32 * WARPS) {
        weight[0][i] = a.q_norm ? a.q_norm[i] : 1.0f;
        weight[1][i] = a.k_norm ? a.k_norm[i] : 1.0f;
    }
    __syncthreads();

    int k = warp / chunks, chunk = warp % chunks;
    Words<T, 8> x;
    T * y = nullptr;
    auto fetch = [&]() {
        y = nullptr;
        if (k >= n) return;
        const bool is_q = chunk < q_chunks;
        const int head = (is_q ? chunk : chunk - q_chunks) * side + sub;
        if (!in || head >= (is_q ? Hq : Hk)) return;
        x = load_words<T, 8>(start[k][is_q ? 0 : 1] + head * (is_q ? a.q.sh : a.k.sh) + at);
        y = start[k][is_q ? 2 : 3] + head * (is_q ? a.q_out.sh : a.k_out.sh) + at;
    };
    fetch();
    while (k < n) {
        const float2 * tr = turn + k * P;
        const bool is_q = chunk < q_chunks;
        T * const to = y;
        float u[8];
        if (to) {
            to_floats<T, 8>(x, u);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = 0.0f;
        }
        for (chunk += WARPS; chunk >= chunks; chunk -= chunks) ++k;
        fetch();   // the next item's heads, while this one is turned
        if (is_q ? a.q_norm != nullptr : a.k_norm != nullptr) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(u[i], u[i], ss);
            for (int o = lph >> 1; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float inv = rsqrtf(fmaf(ss, inv_D, a.eps));
            const float4 * w = (const float4 *) (weight[is_q ? 0 : 1] + (in ? at : 0));
            const float4 w0 = w[0], w1 = w[1];
            u[0] *= inv * w0.x; u[1] *= inv * w0.y; u[2] *= inv * w0.z; u[3] *= inv * w0.w;
            u[4] *= inv * w1.x; u[5] *= inv * w1.y; u[6] *= inv * w1.z; u[7] *= inv * w1.w;
        }
        if (HALF) {
            float * m = mate[warp];
#pragma unroll
            for (int i = 0; i < 8; ++i) m[lane * 9 + i] = u[i];
            __syncwarp();
            const int base = lane - (lane & (lph - 1));   // the head's first lane
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = at + i;
                if (e < 2 * P && in) {
                    const int o = e < P ? e + P : e - P;
                    const float w = m[(base + (o >> 3)) * 9 + (o & 7)];
                    const float2 cs = tr[e < P ? e : e - P];
                    u[i] = fmaf(u[i], cs.x, e < P ? -w * cs.y : w * cs.y);
                }
            }
            __syncwarp();
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const int j = (at + i) >> 1;
                if (j < P) {
                    const float2 cs = tr[j];
                    const float v = u[i];
                    u[i] = v * cs.x - u[i + 1] * cs.y;
                    u[i + 1] = v * cs.y + u[i + 1] * cs.x;
                }
            }
        }
        if (to) store_words<T, 8>(to, u);
    }
}

// Any D, strides and alignment: one warp per head row.
template <class T>
__global__ void __launch_bounds__(32 * WARPS) rope_rows1(const __grid_constant__ tsn_rope_plan_t p, const __grid_constant__ tsn_rope_args a) {
    __shared__ float buf[WARPS][2 * TSN_ROPE_MAX_PAIRS];
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
    if (p.D % 8 == 0 && rows16(a.q, a.Hq) && rows16(a.k, a.Hk) && (!a.q.p || rows16(a.q_out, a.Hq)) && (!a.k.p || rows16(a.k_out, a.Hk))) {
        int lph = 1;
        while (lph * 8 < (int) p.D) lph *= 2;
        // Tokens of a block: as many as give each warp eight rounds, fewer while blocks do not fill the SMs.
        const int chunks = std::max(1, H / (32 / lph));
        int tok = std::min(MAX_TOK, std::max(1, 8 * WARPS / chunks));
        tok = (int) std::min<long long>(tok, std::max(1ll, tokens / (4 * 148)));
        const unsigned blocks = (unsigned) ((tokens + tok - 1) / tok);
        if (p.layout == TSN_ROPE_HALF) rope_rows8<T, true><<<blocks, 32 * WARPS, 0, s>>>(p, a, lph, tok);
        else rope_rows8<T, false><<<blocks, 32 * WARPS, 0, s>>>(p, a, lph, tok);
    } else {
        rope_rows1<T><<<(unsigned) ((tokens * H + WARPS - 1) / WARPS), 32 * WARPS, 0, s>>>(p, a);
    }
    return cudaGetLastError();
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
    if (p.D < 2 || p.D > 2 * TSN_ROPE_MAX_PAIRS || p.D % 2 || 2 * p.P > p.D || p.axes < 1 || p.axes > TSN_ROPE_MAX_AXES)
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

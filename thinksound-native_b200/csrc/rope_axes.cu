// rope_axes.cu — rotary positions with several axes after an optional RMSNorm of each head (tsn_rope_axes).
//
// Pair j of a head turns by pos[axis j] * turn[j] turns, turn[j] a 64-bit fraction of a turn per position:
// the product of the two wraps at whole turns in 64-bit integer arithmetic, so the angle is as exact at
// position 10^6 as at 0 (a 32-bit product of position and frequency is off by 10^6 * 2^-24 rad there).
// One warp per head row.
#include <cmath>

#include "block_ops.h"

namespace tsn {

namespace {

// pos * turn modulo one turn, in [-1/2, 1/2) turns
__device__ __forceinline__ float phase(int pos, uint64_t turn) {
    const uint64_t p = (uint64_t) (long long) pos * turn;
    return (float) (int) (p >> 32) * 0x1p-32f;
}

template <class T>
__global__ void rope_kernel(const __grid_constant__ tsn_rope_plan_t p, const __grid_constant__ tsn_rope_args a) {
    const int lane = threadIdx.x & 31, D = (int) p.D, P = (int) p.P, Hq = a.q.p ? (int) a.Hq : 0, Hk = a.k.p ? (int) a.Hk : 0;
    const long long rows = (long long) a.B * a.S * (Hq + Hk);
    const long long row = (long long) blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int head = (int) (row % (Hq + Hk));
    const long long tok = row / (Hq + Hk), b = tok / a.S, s = tok % a.S;
    const bool is_q = head < Hq;
    const tsn_heads & hi = is_q ? a.q : a.k, & ho = is_q ? a.q_out : a.k_out;
    const int h = is_q ? head : head - Hq;
    const T * x = (const T *) hi.p + b * hi.sb + s * hi.ss + h * hi.sh;
    T * y = (T *) ho.p + b * ho.sb + s * ho.ss + h * ho.sh;
    const float * w = is_q ? a.q_norm : a.k_norm;
    float v[8];   // element 2 i or 2 i + 1 of this lane's pairs of neighbours: e = 64 * i + 2 * lane
    float ss = 0.0f;
    for (int i = 0; i < 4; ++i)
        for (int k = 0; k < 2; ++k) {
            const int e = 64 * i + 2 * lane + k;
            v[2 * i + k] = e < D ? to_f32(x[e]) : 0.0f;
            ss += v[2 * i + k] * v[2 * i + k];
        }
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = w ? rsqrtf(ss / (float) D + a.eps) : 1.0f;
    __shared__ float buf[8][256];
    float * u = buf[threadIdx.x >> 5];
    for (int i = 0; i < 4; ++i)
        for (int k = 0; k < 2; ++k) {
            const int e = 64 * i + 2 * lane + k;
            if (e < D) u[e] = w ? v[2 * i + k] * inv * w[e] : v[2 * i + k];
        }
    __syncwarp();
    const int32_t * pos = a.pos + b * a.pos_sb + s * a.pos_ss;
    for (int j = lane; j < P; j += 32) {
        float sn, cs;
        sincospif(2.0f * phase(pos[p.axis[j]], p.turn[j]), &sn, &cs);
        const int e0 = p.layout == TSN_ROPE_HALF ? j : 2 * j, e1 = p.layout == TSN_ROPE_HALF ? j + P : 2 * j + 1;
        const float p0 = u[e0], p1 = u[e1];
        y[e0] = from_f32<T>(p0 * cs - p1 * sn);
        y[e1] = from_f32<T>(p0 * sn + p1 * cs);
    }
    for (int e = 2 * P + lane; e < D; e += 32) y[e] = from_f32<T>(u[e]);
}

template <class T>
cudaError_t launch(const tsn_rope_plan_t & p, const tsn_rope_args & a, long long rows, cudaStream_t s) {
    rope_kernel<T><<<(unsigned) ((rows + 7) / 8), 256, 0, s>>>(p, a);
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
    if (heads > 65536 || tokens > (0x7fffffffLL * 8) / heads) return fail(TSN_ERR_ARG, "tsn_rope_axes: too many rows");
    if ((a.q.p && a.Hq && !a.q_out.p) || (a.k.p && a.Hk && !a.k_out.p) || (p.P && !a.pos))
        return fail(TSN_ERR_ARG, "tsn_rope_axes: null result or positions");
    auto distinct = [&](const tsn_heads & o, uint32_t H) {
        return (a.B == 1 || o.sb) && (a.S == 1 || o.ss) && (H == 1 || o.sh);
    };
    if ((a.q.p && a.Hq && !distinct(a.q_out, a.Hq)) || (a.k.p && a.Hk && !distinct(a.k_out, a.Hk)))
        return fail(TSN_ERR_ARG, "tsn_rope_axes: a result with a stride of 0");
    const long long rows = tokens * heads;
    cudaError_t e = a.type == TSN_F32   ? launch<float>(p, a, rows, c.stream)
                    : a.type == TSN_F16 ? launch<__half>(p, a, rows, c.stream)
                                        : launch<__nv_bfloat16>(p, a, rows, c.stream);
    if (e != cudaSuccess) return fail(TSN_ERR_CUDA, std::string("tsn_rope_axes: ") + cudaGetErrorString(e));
    return TSN_OK;
}

} // namespace tsn

// block_norm.cu — norms before and after a block, fused with gate and residual scale (tsn_block_norm).
//
// Per row of C elements: x' = r x + act(g) Npost(y), h = Npre(x') (1 + scale) + shift. The row is read
// once and stays on chip between the norms, so DRAM sees x, y and the modulation once, x' and h once.
// One CTA per row; the row's f32 values live in shared memory.
#include "block_ops.h"

namespace tsn {

namespace {

struct NormArgs {
    tsn_block_norm_args a;
    long long rows;
};

__device__ float block_sum(float v, float * red) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
    for (int w = 0; w < (int) (blockDim.x >> 5); ++w) s += red[w];
    return s;
}

template <class T>
__device__ const T * row_of(const tsn_rows & r, long long b, long long t) { return (const T *) r.p + b * r.sb + t * r.st; }

// u (shared, C values) normalised in place
__device__ void norm_row(float * u, int C, int kind, float eps, const float * w, const float * b, float * red) {
    if (kind == TSN_NORM_NONE) return;
    float mean = 0.0f;
    if (kind == TSN_NORM_LAYER) {
        float s = 0.0f;
        for (int i = threadIdx.x; i < C; i += blockDim.x) s += u[i];
        mean = block_sum(s, red) / (float) C;
    }
    float q = 0.0f;
    for (int i = threadIdx.x; i < C; i += blockDim.x) { const float d = u[i] - mean; q += d * d; }
    const float inv = rsqrtf(block_sum(q, red) / (float) C + eps);
    for (int i = threadIdx.x; i < C; i += blockDim.x)
        u[i] = (u[i] - mean) * inv * (w ? w[i] : 1.0f) + (b ? b[i] : 0.0f);
}

template <class TX, class T>
__global__ void block_norm_kernel(const __grid_constant__ NormArgs n) {
    extern __shared__ float u[];
    __shared__ float red[32];
    const tsn_block_norm_args & a = n.a;
    const int C = (int) a.C;
    const long long b = blockIdx.x / a.T, t = blockIdx.x % a.T;
    const TX * x = row_of<TX>(a.x, b, t);
    if (a.y.p) {
        const T * y = row_of<T>(a.y, b, t);
        for (int i = threadIdx.x; i < C; i += blockDim.x) u[i] = to_f32(y[i]);
        norm_row(u, C, a.post, a.post_eps, a.post_w, a.post_b, red);
        if (a.gate.p) {
            const T * g = row_of<T>(a.gate, b, t);
            for (int i = threadIdx.x; i < C; i += blockDim.x) {
                const float v = to_f32(g[i]);
                u[i] *= a.gate_tanh ? tanhf(v) : v;
            }
        }
    } else {
        for (int i = threadIdx.x; i < C; i += blockDim.x) u[i] = 0.0f;
    }
    for (int i = threadIdx.x; i < C; i += blockDim.x) {
        u[i] = fmaf(to_f32(x[i]), a.res_vec ? a.res_vec[i] : a.res_scale, u[i]);
        if (a.x_out.p) ((TX *) a.x_out.p + b * a.x_out.sb + t * a.x_out.st)[i] = from_f32<TX>(u[i]);
    }
    if (!a.h.p) return;
    norm_row(u, C, a.pre, a.pre_eps, a.pre_w, a.pre_b, red);
    T * h = (T *) a.h.p + b * a.h.sb + t * a.h.st;
    for (int i = threadIdx.x; i < C; i += blockDim.x) {
        float v = u[i];
        if (a.scale.p) v *= 1.0f + to_f32(row_of<T>(a.scale, b, t)[i]);
        if (a.shift.p) v += to_f32(row_of<T>(a.shift, b, t)[i]);
        h[i] = from_f32<T>(v);
    }
}

template <class TX, class T>
cudaError_t launch(const NormArgs & n, cudaStream_t s) {
    const size_t smem = n.a.C * sizeof(float);
    static_assert(16384 * sizeof(float) <= 227 * 1024 - 1024, "the longest row fits in shared memory");
    cudaError_t e = cudaFuncSetAttribute(block_norm_kernel<TX, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 16384 * 4);
    if (e != cudaSuccess) return e;
    block_norm_kernel<TX, T><<<(unsigned) n.rows, 256, smem, s>>>(n);
    return cudaGetLastError();
}

} // namespace

int block_norm(DeviceCtx & c, const tsn_block_norm_args & a) {
    if (!known_type(a.type) || (a.xtype != a.type && a.xtype != TSN_F32))
        return fail(TSN_ERR_ARG, "tsn_block_norm: xtype must be type or TSN_F32");
    if (a.C < 1 || a.C > 16384) return fail(TSN_ERR_ARG, "tsn_block_norm: C must lie in 1..16384");
    auto norm_ok = [](int k) { return k == TSN_NORM_NONE || k == TSN_NORM_RMS || k == TSN_NORM_LAYER; };
    if (!norm_ok(a.post) || !norm_ok(a.pre)) return fail(TSN_ERR_ARG, "tsn_block_norm: unknown norm");
    const long long rows = (long long) a.B * a.T;
    if (rows == 0) return TSN_OK;
    if (rows > 0x7fffffffLL) return fail(TSN_ERR_ARG, "tsn_block_norm: more than 2^31 - 1 rows");
    if (!a.x.p) return fail(TSN_ERR_ARG, "tsn_block_norm: null x");
    if (!a.x_out.p && !a.h.p) return fail(TSN_ERR_ARG, "tsn_block_norm: neither x_out nor h");
    if (!a.y.p && a.gate.p) return fail(TSN_ERR_ARG, "tsn_block_norm: a gate without y");
    auto distinct = [&](const tsn_rows & r) {   // rows of a result do not repeat
        return !r.p || ((a.T == 1 || r.st != 0) && (a.B == 1 || r.sb != 0));
    };
    if (!distinct(a.x_out) || !distinct(a.h)) return fail(TSN_ERR_ARG, "tsn_block_norm: a result with a stride of 0");
    const NormArgs n{a, rows};
    cudaError_t e;
    if (a.type == TSN_F32) e = launch<float, float>(n, c.stream);
    else if (a.type == TSN_F16) e = a.xtype == TSN_F32 ? launch<float, __half>(n, c.stream) : launch<__half, __half>(n, c.stream);
    else e = a.xtype == TSN_F32 ? launch<float, __nv_bfloat16>(n, c.stream) : launch<__nv_bfloat16, __nv_bfloat16>(n, c.stream);
    if (e != cudaSuccess) return fail(TSN_ERR_CUDA, std::string("tsn_block_norm: ") + cudaGetErrorString(e));
    return TSN_OK;
}

} // namespace tsn

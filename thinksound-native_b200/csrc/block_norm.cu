// block_norm.cu — norms before and after a block, fused with gate and residual scale (tsn_block_norm).
//
// Per row of C elements: x' = r x + act(g) Npost(y), h = Npre(x') (1 + scale) + shift. Bound by HBM: x, y and
// the modulation rows are read once, x' and h written once. A row stays in registers from the first load to
// the last store, each thread holding NV pieces of V elements (16 bytes of the branch's type). Up to two pieces a
// thread, everything the row needs is requested before the first reduction, so its threads wait for memory
// once; with more the modulation is read when it is needed, as it would not fit in registers. The mean and the sum of
// squared distances from it are two reductions: one pass over squares would lose the variance of a row whose
// mean is large.
#include "block_ops.h"

#include <algorithm>

namespace tsn {

namespace {

struct NormArgs {
    tsn_block_norm_args a;
    unsigned rows;
};

// V elements of type T, held as they lie in memory
template <class T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Piece {
    T v[V];
};
template <class T, int V>
__device__ __forceinline__ Piece<T, V> load(const T * p) {
    Piece<T, V> r;
    if constexpr (sizeof(T) * V >= 16) {
#pragma unroll
        for (int i = 0; i < (int) (sizeof(T) * V / 16); ++i) ((uint4 *) &r)[i] = ((const uint4 *) p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = p[i];
    }
    return r;
}
template <class T, int V>
__device__ __forceinline__ void store(T * p, const float * v) {
    Piece<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = from_f32<T>(v[i]);
    if constexpr (sizeof(T) * V >= 16) {
#pragma unroll
        for (int i = 0; i < (int) (sizeof(T) * V / 16); ++i) ((uint4 *) p)[i] = ((uint4 *) &r)[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = r.v[i];
    }
}

// Sum over the row's threads: a warp, or the whole block (one barrier; red is another array for each sum).
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float v, float * red) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (!BLOCK) return v;
    const int warps = (int) (blockDim.x >> 5);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
    if (warps <= 8) {
        for (int w = 0; w < warps; ++w) s += red[w];
        return s;
    }
    s = (int) (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// u normalised in place. Elements past C are zero and stay so; at(i): whether piece i lies inside the row.
template <int NV, int V, bool BLOCK, class At, class Col>
__device__ __forceinline__ void norm(float (&u)[NV][V], int C, int kind, float eps, const float * w, const float * b, float * red,
                                     At at, Col col) {
    if (kind == TSN_NORM_NONE) return;
    float mean = 0.0f;
    if (kind == TSN_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) s += u[i][k];
        mean = row_sum<BLOCK>(s, red) / (float) C;
    }
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at(i))
#pragma unroll
            for (int k = 0; k < V; ++k) { const float d = u[i][k] - mean; q = fmaf(d, d, q); }
    const float inv = rsqrtf(row_sum<BLOCK>(q, red + 32) / (float) C + eps);
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at(i)) {
            Piece<float, V> wv, bv;
            if (w) wv = load<float, V>(w + col(i));
            if (b) bv = load<float, V>(b + col(i));
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float v = (u[i][k] - mean) * inv;
                if (w) v *= wv.v[k];
                if (b) v += bv.v[k];
                u[i][k] = v;
            }
        }
}

// The most threads of a block: with several 16-byte pieces a thread, half as many at twice the registers.
constexpr int most_threads(int V, int NV, bool block) { return !block ? 128 : V > 1 && NV > 1 ? 512 : 1024; }

// One row per block (BLOCK) or per warp.
template <class TX, class T, int V, int NV, bool BLOCK>
__global__ void __launch_bounds__(most_threads(V, NV, BLOCK)) block_norm_kernel(const __grid_constant__ NormArgs n) {
    __shared__ float red[BLOCK ? 128 : 1];
    const tsn_block_norm_args & a = n.a;
    const int C = (int) a.C;
    const unsigned row = BLOCK ? blockIdx.x : blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (!BLOCK && row >= n.rows) return;
    const int first = (BLOCK ? (int) threadIdx.x : (int) (threadIdx.x & 31)) * V, step = (BLOCK ? (int) blockDim.x : 32) * V;
    auto col = [&](int i) { return first + i * step; };
    auto at = [&](int i) { return col(i) < C; };
    const long long b = row / a.T, t = row % a.T;
    auto in = [&](const tsn_rows & r) { return b * r.sb + t * r.st; };

    Piece<TX, V> x[NV];
    constexpr bool EARLY = NV <= 2;
    Piece<T, V> y[NV], g[EARLY ? NV : 1], sc[EARLY ? NV : 1], sh[EARLY ? NV : 1];
    auto modulation = [&](Piece<T, V> & r, const tsn_rows & m, int i) { r = load<T, V>((const T *) m.p + in(m) + col(i)); };
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at(i)) {
            if (a.y.p) y[i] = load<T, V>((const T *) a.y.p + in(a.y) + col(i));
            x[i] = load<TX, V>((const TX *) a.x.p + in(a.x) + col(i));
            if (EARLY) {
                if (a.gate.p) modulation(g[i], a.gate, i);
                if (a.scale.p) modulation(sc[i], a.scale, i);
                if (a.shift.p) modulation(sh[i], a.shift, i);
            }
        }
    float u[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) u[i][k] = 0.0f;
    if (a.y.p) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at(i))
#pragma unroll
                for (int k = 0; k < V; ++k) u[i][k] = to_f32(y[i].v[k]);
        norm<NV, V, BLOCK>(u, C, a.post, a.post_eps, a.post_w, a.post_b, red, at, col);
        if (a.gate.p)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (at(i)) {
                    Piece<T, V> & gi = g[EARLY ? i : 0];
                    if (!EARLY) modulation(gi, a.gate, i);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float v = to_f32(gi.v[k]);
                        u[i][k] *= a.gate_tanh ? tanhf(v) : v;
                    }
                }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at(i)) {
            Piece<float, V> r;
            if (a.res_vec) r = load<float, V>(a.res_vec + col(i));
#pragma unroll
            for (int k = 0; k < V; ++k) u[i][k] = fmaf(to_f32(x[i].v[k]), a.res_vec ? r.v[k] : a.res_scale, u[i][k]);
            if (a.x_out.p) store<TX, V>((TX *) a.x_out.p + in(a.x_out) + col(i), u[i]);
        }
    if (!a.h.p) return;
    norm<NV, V, BLOCK>(u, C, a.pre, a.pre_eps, a.pre_w, a.pre_b, red + (BLOCK ? 64 : 0), at, col);
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at(i)) {
            Piece<T, V> & si = sc[EARLY ? i : 0], & hi = sh[EARLY ? i : 0];
            if (!EARLY) {
                if (a.scale.p) modulation(si, a.scale, i);
                if (a.shift.p) modulation(hi, a.shift, i);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                if (a.scale.p) u[i][k] *= 1.0f + to_f32(si.v[k]);
                if (a.shift.p) u[i][k] += to_f32(hi.v[k]);
            }
            store<T, V>((T *) a.h.p + in(a.h) + col(i), u[i]);
        }
}

template <class TX, class T, int V>
cudaError_t launch(const NormArgs & n, cudaStream_t s) {
    const int pieces = ((int) n.a.C + V - 1) / V;
    if (pieces <= 32) {
        block_norm_kernel<TX, T, V, 1, false><<<(n.rows + 3) / 4, 128, 0, s>>>(n);
    } else if constexpr (V == 1) {   // unaligned rows
        const int threads = std::min(1024, (pieces + 127) / 128 * 32);
        if (pieces <= 4 * threads) block_norm_kernel<TX, T, V, 4, true><<<n.rows, threads, 0, s>>>(n);
        else block_norm_kernel<TX, T, V, 16, true><<<n.rows, threads, 0, s>>>(n);
    } else {
        // Two pieces a thread where the rows fill the GPU, one where there are few and their latency counts.
        const bool few = n.rows <= 2 * 148;
        const int per = pieces > 2048 ? 8 : pieces > 1024 ? 4 : few ? 1 : 2;
        const int threads = (pieces + 32 * per - 1) / (32 * per) * 32;
        if (per == 1) block_norm_kernel<TX, T, V, 1, true><<<n.rows, threads, 0, s>>>(n);
        else if (per == 2) block_norm_kernel<TX, T, V, 2, true><<<n.rows, threads, 0, s>>>(n);
        else if (per == 4) block_norm_kernel<TX, T, V, 4, true><<<n.rows, threads, 0, s>>>(n);
        else if constexpr (V < 8) block_norm_kernel<TX, T, V, 8, true><<<n.rows, threads, 0, s>>>(n);   // 2048 pieces of 8 are 16384
    }
    return cudaGetLastError();
}

template <class TX, class T>
cudaError_t launch(const NormArgs & n, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const tsn_block_norm_args & a = n.a;
    auto rows16 = [&](const tsn_rows & r, size_t size) {   // every row starts at a 16-byte boundary
        return !r.p || (((uintptr_t) r.p | (uintptr_t) (a.B > 1 ? r.sb : 0) * size | (uintptr_t) (a.T > 1 ? r.st : 0) * size) & 15) == 0;
    };
    auto vec16 = [&](const float * p) { return ((uintptr_t) p & 15) == 0; };
    const bool wide = a.C % V == 0 && rows16(a.x, sizeof(TX)) && rows16(a.x_out, sizeof(TX)) && rows16(a.y, sizeof(T)) &&
                      rows16(a.h, sizeof(T)) && rows16(a.gate, sizeof(T)) && rows16(a.scale, sizeof(T)) &&
                      rows16(a.shift, sizeof(T)) && vec16(a.post_w) && vec16(a.post_b) && vec16(a.pre_w) && vec16(a.pre_b) &&
                      vec16(a.res_vec);
    return wide ? launch<TX, T, V>(n, s) : launch<TX, T, 1>(n, s);
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
    auto aligned = [&](const tsn_rows & r, size_t size) { return ((uintptr_t) r.p & (size - 1)) == 0; };
    const size_t e = type_size(a.type), ex = type_size(a.xtype);
    if (!aligned(a.x, ex) || !aligned(a.x_out, ex) || !aligned(a.y, e) || !aligned(a.h, e) || !aligned(a.gate, e) ||
        !aligned(a.shift, e) || !aligned(a.scale, e) ||
        (((uintptr_t) a.post_w | (uintptr_t) a.post_b | (uintptr_t) a.pre_w | (uintptr_t) a.pre_b | (uintptr_t) a.res_vec) & 3))
        return fail(TSN_ERR_ARG, "tsn_block_norm: an address that is no multiple of its element's size");
    const NormArgs n{a, (unsigned) rows};
    cudaError_t rc;
    if (a.type == TSN_F32) rc = launch<float, float>(n, c.stream);
    else if (a.type == TSN_F16) rc = a.xtype == TSN_F32 ? launch<float, __half>(n, c.stream) : launch<__half, __half>(n, c.stream);
    else rc = a.xtype == TSN_F32 ? launch<float, __nv_bfloat16>(n, c.stream) : launch<__nv_bfloat16, __nv_bfloat16>(n, c.stream);
    if (rc != cudaSuccess) return fail(TSN_ERR_CUDA, std::string("tsn_block_norm: ") + cudaGetErrorString(rc));
    return TSN_OK;
}

} // namespace tsn

// block_norm.cu — norms before and after a block, fused with gate and residual scale (tsn_block_norm).
//
// Per row of C elements: x' = r x + act(g) Npost(y), h = Npre(x') (1 + scale) + shift. Bound by HBM: x, y and
// the modulation rows are read once, x' and h written once. A row stays with its threads from the first load to
// the last store, each holding NV pieces of V elements (16 bytes of the branch's type) in registers; only rows of more
// than 4096 single elements (V 1, NV 16) spill, 290 to 700 bytes a thread. Up to two pieces a
// thread, everything the row needs is requested before the first reduction, so its threads wait for memory
// once; with more the modulation is read when it is needed, as it would not fit in registers. The mean and the sum of
// squared distances from it are two reductions: one pass over squares would lose the variance of a row whose
// mean is large.
// 32 500 rows of 2048 bf16 elements with a modulation of each token take 164 us in one long run of them, 180 us
// with other inputs from call to call (932 MB, 5.7 and 5.2 TB/s, 0.87 and 0.79 of the measured copy), 658 rows of 1024
// 4.0 us (latency: two reductions after the loads).
#include "block_ops.h"
#include "kernels.h"

#include <algorithm>
#include <type_traits>

namespace tsn {

namespace {

struct NormArgs {
    tsn_block_norm_args a;
    unsigned rows;
    int swapped;   // one row a block: the batch runs along x instead of y
};

// V elements of type T: 16-byte words where a piece has some, else a pair in one word or the element itself.
template <class T, int V>
struct Piece {
    static constexpr bool WIDE = sizeof(T) * V >= 16;
    using Pair = typename std::conditional<sizeof(T) == 4, float2, uint32_t>::type;
    typename std::conditional<WIDE, Words<T, WIDE ? V : 16>, typename std::conditional<V == 2, Pair, T>::type>::type r;
    __device__ __forceinline__ void load(const T * p) {
        if constexpr (WIDE) r = load_words<T, V>(p);
        else if constexpr (V == 2) r = *(const Pair *) p;
        else r = *p;
    }
    __device__ __forceinline__ void get(float * v) const {
        if constexpr (WIDE) {
            to_floats<T, V>(r, v);
        } else if constexpr (V == 2) {
            float2 f;
            if constexpr (sizeof(T) == 4) f = r;
            else f = unpack2<T>(r);
            v[0] = f.x;
            v[1] = f.y;
        } else {
            *v = to_f32(r);
        }
    }
};
template <class T, int V>
__device__ __forceinline__ void store(T * p, const float * v) {
    if constexpr (Piece<T, V>::WIDE) store_words<T, V>(p, v);
    else if constexpr (V == 2 && sizeof(T) == 4) *(float2 *) p = make_float2(v[0], v[1]);
    else if constexpr (V == 2) *(uint32_t *) p = pack2<T>(v[0], v[1]);
    else *p = from_f32<T>(*v);
}
// v[k] = f(v[k], ...) over a piece, two at a time where it has two
template <int V, class F2>
__device__ __forceinline__ void each(float * v, F2 f2) {
    if constexpr (V == 1) {
        v[0] = f2(make_float2(v[0], 0.0f), 0).x;
    } else {
#pragma unroll
        for (int k = 0; k < V; k += 2) {
            const float2 r = f2(make_float2(v[k], v[k + 1]), k);
            v[k] = r.x;
            v[k + 1] = r.y;
        }
    }
}
template <int V>
__device__ __forceinline__ float2 at2(const float * v, int k) { return make_float2(v[k], V == 1 ? 0.0f : v[k + (V > 1)]); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// tanh of gates. 16-bit gates: up to 0.4 the odd polynomial x + x^3 p(x^2) of least relative error there (1.2e-7, weighted
// least squares iterated to the maximum norm), beyond it 1 - 2 / (e^(2|x|) + 1), which would cancel near 0. Both are off by
// less than 2^-20 of the value at any size of gate; gates start near zero, and an f32 residual, or a norm after a small
// residual, keeps every bit of them. The library's tanhf, exact to its last bits, would cost more than the row's traffic.
template <class T>
__device__ __forceinline__ float2 gate_tanh(float2 x) {
    if (sizeof(T) == 4) return make_float2(tanhf(x.x), tanhf(x.y));
    auto far = [](float v) {
        float e, r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fabsf(v) * 2.88539008177792681f));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.0f));
        return copysignf(fmaf(-2.0f, r, 1.0f), v);
    };
    const float2 t = mul2(x, x);
    float2 p = fma2(t, make_float2(-0.0477942191f, -0.0477942191f), make_float2(0.13277629f, 0.13277629f));
    p = fma2(t, p, make_float2(-0.33331883f, -0.33331883f));
    p = fma2(mul2(t, p), x, x);
    return make_float2(fabsf(x.x) <= 0.4f ? p.x : far(x.x), fabsf(x.y) <= 0.4f ? p.y : far(x.y));
}

// Sum over the row's threads: a warp, or the whole block (one barrier; red is another array for each sum).
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float v, float * red) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (!BLOCK) return v;
    const int warps = (int) (blockDim.x >> 5), lane = (int) (threadIdx.x & 31);
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = lane < warps ? red[lane] : 0.0f;
    for (int o = 1; o < warps; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);   // lane 0's power of two of lanes
    return __shfl_sync(0xffffffffu, s, 0);
}

// u normalised in place. Elements past C are zero and stay so; at(i): whether piece i lies inside the row.
template <int NV, int V, bool BLOCK, class At, class Col>
__device__ __forceinline__ void norm(float (&u)[NV][V], float inv_C, int kind, float eps, const float * w, const float * b, float * red,
                                     At at, Col col) {
    if (kind == TSN_NORM_NONE) return;
    float mean = 0.0f;
    if (kind == TSN_NORM_LAYER) {
        float2 s = both(0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            each<V>(u[i], [&](float2 v, int) { s = add2(s, v); return v; });
        mean = row_sum<BLOCK>(s.x + s.y, red) * inv_C;
    }
    float2 q = both(0.0f);
    const float2 minus = both(-mean);
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at(i))
            each<V>(u[i], [&](float2 v, int) {
                v = add2(v, minus);
                if (V == 1) v.y = 0.0f;
                q = fma2(v, v, q);
                return v;
            });
    const float2 inv = both(rsqrtf(fmaf(row_sum<BLOCK>(q.x + q.y, red + 32), inv_C, eps)));
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at(i)) {
            each<V>(u[i], [&](float2 v, int) { return mul2(v, inv); });
            float wv[V], bv[V];
            if (w) {
                Piece<float, V> r;
                r.load(w + col(i));
                r.get(wv);
                each<V>(u[i], [&](float2 v, int k) { return mul2(v, at2<V>(wv, k)); });
            }
            if (b) {
                Piece<float, V> r;
                r.load(b + col(i));
                r.get(bv);
                each<V>(u[i], [&](float2 v, int k) { return add2(v, at2<V>(bv, k)); });
            }
        }
}

// The most threads of a block: with several 16-byte pieces a thread, half as many at twice the registers.
constexpr int most_threads(int V, int NV, bool block) { return !block ? 128 : V > 2 && NV > 1 ? 512 : 1024; }

// One row per block (BLOCK) or per warp.
template <class TX, class T, int V, int NV, bool BLOCK>
__global__ void __launch_bounds__(most_threads(V, NV, BLOCK)) block_norm_kernel(const __grid_constant__ NormArgs n) {
    __shared__ float red[BLOCK ? 128 : 1];
    pdl_wait();   // and no trigger: the next kernel's blocks beside this one's made 658 rows take 5.0 us instead of 4.0
    const tsn_block_norm_args & a = n.a;
    const int C = (int) a.C;
    const float inv_C = 1.0f / (float) C;
    const unsigned row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (!BLOCK && row >= n.rows) return;
    const int first = (BLOCK ? (int) threadIdx.x : (int) (threadIdx.x & 31)) * V, step = (BLOCK ? (int) blockDim.x : 32) * V;
    auto col = [&](int i) { return first + i * step; };
    auto at = [&](int i) { return col(i) < C; };
    // a block's row is a block index in each direction: its addresses are the same in all threads and cost them nothing
    const unsigned b = BLOCK ? (n.swapped ? blockIdx.x : blockIdx.y) : row / a.T, t = BLOCK ? (n.swapped ? blockIdx.y : blockIdx.x) : row % a.T;
    auto in = [&](const tsn_rows & r) { return b * r.sb + t * r.st; };

    constexpr bool EARLY = NV <= 2;
    Piece<TX, V> x[NV];
    Piece<T, V> y[NV], g[EARLY ? NV : 1], sc[EARLY ? NV : 1], sh[EARLY ? NV : 1];
    auto modulation = [&](Piece<T, V> & r, const tsn_rows & m, int i) { r.load((const T *) m.p + in(m) + col(i)); };
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at(i)) {
            if (a.y.p) y[i].load((const T *) a.y.p + in(a.y) + col(i));
            x[i].load((const TX *) a.x.p + in(a.x) + col(i));
            if (EARLY && a.gate.p) modulation(g[i], a.gate, i);
        }
    if (EARLY)
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at(i)) {
                if (a.scale.p) modulation(sc[i], a.scale, i);
                if (a.shift.p) modulation(sh[i], a.shift, i);
            }
    float u[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) u[i][k] = 0.0f;
    if (a.y.p) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at(i)) y[i].get(u[i]);
        norm<NV, V, BLOCK>(u, inv_C, a.post, a.post_eps, a.post_w, a.post_b, red, at, col);
        if (a.gate.p)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (at(i)) {
                    Piece<T, V> & gi = g[EARLY ? i : 0];
                    if (!EARLY) modulation(gi, a.gate, i);
                    float gv[V];
                    gi.get(gv);
                    if (a.gate_tanh) each<V>(gv, [](float2 v, int) { return gate_tanh<T>(v); });
                    each<V>(u[i], [&](float2 v, int k) { return mul2(v, at2<V>(gv, k)); });
                }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at(i)) {
            float xv[V], rv[V];
            x[i].get(xv);
            if (a.res_vec) {
                Piece<float, V> r;
                r.load(a.res_vec + col(i));
                r.get(rv);
                each<V>(u[i], [&](float2 v, int k) { return fma2(at2<V>(xv, k), at2<V>(rv, k), v); });
            } else {
                each<V>(u[i], [&](float2 v, int k) { return fma2(at2<V>(xv, k), both(a.res_scale), v); });
            }
            if (a.x_out.p) store<TX, V>((TX *) a.x_out.p + in(a.x_out) + col(i), u[i]);
        }
    if (!a.h.p) return;
    norm<NV, V, BLOCK>(u, inv_C, a.pre, a.pre_eps, a.pre_w, a.pre_b, red + (BLOCK ? 64 : 0), at, col);
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at(i)) {
            float mv[V];
            if (a.scale.p) {
                Piece<T, V> & si = sc[EARLY ? i : 0];
                if (!EARLY) modulation(si, a.scale, i);
                si.get(mv);
                each<V>(u[i], [&](float2 v, int k) { return mul2(v, add2(at2<V>(mv, k), both(1.0f))); });
            }
            if (a.shift.p) {
                Piece<T, V> & hi = sh[EARLY ? i : 0];
                if (!EARLY) modulation(hi, a.shift, i);
                hi.get(mv);
                each<V>(u[i], [&](float2 v, int k) { return add2(v, at2<V>(mv, k)); });
            }
            store<T, V>((T *) a.h.p + in(a.h) + col(i), u[i]);
        }
}

template <class TX, class T, int V>
cudaError_t launch(const NormArgs & n, cudaStream_t s) {
    const int pieces = ((int) n.a.C + V - 1) / V;
    const dim3 grid = n.swapped ? dim3(n.a.B, n.a.T) : dim3(n.a.T, n.a.B);
    cudaError_t e = cudaSuccess;
    auto go = [&](void (*kernel)(NormArgs), int threads) { e = launch_cl(kernel, grid, dim3((unsigned) threads), 0, s, dim3(1), n); };
    if (pieces <= 32) {
        e = launch_cl(block_norm_kernel<TX, T, V, 1, false>, dim3((n.rows + 3) / 4), dim3(128), 0, s, dim3(1), n);
    } else if constexpr (V <= 2) {   // unaligned rows
        const int threads = std::min(1024, (pieces + 127) / 128 * 32);
        if (pieces <= 4 * threads) go(block_norm_kernel<TX, T, V, 4, true>, threads);
        else go(block_norm_kernel<TX, T, V, 16 / V, true>, threads);   // 16384 elements in 1024 threads
    } else {
        // One piece a thread while a block of 512 holds the row: the least latency where there are few rows (658
        // rows of 1024: 4.0 us, 4.8 with two pieces, 8.6 with four). Two, half the reductions, where the rows fill the GPU
        // eight times (with tanh gates 32 500 of 2048 bf16 take 161 us, 195 with one; 2400 of 2048 17.9 and 18.1), and for
        // wide rows of 16 bits from eight rows an SM on (2400 of 4096: 33.1 and 36.7; 600: 12.5 and 12.0).
        const bool two = pieces > 64 && ((long long) n.rows * pieces >= 8ll * 148 * 2048 || (V == 8 && pieces > 256 && n.rows >= 8 * 148));
        const int per = pieces > 2048 ? 8 : pieces > 1024 ? 4 : pieces > 512 || two ? 2 : 1;
        const int threads = (pieces + 32 * per - 1) / (32 * per) * 32;
        if (per == 1) go(block_norm_kernel<TX, T, V, 1, true>, threads);
        else if (per == 2) go(block_norm_kernel<TX, T, V, 2, true>, threads);
        else if (per == 4) go(block_norm_kernel<TX, T, V, 4, true>, threads);
        else if constexpr (V < 8) go(block_norm_kernel<TX, T, V, 8, true>, threads);   // 2048 pieces of 8 are 16384
    }
    if (e != cudaSuccess) cudaGetLastError();
    return e;
}

template <class TX, class T>
cudaError_t launch(const NormArgs & n, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const tsn_block_norm_args & a = n.a;
    // every row, and every vector, starts at a multiple of some elements' bytes, 16 at most
    auto aligned = [&](uintptr_t elements) {
        auto rows = [&](const tsn_rows & r, size_t size) {
            const uintptr_t bytes = std::min<uintptr_t>(16, elements * size);
            return !r.p || (((uintptr_t) r.p | (uintptr_t) (a.B > 1 ? r.sb : 0) * size | (uintptr_t) (a.T > 1 ? r.st : 0) * size) & (bytes - 1)) == 0;
        };
        auto vec = [&](const float * p) { return ((uintptr_t) p & (std::min<uintptr_t>(16, elements * 4) - 1)) == 0; };
        return a.C % elements == 0 && rows(a.x, sizeof(TX)) && rows(a.x_out, sizeof(TX)) && rows(a.y, sizeof(T)) && rows(a.h, sizeof(T)) &&
               rows(a.gate, sizeof(T)) && rows(a.scale, sizeof(T)) && rows(a.shift, sizeof(T)) && vec(a.post_w) && vec(a.post_b) &&
               vec(a.pre_w) && vec(a.pre_b) && vec(a.res_vec);
    };
    // pairs where 16 bytes do not fit: 5400 rows of 1462, f16 with an f32 residual, 50 us (2.9 TB/s); by single elements 89, and
    // 91 for rows of 1461 (1.6 TB/s). Both are bound by narrow loads, which keep few bytes on their way.
    return aligned(V) ? launch<TX, T, V>(n, s) : aligned(2) ? launch<TX, T, 2>(n, s) : launch<TX, T, 1>(n, s);
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
    const NormArgs n{a, (unsigned) rows, a.B > 65535};   // then T is less: there are no more than 2^31 - 1 rows
    cudaError_t rc;
    if (a.type == TSN_F32) rc = launch<float, float>(n, c.stream);
    else if (a.type == TSN_F16) rc = a.xtype == TSN_F32 ? launch<float, __half>(n, c.stream) : launch<__half, __half>(n, c.stream);
    else rc = a.xtype == TSN_F32 ? launch<float, __nv_bfloat16>(n, c.stream) : launch<__nv_bfloat16, __nv_bfloat16>(n, c.stream);
    if (rc != cudaSuccess) return fail(TSN_ERR_CUDA, std::string("tsn_block_norm: ") + cudaGetErrorString(rc));
    return TSN_OK;
}

} // namespace tsn

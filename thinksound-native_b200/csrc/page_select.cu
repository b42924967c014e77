// page_select.cu — which pages a token attends to (the first kernel of tsn_sparse_attn).
//
//   s_x = (sum_g q_g) . mean_x for the pages x before the token's own;  the `picks` best, `first` and `last` ones always
// The picks are whole numbers, and a sum rounded to 32 bits would exchange pages whose scores nearly agree, so scores are
// summed in 64 bits: products of 16-bit values are exact there. A 16-bit value becomes an f64 by shifting its f32 bits
// right by 3 into the high word, which is the value times 2^-896 exactly, subnormals and zero included (a conversion
// instruction has a quarter of the FMAs' rate); q carries a factor of 2^800 against it. Factors that all scores share change no order.
// A block takes one token and kv head. D / 8 lanes read a mean, a warp 16 means a lane at once; their partial sums are
// exchanged so that each lane ends with whole ones. The picks are found by a radix select over the scores' bits in shared memory
// and written in the order of the pages.
#include "kernels.h"
#include "paged.h"

namespace tsn {

namespace {

constexpr int THREADS = 256;

struct Select {
    tsn_sparse_attn_args a;
    int page_log2, G;
};

__device__ __forceinline__ double scaled(float v) {   // v * 2^-896
    const uint32_t x = __float_as_uint(v);
    return __hiloint2double((int) ((x & 0x80000000u) | ((x & 0x7fffffffu) >> 3)), (int) (x << 29));
}

// Sums over the block of two numbers before this thread.
__device__ __forceinline__ int2 before(int2 v, int2 * red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int2 s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(~0u, s.x, o), y = __shfl_up_sync(~0u, s.y, o);
        if (lane >= o) { s.x += x; s.y += y; }
    }
    if (lane == 31) red[warp] = s;
    __syncthreads();
    int2 r = make_int2(s.x - v.x, s.y - v.y);
    for (int w = 0; w < warp; ++w) { r.x += red[w].x; r.y += red[w].y; }
    return r;
}

template <class T, int D>
__global__ void __launch_bounds__(THREADS) page_select_kernel(const __grid_constant__ Select p) {
    extern __shared__ __align__(16) uint64_t keys[];   // [pages]
    __shared__ __align__(16) double qs[D];
    __shared__ int at[2];
    __shared__ int2 red[THREADS / 32];
    __shared__ unsigned int hist[256], found[3];   // found: digit, keys above it, keys of it
    constexpr int LPH = D / 8, SIDE = 32 / LPH;
    const tsn_sparse_attn_args & a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = (int) blockIdx.x, hk = (int) blockIdx.y;
    pdl_wait();
    if (warp == 0) {
        const int b = seq_of_row(a.c, row);
        const int pl = b < 0 ? 0 : place_of_row(a.c, b, row);
        if (lane == 0) {
            at[0] = b;
            at[1] = pl;
        }
    }
    for (int e = tid; e < D; e += THREADS) {
        double s = 0.0;
        for (int g = 0; g < p.G; ++g) s += (double) to_f32(((const T *) a.q.p)[row * a.q.sb + (long long) (hk * p.G + g) * a.q.st + e]);
        qs[e] = s * 0x1p800;
    }
    __syncthreads();
    pdl_trigger();
    const int b = at[0], place = at[1], picks = (int) a.picks;
    if (b < 0) return;   // a row of no sequence
    int * chosen = a.chosen + ((long long) row * a.c.Hk + hk) * picks;
    const int own = place < 0 ? -1 : place >> p.page_log2, n = own >= (int) a.c.M ? 0 : own + 1;
    if (n <= picks) {
        for (int j = tid; j < picks; j += THREADS) chosen[j] = j < n ? j : -1;
        return;
    }
    // pages that compete: first .. top - 1
    const int first = (int) a.first, top = n - (int) a.last, m = top - first;
    const int * table = a.c.table + b * a.c.table_sb;
    const int sub = lane / LPH, e0 = (lane % LPH) * 8;
    double q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = qs[e0 + e];
    constexpr int BATCH = LPH;   // means of a lane at once: as many as lanes share one
    for (int j0 = warp * (BATCH * SIDE); j0 < m; j0 += THREADS / 32 * (BATCH * SIDE)) {
        // lane (sub, l) reads its 8 elements of means j0 + sub * BATCH + y
        double s[BATCH];
        const int mine = first + j0 + sub * BATCH + lane % LPH;
        const int id = mine < top ? table[mine] : -1;
        Words<T, 8> r[BATCH];
        bool there[BATCH];
#pragma unroll
        for (int y = 0; y < BATCH; ++y) {
            const int page = __shfl_sync(~0u, id, sub * LPH + y);
            there[y] = page >= 0 && page < (int) a.c.P;
            if (there[y]) r[y] = load_words<T, 8>((const T *) a.means.p + page * a.means.sb + hk * a.means.st + e0);
        }
#pragma unroll
        for (int y = 0; y < BATCH; ++y) {
            s[y] = 0.0;
            if (there[y]) {
                float u[8];
                to_floats<T, 8>(r[y], u);
#pragma unroll
                for (int e = 0; e < 8; ++e) s[y] = fma(q[e], scaled(u[e]), s[y]);
            }
        }
        // lane l of the mean's lanes ends with the sum of mean l
#pragma unroll
        for (int o = LPH / 2; o; o >>= 1)
#pragma unroll
            for (int y = 0; y < o; ++y) {
                const bool up = (lane & o) != 0;
                const double give = up ? s[y] : s[y + o], keep = up ? s[y + o] : s[y];
                s[y] = keep + __shfl_xor_sync(~0u, give, o);
            }
        if (mine < top) {
            const long long bits = __double_as_longlong(s[0] + 0.0);   // -0 becomes 0
            keys[mine - first] = (uint64_t) (bits < 0 ? ~bits : bits | (long long) 0x8000000000000000ull);
        }
    }
    // the key of rank `need`: bits found from the highest digit on; keys that share the found ones are counted by their next digit
    uint64_t found_bits = 0, known = 0;
    unsigned int need = (unsigned) (picks - first - (int) a.last);
    bool whole = false;   // every key with the found bits is picked
    for (int shift = 56; shift >= 0 && !whole && need; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        for (int j0 = 0; j0 < m; j0 += THREADS) {
            const int j = j0 + tid;
            const uint64_t k = j < m ? keys[j] : 0;
            const bool in = j < m && (k & known) == found_bits;
            const unsigned digit = in ? (unsigned) (k >> shift) & 255u : 256u, same = __match_any_sync(~0u, digit);
            if (in && lane == __ffs(same) - 1) atomicAdd(&hist[digit], (unsigned) __popc(same));
        }
        __syncthreads();
        if (warp == 0) {   // lane l: digits 255 - 8 l .. 248 - 8 l, from the highest down
            unsigned int c[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += c[i] = hist[255 - 8 * lane - i];
            unsigned int upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned int v = __shfl_up_sync(~0u, upto, o);
                if (lane >= o) upto += v;
            }
            unsigned int above = upto - sum;
            if (above < need && need <= upto) {
                int i = 0;
                while (above + c[i] < need) above += c[i++];
                found[0] = (unsigned) (255 - 8 * lane - i);
                found[1] = above;
                found[2] = c[i];
            }
        }
        __syncthreads();
        found_bits |= (uint64_t) found[0] << shift;
        known |= (uint64_t) 255 << shift;
        need -= found[1];
        whole = need == found[2];
        __syncthreads();
    }
    // in the order of the pages: above the found key, and the first `need` of those equal to it in the known bits
    const int per = (n + THREADS - 1) / THREADS, j0 = min(n, tid * per), j1 = min(n, j0 + per);
    auto kind = [&](int j) {   // 2: picked, 1: equal, 0: not
        if (j < first || j >= top) return 2;
        const uint64_t k = keys[j - first] & known;
        return k > found_bits ? 2 : k == found_bits && need ? 1 : 0;
    };
    int2 count = make_int2(0, 0);
    for (int j = j0; j < j1; ++j) {
        const int k = kind(j);
        count.x += k == 2;
        count.y += k == 1;
    }
    int2 pre = before(count, red);
    for (int j = j0; j < j1; ++j) {
        const int k = kind(j);
        if (k == 2 || (k == 1 && pre.y < (int) need)) chosen[pre.x + min(pre.y, (int) need)] = j;
        pre.x += k == 2;
        pre.y += k == 1;
    }
}

template <class T, int D>
cudaError_t launch(const Select & p, cudaStream_t s) {
    return launch_cl(page_select_kernel<T, D>, dim3(p.a.c.N, p.a.c.Hk), dim3(THREADS), (size_t) p.a.c.M * 8, s, dim3(1), p);
}

} // namespace

cudaError_t launch_page_select(const tsn_sparse_attn_args & a, cudaStream_t s) {
    const Select p{a, log2_of(a.c.page), (int) (a.H / a.c.Hk)};
    const bool bf = a.c.type == TSN_BF16;
    if (a.c.D == 64) return bf ? launch<__nv_bfloat16, 64>(p, s) : launch<__half, 64>(p, s);
    return bf ? launch<__nv_bfloat16, 128>(p, s) : launch<__half, 128>(p, s);
}

cudaError_t configure_page_select() {
    cudaError_t e = cudaSuccess;
    auto set = [&](auto * k) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 16384 * 8);
    };
    set(page_select_kernel<__half, 64>);
    set(page_select_kernel<__half, 128>);
    set(page_select_kernel<__nv_bfloat16, 64>);
    set(page_select_kernel<__nv_bfloat16, 128>);
    return e;
}

} // namespace tsn

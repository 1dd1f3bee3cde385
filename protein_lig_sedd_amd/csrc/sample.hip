// Truncated categorical sampling from given uniform numbers: temperature, top-k, top-p and min-p, and the ancestral
// update of the absorbing graph built on it.  Counterpart in the reference: utils/catsample.py:10-13 (Gumbel arg-max over
// the whole vocabulary) and sampling/sampling.py:102-132 (the update that calls it); the truncations are this library's.
//
// Definition, for a row of scores x, noise u and the row's T, k, P, m (all in 64 bits; the token is that of exact
// arithmetic, not of one order of rounding):
//     q_j  = exp((x_j - max x) / T)                          entries of -inf or NaN are no candidates
//     rank = place of j by (x descending, index ascending)
//     kept = rank < k  and  sum of q ranked before j < P * (sum of q over rank < k)  and  q_j >= m;  rank 0 always
//     out  = arg max over kept of q_j / (1e-10 - log(min(u_j + 1e-10, 1)))   (u + 1e-10 rounded to 32 bits), lowest index
// q_j / E_j with E_j exponential has its maximum at j with probability q_j / sum q, so the noise picks among what is kept.
//
// No sort and no running sum: the kept entries are a PREFIX of the order.  The arg-max over everything is found first; one
// pass gives its rank and the mass before it; if it is kept, it is the answer, and if it is not, neither is anything ranked
// behind it, so the next candidate is the arg-max among what is ranked before it.  A row ends after 1/(kept mass) tries
// or about log(V / kept) of them, whichever is less, since each rejection cuts the prefix at a random place.
#include "common.h"

struct SampleArgs {
    const void* x;
    int64_t ld;
    const float* u;
    int64_t ldu;
    const float *T, *P, *m;  // per batch element, or NULL: the scalars below
    const int* k;
    float T0, P0, m0;
    int k0;
    const int64_t* xcur;  // current tokens: only rows that hold mask_id are sampled, the others keep theirs
    int64_t mask_id;
    const float* move;  // per batch element: a masked row is sampled only where u[row][V] < move
    int64_t* out;
    int64_t M, L;
    int V;
};

struct RowParams {
    float T, P, m;
    int k;
};
__device__ __forceinline__ RowParams row_params(const SampleArgs& a, int64_t b) {
    RowParams r;
    r.T = a.T ? a.T[b] : a.T0;
    r.P = a.P ? a.P[b] : a.P0;
    r.m = a.m ? a.m[b] : a.m0;
    r.k = a.k ? a.k[b] : a.k0;
    if (r.k <= 0 || r.k > a.V) r.k = a.V;
    return r;
}
// whether the row is sampled at all; otherwise its token stays
__device__ __forceinline__ bool row_moves(const SampleArgs& a, int64_t row, int64_t b) {
    if (!a.xcur) return true;
    if (a.xcur[row] != a.mask_id) return false;
    return !a.move || a.u[row * a.ldu + a.V] < a.move[b];
}
__device__ __forceinline__ int64_t row_empty(const SampleArgs& a) { return a.xcur ? a.mask_id : (int64_t)-1; }

// fp32 -> unsigned with the same order (both zeros alike); -inf and NaN: 0, no candidate
__device__ __forceinline__ uint32_t order_key(float v) {
    v += 0.0f;
    const uint32_t b = __float_as_uint(v);
    const uint32_t key = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    return v > -INFINITY ? key : 0u;
}
// u + 1e-10 in 32 bits as the reference's catsample rounds it, kept inside (0, 1] whatever u is
__device__ __forceinline__ float noise_arg(float u) { return fminf(fmaxf(u + 1e-10f, 1e-10f), 1.0f); }

// ------------------------------------------------------------------------------- the definition itself, in 64 bits
// NT threads (a power of two of whole waves) work one row together, reading it from memory in every pass.
template <int NT> struct Joint {
    double* sd;  // [NT / 64] each
    int64_t* si;
    template <typename F> __device__ __forceinline__ double dsum(double v, F) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
        if constexpr (NT == 64) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sd[threadIdx.x >> 6] = v;
        __syncthreads();
        v = sd[0];
        for (int w = 1; w < NT / 64; ++w) v += sd[w];
        return v;
    }
    __device__ __forceinline__ double sum(double v) { return dsum(v, 0); }
    __device__ __forceinline__ int64_t isum(int64_t v) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
        if constexpr (NT == 64) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) si[threadIdx.x >> 6] = v;
        __syncthreads();
        v = si[0];
        for (int w = 1; w < NT / 64; ++w) v += si[w];
        return v;
    }
    // largest v, lowest index among equals
    __device__ __forceinline__ void best(double& v, int64_t& i) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const double ov = __shfl_xor(v, o, 64);
            const int64_t oi = __shfl_xor(i, o, 64);
            if (ov > v || (ov == v && oi < i)) { v = ov; i = oi; }
        }
        if constexpr (NT == 64) return;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { sd[threadIdx.x >> 6] = v; si[threadIdx.x >> 6] = i; }
        __syncthreads();
        v = sd[0];
        i = si[0];
        for (int w = 1; w < NT / 64; ++w)
            if (sd[w] > v || (sd[w] == v && si[w] < i)) { v = sd[w]; i = si[w]; }
    }
};

template <typename T, int NT>
__device__ int64_t resolve_row64(const SampleArgs& a, int64_t row, int64_t b, double* sd, int64_t* si) {
    Joint<NT> J{sd, si};
    const int lane = threadIdx.x & (NT - 1), V = a.V;
    const T* x = (const T*)a.x + row * a.ld;
    const float* u = a.u + row * a.ldu;
    const RowParams rp = row_params(a, b);
    const int64_t none = (int64_t)1 << 40;
    // the first entry of the order
    double mxd = -1.0;  // (as an order key, so that one reduction serves)
    int64_t mi = none;
    for (int j = lane; j < V; j += NT) {
        const uint32_t key = order_key(to_f32<T>(x[j]));
        if (key && (double)key > mxd) { mxd = (double)key; mi = j; }
    }
    J.best(mxd, mi);
    if (mi == none) return row_empty(a);
    if (!(rp.T > 0.f)) return mi;  // greedy
    const uint32_t kmax = (uint32_t)mxd;
    const double mx = (double)(to_f32<T>(x[mi]) + 0.0f), rT = (double)rp.T;
    const bool top_inf = isinf(mx);
    auto weight = [&](uint32_t key, float v) -> double {
        if (key == kmax) return 1.0;
        return top_inf ? 0.0 : exp(((double)v - mx) / rT);
    };
    // mass of the k first of the order
    double W = 0.0;
    if (rp.P < 1.f) {
        uint32_t t = 0;  // the k-th largest key, or 0 if there are no k candidates
        if (rp.k < V) {
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t c = t | (1u << bit);
                int64_t n = 0;
                for (int j = lane; j < V; j += NT) n += order_key(to_f32<T>(x[j])) >= c;
                if (J.isum(n) >= rp.k) t = c;
            }
        }
        double s = 0.0, q = 0.0;
        int64_t n = 0;
        for (int j = lane; j < V; j += NT) {
            const float v = to_f32<T>(x[j]);
            const uint32_t key = order_key(v);
            if (key > t) { s += weight(key, v); ++n; }
            else if (key == t && t) q = weight(key, v);
        }
        W = J.sum(s);
        if (t) {
            n = J.isum(n);
            int64_t dummy = 0;
            J.best(q, dummy);
            W += (double)(rp.k - n) * q;  // of equal entries at the border the lowest indices are in; they weigh the same
        }
    }
    uint32_t kc = 0xffffffffu;  // what is still possible: ranked before (kc, ic)
    int64_t ic = none;
    for (;;) {
        double bv = -1.0;
        int64_t bi = none;
        for (int j = lane; j < V; j += NT) {
            const float v = to_f32<T>(x[j]);
            const uint32_t key = order_key(v);
            if (!key || !(key > kc || (key == kc && j < ic) || ic == none)) continue;
            const double r = weight(key, v) / (1e-10 - log((double)noise_arg(u[j])));
            if (r > bv) { bv = r; bi = j; }
        }
        J.best(bv, bi);
        if (bi == none) return mi;  // (cannot be: the first of the order is always kept)
        const float vw = to_f32<T>(x[bi]);
        const uint32_t kw = order_key(vw);
        double S = 0.0;
        int64_t rank = 0;
        for (int j = lane; j < V; j += NT) {
            const float v = to_f32<T>(x[j]);
            const uint32_t key = order_key(v);
            if (key > kw || (key == kw && j < bi)) { S += weight(key, v); ++rank; }
        }
        rank = J.isum(rank);
        if (rank == 0) return bi;
        S = J.sum(S);
        if (rank < rp.k && (!(rp.P < 1.f) || S < (double)rp.P * W) && !(weight(kw, vw) < (double)rp.m)) return bi;
        kc = kw;
        ic = bi;
    }
}

template <typename T, int NT>
__global__ void __launch_bounds__(256) sample_row64_kernel(SampleArgs a) {
    __shared__ double sd[4];
    __shared__ int64_t si[4];
    const int64_t stride = (int64_t)gridDim.x * (256 / NT);
    for (int64_t row = (int64_t)blockIdx.x * (256 / NT) + threadIdx.x / NT; row < a.M; row += stride) {
        const int64_t b = row / a.L;
        int64_t got;
        if (!row_moves(a, row, b)) got = a.xcur[row];
        else got = resolve_row64<T, NT>(a, row, b, sd, si);
        if ((threadIdx.x & (NT - 1)) == 0) a.out[row] = got;
    }
}

template <typename T> static void launch_sample(const SampleArgs& a, hipStream_t st) {
    if (a.V <= 4096)
        hipLaunchKernelGGL((sample_row64_kernel<T, 64>), dim3(sedd_grid_for(a.M, 4, 256 * 8)), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((sample_row64_kernel<T, 256>), dim3(sedd_grid_for(a.M, 1, 256 * 8)), dim3(256), 0, st, a);
}

extern "C" int sedd_sample_truncated(const void* logits, int dtype, int64_t ld, const float* u, int64_t ldu,
                                     const float* temperature, const int32_t* top_k, const float* top_p,
                                     const float* min_p, float temperature0, int top_k0, float top_p0, float min_p0,
                                     const int64_t* x, int64_t mask_id, const float* move, int64_t* out, int64_t M,
                                     int64_t L, int V, sedd_stream_t stream) {
    SEDD_CHECK_ARG(dtype == SEDD_F32 || dtype == SEDD_BF16, "sample_truncated: unknown dtype %d", dtype);
    SEDD_CHECK_ARG(M >= 0 && L > 0 && V > 0 && M % L == 0, "sample_truncated: bad sizes M=%ld L=%ld V=%d", (long)M,
                   (long)L, V);
    SEDD_CHECK_ARG(M <= 1 || (ld >= V && ldu >= V + (move ? 1 : 0)), "sample_truncated: row strides %ld, %ld below V=%d",
                   (long)ld, (long)ldu, V);
    SEDD_CHECK_ARG(!move || x, "sample_truncated: move probabilities without current tokens");
    SEDD_CHECK_ARG(temperature || (temperature0 >= 0.f && temperature0 <= 3.402823466e38f),
                   "sample_truncated: temperature %f", (double)temperature0);
    SEDD_CHECK_ARG(top_p || (top_p0 >= 0.f && top_p0 <= 1.f), "sample_truncated: top_p %f not in [0, 1]", (double)top_p0);
    SEDD_CHECK_ARG(min_p || (min_p0 >= 0.f && min_p0 <= 1.f), "sample_truncated: min_p %f not in [0, 1]", (double)min_p0);
    SEDD_CHECK_ARG(top_k || top_k0 >= 0, "sample_truncated: top_k %d is negative", top_k0);
    if (M == 0) return SEDD_OK;
    SEDD_CHECK_ARG(logits && u && out, "sample_truncated: null pointer");
    const SampleArgs a{logits, ld, u, ldu, temperature, top_p, min_p, top_k, temperature0, top_p0, min_p0, top_k0,
                       x, mask_id, move, out, M, L, V};
    if (dtype == SEDD_F32) launch_sample<float>(a, (hipStream_t)stream);
    else launch_sample<bf16_t>(a, (hipStream_t)stream);
    SEDD_LAUNCH_CHECK();
    return SEDD_OK;
}

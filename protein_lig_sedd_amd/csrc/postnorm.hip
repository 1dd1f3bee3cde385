// Norms before and after a block, fused with its gate and residual scale.  The gated residual is the reference's
// (model/fused_add_dropout_scale.py:13-48) and the norm behind it the next sub-layer's (model/transformer.py:30-38, :186);
// the norm of the branch's own output and the residual scale are this library's (model.post_norm / model.residual_scale).
//   n  = LN(a) * wp                    ahat = (a - pm) * pr
//   x1 = alpha * x + gate_b * keep(n)
//   h  = LN(x1) * w * (1 + scale_b) + shift_b                    (optional)
#include "rowops.h"
#include <initializer_list>

// ================================================================================================ forward
// One wave per row, the row in registers from the branch's output to h: x and a are read once, x1 and h written once, which bounds
// it: 64 x 512 x 768 bf16 with the next norm 61 us, 302 MB at 5.0 TB/s.
template <typename TA, typename TM, int NV, bool NEXT>
__global__ void __launch_bounds__(TPB) post_norm_fwd_kernel(
    const float* __restrict__ res, const TA* __restrict__ a, const float* __restrict__ wp, const TM* __restrict__ gate,
    const TM* __restrict__ shift, const TM* __restrict__ scale, int64_t mod_stride, float alpha, float inv_keep,
    uint64_t seed, uint32_t thr16, const float* __restrict__ w, float* __restrict__ x1, TA* __restrict__ y,
    float* __restrict__ pmean, float* __restrict__ prstd, float* __restrict__ mean, float* __restrict__ rstd, int64_t M,
    int64_t L, int D) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * (TPB / 64) + (threadIdx.x >> 6);
    if (row >= M) return;
    if (thr16) seed = resolve_seed(seed);
    const int64_t b = row / L;
    const float inv_d = 1.0f / (float)D;
    float4 v[NV], rs[NV];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = k * 256 + lane * 4;
        v[k] = rs[k] = f4(0.f);
        if (c < D) {
            v[k] = load4<TA>(a + row * D + c);
            rs[k] = load4<float>(res + row * D + c);
        }
        s += (v[k].x + v[k].y) + (v[k].z + v[k].w);
    }
    const float pm = dpp_sum(s) * inv_d;
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (k * 256 + lane * 4 < D) {
            v[k].x -= pm; v[k].y -= pm; v[k].z -= pm; v[k].w -= pm;
            q += (v[k].x * v[k].x + v[k].y * v[k].y) + (v[k].z * v[k].z + v[k].w * v[k].w);
        }
    }
    const float pr = 1.0f / sqrtf(dpp_sum(q) * inv_d + 1e-5f);
    s = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = k * 256 + lane * 4;
        if (c < D) {
            const int64_t off = row * D + c;
            const float4 ww = load4<float>(wp + c), g = load4<TM>(gate + b * mod_stride + c);
            float4 kk = f4(1.f);
            if (thr16) kk = keep4_hashed(seed, off, thr16, inv_keep);
            v[k].x = alpha * rs[k].x + g.x * (v[k].x * pr * ww.x * kk.x);
            v[k].y = alpha * rs[k].y + g.y * (v[k].y * pr * ww.y * kk.y);
            v[k].z = alpha * rs[k].z + g.z * (v[k].z * pr * ww.z * kk.z);
            v[k].w = alpha * rs[k].w + g.w * (v[k].w * pr * ww.w * kk.w);
            store4<float>(x1 + off, v[k]);
            s += (v[k].x + v[k].y) + (v[k].z + v[k].w);
        }
    }
    if (lane == 0) { pmean[row] = pm; prstd[row] = pr; }
    if constexpr (NEXT) {
        // in the steps of the plain LayerNorm kernel, so that h is to the bit what that makes of x1
        const float mu = wave_sum(s) / (float)D;
        q = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (k * 256 + lane * 4 < D) {
                const float a = v[k].x - mu, b = v[k].y - mu, cc = v[k].z - mu, d = v[k].w - mu;
                q += (a * a + b * b) + (cc * cc + d * d);
            }
        }
        const float r1 = 1.0f / sqrtf(wave_sum(q) / (float)D + 1e-5f);
        if (lane == 0) { mean[row] = mu; rstd[row] = r1; }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = k * 256 + lane * 4;
            if (c < D) {
                const float4 ww = load4<float>(w + c);
                const float4 sc = load4<TM>(scale + b * mod_stride + c), sh = load4<TM>(shift + b * mod_stride + c);
                store4<TA>(y + row * D + c, make_float4((v[k].x - mu) * r1 * ww.x * (1.f + sc.x) + sh.x,
                                                        (v[k].y - mu) * r1 * ww.y * (1.f + sc.y) + sh.y,
                                                        (v[k].z - mu) * r1 * ww.z * (1.f + sc.z) + sh.z,
                                                        (v[k].w - mu) * r1 * ww.w * (1.f + sc.w) + sh.w));
            }
        }
    }
}

// what the vector accesses need: 16 bytes for fp32 rows, 8 for bf16 ones
static bool rows_aligned(int dt, std::initializer_list<const void*> ps) {
    uintptr_t v = 0;
    for (const void* p : ps) v |= (uintptr_t)p;
    return v % (dt == SEDD_F32 ? 16 : 8) == 0;
}
static int post_norm_check(const char* nm, int a_dtype, int mod_dtype, int64_t mod_stride, float p_drop, int64_t M,
                           int64_t L, int D) {
    SEDD_CHECK_ARG(dt_ok(a_dtype) && dt_ok(mod_dtype), "%s: bad dtype", nm);
    SEDD_CHECK_ARG(p_drop >= 0.f && p_drop < 1.f, "%s: p_drop %f", nm, (double)p_drop);
    SEDD_CHECK_ARG(M >= 0 && L > 0 && M % L == 0, "%s: bad sizes M=%ld L=%ld", nm, (long)M, (long)L);
    SEDD_CHECK_ARG(M <= ((int64_t)1 << 26) - 4, "%s: %ld rows", nm, (long)M);  // (a wave each, 2^32 - 1 threads to a launch)
    if (D <= 0 || D % 4 != 0 || D > 2048 || mod_stride % 4 != 0) {
        sedd_set_error("%s: D=%d unsupported (need D %% 4 == 0, D <= 2048)", nm, D);
        return SEDD_ERR_UNSUPPORTED_SHAPE;
    }
    return SEDD_OK;
}
#define DISPATCH_NV(D, ...)                                        \
    do {                                                           \
        if ((D) <= 256) { constexpr int NV = 1; __VA_ARGS__; }     \
        else if ((D) <= 512) { constexpr int NV = 2; __VA_ARGS__; } \
        else if ((D) <= 768) { constexpr int NV = 3; __VA_ARGS__; } \
        else if ((D) <= 1024) { constexpr int NV = 4; __VA_ARGS__; } \
        else { constexpr int NV = 8; __VA_ARGS__; }                \
    } while (0)

extern "C" int sedd_post_norm_residual_fwd(const float* residual, const void* a, int a_dtype, const float* post_w,
                                           const void* gate, const void* shift, const void* scale, int mod_dtype,
                                           int64_t mod_stride, float res_scale, float inv_keep, uint64_t seed,
                                           float p_drop, const float* w, float* x_out, void* y, float* post_mean,
                                           float* post_rstd, float* mean, float* rstd, int64_t M, int64_t L, int D,
                                           sedd_stream_t stream) {
    int rc = post_norm_check("post_norm_residual_fwd", a_dtype, mod_dtype, mod_stride, p_drop, M, L, D);
    if (rc) return rc;
    if (M == 0) return SEDD_OK;
    SEDD_CHECK_ARG(residual && a && post_w && gate && x_out && post_mean && post_rstd,
                   "post_norm_residual_fwd: null pointer");
    SEDD_CHECK_ARG(!w || (shift && scale && y && mean && rstd), "post_norm_residual_fwd: null pointer of the next norm");
    SEDD_CHECK_ARG(rows_aligned(SEDD_F32, {residual, post_w, w, x_out}) && rows_aligned(a_dtype, {a, y}) &&
                       rows_aligned(mod_dtype, {gate, shift, scale}), "post_norm_residual_fwd: misaligned rows");
    const uint32_t thr16 = (uint32_t)(p_drop * 65536.0f + 0.5f);
    const dim3 grid((unsigned)((M + 3) / 4));
#define POST_FWD(NEXT_)                                                                                              \
    hipLaunchKernelGGL((post_norm_fwd_kernel<TA, TM, NV, NEXT_>), grid, dim3(TPB), 0, (hipStream_t)stream, residual,    \
                       (const TA*)a, post_w, (const TM*)gate, (const TM*)shift, (const TM*)scale, mod_stride, res_scale, \
                       inv_keep, seed, thr16, w, x_out, (TA*)y, post_mean, post_rstd, mean, rstd, M, L, D)
    DISPATCH_DT(a_dtype, TA, DISPATCH_DT(mod_dtype, TM, DISPATCH_NV(D, {
        if (w) POST_FWD(true);
        else POST_FWD(false);
    })));
#undef POST_FWD
    SEDD_LAUNCH_CHECK();
    return SEDD_OK;
}

// ================================================================================================ backward
// d   = dx1 + rs * (g - mean(g) - xhat * mean(g xhat)),  g = dh * w * (1 + scale_b)       (d = dx1 without a next norm)
// dx  = alpha * d;  dn = d * gate_b * keep
// da  = pr * (g2 - mean(g2) - ahat * mean(g2 ahat)),     g2 = dn * wp
// dw += dh (1 + scale) xhat;  dshift = sum dh;  dscale = sum dh xhat w;  dgate = sum d keep ahat wp;  dwp += dn ahat;
// dbias += da (before it is rounded: the bias gradient of the Linear that made a)
// A block owns a chunk of rows and a thread four columns of it, so the six column sums are running sums in registers and leave as
// one line of partial sums per chunk: no fold across waves, which a wave-per-row layout needs for all six.  What crosses the
// waves is two pairs of row sums, through LDS.  The next row's operands are loaded before this row's sums are waited for.
// 64 x 512 x 768 bf16: 102 us, 454 MB at 4.4 TB/s, and 8 us for the fold.
// A chunk is a part of one batch element, a whole one where that is shorter than two chunks, or several where they are shorter
// than half of one.  Where no batch element is split, the sums per batch element (dgate, dshift, dscale) are final and go straight
// to their place (2703 x 4 x 1484: 112 us; with a chunk and a fold to each batch element 266 us).
// Rows of a chunk: 32, or fewer where that leaves less than 2560 waves (10 a CU).  Measured with
// half and twice the rows: 64 x 512 x 768 32 rows 113 us (16: 121, 64: 155); 16 x 1024 x 1024 16 rows 71 (8: 80, 32: 86);
// 8 x 512 x 2048 8 rows 36 (4: 46); more waves cover the latency of the row sums, more chunks write more partial sums.
static inline int post_chunk_rows(int64_t M, int D) {
    const int64_t nw = (D + 255) / 256;
    int r = 32;
    while (r > 4 && M / r * nw < 2560) r >>= 1;
    return r;
}
struct PostChunks {
    int64_t n, per_batch, batches;  // chunks; chunks of a batch element; batch elements of a chunk
    int rows;                       // of a chunk at most
};
static PostChunks post_chunks(int64_t M, int64_t L, int D) {
    const int r = post_chunk_rows(M, D);
    const int64_t B = M / L, g = 2 * L <= r ? r / L : 1, per = L < 2 * r ? 1 : (L + r - 1) / r;
    return {g > 1 ? (B + g - 1) / g : B * per, per, g, (int)(g > 1 ? g * L : (L + per - 1) / per)};
}
extern "C" int sedd_post_norm_chunks(int64_t M, int64_t L, int D) {
    return L <= 0 || M <= 0 ? 0 : (int)post_chunks(M, L, D).n;
}
// both sums over the block's nw waves (buf: 2 nw floats; two buffers in turn: the next write to one comes after another barrier)
__device__ __forceinline__ void block_sum2(float& a, float& b, float* buf, int nw) {
    a = dpp_sum(a);
    b = dpp_sum(b);
    if (nw == 1) return;
    if ((threadIdx.x & 63) == 0) {
        const int w = threadIdx.x >> 6;
        buf[2 * w] = a;
        buf[2 * w + 1] = b;
    }
    __syncthreads();
    a = buf[0];
    b = buf[1];
    for (int w = 1; w < nw; ++w) { a += buf[2 * w]; b += buf[2 * w + 1]; }
}

struct PostBwdArgs {
    const float *dx1, *x1, *w, *mean, *rstd, *wp, *pmean, *prstd;
    const void *dh, *a, *scale, *gate;
    float *dx, *ws;
    void* da;
    float* out[6];  // by plane: 0 dgate, 1 dwp, 2 dbias, 3 dw, 4 dshift, 5 dscale; any may be NULL
    int64_t mod_stride, gate_stride, dmod_stride, L, B;
    PostChunks ch;
    float alpha, inv_keep;
    uint64_t seed;
    uint32_t thr16;
    int D, planes;
};
template <typename TA, typename TM, bool NEXT>
__global__ void __launch_bounds__(512) post_norm_bwd_kernel(PostBwdArgs p) {
    __shared__ float sA[2 * 8], sB[2][2 * 8];
    const int nw = blockDim.x >> 6, c = threadIdx.x * 4, D = p.D;
    const bool on = c < D;
    const int64_t chunk = blockIdx.x;
    int64_t b = p.ch.batches > 1 ? chunk * p.ch.batches : chunk / p.ch.per_batch;
    const int64_t row0 = p.ch.batches > 1 ? b * p.L : b * p.L + chunk % p.ch.per_batch * p.ch.rows;
    const int64_t left = (p.ch.batches > 1 ? p.B * p.L : (b + 1) * p.L) - row0;
    const int nrows = left < p.ch.rows ? (int)left : p.ch.rows;
    int batch_end = p.ch.batches > 1 ? (int)p.L : nrows;  // the row behind the batch element at hand
    const float inv_d = 1.0f / (float)D;
    uint64_t seed = p.seed;
    if (p.thr16) seed = resolve_seed(seed);
    const TA *dh = (const TA*)p.dh, *a = (const TA*)p.a;
    TA* da = (TA*)p.da;
    float4 wp = f4(0.f), gt = f4(0.f), ww = f4(0.f), sc1 = f4(0.f);
    auto modulation = [&]() __attribute__((always_inline)) {
        if (!on) return;
        gt = load4<TM>((const TM*)p.gate + b * p.mod_stride + c);
        if constexpr (NEXT) {
            const float4 s = load4<TM>((const TM*)p.scale + b * p.mod_stride + c);
            sc1 = make_float4(1.f + s.x, 1.f + s.y, 1.f + s.z, 1.f + s.w);
        }
    };
    if (on) {
        wp = load4<float>(p.wp + c);
        if constexpr (NEXT) ww = load4<float>(p.w + c);
    }
    modulation();
    float4 aw = f4(0.f), ash = f4(0.f), asc = f4(0.f), ag = f4(0.f), apw = f4(0.f), ab = f4(0.f);
    // the sums of a batch element: final, or a line of partial sums
    auto flush = [&]() __attribute__((always_inline)) {
        if (!on) return;
        if (p.ch.per_batch == 1) {
            auto put = [&](float* o, int64_t stride, const float4& v) {  // (scalar: a gradient slice need not be 16-byte aligned)
                if (!o) return;
                o += b * stride + c;
                o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
            };
            put(p.out[0], p.gate_stride, ag);
            if constexpr (NEXT) {
                put(p.out[4], p.dmod_stride, ash);
                put(p.out[5], p.dmod_stride, asc);
            }
        } else {
            float* o = p.ws + chunk * D + c;
            const int64_t plane = p.ch.n * D;
            store4<float>(o, ag);
            if constexpr (NEXT) {
                store4<float>(o + 4 * plane, ash);
                store4<float>(o + 5 * plane, asc);
            }
        }
    };
    float4 dn = f4(0.f), an = f4(0.f), gn = f4(0.f), xn = f4(0.f);  // the next row
    auto fetch = [&](int i) __attribute__((always_inline)) {
        if (!on) return;
        const int64_t off = (row0 + i) * D + c;
        if (!NEXT || p.dx1) dn = load4<float>(p.dx1 + off);
        an = load4<TA>(a + off);
        if constexpr (NEXT) {
            gn = load4<TA>(dh + off);
            xn = load4<float>(p.x1 + off);
        }
    };
    fetch(0);
    for (int i = 0; i < nrows; ++i) {
        const int64_t row = row0 + i, off = row * D + c;
        float4 d = dn, ah = an, g = gn, xh = xn;
        float rs = 0.f, mu = 0.f;
        if constexpr (NEXT) { mu = p.mean[row]; rs = p.rstd[row]; }
        const float pm = p.pmean[row], pr = p.prstd[row];
        if (i + 1 < nrows) fetch(i + 1);
        float *Dv = &d.x, *A = &ah.x, *G = &g.x, *X = &xh.x;
        const float *W = &ww.x, *S = &sc1.x, *WP = &wp.x, *GT = &gt.x;
        if constexpr (NEXT) {
            float s1 = 0.f, s2 = 0.f;
            if (on) {
                float *AW = &aw.x, *ASH = &ash.x, *ASC = &asc.x;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    X[k] = (X[k] - mu) * rs;
                    ASH[k] += G[k];
                    const float gx = G[k] * X[k];
                    ASC[k] += gx * W[k];
                    AW[k] += gx * S[k];
                    G[k] *= W[k] * S[k];
                    s1 += G[k];
                    s2 += G[k] * X[k];
                }
            }
            block_sum2(s1, s2, sA, nw);
            s1 *= inv_d;
            s2 *= inv_d;
#pragma unroll
            for (int k = 0; k < 4; ++k) Dv[k] += rs * (G[k] - s1 - X[k] * s2);
        }
        float t1 = 0.f, t2 = 0.f;
        if (on) {
            store4<float>(p.dx + off, make_float4(p.alpha * d.x, p.alpha * d.y, p.alpha * d.z, p.alpha * d.w));
            float4 kk = f4(1.f);
            if (p.thr16) kk = keep4_hashed(seed, off, p.thr16, p.inv_keep);
            const float* K = &kk.x;
            float *AG = &ag.x, *APW = &apw.x;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                A[k] = (A[k] - pm) * pr;
                const float dk = Dv[k] * K[k], t = dk * A[k];
                AG[k] += t * WP[k];
                APW[k] += t * GT[k];
                G[k] = dk * GT[k] * WP[k];
                t1 += G[k];
                t2 += G[k] * A[k];
            }
        }
        block_sum2(t1, t2, sB[NEXT ? 0 : i & 1], nw);
        t1 *= inv_d;
        t2 *= inv_d;
        if (on) {
            float4 o;
            float *O = &o.x, *AB = &ab.x;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                O[k] = pr * (G[k] - t1 - A[k] * t2);
                AB[k] += O[k];
            }
            store4<TA>(da + off, o);
        }
        if (i + 1 == batch_end && i + 1 < nrows) {
            flush();
            ag = ash = asc = f4(0.f);
            batch_end += (int)p.L;
            ++b;
            modulation();
        }
    }
    flush();
    if (on) {
        float* o = p.ws + chunk * D + c;
        const int64_t plane = p.ch.n * D;
        store4<float>(o + plane, apw);
        store4<float>(o + 2 * plane, ab);
        if constexpr (NEXT) store4<float>(o + 3 * plane, aw);
    }
}

// Folds the chunks' partial sums in a fixed order: planes 1, 2 and 3 over all chunks (added to what is there) and, where batch
// elements are split, 0, 4 and 5 over each one's (written).  A block folds 64 columns: 16 lanes of four columns each, 16 groups
// of lines that meet in LDS, or, where a batch element has fewer lines than that, 16 batch elements.  The few long folds come
// first, with 8 loads in flight per thread: they are bound by latency.
__host__ __device__ __forceinline__ int64_t fold_batches(const PostChunks& ch) { return ch.per_batch < 16 ? 16 : 1; }
__global__ void __launch_bounds__(TPB) post_norm_reduce_kernel(PostBwdArgs p) {
    const int ncb = (p.D + 63) / 64, nvec = p.planes == 6 ? 3 : 2;
    const int64_t fb = fold_batches(p.ch), nb = (p.B + fb - 1) / fb;
    const bool vec = (int64_t)blockIdx.x < (int64_t)nvec * ncb;
    int64_t i = vec ? blockIdx.x : blockIdx.x - (int64_t)nvec * ncb;
    const int col = (int)(i % ncb) * 64 + (threadIdx.x & 15) * 4, rg = threadIdx.x >> 4;
    i /= ncb;
    const int64_t b = vec ? 0 : i % nb * fb + (fb > 1 ? rg : 0);
    const int k = vec ? 1 + (int)i : (i / nb == 0 ? 0 : 3 + (int)(i / nb));
    float* out = p.out[k];
    if (!out) return;
    auto put = [&](const float4& v) {  // (scalar accesses: a gradient slice need not be 16-byte aligned)
        float* o = out + b * (k == 0 ? p.gate_stride : p.dmod_stride) + col;
        o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
    };
    if (!vec && fb > 1) {
        if (col >= p.D || b >= p.B) return;
        const float* base = p.ws + ((int64_t)k * p.ch.n + b * p.ch.per_batch) * p.D + col;
        float4 s = f4(0.f);
#pragma unroll 8
        for (int64_t c = 0; c < p.ch.per_batch; ++c) {
            const float4 v = load4<float>(base + c * p.D);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        put(s);
        return;
    }
    __shared__ float4 red[16][16];
    const int64_t lines = vec ? p.ch.n : p.ch.per_batch;
    float4 s = f4(0.f);
    if (col < p.D) {
        const float* base = p.ws + ((int64_t)k * p.ch.n + b * p.ch.per_batch) * p.D + col;
        int64_t c = rg;
        for (; c + 7 * 16 < lines; c += 8 * 16) {
            float4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = load4<float>(base + (c + 16 * u) * p.D);
#pragma unroll
            for (int u = 0; u < 8; ++u) { s.x += v[u].x; s.y += v[u].y; s.z += v[u].z; s.w += v[u].w; }
        }
        for (; c < lines; c += 16) {
            const float4 v = load4<float>(base + c * p.D);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
    }
    red[rg][threadIdx.x & 15] = s;
    __syncthreads();
    if (rg == 0 && col < p.D) {
        for (int r = 1; r < 16; ++r) {
            const float4 v = red[r][threadIdx.x];
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        if (vec) { out[col] += s.x; out[col + 1] += s.y; out[col + 2] += s.z; out[col + 3] += s.w; }
        else put(s);
    }
}

extern "C" int sedd_post_norm_residual_bwd(const float* dx1, const void* dh, const float* x1, const float* w,
                                           const void* scale, const float* mean, const float* rstd, const void* a,
                                           int a_dtype, const float* post_w, const void* gate, int mod_dtype,
                                           int64_t mod_stride, const float* post_mean, const float* post_rstd,
                                           float res_scale, float inv_keep, uint64_t seed, float p_drop, float* dx,
                                           void* da, float* dgate, int64_t dgate_stride, float* dshift, float* dscale,
                                           int64_t dmod_stride, float* dpost_w, float* dbias, float* dw, float* ws,
                                           int64_t M, int64_t L, int D, sedd_stream_t stream) {
    int rc = post_norm_check("post_norm_residual_bwd", a_dtype, mod_dtype, mod_stride, p_drop, M, L, D);
    if (rc) return rc;
    if (M == 0) return SEDD_OK;
    SEDD_CHECK_ARG((dx1 || dh) && a && post_w && gate && post_mean && post_rstd && dx && da && ws,
                   "post_norm_residual_bwd: null pointer");
    SEDD_CHECK_ARG(!dh || (x1 && w && scale && mean && rstd), "post_norm_residual_bwd: null pointer of the next norm");
    SEDD_CHECK_ARG(rows_aligned(SEDD_F32, {dx1, post_w, dx, ws}) && rows_aligned(a_dtype, {a, da}) &&
                       rows_aligned(mod_dtype, {gate}) &&
                       (!dh || (rows_aligned(SEDD_F32, {x1, w}) && rows_aligned(a_dtype, {dh}) && rows_aligned(mod_dtype, {scale}))),
                   "post_norm_residual_bwd: misaligned rows");
    PostBwdArgs p;
    p.dx1 = dx1; p.x1 = x1; p.w = w; p.mean = mean; p.rstd = rstd; p.wp = post_w; p.pmean = post_mean; p.prstd = post_rstd;
    p.dh = dh; p.a = a; p.scale = scale; p.gate = gate; p.dx = dx; p.ws = ws; p.da = da;
    float* outs[6] = {dgate, dpost_w, dbias, dw, dshift, dscale};
    for (int k = 0; k < 6; ++k) p.out[k] = outs[k];
    p.mod_stride = mod_stride; p.gate_stride = dgate_stride; p.dmod_stride = dmod_stride; p.L = L; p.B = M / L;
    p.ch = post_chunks(M, L, D); p.alpha = res_scale; p.inv_keep = inv_keep;
    p.seed = seed; p.thr16 = (uint32_t)(p_drop * 65536.0f + 0.5f); p.D = D; p.planes = dh ? 6 : 3;
    const dim3 grid((unsigned)p.ch.n), block((unsigned)((D + 255) / 256 * 64));
    DISPATCH_DT(a_dtype, TA, DISPATCH_DT(mod_dtype, TM, {
        if (dh) hipLaunchKernelGGL((post_norm_bwd_kernel<TA, TM, true>), grid, block, 0, (hipStream_t)stream, p);
        else hipLaunchKernelGGL((post_norm_bwd_kernel<TA, TM, false>), grid, block, 0, (hipStream_t)stream, p);
    }));
    const int64_t fb = fold_batches(p.ch), nb = (p.B + fb - 1) / fb;
    const int64_t folds = (p.planes == 6 ? 3 : 2) + (p.ch.per_batch > 1 ? (p.planes == 6 ? 3 : 1) * nb : 0);
    hipLaunchKernelGGL(post_norm_reduce_kernel, dim3((unsigned)((D + 63) / 64 * folds)), dim3(TPB), 0, (hipStream_t)stream, p);
    SEDD_LAUNCH_CHECK();
    return SEDD_OK;
}

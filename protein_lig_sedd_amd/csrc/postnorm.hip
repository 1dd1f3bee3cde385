// Norms before and after a block, fused with its gate and residual scale.  The gated residual is the reference's
// (model/fused_add_dropout_scale.py:13-48) and the norm behind it the next sub-layer's (model/transformer.py:30-38, :186);
// the norm of the branch's own output and the residual scale are this library's (model.post_norm / model.residual_scale).
//   n  = LN(a) * wp                    ahat = (a - pm) * pr
//   x1 = alpha * x + gate_b * keep(n)
//   h  = LN(x1) * w * (1 + scale_b) + shift_b                    (optional)
#include "rowops.h"
#include <initializer_list>

// ================================================================================================ forward
// One wave per row, the row in registers from the branch's output to h: x and a are read once, x1 and h written once.
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
    const float pm = wave_sum(s) * inv_d;
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (k * 256 + lane * 4 < D) {
            v[k].x -= pm; v[k].y -= pm; v[k].z -= pm; v[k].w -= pm;
            q += (v[k].x * v[k].x + v[k].y * v[k].y) + (v[k].z * v[k].z + v[k].w * v[k].w);
        }
    }
    const float pr = 1.0f / sqrtf(wave_sum(q) * inv_d + 1e-5f);
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
        const float mu = wave_sum(s) * inv_d;
        q = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (k * 256 + lane * 4 < D) {
                v[k].x -= mu; v[k].y -= mu; v[k].z -= mu; v[k].w -= mu;
                q += (v[k].x * v[k].x + v[k].y * v[k].y) + (v[k].z * v[k].z + v[k].w * v[k].w);
            }
        }
        const float r1 = 1.0f / sqrtf(wave_sum(q) * inv_d + 1e-5f);
        if (lane == 0) { mean[row] = mu; rstd[row] = r1; }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = k * 256 + lane * 4;
            if (c < D) {
                const float4 ww = load4<float>(w + c);
                const float4 sc = load4<TM>(scale + b * mod_stride + c), sh = load4<TM>(shift + b * mod_stride + c);
                store4<TA>(y + row * D + c, make_float4(v[k].x * r1 * ww.x * (1.f + sc.x) + sh.x,
                                                        v[k].y * r1 * ww.y * (1.f + sc.y) + sh.y,
                                                        v[k].z * r1 * ww.z * (1.f + sc.z) + sh.z,
                                                        v[k].w * r1 * ww.w * (1.f + sc.w) + sh.w));
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
// A block owns a chunk of at most 32 / 64 rows of one batch element and a thread four columns of it, so the six column
// sums are running sums in registers and leave as one line of partial sums per chunk: no fold across waves, which a
// wave-per-row layout needs for all six.  What crosses the waves is two pairs of row sums, through LDS, for POST_ROWS rows
// at a time.
#ifndef POST_ROWS
#define POST_ROWS 2
#endif
template <int N> __device__ __forceinline__ void block_sums(float (&v)[N], float* buf, int nw) {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if (nw == 1) return;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) buf[wave * N + i] = v[i];
    }
    __syncthreads();  // (two buffers in turn: the next write to this one comes after another such barrier)
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float s = buf[i];
        for (int w = 1; w < nw; ++w) s += buf[w * N + i];
        v[i] = s;
    }
}

struct PostBwdArgs {
    const float *dx1, *x1, *w, *mean, *rstd, *wp, *pmean, *prstd;
    const void *dh, *a, *scale, *gate;
    float *dx, *ws;
    void* da;
    int64_t mod_stride, nchunk, L;
    float alpha, inv_keep;
    uint64_t seed;
    uint32_t thr16;
    int D, CR;
};
template <typename TA, typename TM, bool NEXT>
__global__ void __launch_bounds__(512) post_norm_bwd_kernel(PostBwdArgs p) {
    constexpr int R = POST_ROWS;
    __shared__ float sA[8 * 2 * R], sB[8 * 2 * R];
    const int nw = blockDim.x >> 6, c = threadIdx.x * 4, D = p.D;
    const bool on = c < D;
    const int64_t cpb = (p.L + p.CR - 1) / p.CR;
    const int64_t chunk = blockIdx.x, b = chunk / cpb, c0 = (chunk % cpb) * p.CR;
    const int nrows = (int)((p.L - c0) < p.CR ? (p.L - c0) : p.CR);
    const float inv_d = 1.0f / (float)D;
    uint64_t seed = p.seed;
    if (p.thr16) seed = resolve_seed(seed);
    const TA *dh = (const TA*)p.dh, *a = (const TA*)p.a;
    TA* da = (TA*)p.da;
    float4 wp = f4(0.f), gt = f4(0.f), ww = f4(0.f), sc1 = f4(0.f);
    if (on) {
        wp = load4<float>(p.wp + c);
        gt = load4<TM>((const TM*)p.gate + b * p.mod_stride + c);
        if constexpr (NEXT) {
            ww = load4<float>(p.w + c);
            const float4 s = load4<TM>((const TM*)p.scale + b * p.mod_stride + c);
            sc1 = make_float4(1.f + s.x, 1.f + s.y, 1.f + s.z, 1.f + s.w);
        }
    }
    float4 aw = f4(0.f), ash = f4(0.f), asc = f4(0.f), ag = f4(0.f), apw = f4(0.f), ab = f4(0.f);
    for (int r0 = 0; r0 < nrows; r0 += R) {
        const int64_t row0 = b * p.L + c0 + r0;
        float4 d[R], g[R], xh[R], ah[R];
        float s[2 * R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            d[i] = g[i] = xh[i] = ah[i] = f4(0.f);
            if (on && r0 + i < nrows) {
                const int64_t off = (row0 + i) * D + c;
                if (!NEXT || p.dx1) d[i] = load4<float>(p.dx1 + off);
                ah[i] = load4<TA>(a + off);
                if constexpr (NEXT) {
                    g[i] = load4<TA>(dh + off);
                    xh[i] = load4<float>(p.x1 + off);
                }
            }
        }
        if constexpr (NEXT) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                s[2 * i] = s[2 * i + 1] = 0.f;
                if (on && r0 + i < nrows) {
                    const float mu = p.mean[row0 + i], rs = p.rstd[row0 + i];
                    float* X = &xh[i].x; float* G = &g[i].x;
                    const float *W = &ww.x, *S = &sc1.x;
                    float *AW = &aw.x, *ASH = &ash.x, *ASC = &asc.x;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        X[k] = (X[k] - mu) * rs;
                        ASH[k] += G[k];
                        const float gx = G[k] * X[k];
                        ASC[k] += gx * W[k];
                        AW[k] += gx * S[k];
                        G[k] *= W[k] * S[k];
                        s[2 * i] += G[k];
                        s[2 * i + 1] += G[k] * X[k];
                    }
                }
            }
            block_sums<2 * R>(s, sA, nw);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (on && r0 + i < nrows) {
                    const float rs = p.rstd[row0 + i], m1 = s[2 * i] * inv_d, m2 = s[2 * i + 1] * inv_d;
                    float* Dv = &d[i].x; const float *X = &xh[i].x, *G = &g[i].x;
#pragma unroll
                    for (int k = 0; k < 4; ++k) Dv[k] += rs * (G[k] - m1 - X[k] * m2);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            s[2 * i] = s[2 * i + 1] = 0.f;
            if (on && r0 + i < nrows) {
                const int64_t off = (row0 + i) * D + c;
                const float pm = p.pmean[row0 + i], pr = p.prstd[row0 + i];
                store4<float>(p.dx + off, make_float4(p.alpha * d[i].x, p.alpha * d[i].y, p.alpha * d[i].z, p.alpha * d[i].w));
                float4 kk = f4(1.f);
                if (p.thr16) kk = keep4_hashed(seed, off, p.thr16, p.inv_keep);
                float* A = &ah[i].x; float* G = &g[i].x;
                const float *Dv = &d[i].x, *K = &kk.x, *WP = &wp.x, *GT = &gt.x;
                float *AG = &ag.x, *APW = &apw.x;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    A[k] = (A[k] - pm) * pr;
                    const float dk = Dv[k] * K[k], da_ = dk * A[k];
                    AG[k] += da_ * WP[k];
                    APW[k] += da_ * GT[k];
                    G[k] = dk * GT[k] * WP[k];
                    s[2 * i] += G[k];
                    s[2 * i + 1] += G[k] * A[k];
                }
            }
        }
        block_sums<2 * R>(s, sB, nw);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (on && r0 + i < nrows) {
                const float pr = p.prstd[row0 + i], m1 = s[2 * i] * inv_d, m2 = s[2 * i + 1] * inv_d;
                float4 o;
                float* O = &o.x; const float *A = &ah[i].x, *G = &g[i].x;
                float* AB = &ab.x;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    O[k] = pr * (G[k] - m1 - A[k] * m2);
                    AB[k] += O[k];
                }
                store4<TA>(da + (row0 + i) * D + c, o);
            }
        }
        if (!NEXT && nw > 1) __syncthreads();  // (one buffer only in this form)
    }
    if (on) {
        float* o = p.ws + chunk * D + c;
        const int64_t plane = p.nchunk * D;
        store4<float>(o, ag);
        store4<float>(o + plane, apw);
        store4<float>(o + 2 * plane, ab);
        if constexpr (NEXT) {
            store4<float>(o + 3 * plane, aw);
            store4<float>(o + 4 * plane, ash);
            store4<float>(o + 5 * plane, asc);
        }
    }
}

// Folds the chunk partials in a fixed order.  Planes: 0 dgate, 1 dwp, 2 dbias, 3 dw, 4 dshift, 5 dscale; 0, 4 and 5 are sums
// per batch element (written), 1, 2 and 3 over all chunks (added to what is there).  Any output may be NULL.
struct PostReduceArgs {
    const float* ws;
    float* out[6];
    int64_t gate_stride, mod_stride, nchunk, cpb, B;
    int D, np;
};
__global__ void __launch_bounds__(TPB) post_norm_reduce_kernel(PostReduceArgs p) {
    const int nxb = (p.D + 255) / 256;
    const int64_t nbatch = (int64_t)nxb * p.B;
    const int64_t plane = p.nchunk * p.D;
    if ((int64_t)blockIdx.x < nbatch) {
        const int j = (int)(blockIdx.x % nxb) * 256 + threadIdx.x;
        const int64_t b = blockIdx.x / nxb;
        if (j >= p.D) return;
        for (int k = 0; k < p.np; ++k) {
            if ((k >= 1 && k <= 3) || !p.out[k]) continue;
            const float* base = p.ws + k * plane + b * p.cpb * p.D + j;
            float s = 0.f;
            for (int64_t c = 0; c < p.cpb; ++c) s += base[c * p.D];
            p.out[k][b * (k == 0 ? p.gate_stride : p.mod_stride) + j] = s;
        }
        return;
    }
    // 16 columns per block and plane: 16 row groups of 16 lanes
    __shared__ float red[16][17];
    const int64_t i = blockIdx.x - nbatch;
    const int ncb = (p.D + 15) / 16, k = 1 + (int)(i / ncb), col = (int)(i % ncb) * 16 + (threadIdx.x & 15);
    const int rg = threadIdx.x >> 4;
    float* out = p.out[k];
    if (!out) return;
    float s0 = 0.f, s1 = 0.f;
    if (col < p.D) {
        const float* base = p.ws + k * plane + col;
        int64_t c = rg;
        for (; c + 16 < p.nchunk; c += 32) { s0 += base[c * p.D]; s1 += base[(c + 16) * p.D]; }
        if (c < p.nchunk) s0 += base[c * p.D];
    }
    red[rg][threadIdx.x & 15] = s0 + s1;
    __syncthreads();
    if (rg == 0 && col < p.D) {
        float t = red[0][threadIdx.x];
        for (int r = 1; r < 16; ++r) t += red[r][threadIdx.x];
        out[col] += t;
    }
}

extern "C" int sedd_post_norm_residual_bwd(const float* dx1, const void* dh, const float* x1, const float* w,
                                           const void* scale, const float* mean, const float* rstd, const void* a,
                                           int a_dtype, const float* post_w, const void* gate, int mod_dtype,
                                           int64_t mod_stride, const float* post_mean, const float* post_rstd,
                                           float res_scale, float inv_keep, uint64_t seed, float p_drop, float* dx,
                                           void* da, float* ws, int64_t M, int64_t L, int D, sedd_stream_t stream) {
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
    p.mod_stride = mod_stride; p.nchunk = sedd_ln_bwd_chunks(M, L); p.L = L; p.alpha = res_scale; p.inv_keep = inv_keep;
    p.seed = seed; p.thr16 = (uint32_t)(p_drop * 65536.0f + 0.5f); p.D = D; p.CR = chunk_rows(M);
    const dim3 grid((unsigned)p.nchunk), block((unsigned)((D + 255) / 256 * 64));
    DISPATCH_DT(a_dtype, TA, DISPATCH_DT(mod_dtype, TM, {
        if (dh) hipLaunchKernelGGL((post_norm_bwd_kernel<TA, TM, true>), grid, block, 0, (hipStream_t)stream, p);
        else hipLaunchKernelGGL((post_norm_bwd_kernel<TA, TM, false>), grid, block, 0, (hipStream_t)stream, p);
    }));
    SEDD_LAUNCH_CHECK();
    return SEDD_OK;
}

extern "C" int sedd_post_norm_residual_bwd_reduce(const float* ws, float* dgate, int64_t dgate_stride, float* dshift,
                                                  float* dscale, int64_t dmod_stride, float* dpost_w, float* dbias,
                                                  float* dw, int64_t M, int64_t L, int D, sedd_stream_t stream) {
    SEDD_CHECK_ARG(M >= 0 && L > 0 && M % L == 0 && D > 0 && D % 4 == 0, "post_norm_residual_bwd_reduce: bad sizes");
    if (M == 0) return SEDD_OK;
    SEDD_CHECK_ARG(ws, "post_norm_residual_bwd_reduce: ws is null");
    PostReduceArgs p;
    p.ws = ws;
    float* outs[6] = {dgate, dpost_w, dbias, dw, dshift, dscale};
    for (int k = 0; k < 6; ++k) p.out[k] = outs[k];
    p.gate_stride = dgate_stride; p.mod_stride = dmod_stride; p.nchunk = sedd_ln_bwd_chunks(M, L); p.B = M / L; p.cpb = p.nchunk / p.B; p.D = D;
    p.np = (dw || dshift || dscale) ? 6 : 3;
    const int64_t blocks = (int64_t)((D + 255) / 256) * p.B + (int64_t)((D + 15) / 16) * (p.np == 6 ? 3 : 2);
    hipLaunchKernelGGL(post_norm_reduce_kernel, dim3((unsigned)blocks), dim3(TPB), 0, (hipStream_t)stream, p);
    SEDD_LAUNCH_CHECK();
    return SEDD_OK;
}

// Norm of the gradients over many tensors and their clipping in place.  Reference: processing/losses.py:65-66
// (torch.nn.utils.clip_grad_norm_ over the parameter list).
//   norm = sqrt(sum over tensors and elements of g^2),  g *= min(1, max_norm / (norm + 1e-6))
// HBM-bound: the gradients are read once for the norm and read and written once for the scaling.  The scaling goes through them
// backwards: what the norm read last still lies in the Infinity Cache (256 MB).  655 MB of fp32 gradients in 78 tensors: norm
// 115 us (5.7 TB/s), both 405 us (forwards 440 us); 302 MB 49 us (6.1 TB/s) and 172 us; 101 MB 19 us and 63 us.  Eight loads in
// flight per thread instead of the compiler's choice changed nothing (115 us).  Squares are summed in 64 bits: a 32-bit sum overflows at gradients
// of 1e19 and drops what is below 1e-23, and 64-bit adds are free beside the loads.  The partial sums have fixed places
// and are added in a fixed order (no atomics), so the norm is the same from run to run.
#include "common.h"

#define TPB 256
// The tensor table travels as a kernel argument (at most 4 KB): nothing is copied to the device and nothing has to
// outlive the call, so a captured launch holds its own table.  More tensors than this take several launches.
#define MT_MAX 176
struct TensorTable {
    int64_t chunk;           // elements per block
    int n, base;             // tensors; partial sum of block 0
    int backwards;           // the chunks of a tensor from its last to its first
    void* ptr[MT_MAX];
    int64_t numel[MT_MAX];
    int first[MT_MAX];       // first block of each tensor
    uint8_t bf16[MT_MAX];
};

// the tensor of this block (the last one whose first block is not behind it) and its element range
struct Piece {
    int t;
    int64_t lo, hi;
};
__device__ __forceinline__ Piece piece_of(const TensorTable& tab) {
    int lo = 0, hi = tab.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.first[mid] <= (int)blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    int64_t c = (int)blockIdx.x - tab.first[lo];
    if (tab.backwards) c = (tab.numel[lo] + tab.chunk - 1) / tab.chunk - 1 - c;
    const int64_t s = c * tab.chunk;
    const int64_t e = s + tab.chunk;
    return {lo, s, e < tab.numel[lo] ? e : tab.numel[lo]};
}
// elements of [lo, hi) before the first 16-byte boundary
template <typename T> __device__ __forceinline__ int64_t head_of(const T* p, int64_t lo, int64_t hi) {
    const int64_t h = (int64_t)((16 - ((uintptr_t)(p + lo) & 15)) & 15) / (int64_t)sizeof(T);
    return h < hi - lo ? h : hi - lo;
}

template <typename T> __device__ __forceinline__ double sumsq_piece(const T* p, int64_t lo, int64_t hi) {
    double s = 0.0;
    const int64_t h = head_of<T>(p, lo, hi);
    constexpr int E = 16 / sizeof(T);
    const int64_t v0 = lo + h, nv = (hi - v0) / E, tail = v0 + nv * E;
    for (int64_t i = lo + threadIdx.x; i < lo + h; i += TPB) { const double x = (double)to_f32<T>(p[i]); s += x * x; }
    for (int64_t i = threadIdx.x; i < nv; i += TPB) {
        union { uint4 u; T e[E]; } r;
        r.u = reinterpret_cast<const uint4*>(p + v0)[i];
#pragma unroll
        for (int k = 0; k < E; ++k) { const double x = (double)to_f32<T>(r.e[k]); s += x * x; }
    }
    for (int64_t i = tail + threadIdx.x; i < hi; i += TPB) { const double x = (double)to_f32<T>(p[i]); s += x * x; }
    return s;
}

__global__ void __launch_bounds__(TPB) multi_sumsq_kernel(TensorTable tab, double* __restrict__ ws) {
    __shared__ double red[TPB / 64];
    const Piece pc = piece_of(tab);
    double s = tab.bf16[pc.t] ? sumsq_piece<bf16_t>((const bf16_t*)tab.ptr[pc.t], pc.lo, pc.hi)
                              : sumsq_piece<float>((const float*)tab.ptr[pc.t], pc.lo, pc.hi);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) ws[tab.base + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// out[0] = norm, out[1] = clip coefficient
__global__ void __launch_bounds__(1024) multi_norm_kernel(const double* __restrict__ ws, int n, double max_norm,
                                                          float* __restrict__ out) {
    __shared__ double red[16];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) s += ws[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = red[0];
        for (int w = 1; w < 16; ++w) t += red[w];
        const double norm = sqrt(t), c = max_norm / (norm + 1e-6);
        out[0] = (float)norm;
        out[1] = c > 1.0 ? 1.0f : (float)c;  // a NaN norm stays one and reaches the gradients, as in torch
    }
}

template <typename T> __device__ __forceinline__ void scale_piece(T* p, int64_t lo, int64_t hi, float c) {
    const int64_t h = head_of<T>(p, lo, hi);
    constexpr int E = 16 / sizeof(T);
    const int64_t v0 = lo + h, nv = (hi - v0) / E, tail = v0 + nv * E;
    for (int64_t i = lo + threadIdx.x; i < lo + h; i += TPB) p[i] = from_f32<T>(to_f32<T>(p[i]) * c);
    for (int64_t i = threadIdx.x; i < nv; i += TPB) {
        union { uint4 u; T e[E]; } r;
        r.u = reinterpret_cast<const uint4*>(p + v0)[i];
#pragma unroll
        for (int k = 0; k < E; ++k) r.e[k] = from_f32<T>(to_f32<T>(r.e[k]) * c);
        reinterpret_cast<uint4*>(p + v0)[i] = r.u;
    }
    for (int64_t i = tail + threadIdx.x; i < hi; i += TPB) p[i] = from_f32<T>(to_f32<T>(p[i]) * c);
}

// round_coef: a bf16 tensor is multiplied by the coefficient as bf16 holds it, which is what `grad.mul_(coef)` does
__global__ void __launch_bounds__(TPB) multi_scale_kernel(TensorTable tab, const float* __restrict__ coef, int round_coef) {
    const float c = coef[0];
    if (c == 1.0f) return;  // (x * 1 is x)
    const Piece pc = piece_of(tab);
    if (tab.bf16[pc.t]) scale_piece<bf16_t>((bf16_t*)tab.ptr[pc.t], pc.lo, pc.hi, round_coef ? (float)(bf16_t)c : c);
    else scale_piece<float>((float*)tab.ptr[pc.t], pc.lo, pc.hi, c);
}

// At most MULTI_PIECES blocks over all tensors, besides one for the rest of each: 16384 elements per block or more.
#define MULTI_PIECES SEDD_MULTI_WS_DOUBLES
static int64_t chunk_for(const int64_t* numel, int n) {
    int64_t total = 0;
    for (int t = 0; t < n; ++t) total += numel[t];
    const int64_t c = ((total + MULTI_PIECES - 1) / MULTI_PIECES + 2047) / 2048 * 2048;
    return c < 16384 ? 16384 : c;
}
static int check_table(const char* nm, const void* const* ptrs, const int64_t* numel, const int32_t* dtype, int n) {
    SEDD_CHECK_ARG(n >= 0 && (n == 0 || (ptrs && numel && dtype)), "%s: bad tensor list", nm);
    for (int t = 0; t < n; ++t) {
        SEDD_CHECK_ARG(numel[t] >= 0 && (numel[t] == 0 || ptrs[t]), "%s: tensor %d is null", nm, t);
        SEDD_CHECK_ARG(dtype[t] == SEDD_F32 || dtype[t] == SEDD_BF16, "%s: tensor %d: unknown dtype %d", nm, t, dtype[t]);
        SEDD_CHECK_ARG((uintptr_t)ptrs[t] % (dtype[t] == SEDD_F32 ? 4 : 2) == 0, "%s: tensor %d is not aligned to its type", nm, t);
    }
    return SEDD_OK;
}
// calls f(table, blocks) for each launch; returns the number of blocks in all.  Backwards: from the last element of the last
// tensor to the first of the first
template <typename F>
static int for_each_table(const void* const* ptrs, const int64_t* numel, const int32_t* dtype, int n, bool backwards, F f) {
    TensorTable tab;
    tab.backwards = backwards;
    tab.chunk = chunk_for(numel, n);
    int base = 0, blocks = 0;
    tab.n = 0;
    for (int k = 0; k < n; ++k) {
        const int t = backwards ? n - 1 - k : k;
        if (numel[t] == 0) continue;
        tab.ptr[tab.n] = const_cast<void*>(ptrs[t]);
        tab.numel[tab.n] = numel[t];
        tab.bf16[tab.n] = dtype[t] == SEDD_BF16;
        tab.first[tab.n] = blocks;
        blocks += (int)((numel[t] + tab.chunk - 1) / tab.chunk);
        if (++tab.n == MT_MAX) {
            tab.base = base;
            f(tab, blocks);
            base += blocks;
            blocks = tab.n = 0;
        }
    }
    if (tab.n) {
        tab.base = base;
        f(tab, blocks);
        base += blocks;
    }
    return base;
}

extern "C" int sedd_multi_norm_clip_f64(const void* const* ptrs_host, const int64_t* numel_host, const int32_t* dtype_host,
                                        int ntensors, const double* max_norm_host, double* ws, int64_t ws_doubles, float* out,
                                        sedd_stream_t stream) {
    int rc = check_table("multi_norm_clip", ptrs_host, numel_host, dtype_host, ntensors);
    if (rc) return rc;
    SEDD_CHECK_ARG(ws && out && max_norm_host, "multi_norm_clip: null pointer");
    const double max_norm = *max_norm_host;
    SEDD_CHECK_ARG(max_norm >= 0.0, "multi_norm_clip: max_norm %f", max_norm);
    SEDD_CHECK_ARG(ws_doubles >= MULTI_PIECES + (int64_t)ntensors, "multi_norm_clip: workspace of %ld doubles, need %ld",
                   (long)ws_doubles, (long)MULTI_PIECES + ntensors);
    hipStream_t st = (hipStream_t)stream;
    const int n = for_each_table(ptrs_host, numel_host, dtype_host, ntensors, false, [&](const TensorTable& tab, int blocks) {
        hipLaunchKernelGGL(multi_sumsq_kernel, dim3(blocks), dim3(TPB), 0, st, tab, ws);
    });
    hipLaunchKernelGGL(multi_norm_kernel, dim3(1), dim3(1024), 0, st, ws, n, max_norm, out);
    SEDD_LAUNCH_CHECK();
    return SEDD_OK;
}
extern "C" int sedd_multi_norm_clip(const void* const* ptrs_host, const int64_t* numel_host, const int32_t* dtype_host,
                                    int ntensors, float max_norm, double* ws, int64_t ws_doubles, float* out,
                                    sedd_stream_t stream) {
    const double limit = max_norm;
    return sedd_multi_norm_clip_f64(ptrs_host, numel_host, dtype_host, ntensors, &limit, ws, ws_doubles, out, stream);
}

extern "C" int sedd_multi_scale(void* const* ptrs_host, const int64_t* numel_host, const int32_t* dtype_host, int ntensors,
                                const float* coef, int round_coef, sedd_stream_t stream) {
    int rc = check_table("multi_scale", ptrs_host, numel_host, dtype_host, ntensors);
    if (rc) return rc;
    SEDD_CHECK_ARG(coef, "multi_scale: null pointer");
    hipStream_t st = (hipStream_t)stream;
    const int n = for_each_table(ptrs_host, numel_host, dtype_host, ntensors, true, [&](const TensorTable& tab, int blocks) {
        hipLaunchKernelGGL(multi_scale_kernel, dim3(blocks), dim3(TPB), 0, st, tab, coef, round_coef);
    });
    if (n) SEDD_LAUNCH_CHECK();
    return SEDD_OK;
}

// Helpers of the kernels that work row by row over the residual stream: 4-wide vector access, dtype dispatch, the
// backward passes' row chunks and the counter-based dropout mask.
#pragma once
#include "common.h"

#define TPB 256
// rows per backward chunk (never straddles a batch element): 32, or 64 once there are enough rows to fill the chip
// with the longer chunks (fewer block prologues / partial-sum folds per byte)
__host__ __device__ static inline int chunk_rows(int64_t M) { return M >= 16384 ? 64 : 32; }

// ---- 4-wide vector access helpers -------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float4 load4(const T* p);
template <> __device__ __forceinline__ float4 load4<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <> __device__ __forceinline__ float4 load4<bf16_t>(const bf16_t* p) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    float4 o;
    o.x = __uint_as_float(r.x << 16);
    o.y = __uint_as_float(r.x & 0xffff0000u);
    o.z = __uint_as_float(r.y << 16);
    o.w = __uint_as_float(r.y & 0xffff0000u);
    return o;
}
template <typename T> __device__ __forceinline__ void store4(T* p, float4 v);
template <> __device__ __forceinline__ void store4<float>(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
template <> __device__ __forceinline__ void store4<bf16_t>(bf16_t* p, float4 v) {
    union { bf16_t h[4]; uint2 u; } c;
    c.h[0] = (bf16_t)v.x; c.h[1] = (bf16_t)v.y; c.h[2] = (bf16_t)v.z; c.h[3] = (bf16_t)v.w;
    *reinterpret_cast<uint2*>(p) = c.u;
}
__device__ __forceinline__ float4 f4(float a) { return make_float4(a, a, a, a); }
// v as it reads back after a store in type T
template <typename T> __device__ __forceinline__ float4 round4(float4 v) {
    if constexpr (sizeof(T) == 2)
        return make_float4((float)(bf16_t)v.x, (float)(bf16_t)v.y, (float)(bf16_t)v.z, (float)(bf16_t)v.w);
    else return v;
}

#define DISPATCH_DT(code, TT, ...)                              \
    do {                                                        \
        if ((code) == SEDD_F32) { using TT = float; __VA_ARGS__; } \
        else { using TT = bf16_t; __VA_ARGS__; }                \
    } while (0)

static bool dt_ok(int d) { return d == SEDD_F32 || d == SEDD_BF16; }

// Counter-based dropout: the keep decision of element e is a pure function of (seed, e), so forward and backward
// regenerate the same mask instead of writing / reading a [M, D] byte mask (and no torch RNG kernel runs per block).
// Two rounds of a 32-bit avalanche hash (lowbias32) per group of 4 consecutive elements give four 16-bit uniforms;
// keep <=> u16 >= thr16 with thr16 = round(p * 65536).
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x ^= x >> 16; x *= 0x7feb352dU; x ^= x >> 15; x *= 0x846ca68bU; x ^= x >> 16;
    return x;
}
// A seed with bit 63 set is INDIRECT: bits 47..0 hold the device address of a uint64 salt, bits 62..48 a site number, and
// the effective seed is salt + site * odd constant — a step captured in a HIP graph replays with fresh masks when the host
// (or a node of the graph) changes the salt in device memory, while the launch arguments stay what they were at capture.
__device__ __forceinline__ uint64_t resolve_seed(uint64_t seed) {
    if ((seed >> 63) == 0) return seed;
    const uint64_t salt = *reinterpret_cast<const uint64_t*>(seed & 0x0000FFFFFFFFFFFFull);
    return (salt + ((seed >> 48) & 0x7FFFull) * 0xD1B54A32D192ED03ull) & 0x7FFFFFFFFFFFFFFFull;
}
__device__ __forceinline__ float4 keep4_hashed(uint64_t seed, int64_t off, uint32_t thr16, float inv_keep) {
    const uint64_t q = (uint64_t)off >> 2;
    const uint32_t h0 = mix32(mix32((uint32_t)q ^ (uint32_t)seed) + (uint32_t)(q >> 32) + (uint32_t)(seed >> 32));
    const uint32_t h1 = mix32(h0 ^ 0x9e3779b9U);
    return make_float4((h0 & 0xffffU) >= thr16 ? inv_keep : 0.f, (h0 >> 16) >= thr16 ? inv_keep : 0.f,
                       (h1 & 0xffffU) >= thr16 ? inv_keep : 0.f, (h1 >> 16) >= thr16 ? inv_keep : 0.f);
}

// int8.cuh -- device helpers of the 8-bit serving operators.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "int8.h"

namespace evl {

// Two or four consecutive values of an activation tensor as f32 (exact for the 16-bit types).
__device__ __forceinline__ void unpack2(uint32_t w, __half, float& a, float& b) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x, b = f.y;
}
__device__ __forceinline__ void unpack2(uint32_t w, __nv_bfloat16, float& a, float& b) {
    a = __uint_as_float(w << 16), b = __uint_as_float(w & 0xffff0000u);
}
template <class T> __device__ __forceinline__ void load2(const T* p, float& a, float& b) {
    if constexpr (sizeof(T) == 4) {
        const float2 f = *reinterpret_cast<const float2*>(p);
        a = f.x, b = f.y;
    } else {
        unpack2(*reinterpret_cast<const uint32_t*>(p), T{}, a, b);
    }
}
template <class T> __device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
    if constexpr (sizeof(T) == 4) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        unpack2(w.x, T{}, v[0], v[1]);
        unpack2(w.y, T{}, v[2], v[3]);
    }
}
template <class T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 f = reinterpret_cast<const float4*>(p)[0], g = reinterpret_cast<const float4*>(p)[1];
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w, v[4] = g.x, v[5] = g.y, v[6] = g.z, v[7] = g.w;
    } else {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        unpack2(w.x, T{}, v[0], v[1]);
        unpack2(w.y, T{}, v[2], v[3]);
        unpack2(w.z, T{}, v[4], v[5]);
        unpack2(w.w, T{}, v[6], v[7]);
    }
}
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
// the output type's one rounding (to nearest, ties to even)
template <class T> __device__ __forceinline__ T from_f32(float x) {
    if constexpr (sizeof(T) == 4) return x;
    else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}
template <class T> __device__ __forceinline__ void store2(T* p, float a, float b) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float2*>(p) = make_float2(a, b);
    } else {
        T v[2] = {from_f32<T>(a), from_f32<T>(b)};
        *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<uint32_t*>(v);
    }
}

template <class T> __device__ __forceinline__ void store4(T* p, const float (&x)[4]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        T v[4] = {from_f32<T>(x[0]), from_f32<T>(x[1]), from_f32<T>(x[2]), from_f32<T>(x[3])};
        *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(v);
    }
}

// A launch that may begin while the kernel before it in the stream ends: every kernel of these operators
// first waits (pdl_wait, every CTA, before it reads or writes anything of the caller's) until that
// kernel has ended and its writes can be seen, and most let the next one begin once they hold their own
// resources (pdl_launch_dependents). Launching, and the product's barriers and tensor memory, then cost no time of their own: the
// attention half of a layer, one token over 600 positions, took 36.8 us without and 34.4 with it; 32 over 2100, 65.8 and 63.9.
template <class... P>
cudaError_t launch_chained(void (*kernel)(P...), dim3 grid, uint32_t threads, uint32_t smem, cudaStream_t s, const P&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// |x| as bits: unsigned order is the order of magnitudes, with the infinity above every
// finite number and NaN above it, so one integer maximum finds both the largest magnitude
// and whether all values are finite.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// the scale of a group of values whose largest magnitude has these bits
__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    const float a = __uint_as_float(amax_bits);
    return a < kInt8Tiny ? 0.f : __fdiv_rn(a, 127.f);
}
// 1 / scale for codes; 0 where the group holds zeros or is not finite
__device__ __forceinline__ float inverse_of(float scale) { return scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f; }
// The code of x in the low byte: adding 1.5 * 2^23 rounds the product (|x inv| < 127.5, ties
// to even) into the last mantissa bits. `inv` 0 must not meet an infinite or NaN x.
__device__ __forceinline__ uint32_t code_bits(float x, float inv) {
    return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f));
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

__device__ __forceinline__ void flag_error(int32_t* err, int code) {
    if (err) atomicMax(err, code);
}

// The sequence of token t: the last s with cu[s] <= t, found 32 boundaries at a time by the
// whole warp; -1 if there is none. cu is read within [0, n_seqs].
__device__ __forceinline__ int find_seq(const int32_t* cu, uint32_t n_seqs, int32_t t, uint32_t lane) {
    uint32_t lo = 0, n = n_seqs;
    while (n > 32) {
        const uint32_t step = (n + 31) / 32, at = lane * step;
        const bool in = at < n && cu[lo + at] <= t;
        const uint32_t hit = __popc(__ballot_sync(0xffffffffu, in));
        if (!hit) return -1;
        lo += (hit - 1) * step;
        n = min(step, n - (hit - 1) * step);
    }
    const bool in = lane < n && cu[lo + lane] <= t;
    const uint32_t hit = __popc(__ballot_sync(0xffffffffu, in));
    return hit ? (int)(lo + hit - 1) : -1;
}

}  // namespace evl

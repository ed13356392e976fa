// Element types of the token operators: conversions to and from fp32 and 16-byte vectors of values.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>
#include "common.cuh"

namespace msnh {

// First thing in a kernel that is launched while the one before it may still run: waits until that one has ended and its writes are
// visible, then lets the next launch be scheduled. In this order the next one may take it that everything before this kernel has ended.
__device__ __forceinline__ void pdl_enter() {
    pdl_wait();
    pdl_launch_dependents();
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__nv_fp8_e4m3 v) { return static_cast<float>(v); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two values to the nearest 8-bit ones (ties to even), the first in the low byte
__device__ __forceinline__ uint16_t to_e4m3x2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// kVec values of T in 16 bytes
template <typename T> struct Vec16 {
    static constexpr int kVec = 16 / sizeof(T);
    __device__ __forceinline__ static void unpack(const uint4 &raw, float (&v)[kVec]) {
        const T *p = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = to_float(p[i]);
    }
    __device__ __forceinline__ static uint4 pack(const float (&v)[kVec]) {
        uint4 raw;
        T *p = reinterpret_cast<T *>(&raw);
#pragma unroll
        for (int i = 0; i < kVec; ++i) p[i] = from_float<T>(v[i]);
        return raw;
    }
};

}  // namespace msnh

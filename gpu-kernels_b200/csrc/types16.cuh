// types16.cuh — the 16-bit element types of the linear and mixture-of-experts operators:
// 16-byte vectors of eight values, widened to fp32 for every computation and rounded once.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace nvfp4 {

template <typename T>
struct Type16;

template <>
struct Type16<__nv_bfloat16> {
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t *>(&h);
    }
    static __device__ __forceinline__ float load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ __nv_bfloat16 round(float a) { return __float2bfloat16_rn(a); }
};

template <>
struct Type16<__half> {
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t *>(&h);
    }
    static __device__ __forceinline__ float load(const __half *p) { return __half2float(*p); }
    static __device__ __forceinline__ __half round(float a) { return __float2half_rn(a); }
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4 &v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 p = Type16<T>::unpack(w[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(Type16<T>::pack(f[0], f[1]), Type16<T>::pack(f[2], f[3]), Type16<T>::pack(f[4], f[5]),
                      Type16<T>::pack(f[6], f[7]));
}

}  // namespace nvfp4

// Tensor elements as fp32, single ones and neighbours through wide accesses.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace rwkv7 {

__device__ __forceinline__ float ldf(const float *p) { return *p; }
__device__ __forceinline__ float ldf(const __nv_bfloat16 *p) {
    return __uint_as_float((uint32_t)*reinterpret_cast<const unsigned short *>(p) << 16);
}
__device__ __forceinline__ void stf(float *p, float x) { *p = x; }
__device__ __forceinline__ void stf(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void st8(float *p, const float (&v)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void st8(__nv_bfloat16 *p, const float (&v)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
}
// Four elements to shared memory as fp32; N (2 or 4) neighbours.
__device__ __forceinline__ void st4(float *to, const float *from) { *reinterpret_cast<float4 *>(to) = *reinterpret_cast<const float4 *>(from); }
__device__ __forceinline__ void st4(float *to, const __nv_bfloat16 *from) {
    const uint2 u = *reinterpret_cast<const uint2 *>(from);
    *reinterpret_cast<float4 *>(to) = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                                                  __uint_as_float(u.y & 0xffff0000u));
}
template <int N>
__device__ __forceinline__ void ldn(float (&v)[N], const float *p) {
    if constexpr (N == 4) {
        const float4 x = *reinterpret_cast<const float4 *>(p);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
        const float2 x = *reinterpret_cast<const float2 *>(p);
        v[0] = x.x; v[1] = x.y;
    }
}
template <int N>
__device__ __forceinline__ void stn(float *p, const float (&v)[N]) {
    if constexpr (N == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
}
template <int N>
__device__ __forceinline__ void stn(__nv_bfloat16 *p, const float (&v)[N]) {
    if constexpr (N == 4) *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]));
    else *reinterpret_cast<uint32_t *>(p) = pack_bf2(v[0], v[1]);
}

}  // namespace rwkv7

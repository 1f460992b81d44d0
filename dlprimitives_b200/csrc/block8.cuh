// What the operators with typed operands share: element types, eight consecutive elements as fp32, and the 8-bit form of a block.
#pragma once
#include "common.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace dlp {

constexpr int SCALE_BLOCK = 128;                  // elements under one scale

inline bool is_real_type(int t) { return t == DLP_TYPE_F32 || t == DLP_TYPE_F16 || t == DLP_TYPE_BF16; }
inline int type_size(int t) { return t == DLP_TYPE_F32 ? 4 : (t == DLP_TYPE_E4M3 ? 1 : 2); }
inline bool aligned_to(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template<typename T> __device__ __forceinline__ T from_float(float v);
template<> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template<> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template<> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight consecutive elements; VEC: 16-byte accesses, all eight there (p aligned to 16 bytes).  Otherwise one by one, the first `count` of them, and
// zeros for the rest.
template<typename T, bool VEC> __device__ __forceinline__ void load8(const T *p, int count, float (&v)[8])
{
    if(VEC) {
        union { uint4 w[sizeof(T) / 2]; T e[8]; } u;
        #pragma unroll
        for(int i = 0; i < int(sizeof(T)) / 2; i++) u.w[i] = ld_plain(reinterpret_cast<const uint4 *>(p) + i);
        #pragma unroll
        for(int j = 0; j < 8; j++) v[j] = to_float(u.e[j]);
    }
    else {
        #pragma unroll
        for(int j = 0; j < 8; j++) v[j] = j < count ? to_float(ld_plain(p + j)) : 0.0f;
    }
}
template<typename T, bool VEC> __device__ __forceinline__ void store8(T *p, int count, const float (&v)[8])
{
    if(VEC) {
        union { uint4 w[sizeof(T) / 2]; T e[8]; } u;
        #pragma unroll
        for(int j = 0; j < 8; j++) u.e[j] = from_float<T>(v[j]);
        #pragma unroll
        for(int i = 0; i < int(sizeof(T)) / 2; i++) reinterpret_cast<uint4 *>(p)[i] = u.w[i];
    }
    else {
        #pragma unroll
        for(int j = 0; j < 8; j++)
            if(j < count) p[j] = from_float<T>(v[j]);
    }
}

// The 8-bit form of a block of values v is a scale s = max|v| / 448 (448: the largest e4m3) and the numbers e4m3(v / s): the largest value
// meets the largest number.  s is no smaller than 2^-126, so that a block of zeros, or of subnormals, has a finite 1 / s; a NaN or
// an infinity in the block makes s NaN or infinite and with it whatever is computed from the block.
// Largest magnitude of the thread's values, as bits: magnitudes are ordered as their bits are, a NaN above all of them.
__device__ __forceinline__ unsigned magnitude_bits(const float (&v)[8])
{
    unsigned m = 0;
    #pragma unroll
    for(int j = 0; j < 8; j++) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    return m;
}
__device__ __forceinline__ float block_scale(unsigned magnitude)
{
    const float s = __uint_as_float(magnitude) / 448.0f;
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}
// Eight numbers of the block, the first in the lowest byte.  v * (1 / s) is within one and a half units in the last place of v / s in fp32, a
// twenty-thousandth part of a step of e4m3: only a value that close to the middle of two numbers may go to the other one.
__device__ __forceinline__ uint2 pack_e4m3(const float (&v)[8], float inverse_scale)
{
    uint32_t w[2];
    #pragma unroll
    for(int i = 0; i < 2; i++) {
        unsigned short a, b;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a) : "f"(v[4 * i + 1] * inverse_scale), "f"(v[4 * i] * inverse_scale));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(v[4 * i + 3] * inverse_scale), "f"(v[4 * i + 2] * inverse_scale));
        w[i] = uint32_t(a) | uint32_t(b) << 16;
    }
    return make_uint2(w[0], w[1]);
}
// VEC: one 8-byte store (p aligned to 8 bytes)
template<bool VEC> __device__ __forceinline__ void store_e4m3(unsigned char *p, int count, uint2 w)
{
    if(VEC) *reinterpret_cast<uint2 *>(p) = w;
    else {
        #pragma unroll
        for(int j = 0; j < 8; j++)
            if(j < count) p[j] = (unsigned char)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
    }
}

} // namespace dlp

// What the operators with typed operands share: element types, eight consecutive elements as fp32, and the 8-bit form of a block.
#pragma once
#include "common.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>

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

// Two fp32 operations to an instruction: what bounds these kernels beside memory is the issue of instructions.
struct Pair { unsigned long long v; };
__device__ __forceinline__ Pair pair(float a, float b)
{
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ Pair both(float a) { return pair(a, a); }
__device__ __forceinline__ void apart(Pair r, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r.v)); }
__device__ __forceinline__ Pair operator*(Pair a, Pair b)
{
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b)
{
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c)
{
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// ---- Rows.  What one is known to be: WHOLE, on a 16-byte boundary and a multiple of eight elements long, as all others of the call: a lane has eight
// consecutive elements, all there or none, in 16-byte pieces.  Or ANY: a lane has every 32nd of 256 elements, so that whatever the boundaries a
// warp's load or store is of consecutive ones; where all 256 are there, without a condition (a condition at each load holds the loads apart: weights
// 11000 x 4097 56 us for 41).  (Those in 16-byte pieces too, with the words shifted between lanes to where they belong, took more
// instructions than the loads that they saved, and twice the registers: norm of 4000 x 5001 82 us for 41, of 30000 x 777 90 for 53.)
enum { ROW_WHOLE, ROW_ANY };
template<typename T> constexpr int WORDS = 2 * int(sizeof(T));                // 32-bit words of eight elements

// A lane's eight of 256 elements from column c0 of a row, in two steps, so that a thread can ask for all it reads before it waits for any of it: ask(),
// and settle() when the values are used: zeros beyond the row's end.
template<typename T, int KIND> struct Row8 {
    union { uint4 w[WORDS<T> / 4]; T e[8]; };
    __device__ __forceinline__ void ask(const T *row, int c0, int lane, int cols)
    {
        if constexpr(KIND == ROW_WHOLE) {
            const int c = c0 + lane * 8;
            if(c < cols) {
                #pragma unroll
                for(int i = 0; i < WORDS<T> / 4; i++) w[i] = ld_plain(reinterpret_cast<const uint4 *>(row + c) + i);
            }
            else {
                #pragma unroll
                for(int i = 0; i < WORDS<T> / 4; i++) w[i] = make_uint4(0, 0, 0, 0);
            }
        }
        else if(c0 + 256 <= cols) {
            #pragma unroll
            for(int j = 0; j < 8; j++) e[j] = ld_plain(row + c0 + lane + 32 * j);
        }
        else {
            #pragma unroll
            for(int j = 0; j < 8; j++) e[j] = c0 + lane + 32 * j < cols ? ld_plain(row + c0 + lane + 32 * j) : from_float<T>(0.0f);
        }
    }
    __device__ __forceinline__ void settle(float (&v)[8]) const
    {
        #pragma unroll
        for(int j = 0; j < 8; j++) v[j] = to_float(e[j]);
    }
};
template<typename T, int KIND> __device__ __forceinline__ void store8(T *row, int c0, int lane, int cols, const float (&v)[8])
{
    if constexpr(KIND == ROW_WHOLE) {
        union { uint32_t w[WORDS<T>]; T e[8]; } u;
        #pragma unroll
        for(int j = 0; j < 8; j++) u.e[j] = from_float<T>(v[j]);
        const int c = c0 + lane * 8;
        if(c < cols) {
            #pragma unroll
            for(int g = 0; g < WORDS<T> / 4; g++)
                reinterpret_cast<uint4 *>(row + c)[g] = make_uint4(u.w[4 * g], u.w[4 * g + 1], u.w[4 * g + 2], u.w[4 * g + 3]);
        }
    }
    else if(c0 + 256 <= cols) {
        #pragma unroll
        for(int j = 0; j < 8; j++) row[c0 + lane + 32 * j] = from_float<T>(v[j]);
    }
    else {
        #pragma unroll
        for(int j = 0; j < 8; j++)
            if(c0 + lane + 32 * j < cols) row[c0 + lane + 32 * j] = from_float<T>(v[j]);
    }
}

// The 8-bit form of a block of values v is a scale s = max|v| / 448 (448: the largest e4m3) and the numbers e4m3(v / s): the largest value
// meets the largest number.  s is no smaller than 2^-126, so that a block of zeros, or of subnormals, has a finite 1 / s; a NaN or
// an infinity in the block makes s NaN or infinite and with it whatever is computed from the block.
// Largest magnitude of the thread's values from `first` on, as bits (magnitudes are ordered as their bits are); a NaN if one of them is.
template<int N = 8> __device__ __forceinline__ unsigned magnitude_bits(const float (&v)[8], int first = 0)
{
    float m = 0.0f;
    #pragma unroll
    for(int j = 0; j < N; j += 2) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(v[first + j]), "f"(v[first + j + 1]));
    return __float_as_uint(m);
}
// The quotient by 448 is the product with its reciprocal, corrected by the remainder: rounded as a division would, without its length.
__device__ __forceinline__ float block_scale(unsigned magnitude)
{
    const float m = __uint_as_float(magnitude);
    const float s0 = m * (1.0f / 448.0f), s = fmaf(fmaf(-448.0f, s0, m), 1.0f / 448.0f, s0);
    return m < 0x1.cp-118f ? 0x1p-126f : (magnitude < 0x7f800000u ? s : m);                // under 448 * 2^-126: 2^-126; infinite and NaN stay
}
// Four numbers of the block, the first in the lowest byte: v / s, by a product with the approximate 1 / s and a correction of its remainder (a Newton step
// of the quotient, after which it is the rounded one but for rare last units), then to the nearest e4m3, ties to even.
struct Quotient {
    Pair back, inv;
    __device__ __forceinline__ explicit Quotient(float scale)
    {
        // (an infinite scale takes the correction out: finite values give 0, infinite ones and NaN a NaN)
        back = both(scale < __int_as_float(0x7f800000) ? -scale : 0.0f);
        float inverse;
        asm("rcp.approx.f32 %0, %1;" : "=f"(inverse) : "f"(scale));
        inv = both(inverse);
    }
    __device__ __forceinline__ uint32_t pack(const float (&v)[8], int first) const
    {
        unsigned short part[2];
        #pragma unroll
        for(int i = 0; i < 2; i++) {
            const Pair x = pair(v[first + 2 * i], v[first + 2 * i + 1]), q0 = x * inv;
            float lo, hi;
            apart(fma2(fma2(back, q0, x), inv, q0), lo, hi);
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(part[i]) : "f"(hi), "f"(lo));
        }
        return uint32_t(part[0]) | uint32_t(part[1]) << 16;
    }
};
// The 8-bit form of a warp's 256 elements in blocks of one row; `scales` at the row's first one.
template<int KIND> __device__ __forceinline__ void store_e4m3(unsigned char *row, float *scales, long long scale_stride, int c0, int lane, int cols, const float (&v)[8])
{
    if constexpr(KIND == ROW_WHOLE) {
        const int c = c0 + lane * 8;
        const float s = block_scale(__reduce_max_sync(lane < 16 ? 0xffffu : 0xffff0000u, magnitude_bits(v)));
        if((lane & 15) == 0 && c < cols) scales[(c / SCALE_BLOCK) * scale_stride] = s;
        const Quotient by(s);
        const uint2 q = make_uint2(by.pack(v, 0), by.pack(v, 4));
        if(c < cols) *reinterpret_cast<uint2 *>(row + c) = q;
    }
    else {
        #pragma unroll
        for(int h = 0; h < 2; h++) {                         // elements 4 h to 4 h + 3 are of block h of the two
            const int c = c0 + h * SCALE_BLOCK + lane;
            const float s = block_scale(__reduce_max_sync(0xffffffffu, magnitude_bits<4>(v, 4 * h)));
            if(lane == 0 && c < cols) scales[(c / SCALE_BLOCK) * scale_stride] = s;
            const uint32_t q = Quotient(s).pack(v, 4 * h);
            if(c0 + 256 <= cols) {
                #pragma unroll
                for(int j = 0; j < 4; j++) row[c + 32 * j] = (unsigned char)(q >> (8 * j));
            }
            else {
                #pragma unroll
                for(int j = 0; j < 4; j++)
                    if(c + 32 * j < cols) row[c + 32 * j] = (unsigned char)(q >> (8 * j));
            }
        }
    }
}

} // namespace dlp

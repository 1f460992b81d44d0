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

// ---- Rows, eight consecutive elements to a lane: lane l of WIDTH (32, or 16: two rows to a warp) has the elements from column c = c0 + 8 l.
// Memory is read and written in 16-byte pieces on their boundaries, also where a row starts off one (any length and stride of 16-bit elements):
// then a lane's elements lie in its own pieces and the first one of the lane after it, m elements on.  Stores that a row's ends cut go element by element,
// and so do loads of pieces that reach beyond the tensor.  All lanes take part (with c >= cols where there is nothing).
template<typename T> constexpr int PIECE = 16 / int(sizeof(T));               // elements of a piece
template<typename T> constexpr int WORDS = 2 * int(sizeof(T));                // 32-bit words of eight elements
template<typename T> __device__ __forceinline__ int off_boundary(const T *row) { return int(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T)); }

// N words from `bytes` (even, under 16) on in N + 4
template<int N> __device__ __forceinline__ void shift_words(uint32_t (&w)[N + 4], int bytes)
{
    #pragma unroll
    for(int i = 0; i < N + 2; i++) w[i] = bytes & 8 ? w[i + 2] : w[i];
    #pragma unroll
    for(int i = 0; i < N + 1; i++) w[i] = bytes & 4 ? w[i + 1] : w[i];
    #pragma unroll
    for(int i = 0; i < N; i++) w[i] = bytes & 2 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
}
// What a row is known to be: WHOLE, on a 16-byte boundary and a multiple of eight elements long, so that a lane's eight are all there or none; or ANY.
enum { ROW_WHOLE, ROW_ANY };
// A load in two steps, so that a thread can ask for all it reads before it waits for any of it: ask(), and settle() when the values are used.
template<typename T, int KIND, int WIDTH = 32> struct Row8 {
    uint32_t w[WORDS<T> + (KIND == ROW_ANY ? 4 : 0)];
    static __device__ __forceinline__ int lane() { return threadIdx.x & (WIDTH - 1); }
    __device__ __forceinline__ void put(int i, uint4 v) { w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w; }
    // the elements of a piece that the row's ends cut
    __device__ __forceinline__ void cut_piece(int i, const T *row, int e, int cols)
    {
        union { T e[PIECE<T>]; uint4 w; } u;
        u.w = make_uint4(0, 0, 0, 0);
        if(e >= 0 && e + PIECE<T> <= cols) u.w = ld_plain(reinterpret_cast<const uint4 *>(row + e));
        else {
            #pragma unroll
            for(int k = 0; k < PIECE<T>; k++)
                if(e + k >= 0 && e + k < cols) u.e[k] = ld_plain(row + e + k);
        }
        put(i, u.w);
    }
    // from, to: what may be read, the memory between the first row's start and the last one's end (a piece that a row's end cuts is read whole where
    // it lies in it)
    __device__ __forceinline__ void ask(const T *row, int c, int cols, const T *from, const T *to)
    {
        if constexpr(KIND == ROW_WHOLE) {
            if(c < cols) {
                #pragma unroll
                for(int i = 0; i < WORDS<T>; i += 4) put(i, ld_plain(reinterpret_cast<const uint4 *>(row + c) + i / 4));
            }
            else {
                #pragma unroll
                for(int i = 0; i < WORDS<T>; i += 4) put(i, make_uint4(0, 0, 0, 0));
            }
        }
        else {
            const int m = off_boundary(row), first = c - lane() * 8;
            if(row + first - m >= from && row + first - m + WIDTH * 8 + PIECE<T> <= to) {
                const uint4 *p = reinterpret_cast<const uint4 *>(row + c - m);
                if(c - m < cols) {
                    #pragma unroll
                    for(int i = 0; i < WORDS<T>; i += 4) put(i, ld_plain(p + i / 4));
                }
                if(lane() == WIDTH - 1 && c - m + 8 < cols) put(WORDS<T>, ld_plain(p + WORDS<T> / 4));
            }
            else {
                #pragma unroll
                for(int i = 0; i < WORDS<T>; i += 4) cut_piece(i, row, c - m + i / 4 * PIECE<T>, cols);
                if(lane() == WIDTH - 1) cut_piece(WORDS<T>, row, c - m + 8, cols);
            }
        }
    }
    // the eight elements, zeros beyond the row's end; all lanes take part
    __device__ __forceinline__ void settle(const T *row, int c, int cols, float (&v)[8])
    {
        if constexpr(KIND == ROW_ANY) {
            const int m = off_boundary(row);
            #pragma unroll
            for(int i = 0; i < 4; i++) {
                const uint32_t next = __shfl_down_sync(0xffffffffu, w[i], 1, WIDTH);
                w[WORDS<T> + i] = lane() == WIDTH - 1 ? w[WORDS<T> + i] : next;
            }
            shift_words<WORDS<T>>(w, m * int(sizeof(T)));
        }
        union { uint32_t w[WORDS<T>]; T e[8]; } u;
        #pragma unroll
        for(int i = 0; i < WORDS<T>; i++) u.w[i] = w[i];
        #pragma unroll
        for(int j = 0; j < 8; j++) v[j] = to_float(u.e[j]);
        if(KIND == ROW_ANY && c + 8 > cols) {
            #pragma unroll
            for(int j = 0; j < 8; j++) v[j] = c + j < cols ? v[j] : 0.0f;
        }
    }
};

template<typename T> __device__ __forceinline__ void store_piece(T *row, int e, int from, int cols, const uint32_t *w)
{
    if(e >= from && e + PIECE<T> <= cols) *reinterpret_cast<uint4 *>(row + e) = make_uint4(w[0], w[1], w[2], w[3]);
    else {
        union { uint32_t w[4]; T e[PIECE<T>]; } u;
        #pragma unroll
        for(int i = 0; i < 4; i++) u.w[i] = w[i];
        #pragma unroll
        for(int i = 0; i < PIECE<T>; i++)
            if(e + i >= from && e + i < cols) row[e + i] = u.e[i];
    }
}
template<typename T> __device__ __forceinline__ void store_words_off(T *row, int c, int cols, const uint32_t (&w)[WORDS<T>])
{
    // a lane stores the pieces that begin with the last m elements of the lane before; the first and the last lane what is theirs of the outer ones
    const int m = off_boundary(row), lane = threadIdx.x & 31;
    uint32_t all[WORDS<T> + 4];
    #pragma unroll
    for(int i = 0; i < WORDS<T>; i++) all[i + 4] = w[i];
    #pragma unroll
    for(int i = 0; i < 4; i++) all[i] = __shfl_up_sync(0xffffffffu, w[WORDS<T> - 4 + i], 1);
    shift_words<WORDS<T>>(all, 16 - m * int(sizeof(T)));
    #pragma unroll
    for(int g = 0; g < WORDS<T> / 4; g++) store_piece(row, c - m + g * PIECE<T>, lane == 0 ? c : 0, cols, all + g * 4);
    if(lane == 31) {
        union { uint32_t w[4]; T e[PIECE<T>]; } u;
        #pragma unroll
        for(int i = 0; i < 4; i++) u.w[i] = w[WORDS<T> - 4 + i];
        #pragma unroll
        for(int i = 0; i < PIECE<T>; i++)
            if(i >= PIECE<T> - m && c + 8 - PIECE<T> + i < cols) row[c + 8 - PIECE<T> + i] = u.e[i];
    }
}
template<typename T, int KIND> __device__ __forceinline__ void store8(T *row, int c, int cols, const float (&v)[8])
{
    union { uint32_t w[WORDS<T>]; T e[8]; } u;
    #pragma unroll
    for(int j = 0; j < 8; j++) u.e[j] = from_float<T>(v[j]);
    if constexpr(KIND == ROW_WHOLE) {
        if(c < cols) {
            #pragma unroll
            for(int g = 0; g < WORDS<T> / 4; g++)
                reinterpret_cast<uint4 *>(row + c)[g] = make_uint4(u.w[4 * g], u.w[4 * g + 1], u.w[4 * g + 2], u.w[4 * g + 3]);
        }
    }
    else if(off_boundary(row) != 0) store_words_off(row, c, cols, u.w);
    else {
        #pragma unroll
        for(int g = 0; g < WORDS<T> / 4; g++) store_piece(row, c + g * PIECE<T>, 0, cols, u.w + g * 4);
    }
}

// The 8-bit form of a block of values v is a scale s = max|v| / 448 (448: the largest e4m3) and the numbers e4m3(v / s): the largest value
// meets the largest number.  s is no smaller than 2^-126, so that a block of zeros, or of subnormals, has a finite 1 / s; a NaN or
// an infinity in the block makes s NaN or infinite and with it whatever is computed from the block.
// Largest magnitude of the thread's values, as bits (magnitudes are ordered as their bits are); a NaN if one of them is.
__device__ __forceinline__ unsigned magnitude_bits(const float (&v)[8])
{
    float m = 0.0f;
    #pragma unroll
    for(int j = 0; j < 8; j += 2) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(v[j]), "f"(v[j + 1]));
    return __float_as_uint(m);
}
// The quotient by 448 is the product with its reciprocal, corrected by the remainder: rounded as a division would, without its length.
__device__ __forceinline__ float block_scale(unsigned magnitude)
{
    const float m = __uint_as_float(magnitude);
    const float s0 = m * (1.0f / 448.0f), s = fmaf(fmaf(-448.0f, s0, m), 1.0f / 448.0f, s0);
    return m < 5.2656e-36f ? 1.17549435e-38f : (magnitude < 0x7f800000u ? s : m);          // 448 * 2^-126 (under it 2^-126); infinite and NaN stay
}
// Eight numbers of the block, the first in the lowest byte: v / s, by a product with the approximate 1 / s and a correction of its remainder (a Newton step
// of the quotient, after which it is the rounded one but for rare last units), then to the nearest e4m3, ties to even.
__device__ __forceinline__ uint2 pack_e4m3(const float (&v)[8], float scale)
{
    // (an infinite scale takes the correction out: finite values give 0, infinite ones and NaN a NaN)
    const Pair back = both(scale < __int_as_float(0x7f800000) ? -scale : 0.0f);
    float inverse;
    asm("rcp.approx.f32 %0, %1;" : "=f"(inverse) : "f"(scale));
    const Pair inv = both(inverse);
    unsigned short part[4];
    #pragma unroll
    for(int i = 0; i < 4; i++) {
        const Pair x = pair(v[2 * i], v[2 * i + 1]), q0 = x * inv;
        float lo, hi;
        apart(fma2(fma2(back, q0, x), inv, q0), lo, hi);
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(part[i]) : "f"(hi), "f"(lo));
    }
    return make_uint2(uint32_t(part[0]) | uint32_t(part[1]) << 16, uint32_t(part[2]) | uint32_t(part[3]) << 16);
}
// The row is on an 8-byte boundary and a multiple of eight long (ROW_WHOLE), or anything.
template<int KIND> __device__ __forceinline__ void store_e4m3(unsigned char *row, int c, int cols, uint2 w)
{
    if(KIND == ROW_WHOLE ? c < cols : (reinterpret_cast<uintptr_t>(row) % 8 == 0 && c + 8 <= cols)) *reinterpret_cast<uint2 *>(row + c) = w;
    else if(KIND != ROW_WHOLE) {
        #pragma unroll
        for(int j = 0; j < 8; j++)
            if(c + j < cols) row[c + j] = (unsigned char)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
    }
}

} // namespace dlp

// Root-mean-square norm of rows, with the addition of a residual before it and an 8-bit form of the result:
//     h = x + residual,   y = h / sqrt(mean(h^2) + eps) * weight.
// A block of threads has a row in its registers between the sum of squares and the outputs, so that a row is read once (up to 32768 columns; longer
// ones are read a second time, from L2).  What bounds it is memory: 8192 x 5120 bf16 with residual and 8-bit output take 52 us, 5.7 TB/s of the
// 6.5 that a copy reaches (82 us before a row stayed in registers and the next one's loads were under way, 60 before the arithmetic went two values to an
// instruction); 8192 x 4096 fp32 without a residual, 8-bit output, 39 us, 4.3 TB/s (45 with the weights kept, for which there are no registers: 36 bytes a
// thread are spilled as it is, and 760 in fp32 rows of 16385 to 32768).  Rows off 16-byte boundaries are read element by element, a warp's 32 at a
// time, and then it is the number of loads: 4000 x 5001 with residual and 8-bit output bf16 41 us, 3.4 TB/s, fp32 49, 5.3.  1500 x 15001 63 us (68 in 512
// threads).  One row of 4096: 1.8 us, the launch.
#include "block8.cuh"

namespace dlp {
namespace {

struct NormArgs {
    const void *x, *residual, *weight;
    void *total, *y;
    float *scales;
    long long x_stride, residual_stride, total_stride, y_stride, scale_stride;
    int cols, y_type;
    float eps;
};

// Threads of a block at most.  (ANY: see Row8.  Two pieces to a thread and its registers at 64 fill an SM with 1024 threads, in one block or more.)
constexpr int MAX_THREADS = 512;
constexpr int most_threads(int nv, int kind) { return kind == ROW_ANY && nv <= 2 ? 1024 : MAX_THREADS; }

// Sum over the block; `part` is used in turn from call to call, so that one barrier a call is enough.
template<int WARPS> __device__ __forceinline__ float block_sum(float v, float (&part)[WARPS])
{
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    #pragma unroll
    for(int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if(warps == 1) return v;
    if(lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (lane & (WARPS - 1)) < warps ? part[lane & (WARPS - 1)] : 0.0f;
    #pragma unroll
    for(int o = WARPS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// 1 / sqrt(v), with a Newton step for the last bits of the approximation
__device__ __forceinline__ float inverse_root(float v)
{
    const float f = rsqrtf(v);
    return v < __int_as_float(0x7f800000) ? fmaf(0.5f * f, fmaf(-v * f, f, 1.0f), f) : f;
}

// Where finite values have a sum of squares beyond fp32 (their rms is over 2^64 / sqrt(cols) then), 1 / sqrt(mean(h^2) + eps) comes out as 0.  The row is read again
// then for the sum of (2^-96 h)^2, which is neither beyond fp32 nor lost; an infinity among the values makes that one infinite, too, and the result 0 again.
// The sum is the same in every thread of the block, so all of them come here together, and nobody has written a total yet.
// (Out of line and element by element, so that it takes no registers from the path without: the same from the row in registers cost bf16 rows of 20480 with
// residual 85 -> 100 us.)
template<typename T, int WARPS> __device__ __noinline__ float inverse_of_large(const T *x, const T *r, int cols, float eps, float (&part)[WARPS])
{
    constexpr float S = 0x1p-96f;
    float again = 0.0f;
    #pragma unroll 1
    for(int c = threadIdx.x; c < cols; c += blockDim.x) {
        const float h = (to_float(ld_plain(x + c)) + (r ? to_float(ld_plain(r + c)) : 0.0f)) * S;
        again = fmaf(h, h, again);
    }
    return inverse_root(block_sum(again, part) / float(cols) + eps * S * S) * S;
}
template<typename T, int WARPS> __device__ __forceinline__ float inverse_rms(float sum, const NormArgs &a, long long row, float (&part)[WARPS])
{
    float f = inverse_root(sum / float(a.cols) + a.eps);
    if(f == 0.0f)
        f = inverse_of_large(static_cast<const T *>(a.x) + row * a.x_stride, a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr,
                             a.cols, a.eps, part);
    return f;
}

// What becomes of a lane's eight of 256 values h of a row: total, and the output in its type.
template<typename T, int KIND>
__device__ __forceinline__ void norm_out(const NormArgs &a, long long row, int c0, int lane, float (&v)[8], const float (&g)[8], float f)
{
    if(a.total) store8<T, KIND>(static_cast<T *>(a.total) + row * a.total_stride, c0, lane, a.cols, v);
    #pragma unroll
    for(int j = 0; j < 8; j += 2) apart(pair(v[j], v[j + 1]) * both(f) * pair(g[j], g[j + 1]), v[j], v[j + 1]);
    if(a.y_type == DLP_TYPE_E4M3) store_e4m3<KIND>(static_cast<unsigned char *>(a.y) + row * a.y_stride, a.scales + row, a.scale_stride, c0, lane, a.cols, v);
    else if(a.y_type == DLP_TYPE_F32) store8<float, KIND>(static_cast<float *>(a.y) + row * a.y_stride, c0, lane, a.cols, v);
    else if(a.y_type == DLP_TYPE_F16) store8<__half, KIND>(static_cast<__half *>(a.y) + row * a.y_stride, c0, lane, a.cols, v);
    else store8<__nv_bfloat16, KIND>(static_cast<__nv_bfloat16 *>(a.y) + row * a.y_stride, c0, lane, a.cols, v);
}

// NV: pieces of 256 columns, two blocks of the 8-bit form, that a warp keeps, a block's width apart.  KIND: see Row8, of all tensors together.
// WHOLE: a block takes rows in turn and asks for the next one as soon as the registers of this one's words are free: the reduction, the
// arithmetic and the stores of a row run under the loads of the next; the weights stay as far as registers go.  ANY: a row to a block, so that more of them
// fit an SM and run under one another.
template<typename T, int NV, int KIND>
__global__ void __launch_bounds__(most_threads(NV, KIND), (NV <= 2 ? 1024 : MAX_THREADS) / most_threads(NV, KIND)) rms_norm_kernel(const NormArgs a, unsigned rows)
{
    pdl_wait();
    __shared__ float part[3][most_threads(NV, KIND) / 32];           // in turn from row to row, and for a second sum
    typedef Row8<T, KIND> Row;
    const int cols = a.cols, lane = threadIdx.x & 31, stride = blockDim.x * 8, c0 = (threadIdx.x >> 5) * 256;
    const T *weight = static_cast<const T *>(a.weight);
    constexpr bool KEEP_WEIGHT = KIND == ROW_WHOLE ? NV * WORDS<T> <= (NV > 2 ? 16 : 8) : NV <= 2;
    Row xw[NV], rw[NV], ww[KEEP_WEIGHT ? NV : 1];
    auto ask = [&](unsigned row) {
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride, *r = static_cast<const T *>(a.residual) + row * a.residual_stride;
        #pragma unroll
        for(int i = 0; i < NV; i++) {
            xw[i].ask(x, c0 + i * stride, lane, cols);
            if(a.residual) rw[i].ask(r, c0 + i * stride, lane, cols);
        }
    };
    ask(blockIdx.x);
    if(KEEP_WEIGHT) {
        #pragma unroll
        for(int i = 0; i < NV; i++) ww[KEEP_WEIGHT ? i : 0].ask(weight, c0 + i * stride, lane, cols);
    }
    int turn = 0;
    #pragma unroll 1
    for(unsigned row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
        float h[NV][8];
        Pair squares = both(0.0f);
        #pragma unroll
        for(int i = 0; i < NV; i++) {
            xw[i].settle(h[i]);
            if(a.residual) {
                float b[8];
                rw[i].settle(b);
                #pragma unroll
                for(int j = 0; j < 8; j += 2) apart(pair(h[i][j], h[i][j + 1]) + pair(b[j], b[j + 1]), h[i][j], h[i][j + 1]);
            }
            #pragma unroll
            for(int j = 0; j < 8; j += 2) squares = fma2(pair(h[i][j], h[i][j + 1]), pair(h[i][j], h[i][j + 1]), squares);
        }
        float sum, odd;
        apart(squares, sum, odd);
        sum += odd;
        if(KIND == ROW_WHOLE && row + gridDim.x < rows) ask(row + gridDim.x);
        const float f = inverse_rms<T>(block_sum(sum, part[turn]), a, row, part[2]);
        #pragma unroll
        for(int i = 0; i < NV; i++) {
            Row w;
            if(KEEP_WEIGHT) w = ww[KEEP_WEIGHT ? i : 0];
            else w.ask(weight, c0 + i * stride, lane, cols);
            float g[8];
            w.settle(g);
            norm_out<T, KIND>(a, row, c0 + i * stride, lane, h[i], g, f);
        }
        if(KIND == ROW_ANY) return;
    }
}

// Rows of more than a block's registers: read twice, the second time from L2.
template<typename T, int KIND>
__global__ void __launch_bounds__(MAX_THREADS, 2) rms_norm_long_kernel(const NormArgs a)
{
    pdl_wait();
    __shared__ float part[2][MAX_THREADS / 32];
    const long long row = blockIdx.x;
    const int cols = a.cols, lane = threadIdx.x & 31, stride = blockDim.x * 8, first = (threadIdx.x >> 5) * 256;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride, *weight = static_cast<const T *>(a.weight);
    const T *r = a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
    auto fetch = [&](int c0, float (&h)[8]) {
        Row8<T, KIND> xw, rw;
        xw.ask(x, c0, lane, cols);
        if(r) rw.ask(r, c0, lane, cols);
        xw.settle(h);
        if(r) {
            float b[8];
            rw.settle(b);
            #pragma unroll
            for(int j = 0; j < 8; j++) h[j] += b[j];
        }
    };
    float sum = 0.0f;
    for(int c0 = first; c0 < cols; c0 += stride) {
        float h[8];
        fetch(c0, h);
        #pragma unroll
        for(int j = 0; j < 8; j++) sum += h[j] * h[j];
    }
    const float f = inverse_rms<T>(block_sum(sum, part[0]), a, row, part[1]);
    for(int c0 = first; c0 < cols; c0 += stride) {
        float h[8], g[8];
        Row8<T, KIND> w;
        w.ask(weight, c0, lane, cols);
        fetch(c0, h);
        w.settle(g);
        norm_out<T, KIND>(a, row, c0, lane, h, g, f);
    }
}

template<typename T, int NV>
dlp_status launch_nv(const NormArgs &a, int rows, int threads, bool off, cudaStream_t stream)
{
    const int resident = std::min(rows, sm_count() * std::max(1, (NV <= 2 ? 2 : 1) * MAX_THREADS / threads));
    if constexpr(NV != 4) {                                  // (what is ANY has two pieces in 1024 threads where four would be in 512)
        if(off) {
            DLP_LAUNCH_PDL(launch_pdl(one_wave(rows, threads), rms_norm_kernel<T, NV, ROW_ANY>, rows, threads, 0, stream, a, unsigned(rows)), "rms_norm_kernel");
            return DLP_OK;
        }
    }
    DLP_LAUNCH_PDL(launch_pdl(true, rms_norm_kernel<T, NV, ROW_WHOLE>, resident, threads, 0, stream, a, unsigned(rows)), "rms_norm_kernel");
    return DLP_OK;
}
template<typename T>
dlp_status launch_norm(const NormArgs &a, int rows, bool off, cudaStream_t stream)
{
    // With few rows each has as many warps as it can use (latency); with many, warps that keep two pieces or more have more loads under way.
    const int pieces = ceil_div(a.cols, 256), least = rows <= 2 * sm_count() ? 1 : 2;
    int nv = 1;
    while(nv < 8 && (nv < least || ceil_div(pieces, nv) > most_threads(nv, off ? ROW_ANY : ROW_WHOLE) / 32)) nv *= 2;
    const int threads = ceil_div(pieces, nv) * 32;
    if(threads > most_threads(nv, off ? ROW_ANY : ROW_WHOLE)) {
        const bool early = one_wave(rows, MAX_THREADS);
        if(off) DLP_LAUNCH_PDL(launch_pdl(early, rms_norm_long_kernel<T, ROW_ANY>, rows, MAX_THREADS, 0, stream, a), "rms_norm_long_kernel");
        else DLP_LAUNCH_PDL(launch_pdl(early, rms_norm_long_kernel<T, ROW_WHOLE>, rows, MAX_THREADS, 0, stream, a), "rms_norm_long_kernel");
        return DLP_OK;
    }
    switch(nv) {
    case 1: return launch_nv<T, 1>(a, rows, threads, off, stream);
    case 2: return launch_nv<T, 2>(a, rows, threads, off, stream);
    case 4: return launch_nv<T, 4>(a, rows, threads, off, stream);
    default: return launch_nv<T, 8>(a, rows, threads, off, stream);
    }
}

} // namespace
} // namespace dlp

using namespace dlp;

extern "C" {

dlp_status dlp_rms_norm_fwd(const dlp_rms_norm_args *args, void *stream)
{
    DLP_REQUIRE(args != nullptr, "null arguments");
    const auto [x, residual, weight, total, y, scales, x_stride, residual_stride, total_stride, y_stride, scale_stride, rows, cols, type, y_type, eps] = *args;
    DLP_REQUIRE(rows >= 0 && cols > 0 && cols < (1 << 30), "bad norm shape");
    DLP_REQUIRE(is_real_type(type), "the input's type must be fp32, fp16 or bf16");
    DLP_REQUIRE(is_real_type(y_type) || y_type == DLP_TYPE_E4M3, "unknown output type");
    DLP_REQUIRE(eps > 0.0f && eps < 1e30f, "eps must be positive and finite");
    DLP_REQUIRE(!total || residual, "a total is written only where a residual is added");
    if(rows == 0) return DLP_OK;
    DLP_REQUIRE(x && weight && y, "null tensor");
    DLP_REQUIRE((y_type == DLP_TYPE_E4M3) == (scales != nullptr), "scales go with the 8-bit output and with no other");
    DLP_REQUIRE(rows <= 1 || (x_stride >= cols && y_stride >= cols && (!residual || residual_stride >= cols) && (!total || total_stride >= cols)),
                "rows overlap");
    DLP_REQUIRE(!scales || cols <= SCALE_BLOCK || scale_stride >= rows, "blocks of scales overlap");
    const size_t size = type_size(type), y_size = type_size(y_type);
    DLP_REQUIRE(aligned_to(x, size) && aligned_to(weight, size) && aligned_to(y, y_size) && (!residual || aligned_to(residual, size)) &&
                (!total || aligned_to(total, size)) && (!scales || aligned_to(scales, 4)), "a tensor is not aligned to its elements");
    NormArgs a = { x, residual, weight, total, y, scales, x_stride, residual_stride, total_stride, y_stride, scale_stride, cols, y_type, eps };
    const auto rows_on = [rows = args->rows](const void *p, long long stride, size_t element, size_t n) { return aligned_to(p, n) && (rows == 1 || stride * element % n == 0); };
    const bool off = !(cols % 8 == 0 && rows_on(x, x_stride, size, 16) && aligned_to(weight, 16) && (!residual || rows_on(residual, residual_stride, size, 16)) &&
                       (!total || rows_on(total, total_stride, size, 16)) && rows_on(y, y_stride, y_size, y_type == DLP_TYPE_E4M3 ? 8 : 16));
    if(type == DLP_TYPE_F32) return launch_norm<float>(a, rows, off, (cudaStream_t)stream);
    if(type == DLP_TYPE_F16) return launch_norm<__half>(a, rows, off, (cudaStream_t)stream);
    return launch_norm<__nv_bfloat16>(a, rows, off, (cudaStream_t)stream);
}

} // extern "C"

// Root-mean-square norm of rows, with the addition of a residual before it and an 8-bit form of the result:
//     h = x + residual,   y = h / sqrt(mean(h^2) + eps) * weight.
// The row's sum of squares has to be complete before the first output, so a row is read twice: simple, the second time from L2.
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

constexpr int MAX_THREADS = 512;

// A block of threads per row; a thread takes eight consecutive columns at a time, so that sixteen lanes hold a block of the 8-bit form.
template<typename T, bool VEC>
__global__ void __launch_bounds__(MAX_THREADS) rms_norm_kernel(const NormArgs a)
{
    pdl_wait();
    __shared__ float part[MAX_THREADS / 32];
    const long long row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *r = a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    auto fetch = [&](int c, float (&h)[8]) {
        load8<T, VEC>(x + c, a.cols - c, h);
        if(r) {
            float b[8];
            load8<T, VEC>(r + c, a.cols - c, b);
            #pragma unroll
            for(int j = 0; j < 8; j++) h[j] += b[j];
        }
    };
    float sum = 0.0f;
    for(int c = threadIdx.x * 8; c < a.cols; c += blockDim.x * 8) {
        float h[8];
        fetch(c, h);
        #pragma unroll
        for(int j = 0; j < 8; j++) sum += h[j] * h[j];
    }
    #pragma unroll
    for(int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if(lane == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0.0f;
    for(int i = 0; i < warps; i++) sum += part[i];
    const float f = rsqrtf(sum / float(a.cols) + a.eps);
    // (whole blocks of lanes stay in the loop for the maximum over a block)
    for(int c0 = 0; c0 < a.cols; c0 += blockDim.x * 8) {
        const int c = c0 + threadIdx.x * 8;
        const bool in = c < a.cols;
        const int count = a.cols - c;
        float v[8] = {};
        if(in) {
            float w[8];
            fetch(c, v);
            load8<T, VEC>(static_cast<const T *>(a.weight) + c, count, w);
            if(a.total) store8<T, VEC>(static_cast<T *>(a.total) + row * a.total_stride + c, count, v);
            #pragma unroll
            for(int j = 0; j < 8; j++) v[j] = v[j] * f * w[j];
        }
        if(a.y_type == DLP_TYPE_E4M3) {
            const unsigned m = __reduce_max_sync(lane < 16 ? 0xffffu : 0xffff0000u, magnitude_bits(v));
            const float s = block_scale(m);
            if(in) {
                if((threadIdx.x & 15) == 0) a.scales[(c / SCALE_BLOCK) * a.scale_stride + row] = s;
                store_e4m3<VEC>(static_cast<unsigned char *>(a.y) + row * a.y_stride + c, count, pack_e4m3(v, 1.0f / s));
            }
        }
        else if(in) {
            if(a.y_type == DLP_TYPE_F32) store8<float, VEC>(static_cast<float *>(a.y) + row * a.y_stride + c, count, v);
            else if(a.y_type == DLP_TYPE_F16) store8<__half, VEC>(static_cast<__half *>(a.y) + row * a.y_stride + c, count, v);
            else store8<__nv_bfloat16, VEC>(static_cast<__nv_bfloat16 *>(a.y) + row * a.y_stride + c, count, v);
        }
    }
}

template<typename T>
dlp_status launch_norm(const NormArgs &a, int rows, bool vec, cudaStream_t stream)
{
    const int threads = std::min(MAX_THREADS, round_up(ceil_div(a.cols, 8), 32));
    const bool early = one_wave(rows, threads);
    if(vec) DLP_LAUNCH_PDL(launch_pdl(early, rms_norm_kernel<T, true>, rows, threads, 0, stream, a), "rms_norm_kernel");
    else DLP_LAUNCH_PDL(launch_pdl(early, rms_norm_kernel<T, false>, rows, threads, 0, stream, a), "rms_norm_kernel");
    return DLP_OK;
}

} // namespace
} // namespace dlp

using namespace dlp;

extern "C" {

dlp_status dlp_rms_norm_fwd(const dlp_rms_norm_args *args, void *stream)
{
    DLP_REQUIRE(args != nullptr, "null arguments");
    const auto [x, residual, weight, total, y, scales, x_stride, residual_stride, total_stride, y_stride, scale_stride, rows, cols, type, y_type, eps] = *args;
    DLP_REQUIRE(rows >= 0 && cols > 0, "bad norm shape");
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
    // 16-byte accesses (8 for the 8-bit output): every row and its end on such a boundary
    const auto rows_on = [rows = args->rows](const void *p, long long stride, size_t element, size_t n) { return aligned_to(p, n) && (rows == 1 || stride * element % n == 0); };
    const bool vec = cols % 8 == 0 && rows_on(x, x_stride, size, 16) && aligned_to(weight, 16) && (!residual || rows_on(residual, residual_stride, size, 16)) &&
                     (!total || rows_on(total, total_stride, size, 16)) && rows_on(y, y_stride, y_size, y_type == DLP_TYPE_E4M3 ? 8 : 16);
    if(type == DLP_TYPE_F32) return launch_norm<float>(a, rows, vec, (cudaStream_t)stream);
    if(type == DLP_TYPE_F16) return launch_norm<__half>(a, rows, vec, (cudaStream_t)stream);
    return launch_norm<__nv_bfloat16>(a, rows, vec, (cudaStream_t)stream);
}

} // extern "C"

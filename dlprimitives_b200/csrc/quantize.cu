// The 8-bit form of a matrix, or of what a gated activation makes of a pair of matrices side by side: blocks of 128 columns of one row
// (the left operand of an 8-bit product) or of 128 x 128 (its weights).
#include "block8.cuh"

namespace dlp {
namespace {

struct QuantArgs {
    const void *x;
    unsigned char *q;
    float *scales;
    long long x_stride, q_stride, scale_stride;
    int rows, cols, gate;
};

// silu(a) = a / (1 + e^-a);  gelu(a) = a / 2 (1 + tanh(sqrt(2 / pi) (a + 0.044715 a^3)))
__device__ __forceinline__ float gated(float a, float up, int gate)
{
    if(gate == DLP_GATE_SILU) return a / (1.0f + expf(-a)) * up;
    return 0.5f * a * (1.0f + tanhf(0.7978845608f * (a + 0.044715f * a * a * a))) * up;
}

constexpr int ROW_THREADS = 256;

// A warp takes 256 columns of a row, eight a lane; sixteen lanes hold a block.
template<typename T, bool VEC>
__global__ void __launch_bounds__(ROW_THREADS) quantize_rows_kernel(const QuantArgs a, unsigned pieces, long long items)
{
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long step = (long long)gridDim.x * (ROW_THREADS / 32);
    for(long long item = blockIdx.x * (long long)(ROW_THREADS / 32) + (threadIdx.x >> 5); item < items; item += step) {
        const long long row = item / pieces;
        const int c = int(item - row * pieces) * 256 + lane * 8, count = a.cols - c;
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
        float v[8] = {};
        if(count > 0) {
            load8<T, VEC>(x + c, count, v);
            if(a.gate != DLP_GATE_NONE) {
                float up[8];
                load8<T, VEC>(x + a.cols + c, count, up);
                #pragma unroll
                for(int j = 0; j < 8; j++) v[j] = gated(v[j], up[j], a.gate);
            }
        }
        const float s = block_scale(__reduce_max_sync(lane < 16 ? 0xffffu : 0xffff0000u, magnitude_bits(v)));
        if(count > 0) {
            if((lane & 15) == 0) a.scales[(c / SCALE_BLOCK) * a.scale_stride + row] = s;
            store_e4m3<VEC>(a.q + row * a.q_stride + c, count, pack_e4m3(v, 1.0f / s));
        }
    }
}

// A block of 256 threads takes a block of 128 x 128 and keeps it in registers: sixteen lanes hold a row, a thread eight rows.
template<typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const QuantArgs a)
{
    pdl_wait();
    __shared__ unsigned most[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = blockIdx.x * SCALE_BLOCK + (lane & 15) * 8, count = a.cols - c;
    const int row0 = blockIdx.y * SCALE_BLOCK + warp * 2 + (lane >> 4);
    float v[8][8];
    unsigned m = 0;
    #pragma unroll
    for(int i = 0; i < 8; i++) {
        #pragma unroll
        for(int j = 0; j < 8; j++) v[i][j] = 0.0f;
        if(count > 0 && row0 + i * 16 < a.rows) load8<T, VEC>(static_cast<const T *>(a.x) + (row0 + i * 16) * a.x_stride + c, count, v[i]);
    }
    #pragma unroll
    for(int i = 0; i < 8; i++) m = max(m, magnitude_bits(v[i]));
    m = __reduce_max_sync(0xffffffffu, m);
    if(lane == 0) most[warp] = m;
    __syncthreads();
    #pragma unroll
    for(int i = 0; i < 8; i++) m = max(m, most[i]);
    const float s = block_scale(m), inverse = 1.0f / s;
    if(threadIdx.x == 0) a.scales[blockIdx.y * a.scale_stride + blockIdx.x] = s;
    #pragma unroll
    for(int i = 0; i < 8; i++)
        if(count > 0 && row0 + i * 16 < a.rows) store_e4m3<VEC>(a.q + (row0 + i * 16) * a.q_stride + c, count, pack_e4m3(v[i], inverse));
}

template<typename T>
dlp_status launch_quantize(const QuantArgs &a, int block_rows, bool vec, cudaStream_t stream)
{
    if(block_rows == 1) {
        const int pieces = ceil_div(a.cols, 256);
        const long long items = (long long)a.rows * pieces, blocks = ceil_div<long long>(items, ROW_THREADS / 32);
        const unsigned grid = unsigned(std::min<long long>(blocks, (long long)sm_count() * 64));
        const bool early = one_wave(grid, ROW_THREADS);
        if(vec) DLP_LAUNCH_PDL(launch_pdl(early, quantize_rows_kernel<T, true>, grid, ROW_THREADS, 0, stream, a, unsigned(pieces), items), "quantize_rows_kernel");
        else DLP_LAUNCH_PDL(launch_pdl(early, quantize_rows_kernel<T, false>, grid, ROW_THREADS, 0, stream, a, unsigned(pieces), items), "quantize_rows_kernel");
        return DLP_OK;
    }
    const dim3 grid(ceil_div(a.cols, SCALE_BLOCK), ceil_div(a.rows, SCALE_BLOCK));
    const bool early = one_wave((long long)grid.x * grid.y, 256);
    if(vec) DLP_LAUNCH_PDL(launch_pdl(early, quantize_blocks_kernel<T, true>, grid, 256, 0, stream, a), "quantize_blocks_kernel");
    else DLP_LAUNCH_PDL(launch_pdl(early, quantize_blocks_kernel<T, false>, grid, 256, 0, stream, a), "quantize_blocks_kernel");
    return DLP_OK;
}

} // namespace
} // namespace dlp

using namespace dlp;

extern "C" {

dlp_status dlp_quantize_fwd(const dlp_quantize_args *args, void *stream)
{
    DLP_REQUIRE(args != nullptr, "null arguments");
    const auto [x, q, scales, x_stride, q_stride, scale_stride, rows, cols, type, gate, block_rows] = *args;
    DLP_REQUIRE(rows >= 0 && cols > 0 && cols < (1 << 30), "bad shape");
    DLP_REQUIRE(is_real_type(type), "the input's type must be fp32, fp16 or bf16");
    DLP_REQUIRE(gate >= DLP_GATE_NONE && gate <= DLP_GATE_GELU, "unknown gate");
    DLP_REQUIRE(block_rows == 1 || block_rows == SCALE_BLOCK, "blocks have 1 or 128 rows");
    DLP_REQUIRE(gate == DLP_GATE_NONE || block_rows == 1, "a gated pair has blocks of one row");
    if(rows == 0) return DLP_OK;
    DLP_REQUIRE(x && q && scales, "null tensor");
    DLP_REQUIRE(rows <= 1 || (x_stride >= (gate == DLP_GATE_NONE ? 1ll : 2ll) * cols && q_stride >= cols), "rows overlap");
    DLP_REQUIRE(block_rows == 1 ? cols <= SCALE_BLOCK || scale_stride >= rows : rows <= SCALE_BLOCK || scale_stride >= ceil_div(cols, SCALE_BLOCK),
                "lines of scales overlap");
    DLP_REQUIRE(block_rows == 1 || rows <= 65535 * SCALE_BLOCK, "too many rows");
    const size_t size = type_size(type);
    DLP_REQUIRE(aligned_to(x, size) && aligned_to(scales, 4), "a tensor is not aligned to its elements");
    const QuantArgs a = { x, static_cast<unsigned char *>(q), scales, x_stride, q_stride, scale_stride, rows, cols, gate };
    // 16-byte loads and 8-byte stores: every row and its end on such a boundary
    const bool vec = cols % 8 == 0 && aligned_to(x, 16) && aligned_to(q, 8) && (rows == 1 || (x_stride * size % 16 == 0 && q_stride % 8 == 0));
    if(type == DLP_TYPE_F32) return launch_quantize<float>(a, block_rows, vec, (cudaStream_t)stream);
    if(type == DLP_TYPE_F16) return launch_quantize<__half>(a, block_rows, vec, (cudaStream_t)stream);
    return launch_quantize<__nv_bfloat16>(a, block_rows, vec, (cudaStream_t)stream);
}

} // extern "C"

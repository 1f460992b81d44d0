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

// silu(a) = a / (1 + e^-a);  gelu(a) = a / 2 (1 + tanh z) = a / (1 + e^-2z), z = sqrt(2 / pi) (a + 0.044715 a^3): no difference of nearly equal numbers
// where tanh is near -1.  The quotient is a product with the approximate reciprocal (within a unit): with the division, 8192 x 12288 pairs
// took longer for their arithmetic than for memory.  Where the exponential overflows the reciprocal is 0.
__device__ __forceinline__ float gated(float a, float up, int gate)
{
    const float t = gate == DLP_GATE_SILU ? a : 1.5957691216f * fmaf(0.044715f * a * a, a, a);
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + expf(-t)));
    return a * r * up;
}

constexpr int ROW_THREADS = 256;

// A warp takes NP pieces of 256 columns of a row, eight a lane of each; sixteen lanes hold a block.  All its loads are under way before the first is
// used.  OFF: rows start off 16-byte boundaries.
template<typename T, bool GATED, bool OFF>
__global__ void __launch_bounds__(ROW_THREADS) quantize_rows_kernel(const QuantArgs a, unsigned groups, unsigned items)
{
    pdl_wait();
    constexpr int NP = GATED || sizeof(T) == 4 ? 2 : 4;
    const int lane = threadIdx.x & 31, cols = a.cols;
    const unsigned step = gridDim.x * (ROW_THREADS / 32);
    for(unsigned item = blockIdx.x * (ROW_THREADS / 32) + (threadIdx.x >> 5); item < items; item += step) {
        const unsigned row = item / groups;
        const int c0 = int(item - row * groups) * (256 * NP) + lane * 8;
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
        Row8<T, OFF> w[NP], u[GATED ? NP : 1];
        #pragma unroll
        for(int i = 0; i < NP; i++) {
            w[i].ask(x, c0 + i * 256, cols);
            if(GATED) u[GATED ? i : 0].ask(x + cols, c0 + i * 256, cols);
        }
        #pragma unroll
        for(int i = 0; i < NP; i++) {
            w[i].patch(x, c0 + i * 256, cols);
            if(GATED) u[GATED ? i : 0].patch(x + cols, c0 + i * 256, cols);
        }
        unsigned char *q = a.q + row * a.q_stride;
        const bool aligned = reinterpret_cast<uintptr_t>(q) % 8 == 0;
        #pragma unroll
        for(int i = 0; i < NP; i++) {
            const int c = c0 + i * 256;
            float v[8];
            w[i].settle(x, v);
            if(GATED) {
                float up[8];
                u[GATED ? i : 0].settle(x + cols, up);
                if(a.gate == DLP_GATE_SILU) {
                    #pragma unroll
                    for(int j = 0; j < 8; j++) v[j] = gated(v[j], up[j], DLP_GATE_SILU);
                }
                else {
                    #pragma unroll
                    for(int j = 0; j < 8; j++) v[j] = gated(v[j], up[j], DLP_GATE_GELU);
                }
            }
            const float s = block_scale(__reduce_max_sync(lane < 16 ? 0xffffu : 0xffff0000u, magnitude_bits(v)));
            if((lane & 15) == 0 && c < cols) a.scales[(c / SCALE_BLOCK) * a.scale_stride + row] = s;
            store_e4m3(q, c, cols, aligned, pack_e4m3(v, s));
        }
    }
}

// A block of 256 threads takes a block of 128 x 128 and keeps it in registers: sixteen lanes hold a row, a thread eight rows.
template<typename T, bool OFF>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const QuantArgs a)
{
    pdl_wait();
    __shared__ unsigned most[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = blockIdx.x * SCALE_BLOCK + (lane & 15) * 8, row0 = blockIdx.y * SCALE_BLOCK + warp * 2 + (lane >> 4);
    Row8<T, OFF, 16> w[8];
    const T *x[8];
    const auto cols_of = [&](int i) { return row0 + i * 16 < a.rows ? a.cols : 0; };       // a row that is not there has no columns
    #pragma unroll
    for(int i = 0; i < 8; i++) {
        x[i] = static_cast<const T *>(a.x) + (row0 + i * 16 < a.rows ? row0 + i * 16 : 0) * a.x_stride;
        w[i].ask(x[i], c, cols_of(i));
    }
    #pragma unroll
    for(int i = 0; i < 8; i++) w[i].patch(x[i], c, cols_of(i));
    float v[8][8];
    unsigned m = 0;
    #pragma unroll
    for(int i = 0; i < 8; i++) {
        w[i].settle(x[i], v[i]);
        m = max(m, magnitude_bits(v[i]));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if(lane == 0) most[warp] = m;
    __syncthreads();
    #pragma unroll
    for(int i = 0; i < 8; i++) m = max(m, most[i]);
    const float s = block_scale(m);
    if(threadIdx.x == 0) a.scales[blockIdx.y * a.scale_stride + blockIdx.x] = s;
    #pragma unroll
    for(int i = 0; i < 8; i++) {
        const int row = row0 + i * 16;
        const uint2 q = pack_e4m3(v[i], s);
        unsigned char *to = a.q + (row < a.rows ? row : 0) * a.q_stride;
        if(row < a.rows) store_e4m3(to, c, a.cols, reinterpret_cast<uintptr_t>(to) % 8 == 0, q);
    }
}

template<typename T, bool GATED>
dlp_status launch_rows(const QuantArgs &a, bool off, cudaStream_t stream)
{
    const int groups = ceil_div(a.cols, 256 * (GATED || sizeof(T) == 4 ? 2 : 4));
    const long long items = (long long)a.rows * groups, blocks = ceil_div<long long>(items, ROW_THREADS / 32);
    DLP_REQUIRE(items < (1ll << 32) - (1 << 24), "too many rows");
    const unsigned grid = unsigned(std::min<long long>(blocks, (long long)sm_count() * 64));
    const bool early = one_wave(grid, ROW_THREADS);
    if(off) DLP_LAUNCH_PDL(launch_pdl(early, quantize_rows_kernel<T, GATED, true>, grid, ROW_THREADS, 0, stream, a, unsigned(groups), unsigned(items)), "quantize_rows_kernel");
    else DLP_LAUNCH_PDL(launch_pdl(early, quantize_rows_kernel<T, GATED, false>, grid, ROW_THREADS, 0, stream, a, unsigned(groups), unsigned(items)), "quantize_rows_kernel");
    return DLP_OK;
}
template<typename T>
dlp_status launch_quantize(const QuantArgs &a, int block_rows, bool off, cudaStream_t stream)
{
    if(block_rows == 1) return a.gate == DLP_GATE_NONE ? launch_rows<T, false>(a, off, stream) : launch_rows<T, true>(a, off, stream);
    const dim3 grid(ceil_div(a.cols, SCALE_BLOCK), ceil_div(a.rows, SCALE_BLOCK));
    const bool early = one_wave((long long)grid.x * grid.y, 256);
    if(off) DLP_LAUNCH_PDL(launch_pdl(early, quantize_blocks_kernel<T, true>, grid, 256, 0, stream, a), "quantize_blocks_kernel");
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
    // every row, and the second half of a pair's, on a 16-byte boundary?
    const bool off = !(aligned_to(x, 16) && (rows == 1 || x_stride * size % 16 == 0) && (gate == DLP_GATE_NONE || cols * size % 16 == 0));
    if(type == DLP_TYPE_F32) return launch_quantize<float>(a, block_rows, off, (cudaStream_t)stream);
    if(type == DLP_TYPE_F16) return launch_quantize<__half>(a, block_rows, off, (cudaStream_t)stream);
    return launch_quantize<__nv_bfloat16>(a, block_rows, off, (cudaStream_t)stream);
}

} // extern "C"

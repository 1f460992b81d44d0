// The 8-bit form of a matrix, or of what a gated activation makes of a pair of matrices side by side: blocks of 128 columns of one row
// (the left operand of an 8-bit product) or of 128 x 128 (its weights).  Memory bounds it where there is no gate (8192 x 8192: fp32 50 us, 6.8 TB/s; bf16
// 39 us, 5.2 TB/s; weights 11000 x 4096 bf16 25 us, 5.4 TB/s); with one, the arithmetic does not quite go under it: 8192 x 12288 pairs 119 us, 4.3 TB/s,
// of which memory alone would take 77.  Rows off 16-byte boundaries: 4000 x 5001 pairs 40 us, weights 11000 x 4097 41 us, 3.3 TB/s.
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
// took longer for their arithmetic than for memory.  (Silu of N(0, 9) times N(0, 1): off by 1.1 halves of an fp32 unit, at most 5.3; with expf and
// a division 0.85 and 3.7.)  Where the exponential overflows the reciprocal is 0.
// e^-t is 2^s with s = -t log2(e) rounded, and what the rounding (and log2(e) in 24 bits) left out goes in as a factor 1 + left ln 2.  Past |t| = 200
// nothing changes any more.
__device__ __forceinline__ void gated2(float &a0, float &a1, float up0, float up1, int gate)
{
    const Pair a = pair(a0, a1);
    float t0 = a0, t1 = a1, s0, s1, e0, e1, r0, r1;
    if(gate == DLP_GATE_GELU) apart(both(1.5957691216f) * fma2(both(0.044715f) * a * a, a, a), t0, t1);
    const Pair t = pair(fminf(fmaxf(t0, -200.0f), 200.0f), fminf(fmaxf(t1, -200.0f), 200.0f));
    const Pair s = t * both(-1.44269502f), left = fma2(t, both(-1.92596299e-8f), fma2(t, both(-1.44269502f), s * both(-1.0f)));
    apart(s, s0, s1);
    asm("ex2.approx.f32 %0, %1;" : "=f"(e0) : "f"(s0));
    asm("ex2.approx.f32 %0, %1;" : "=f"(e1) : "f"(s1));
    apart(fma2(pair(e0, e1), fma2(left, both(0.693147181f), both(1.0f)), both(1.0f)), e0, e1);
    asm("rcp.approx.f32 %0, %1;" : "=f"(r0) : "f"(e0));
    asm("rcp.approx.f32 %0, %1;" : "=f"(r1) : "f"(e1));
    apart(a * pair(r0, r1) * pair(up0, up1), a0, a1);
}

constexpr int ROW_THREADS = 256, ROW_WARPS = ROW_THREADS / 32, ROW_PIECES = 2;

// A warp takes ROW_PIECES pieces of 256 columns of a row, two blocks, eight columns a lane of each.  All its loads are under way before the
// first is used.  2^per_row_log2: warps of a block that share a row; blockIdx.y: blocks that do; KIND: see Row8.  (Blocks that stay, go from row to
// row and have the next pieces' loads under way were slower, 139 against 121 us for 8192 x 12288 pairs: a block that ends makes room for one that
// starts with its loads, which keeps memory busy under the others' arithmetic better than a fixed order within each warp.)
template<typename T, bool GATED, int KIND>
__global__ void __launch_bounds__(ROW_THREADS, 4) quantize_rows_kernel(const QuantArgs a, int per_row_log2)
{
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cols = a.cols, per_row = 1 << per_row_log2;
    const long long row = (long long)blockIdx.x * (ROW_WARPS >> per_row_log2) + (warp >> per_row_log2);
    if(row >= a.rows) return;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    unsigned char *q = a.q + row * a.q_stride;
    float *scale = a.scales + row;
    const int step = gridDim.y * per_row * (256 * ROW_PIECES);
    #pragma unroll 1
    for(int c0 = (blockIdx.y * per_row + (warp & (per_row - 1))) * (256 * ROW_PIECES); c0 < cols; c0 += step) {
        Row8<T, KIND> w[ROW_PIECES], u[GATED ? ROW_PIECES : 1];
        #pragma unroll
        for(int i = 0; i < ROW_PIECES; i++) {
            w[i].ask(x, c0 + i * 256, lane, cols);
            if(GATED) u[GATED ? i : 0].ask(x + cols, c0 + i * 256, lane, cols);
        }
        #pragma unroll
        for(int i = 0; i < ROW_PIECES; i++) {
            float v[8];
            w[i].settle(v);
            if(GATED) {
                float up[8];
                u[GATED ? i : 0].settle(up);
                if(a.gate == DLP_GATE_SILU) {
                    #pragma unroll
                    for(int j = 0; j < 8; j += 2) gated2(v[j], v[j + 1], up[j], up[j + 1], DLP_GATE_SILU);
                }
                else {
                    #pragma unroll
                    for(int j = 0; j < 8; j += 2) gated2(v[j], v[j + 1], up[j], up[j + 1], DLP_GATE_GELU);
                }
            }
            store_e4m3<KIND>(q, scale, a.scale_stride, c0 + i * 256, lane, cols, v);
        }
    }
}

// A block of threads takes a block of 128 x 128 and keeps it in registers, pairs of rows to a warp: sixteen lanes hold a row each in eight consecutive
// columns of a lane (WHOLE), or all of them the one and then the other in every 32nd column (ANY: half as many pairs to a warp, since a load brings a
// register one element).
constexpr int block_threads(int kind) { return kind == ROW_WHOLE ? 256 : 512; }
template<typename T, int KIND>
__global__ void __launch_bounds__(block_threads(KIND), KIND == ROW_WHOLE ? 3 : 2) quantize_blocks_kernel(const QuantArgs a, int across)
{
    pdl_wait();
    constexpr int BLOCK_WARPS = block_threads(KIND) / 32, PAIRS = SCALE_BLOCK / 2 / BLOCK_WARPS;
    __shared__ unsigned most[BLOCK_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int block_row = blockIdx.x / across, block_col = blockIdx.x - block_row * across;       // (a grid's second axis ends at 65535)
    const int row0 = block_row * SCALE_BLOCK + warp * PAIRS * 2 + (KIND == ROW_WHOLE ? lane >> 4 : 0);
    const int col = block_col * SCALE_BLOCK + (KIND == ROW_WHOLE ? (lane & 15) * 8 : lane);
    // element j of pair i, as far as it is another one's place: row and column after row0 and col
    const auto row_of = [](int i, int j) { return 2 * i + (KIND == ROW_WHOLE ? 0 : j >> 2); };
    const auto col_of = [](int j) { return KIND == ROW_WHOLE ? 0 : 32 * (j & 3); };
    const auto there = [&](int i, int j) { return row0 + row_of(i, j) < a.rows && col + col_of(j) < a.cols; };
    const bool full = (block_row + 1) * SCALE_BLOCK <= a.rows && (block_col + 1) * SCALE_BLOCK <= a.cols;
    const T *x = static_cast<const T *>(a.x) + row0 * a.x_stride + col;
    float v[PAIRS][8];
    {
        union { uint4 w[WORDS<T> / 4]; T e[8]; } u[PAIRS];
        #pragma unroll
        for(int i = 0; i < PAIRS; i++) {
            if constexpr(KIND == ROW_WHOLE) {
                #pragma unroll
                for(int g = 0; g < WORDS<T> / 4; g++)
                    u[i].w[g] = there(i, 0) ? ld_plain(reinterpret_cast<const uint4 *>(x + row_of(i, 0) * a.x_stride) + g) : make_uint4(0, 0, 0, 0);
            }
            else if(!full) {
                #pragma unroll
                for(int j = 0; j < 8; j++) u[i].e[j] = there(i, j) ? ld_plain(x + row_of(i, j) * a.x_stride + col_of(j)) : from_float<T>(0.0f);
            }
        }
        if(KIND == ROW_ANY && full) {
            #pragma unroll
            for(int i = 0; i < PAIRS; i++)
                #pragma unroll
                for(int j = 0; j < 8; j++) u[i].e[j] = ld_plain(x + row_of(i, j) * a.x_stride + col_of(j));
        }
        #pragma unroll
        for(int i = 0; i < PAIRS; i++)
            #pragma unroll
            for(int j = 0; j < 8; j++) v[i][j] = to_float(u[i].e[j]);
    }
    unsigned m = 0;
    #pragma unroll
    for(int i = 0; i < PAIRS; i++) m = max(m, magnitude_bits(v[i]));
    m = __reduce_max_sync(0xffffffffu, m);
    if(lane == 0) most[warp] = m;
    __syncthreads();
    #pragma unroll
    for(int i = 0; i < BLOCK_WARPS; i++) m = max(m, most[i]);
    const float s = block_scale(m);
    const Quotient by(s);
    if(threadIdx.x == 0) a.scales[block_row * a.scale_stride + block_col] = s;
    unsigned char *to = a.q + row0 * a.q_stride + col;
    if(KIND == ROW_ANY && full) {
        #pragma unroll
        for(int i = 0; i < PAIRS; i++) {
            const uint32_t q[2] = { by.pack(v[i], 0), by.pack(v[i], 4) };
            #pragma unroll
            for(int j = 0; j < 8; j++) to[row_of(i, j) * a.q_stride + col_of(j)] = (unsigned char)(q[j >> 2] >> (8 * (j & 3)));
        }
        return;
    }
    #pragma unroll
    for(int i = 0; i < PAIRS; i++) {
        const uint32_t q[2] = { by.pack(v[i], 0), by.pack(v[i], 4) };
        if constexpr(KIND == ROW_WHOLE) {
            if(there(i, 0)) *reinterpret_cast<uint2 *>(to + row_of(i, 0) * a.q_stride) = make_uint2(q[0], q[1]);
        }
        else {
            #pragma unroll
            for(int j = 0; j < 8; j++)
                if(there(i, j)) to[row_of(i, j) * a.q_stride + col_of(j)] = (unsigned char)(q[j >> 2] >> (8 * (j & 3)));
        }
    }
}

template<typename T, bool GATED>
dlp_status launch_rows(const QuantArgs &a, bool off, cudaStream_t stream)
{
    const int groups = ceil_div(a.cols, 256 * ROW_PIECES);
    int log2 = 0;
    while((1 << log2) < std::min(groups, ROW_WARPS)) log2++;
    const int blocks = int(ceil_div<long long>(a.rows, ROW_WARPS >> log2));      // (rows may be up to 2^31 - 1)
    // few rows: more blocks to a row, until the GPU is full
    const int across = std::max(1, std::min(ceil_div(groups, 1 << log2), sm_count() * 4 / blocks));
    const dim3 grid(blocks, across);
    const bool early = one_wave((long long)blocks * across, ROW_THREADS);
    if(off) DLP_LAUNCH_PDL(launch_pdl(early, quantize_rows_kernel<T, GATED, ROW_ANY>, grid, ROW_THREADS, 0, stream, a, log2), "quantize_rows_kernel");
    else DLP_LAUNCH_PDL(launch_pdl(early, quantize_rows_kernel<T, GATED, ROW_WHOLE>, grid, ROW_THREADS, 0, stream, a, log2), "quantize_rows_kernel");
    return DLP_OK;
}
template<typename T>
dlp_status launch_quantize(const QuantArgs &a, int block_rows, bool off, cudaStream_t stream)
{
    if(block_rows == 1) return a.gate == DLP_GATE_NONE ? launch_rows<T, false>(a, off, stream) : launch_rows<T, true>(a, off, stream);
    const int across = ceil_div(a.cols, SCALE_BLOCK);
    const long long grid = (long long)across * ceil_div(a.rows, SCALE_BLOCK);
    DLP_REQUIRE(grid < 1ll << 31, "too large");
    const bool early = one_wave(grid, block_threads(off ? ROW_ANY : ROW_WHOLE));
    if(off) DLP_LAUNCH_PDL(launch_pdl(early, quantize_blocks_kernel<T, ROW_ANY>, unsigned(grid), block_threads(ROW_ANY), 0, stream, a, across), "quantize_blocks_kernel");
    else DLP_LAUNCH_PDL(launch_pdl(early, quantize_blocks_kernel<T, ROW_WHOLE>, unsigned(grid), block_threads(ROW_WHOLE), 0, stream, a, across), "quantize_blocks_kernel");
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
    DLP_REQUIRE(block_rows == 1 || rows <= (1 << 30), "too many rows");
    const size_t size = type_size(type);
    DLP_REQUIRE(aligned_to(x, size) && aligned_to(scales, 4), "a tensor is not aligned to its elements");
    const QuantArgs a = { x, static_cast<unsigned char *>(q), scales, x_stride, q_stride, scale_stride, rows, cols, gate };
    // every row, and the second half of a pair's, on a 16-byte boundary (8 for the numbers) and a multiple of eight long?
    const bool off = !(cols % 8 == 0 && aligned_to(x, 16) && aligned_to(q, 8) && (rows == 1 || (x_stride * size % 16 == 0 && q_stride % 8 == 0)));
    if(type == DLP_TYPE_F32) return launch_quantize<float>(a, block_rows, off, (cudaStream_t)stream);
    if(type == DLP_TYPE_F16) return launch_quantize<__half>(a, block_rows, off, (cudaStream_t)stream);
    return launch_quantize<__nv_bfloat16>(a, block_rows, off, (cudaStream_t)stream);
}

} // extern "C"

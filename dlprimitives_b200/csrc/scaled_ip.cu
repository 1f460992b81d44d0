// InnerProduct of 8-bit operands with a scale for each block of 128, on the sm_100a tensor cores:
//     y[r][o] = act( sum_b xs[b][r] ws[o / 128][b] sum_{k in block b} x[r][k] w[o][k]  + bias[o] ).
// The scales differ from block to block of K, so the tensor core sums one block (four tcgen05.mma of K = 32) into tensor memory and
// the sum over blocks is kept in fp32 registers: warps read a block's products from tensor memory, multiply by the two scales
// and add, while the tensor core works on the next block in another part of tensor memory.  Both operands are K-major and come in
// by tensor-map copies, 128 bytes (a block of K) wide, zero-filled beyond the matrices, so that no size needs padding.
//
// This file has the entry point, the choice of kernel, and the kernel for few rows; scaled_ip_pair.cu has the one for many.  With few rows the weights
// are what is read, and a tile is 128 rows of w (the MMA's M) by 16 to 64 rows of x (its N): a batch of 16 rows fills a tile's 16 columns instead
// of an eighth of its 128 rows.  K is cut into parts over the blocks of a cluster, so that a product of few tiles reads its weights with the whole GPU; the parts
// are added through distributed shared memory in a fixed order.  Measured (captured, us; in brackets the bytes' time at a copy's 6.5 TB/s): one row 4096 -> 4096
// 5.1 (2.6: launch, set-up and the cluster's sum are the rest), one row 4096 -> 24576 19.2 (15.4), 48 rows 23.4 (15.8), 64 rows 24.7 (16.0).
// Every wait is bounded (device status word + abort flag).
#include "scaled_ip.cuh"
#include <algorithm>

namespace dlp {
namespace sip {

constexpr int SC_CHUNK = 16;                // blocks of K whose scales are brought in at a time
constexpr int MAX_STAGES = 8;
constexpr int MAX_CLUSTER = 8;

struct Shared {
    unsigned long long full[MAX_STAGES], empty[MAX_STAGES], acc_full[4], acc_empty[4], drain;
    uint32_t tmem_base;
    int abort_flag;
};

struct Params {
    const float *x_scales, *w_scales, *bias;
    void *y;
    long long x_scale_stride, w_scale_stride, y_stride;
    int rows, outputs;
    int kblocks;            // of the whole K
    int per_part;           // of a part of K
    int n_tiles;            // tiles of rows of x
    int y_type, act;
};

// Warps that sum and store, beside the two that copy and issue: four have a quarter of the tile's rows each; with many columns eight, half of
// the columns each.
constexpr int sum_warps_for(int bn) { return bn == 64 ? 8 : 4; }
constexpr int threads_for(int bn) { return 64 + 32 * sum_warps_for(bn); }
// Two blocks on an SM, with half of its shared memory each: what bounds this kernel is the stream of weights, and they fill one another's pauses.
constexpr int PER_SM = 2;
constexpr int fixed_for(int bn) { return 2048 + 2 * SC_CHUNK * bn * 4; }                          // alignment slack, barriers, scales
constexpr int stages_for(int bn) { return std::min(MAX_STAGES, ((SMEM_LIMIT + 1024) / PER_SM - 1024 - fixed_for(bn)) / ((BM + bn) * BK)); }

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const void *tmap, int x, int y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(place_in(addr, rank)) : "memory");
    return v;
}

__device__ __forceinline__ void store_out(void *y, long long at, int type, float v)
{
    if(type == DLP_TYPE_F32) static_cast<float *>(y)[at] = v;
    else if(type == DLP_TYPE_F16) static_cast<__half *>(y)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(y)[at] = __float2bfloat16_rn(v);
}

// A tile is 128 rows of w by BN rows of x.
template<int BN>
__global__ void __launch_bounds__(threads_for(BN), PER_SM)
scaled_ip_few_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Params q, int *status)
{
    extern __shared__ unsigned char smem_raw[];
    constexpr int ACC = 4;                                   // accumulators in tensor memory
    constexpr int SUM = sum_warps_for(BN), SUM_THREADS = 32 * SUM, COLS = BN * 4 / SUM;      // columns of a summing warp
    constexpr int TMEM_COLS = ACC * BN;
    constexpr int S = stages_for(BN), STAGE_BYTES = (BM + BN) * BK;
    unsigned char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    Shared *sh = reinterpret_cast<Shared *>(smem);
    float *scale_ring = reinterpret_cast<float *>(smem + 1024);           // two chunks of SC_CHUNK x BN
    unsigned char *ring = smem + 1024 + 2 * SC_CHUNK * BN * 4;
    static_assert(sizeof(Shared) <= 1024 && (SC_CHUNK * BN * 8) % 1024 == 0 && S >= 4, "ring");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = int(cluster_size()), part = int(cluster_rank());
    const int tile = int(blockIdx.x) / parts, w_tile = tile / q.n_tiles, x_tile = tile - w_tile * q.n_tiles;
    const int kb0 = part * q.per_part, kblocks = max(0, min(q.per_part, q.kblocks - kb0));
    int *abort_flag = &sh->abort_flag;

    if(threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_x) : "memory");
        for(int s = 0; s < S; s++) { mbar_init(&sh->full[s], 1); mbar_init(&sh->empty[s], 1); }
        for(int a = 0; a < ACC; a++) { mbar_init(&sh->acc_full[a], 1); mbar_init(&sh->acc_empty[a], SUM); }
        mbar_init(&sh->drain, 1);
        sh->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if(warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem_base)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *(volatile uint32_t *)&sh->tmem_base;
    pdl_wait();

    constexpr int MINE = BN * SC_CHUNK / SUM_THREADS;                // scale products a summing thread brings in per chunk
    float acc[COLS];
    #pragma unroll
    for(int j = 0; j < COLS; j++) acc[j] = 0.0f;
    const int quad = warp & 3, row_in_tile = quad * 32 + lane, col0 = warp >= 6 ? COLS : 0;

    // (One elected thread copies and one issues; the compiler then knows that it is one, and takes the operands of a tcgen05.mma as they are.  Chosen by
    // its lane number it brings them together for each instruction: 370 instead of 170 cycles for four of them and two commits.)
    if(warp == 0) {
        if(elect_one()) {
            const uint32_t full0 = smem_u32(&sh->full[0]), empty0 = smem_u32(&sh->empty[0]), ring0 = smem_u32(ring);
            uint32_t s = 0, phase = 1;
            int kb = 0;
            #pragma unroll 1
            for(; kb < kblocks; kb++) {
                if(!wait_quietly(empty0 + 8 * s, phase, abort_flag, status, SIP_EMPTY)) break;
                mbar_arrive_expect_tx(&sh->full[s], STAGE_BYTES);
                tma_load_2d(ring0 + s * STAGE_BYTES, &tm_w, (kb0 + kb) * BK, w_tile * BM, full0 + 8 * s);
                tma_load_2d(ring0 + s * STAGE_BYTES + BM * BK, &tm_x, (kb0 + kb) * BK, x_tile * BN, full0 + 8 * s);
                if(++s == S) { s = 0; phase ^= 1; }
            }
            // nothing may still be on its way into shared memory when the block ends
            for(int n = max(0, kb - S); n < kb; n++) {
                const long long t0 = global_ns();
                while(!mbar_try_wait(&sh->full[n % S], (n / S) & 1)) {
                    __nanosleep(256);
                    if(global_ns() - t0 > WAIT_LIMIT_NS) { atomicCAS(status, 0, SIP_DRAIN); break; }
                }
            }
        }
        __syncwarp();
    }
    else if(warp == 1) {
        if(elect_one()) {
            constexpr uint32_t IDESC = (1u << 4) | (uint32_t(BN >> 3) << 17) | (uint32_t(BM >> 4) << 24);     // fp32 sums of e4m3, K-major, M 128
            constexpr uint64_t DESC_HI = uint64_t((1024u >> 4) | (1u << 14) | (2u << 29)) << 32;   // 8-row groups 1024 bytes apart, version 1, SWIZZLE_128B
            const uint32_t full0 = smem_u32(&sh->full[0]), empty0 = smem_u32(&sh->empty[0]), acc_full0 = smem_u32(&sh->acc_full[0]),
                           acc_empty0 = smem_u32(&sh->acc_empty[0]), ring0 = ((smem_u32(ring) & 0x3FFFF) >> 4) | (1u << 16);
            uint32_t s = 0, phase = 0, b = 0, b_phase = 1;
            #pragma unroll 1
            for(int kb = 0; kb < kblocks; kb++) {
                if(!wait_quietly(acc_empty0 + 8 * b, b_phase, abort_flag, status, SIP_ACC_EMPTY)) break;
                const uint32_t wd = ring0 + s * (STAGE_BYTES >> 4), xd = wd + (BM * BK >> 4), d = tmem_base + b * BN;
                if(!wait_quietly(full0 + 8 * s, phase, abort_flag, status, SIP_FULL)) break;
                tc_fence_after();
                #pragma unroll
                for(int j = 0; j < 4; j++)
                    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                                 "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                                 ::"r"(d), "l"(DESC_HI | (wd + 2 * j)), "l"(DESC_HI | (xd + 2 * j)), "r"(IDESC), "r"(j) : "memory");
                mma_commit(empty0 + 8 * s);
                mma_commit(acc_full0 + 8 * b);
                if(++s == S) { s = 0; phase ^= 1; }
                if(++b == ACC) { b = 0; b_phase ^= 1; }
            }
        }
        __syncwarp();
    }
    else {
        const int t = threadIdx.x - 64;
        const uint32_t acc_full0 = smem_u32(&sh->acc_full[0]), acc_empty0 = smem_u32(&sh->acc_empty[0]);
        // Products of the scales for the chunk of blocks of K at kb, [block][row of x]; zero beyond the matrices.
        float next_x[MINE], next_w[MINE];
        auto fetch = [&](int kb) {
            #pragma unroll
            for(int i = 0; i < MINE; i++) {
                const int at = i * SUM_THREADS + t, k = kb + at / BN, r = x_tile * BN + at % BN;
                const bool there = k < kblocks && r < q.rows;
                next_x[i] = there ? ld_plain(q.x_scales + (kb0 + k) * q.x_scale_stride + r) : 0.0f;
                next_w[i] = there ? ld_plain(q.w_scales + w_tile * q.w_scale_stride + kb0 + k) : 0.0f;
            }
        };
        if(kblocks > 0) fetch(0);
        uint32_t b = 0, b_phase = 0;
        #pragma unroll 1
        for(int kb = 0; kb < kblocks; kb++) {
            const int in = kb % SC_CHUNK;
            const float *sc = scale_ring + ((kb / SC_CHUNK & 1) * SC_CHUNK + in) * BN + col0;
            if(in == 0) {
                #pragma unroll
                for(int i = 0; i < MINE; i++) scale_ring[(kb / SC_CHUNK & 1) * SC_CHUNK * BN + i * SUM_THREADS + t] = next_x[i] * next_w[i];
                asm volatile("bar.sync 1, %0;" ::"n"(SUM_THREADS) : "memory");
                if(kb + SC_CHUNK < kblocks) fetch(kb + SC_CHUNK);
            }
            // (no vote: should the wait give up, the others do so at once, and what is read means nothing)
            warp_wait_quietly(acc_full0 + 8 * b, b_phase, abort_flag, status, SIP_ACC_FULL, lane == 0);
            tc_fence_after();
            const uint32_t taddr = tmem_base + (uint32_t(quad * 32) << 16) + b * BN + col0;
            constexpr int W = 16;
            #pragma unroll
            for(int g = 0; g < COLS / W; g++) {
                uint32_t v[W];
                tmem_ld(taddr + g * W, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if(g + 1 == COLS / W) {
                    tc_fence_before();
                    __syncwarp();
                    arrive_if(lane == 0, acc_empty0 + 8 * b);
                }
                #pragma unroll
                for(int j = 0; j < W; j += 4) {
                    const float4 f = *reinterpret_cast<const float4 *>(sc + g * W + j);
                    acc[g * W + j] += __uint_as_float(v[j]) * f.x;
                    acc[g * W + j + 1] += __uint_as_float(v[j + 1]) * f.y;
                    acc[g * W + j + 2] += __uint_as_float(v[j + 2]) * f.z;
                    acc[g * W + j + 3] += __uint_as_float(v[j + 3]) * f.w;
                }
            }
            if(++b == ACC) { b = 0; b_phase ^= 1; }
        }
    }

    // ---- tensor memory goes back
    tc_fence_before();
    __syncthreads();
    if(*(volatile int *)abort_flag) {
        // a wait gave up: let the MMAs already issued retire (bounded) before tensor memory goes away
        if(warp == 1 && elect_one()) {
            mma_commit(smem_u32(&sh->drain));
            const long long t0 = global_ns();
            while(!mbar_try_wait(&sh->drain, 0)) {
                __nanosleep(256);
                if(global_ns() - t0 > WAIT_LIMIT_NS) { atomicCAS(status, 0, SIP_DRAIN); break; }
            }
        }
        __syncthreads();
    }
    if(warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }

    // ---- sum over the parts of K, bias, activation, store: a warp stores 32 outputs of a row of x.  The sums pass through shared memory in any case, where
    // the operands were: from there a short loop takes them row by row (unrolled over registers, with three types and five activations, the code was
    // longer than the rest of the kernel, and fetching it took 6 us).
    const int o = w_tile * BM + row_in_tile, rows = min(BN, q.rows - x_tile * BN);
    float *partial = reinterpret_cast<float *>(ring);        // [row of x][row of w]
    if(warp >= 2) {
        #pragma unroll
        for(int j = 0; j < COLS; j++)
            if(col0 + j < rows) partial[(col0 + j) * BM + row_in_tile] = acc[j];
    }
    if(parts > 1) cluster_sync();
    else __syncthreads();
    if(warp >= 2 && o < q.outputs) {
        // part p of the cluster finishes rows p, p + parts, ...; of two warps with the same rows of w each takes every other one
        const uint32_t base = smem_u32(partial) + row_in_tile * 4;
        const float bias = q.bias ? ld_plain(q.bias + o) : 0.0f;
        const int step = parts * (SUM / 4);
        int j = part + (warp >= 6 ? parts : 0);
        long long at = (long long)(x_tile * BN + j) * q.y_stride + o;
        #pragma unroll 1
        for(; j < rows; j += step, at += step * q.y_stride) {
            float v;
            if(parts > 1) {
                float p[MAX_CLUSTER];
                #pragma unroll
                for(int i = 0; i < MAX_CLUSTER; i++) p[i] = i < parts ? ld_cluster(base + j * (BM * 4), i) : 0.0f;
                v = p[0];
                #pragma unroll
                for(int i = 1; i < MAX_CLUSTER; i++) v += p[i];
            }
            else v = partial[j * BM + row_in_tile];
            store_out(q.y, at, q.y_type, apply_act(v + bias, q.act));
        }
    }
    if(parts > 1) cluster_sync();                            // nobody leaves while its sums are being read
}

// ---------------------------------------------------------------------------------------------- host
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);
static EncodeTiledFn encode_fn()
{
    static std::mutex mutex;
    static EncodeTiledFn fn = nullptr;
    std::lock_guard<std::mutex> lock(mutex);
    if(!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult res;
        if(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &res) == cudaSuccess && res == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    }
    return fn;
}
static dlp_status encode_2d(CUtensorMap &map, CUtensorMapDataType type, const void *p, long long cols, long long rows, long long stride_bytes, int box_cols,
                            int box_rows)
{
    EncodeTiledFn enc = encode_fn();
    if(!enc) return fail(DLP_CUDA_ERROR, "cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t dims[2] = { cuuint64_t(cols), cuuint64_t(rows) }, strides[1] = { cuuint64_t(stride_bytes) };
    cuuint32_t box[2] = { cuuint32_t(box_cols), cuuint32_t(box_rows) }, elem[2] = { 1, 1 };
    const CUresult r = enc(&map, type, 2, const_cast<void *>(p), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if(r != CUDA_SUCCESS) return fail(DLP_CUDA_ERROR, "cuTensorMapEncodeTiled failed with code " + std::to_string(int(r)));
    return DLP_OK;
}
dlp_status encode_operand(CUtensorMap &map, const void *p, long long stride, int rows, int cols, int box_rows)
{
    return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, p, cols, rows, rows > 1 ? stride : round_up(cols, 16), BK, box_rows);
}
dlp_status encode_result(CUtensorMap &map, const Problem &p)
{
    const int size = type_size(p.y_type);
    const CUtensorMapDataType type = p.y_type == DLP_TYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                                              : (p.y_type == DLP_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
    return encode_2d(map, type, p.y, p.outputs, p.rows, p.y_stride * size, 128 / size, 32);
}

// Parts of K that give every SM a block; and a second one where parts stay ten blocks of K long (us, parts: 8 rows, 2000 -> 12000 7.8 one, 9.4 two; 32 rows,
// 5000 -> 7100 15.0 two, 12.9 four; one row, 4096 -> 4096 8.2 one, 6.5 two, 5.5 four, 5.5 eight).  Parts that start a second round do not pay (48 rows,
// 4096 -> 24576 24 one, 35 two, 36 three).
static int few_parts(const Problem &p, int bn)
{
    const long long tiles = (long long)ceil_div(p.outputs, BM) * ceil_div(p.rows, bn), sms = sm_count();
    int parts = 1;
    while(parts < MAX_CLUSTER && tiles * parts * 2 <= (p.kblocks >= parts * 2 * 10 ? 2 * sms : sms) && parts * 2 <= p.kblocks) parts *= 2;
    return parts;
}

template<int BN> static dlp_status launch_few(const Problem &p, cudaStream_t stream)
{
    dlp_status st = allow_shared<scaled_ip_few_kernel<BN>>(SMEM_LIMIT);
    if(st != DLP_OK) return st;
    int *status = device_status_word();
    if(!status) return fail(DLP_CUDA_ERROR, "cannot resolve the device status word");
    const int x_tiles = ceil_div(p.rows, BN), parts = few_parts(p, BN);
    const Params q = { p.x_scales, p.w_scales, p.bias, p.y, p.x_scale_stride, p.w_scale_stride, p.y_stride, p.rows, p.outputs, p.kblocks,
                       ceil_div(p.kblocks, parts), x_tiles, p.y_type, p.act };
    CUtensorMap mx, mw;
    st = encode_operand(mx, p.x, p.x_stride, p.rows, p.inputs, BN);
    if(st == DLP_OK) st = encode_operand(mw, p.w, p.w_stride, p.outputs, p.inputs, BM);
    if(st != DLP_OK) return st;
    const long long blocks = (long long)ceil_div(p.outputs, BM) * x_tiles * parts;
    DLP_REQUIRE(blocks < (1ll << 31), "too many tiles");
    // (a short part of K needs no more stages than it has blocks; the places left let the next kernel's blocks be set up early)
    const int smem = fixed_for(BN) + std::max(std::min(stages_for(BN), q.per_part), ceil_div(BN * BM * 4, (BM + BN) * BK)) * (BM + BN) * BK;
    note_route("scaled_few", BN, parts);
    DLP_LAUNCH_PDL(launch_pdl_cluster(blocks <= sm_count() * 2, parts, scaled_ip_few_kernel<BN>, unsigned(blocks), threads_for(BN), smem, stream, mw, mx, q,
                                      status), "scaled_ip_few_kernel");
    return DLP_OK;
}

// Which kernel.  Up to 64 rows one tile of the few-rows kernel covers them all.  Beyond, it is measured time per block of K and round of tiles (us,
// at full clocks): 0.64 for its 64-column tiles, two on an SM, which can be cut along K; 0.33 and 0.52 for pair tiles of 128 and 256 outputs, which
// cannot, and have an end of 0.5 and 1.2 a round.  (Measured, each of the three, us: 128 rows, 4096 -> 24576 39.7, 34.5, 38.9; 256 rows, 8192 -> 1000 10.9,
// 22.5, 33.5; 517 rows, 4096 -> 4096 23.5, 24.2, 21.5; 517 rows, 5000 -> 7100 61.8, 44.5, 47.8; 4096 rows, 4096 -> 24576 837, 447, 387.)
static dlp_status dispatch(const Problem &p, cudaStream_t stream)
{
    if(p.rows <= 16) return launch_few<16>(p, stream);
    if(p.rows <= 32) return launch_few<32>(p, stream);
    if(p.rows <= 64) return launch_few<64>(p, stream);
    const auto rounds = [](long long tiles, int places) { return double((tiles + places - 1) / places); };
    const int parts = few_parts(p, 64);
    const double few = rounds((long long)ceil_div(p.outputs, BM) * ceil_div(p.rows, 64) * parts, sm_count() * 2) * ceil_div(p.kblocks, parts) * 0.64;
    const long long row_tiles = ceil_div(p.rows, 2 * BM);
    const double narrow = rounds(row_tiles * ceil_div(p.outputs, 128), sm_count() / 2) * (p.kblocks * 0.33 + 0.5);
    const double wide = rounds(row_tiles * ceil_div(p.outputs, 256), sm_count() / 2) * (p.kblocks * 0.52 + 1.2);
    if(few <= narrow && few <= wide) return launch_few<64>(p, stream);
    return launch_pair(p, narrow < wide ? 128 : 256, stream);
}

} // namespace sip
} // namespace dlp

using namespace dlp;

extern "C" {

dlp_status dlp_scaled_ip_fwd(const dlp_scaled_ip_args *args, void *stream)
{
    DLP_REQUIRE(args != nullptr, "null arguments");
    const auto [x, x_scales, w, w_scales, bias, y, x_stride, x_scale_stride, w_stride, w_scale_stride, y_stride, rows, inputs, outputs, y_type, activation] = *args;
    DLP_REQUIRE(rows >= 0 && inputs > 0 && outputs > 0, "bad shape");
    DLP_REQUIRE(inputs <= (1 << 30) && outputs <= (1 << 30) && rows <= (1 << 30), "too large");
    DLP_REQUIRE(is_real_type(y_type), "the result's type must be fp32, fp16 or bf16");
    DLP_REQUIRE(activation >= DLP_ACT_IDENTITY && activation <= DLP_ACT_RELU6, "unknown activation");
    if(rows == 0) return DLP_OK;
    DLP_REQUIRE(x && x_scales && w && w_scales && y, "null tensor");
    const int kblocks = ceil_div(inputs, SCALE_BLOCK), oblocks = ceil_div(outputs, SCALE_BLOCK);
    DLP_REQUIRE((rows <= 1 || (x_stride >= inputs && y_stride >= outputs)) && (outputs == 1 || w_stride >= inputs), "rows overlap");
    DLP_REQUIRE((kblocks == 1 || x_scale_stride >= rows) && (oblocks == 1 || w_scale_stride >= kblocks), "lines of scales overlap");
    DLP_REQUIRE(aligned_to(x, 16) && (rows <= 1 || x_stride % 16 == 0) && aligned_to(w, 16) && (outputs == 1 || w_stride % 16 == 0),
                "rows of 8-bit operands must start on 16-byte boundaries");
    DLP_REQUIRE((rows <= 1 || x_stride < (1ll << 40)) && (outputs == 1 || w_stride < (1ll << 40)), "a row stride must be under 2^40");
    DLP_REQUIRE(aligned_to(x_scales, 4) && aligned_to(w_scales, 4) && (!bias || aligned_to(bias, 4)) && aligned_to(y, type_size(y_type)),
                "a tensor is not aligned to its elements");
    const sip::Problem p = { x, w, x_stride, w_stride, x_scales, w_scales, bias, y, x_scale_stride, w_scale_stride, y_stride, rows, inputs, outputs,
                             kblocks, y_type, activation };
    return sip::dispatch(p, (cudaStream_t)stream);
}

} // extern "C"

// InnerProduct of 8-bit operands with a scale for each block of 128, on the sm_100a tensor cores:
//     y[r][o] = act( sum_b xs[b][r] ws[o / 128][b] sum_{k in block b} x[r][k] w[o][k]  + bias[o] ).
// The scales differ from block to block of K, so the tensor core sums one block (four tcgen05.mma of K = 32) into tensor memory and
// the sum over blocks is kept in fp32 registers: warps read a block's 128 x BN products from tensor memory, multiply by the two scales
// and add, while the tensor core works on the next block in another part of tensor memory.  Both operands are K-major and come in
// by tensor-map copies, 128 bytes (a block of K) wide, zero-filled beyond the matrices, so that no size needs padding.
//   * rows of x are the tile's rows (many rows): a thread's products share one pair of scales;
//   * rows of w are the tile's rows (few rows of x): a batch of 16 rows fills a tile's 16 columns instead of an eighth of its 128 rows.
//     K is cut into parts over the blocks of a cluster, so that a product of few tiles reads its weights with the whole GPU; the parts are
//     added through distributed shared memory in a fixed order.
// Every wait is bounded (device status word + abort flag).
#include "scaled_ip.cuh"
#include <cstring>

namespace dlp {
namespace sip {

constexpr int SC_CHUNK = 16;                // blocks of K whose scales are brought in at a time
constexpr int MAX_STAGES = 12;
constexpr int NUM_THREADS = 192;            // copies, MMA issue, four warps that sum and store
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
    int n_tiles;            // tiles along the columns (of the tile's frame)
    int y_type, act, stages;
};

constexpr uint32_t idesc_e4m3(int bn) { return (1u << 4) | (uint32_t(bn >> 3) << 17) | (uint32_t(BM >> 4) << 24); }

__device__ __forceinline__ void tma_load_2d(void *dst, const void *tmap, int x, int y, unsigned long long *bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_u32(dst)), "l"(tmap), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}
// the four MMAs of a block of K
template<int BN> __device__ __forceinline__ void mma_block(uint32_t d, uint64_t a, uint64_t b)
{
    #pragma unroll
    for(int j = 0; j < 4; j++)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a + 2 * j), "l"(b + 2 * j), "r"(idesc_e4m3(BN)), "r"(j) : "memory");
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

// SWAP: the tile's rows are rows of w (and its columns rows of x).
template<int BN, bool SWAP>
__global__ void __launch_bounds__(NUM_THREADS, 1)
scaled_ip_kernel(const __grid_constant__ CUtensorMap tm_r, const __grid_constant__ CUtensorMap tm_c, const Params q, int *status)
{
    extern __shared__ unsigned char smem_raw[];
    constexpr int ACC = BN <= 64 ? 4 : 2;                    // accumulators in tensor memory
    constexpr int TMEM_COLS = ACC * BN < 32 ? 32 : ACC * BN;
    constexpr int STAGE_BYTES = (BM + BN) * BK;
    constexpr int SC = SWAP ? BN : BM;                       // scale products of a block of K
    unsigned char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    Shared *sh = reinterpret_cast<Shared *>(smem);
    float *scale_ring = reinterpret_cast<float *>(smem + 1024);           // two chunks of SC_CHUNK x SC
    unsigned char *ring = smem + 1024 + 2 * SC_CHUNK * SC * 4;
    static_assert(sizeof(Shared) <= 1024 && (SC_CHUNK * SC * 8) % 1024 == 0, "ring alignment");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = q.stages;
    const int parts = int(cluster_size()), part = int(cluster_rank());
    const int tile = int(blockIdx.x) / parts, row_tile = tile / q.n_tiles, col_tile = tile - row_tile * q.n_tiles;
    const int kb0 = part * q.per_part, kblocks = max(0, min(q.per_part, q.kblocks - kb0));
    int *abort_flag = &sh->abort_flag;

    if(threadIdx.x == 0) {
        for(int s = 0; s < S; s++) { mbar_init(&sh->full[s], 1); mbar_init(&sh->empty[s], 1); }
        for(int a = 0; a < 4; a++) { mbar_init(&sh->acc_full[a], 1); mbar_init(&sh->acc_empty[a], 4); }
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

    constexpr int MINE = SC * SC_CHUNK / 128;                // scale products a summing thread brings in per chunk
    float acc[BN];
    #pragma unroll
    for(int j = 0; j < BN; j++) acc[j] = 0.0f;
    const int quad = warp & 3, row_in_tile = quad * 32 + lane;

    if(warp == 0) {
        if(lane == 0) {
            int kb = 0;
            for(; kb < kblocks; kb++) {
                const int s = kb % S;
                if(!mbar_wait(&sh->empty[s], ((kb / S) & 1) ^ 1, abort_flag, status, SIP_EMPTY)) break;
                mbar_arrive_expect_tx(&sh->full[s], STAGE_BYTES);
                tma_load_2d(ring + s * STAGE_BYTES, &tm_r, (kb0 + kb) * BK, row_tile * BM, &sh->full[s]);
                tma_load_2d(ring + s * STAGE_BYTES + BM * BK, &tm_c, (kb0 + kb) * BK, col_tile * BN, &sh->full[s]);
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
    }
    else if(warp == 1) {
        if(lane == 0) {
            constexpr uint64_t DESC_HI = uint64_t((1024u >> 4) | (1u << 14) | (2u << 29)) << 32;   // 8-row groups 1024 bytes apart, version 1, SWIZZLE_128B
            for(int kb = 0; kb < kblocks; kb++) {
                const int s = kb % S, b = kb % ACC;
                if(!mbar_wait(&sh->acc_empty[b], ((kb / ACC) & 1) ^ 1, abort_flag, status, SIP_ACC_EMPTY)) break;
                if(!mbar_wait(&sh->full[s], (kb / S) & 1, abort_flag, status, SIP_FULL)) break;
                tc_fence_after();
                const uint32_t base = ((smem_u32(ring + s * STAGE_BYTES) & 0x3FFFF) >> 4) | (1u << 16);
                mma_block<BN>(tmem_base + b * BN, DESC_HI | base, DESC_HI | (base + (BM * BK >> 4)));
                mma_commit(smem_u32(&sh->empty[s]));
                mma_commit(smem_u32(&sh->acc_full[b]));
            }
        }
    }
    else {
        const int t = threadIdx.x - 64;
        // Products of the scales for the chunk of blocks of K at kb, [block][row of the tile, or column]; zero beyond the matrices.
        float next[MINE];
        auto fetch = [&](int kb) {
            #pragma unroll
            for(int i = 0; i < MINE; i++) {
                const int at = i * 128 + t, b = kb0 + kb + at / SC, j = at % SC;
                const int r = SWAP ? col_tile * BN + j : row_tile * BM + j;
                const int o = SWAP ? row_tile : col_tile * BN / SCALE_BLOCK;
                next[i] = kb + at / SC < kblocks && r < q.rows ? ld_plain(q.x_scales + b * q.x_scale_stride + r) * ld_plain(q.w_scales + o * q.w_scale_stride + b)
                                                               : 0.0f;
            }
        };
        static_assert(SWAP || BN <= SCALE_BLOCK, "one scale of w per tile");
        if(kblocks > 0) fetch(0);
        bool live = true;
        for(int kb = 0; kb < kblocks; kb++) {
            const int in = kb % SC_CHUNK, b = kb % ACC;
            float *sc = scale_ring + (kb / SC_CHUNK & 1) * SC_CHUNK * SC;
            if(in == 0) {
                #pragma unroll
                for(int i = 0; i < MINE; i++) sc[i * 128 + t] = next[i];
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if(kb + SC_CHUNK < kblocks) fetch(kb + SC_CHUNK);
            }
            if(live && !warp_wait(&sh->acc_full[b], (kb / ACC) & 1, abort_flag, status, SIP_ACC_FULL, lane)) live = false;
            if(!live) continue;                              // (the barriers above are met on every path)
            tc_fence_after();
            const uint32_t taddr = tmem_base + (uint32_t(quad * 32) << 16) + b * BN;
            const float mine = SWAP ? 0.0f : sc[in * SC + row_in_tile];
            #pragma unroll
            for(int g = 0; g < BN / 16; g++) {
                uint32_t v[16];
                tmem_ld16(taddr + g * 16, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                #pragma unroll
                for(int j = 0; j < 16; j += 4) {
                    const float4 f = SWAP ? *reinterpret_cast<const float4 *>(sc + in * SC + g * 16 + j) : make_float4(mine, mine, mine, mine);
                    acc[g * 16 + j] += __uint_as_float(v[j]) * f.x;
                    acc[g * 16 + j + 1] += __uint_as_float(v[j + 1]) * f.y;
                    acc[g * 16 + j + 2] += __uint_as_float(v[j + 2]) * f.z;
                    acc[g * 16 + j + 3] += __uint_as_float(v[j + 3]) * f.w;
                }
            }
            tc_fence_before();
            __syncwarp();
            if(lane == 0) mbar_arrive(&sh->acc_empty[b]);
        }
    }

    // ---- tensor memory goes back
    tc_fence_before();
    __syncthreads();
    if(*(volatile int *)abort_flag) {
        // a wait gave up: let the MMAs already issued retire (bounded) before tensor memory goes away
        if(warp == 1 && lane == 0) {
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

    // ---- sum over the parts of K, bias, activation, store
    if(parts > 1) {
        // a part's sums as [column][row of the tile], where its operands were
        float *partial = reinterpret_cast<float *>(ring);
        if(warp >= 2) {
            #pragma unroll
            for(int j = 0; j < BN; j++) partial[j * BM + row_in_tile] = acc[j];
        }
        __syncthreads();
        cluster_sync();
        if(warp >= 2) {
            // part p of the cluster finishes columns p, p + parts, ...
            const uint32_t base = smem_u32(partial);
            const int o = row_tile * BM + row_in_tile;
            const float bias = q.bias && o < q.outputs ? ld_plain(q.bias + o) : 0.0f;
            for(int j = part; j < BN && col_tile * BN + j < q.rows; j += parts) {
                float sum = 0.0f;
                for(int p = 0; p < parts; p++) sum += ld_cluster(base + (j * BM + row_in_tile) * 4, p);
                if(o < q.outputs) store_out(q.y, (long long)(col_tile * BN + j) * q.y_stride + o, q.y_type, apply_act(sum + bias, q.act));
            }
        }
        __syncthreads();
        cluster_sync();                                      // nobody leaves while its sums are being read
    }
    else if(warp >= 2) {
        if(SWAP) {
            const int o = row_tile * BM + row_in_tile;
            const float bias = q.bias && o < q.outputs ? ld_plain(q.bias + o) : 0.0f;
            if(o < q.outputs) {
                #pragma unroll
                for(int j = 0; j < BN; j++)
                    if(col_tile * BN + j < q.rows)
                        store_out(q.y, (long long)(col_tile * BN + j) * q.y_stride + o, q.y_type, apply_act(acc[j] + bias, q.act));
            }
        }
        else {
            const int r = row_tile * BM + row_in_tile;
            if(r < q.rows) {
                #pragma unroll
                for(int j = 0; j < BN; j++) {
                    const int o = col_tile * BN + j;
                    if(o < q.outputs) store_out(q.y, r * q.y_stride + o, q.y_type, apply_act(acc[j] + (q.bias ? ld_plain(q.bias + o) : 0.0f), q.act));
                }
            }
        }
    }
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
                           CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
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

template<int BN, bool SWAP>
static dlp_status launch(const Problem &p, int parts, cudaStream_t stream)
{
    dlp_status st = allow_shared<scaled_ip_kernel<BN, SWAP>>(SMEM_LIMIT);
    if(st != DLP_OK) return st;
    int *status = device_status_word();
    if(!status) return fail(DLP_CUDA_ERROR, "cannot resolve the device status word");
    Params q = { p.x_scales, p.w_scales, p.bias, p.y, p.x_scale_stride, p.w_scale_stride, p.y_stride, p.rows, p.outputs, p.kblocks,
                 ceil_div(p.kblocks, parts), 0, p.y_type, p.act, 0 };
    CUtensorMap mx, mw;
    st = encode_operand(mx, p.x, p.x_stride, p.rows, p.inputs, SWAP ? BN : BM);
    if(st == DLP_OK) st = encode_operand(mw, p.w, p.w_stride, p.outputs, p.inputs, SWAP ? BM : BN);
    if(st != DLP_OK) return st;
    const int fixed = 2048 + 2 * SC_CHUNK * (SWAP ? BN : BM) * 4, stage = (BM + BN) * BK;
    q.stages = std::min(MAX_STAGES, (SMEM_LIMIT - fixed) / stage);
    q.n_tiles = SWAP ? ceil_div(q.rows, BN) : ceil_div(q.outputs, BN);
    const long long blocks = (long long)q.n_tiles * ceil_div(SWAP ? q.outputs : q.rows, BM) * parts;
    DLP_REQUIRE(blocks < (1ll << 31), "too many tiles");
    const int smem = fixed + q.stages * stage;
    DLP_LAUNCH_PDL(launch_pdl_cluster(few_items(blocks), parts, scaled_ip_kernel<BN, SWAP>, unsigned(blocks), NUM_THREADS, smem, stream, SWAP ? mw : mx,
                                      SWAP ? mx : mw, q, status), "scaled_ip_kernel");
    return DLP_OK;
}

} // namespace sip
} // namespace dlp

using namespace dlp;

extern "C" {

dlp_status dlp_scaled_ip_fwd(const void *x, long long x_stride, const float *x_scales, long long x_scale_stride, const void *w,
                             long long w_stride, const float *w_scales, long long w_scale_stride, const float *bias, void *y,
                             long long y_stride, int y_type, int activation, int rows, int inputs, int outputs, void *stream)
{
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
    cudaStream_t s = (cudaStream_t)stream;
    if(rows > 128) return sip::launch_pair(p, s);
    // parts of K until every SM has a tile
    int parts = 1;
    while(parts < sip::MAX_CLUSTER && parts * 2 <= kblocks && oblocks * parts * 2 <= sm_count()) parts *= 2;
    if(rows <= 16) return sip::launch<16, true>(p, parts, s);
    if(rows <= 32) return sip::launch<32, true>(p, parts, s);
    if(rows <= 64) return sip::launch<64, true>(p, parts, s);
    return sip::launch<128, true>(p, parts, s);
}

} // extern "C"

// InnerProduct of 8-bit operands with block scales, many rows: pairs of SMs share a tile of 256 rows x BN outputs (tcgen05 cta_group::2).
//
// A block of K (128) is four tcgen05.mma (M 256, N BN, K 32), into one of 512 / BN accumulators in tensor memory; the sum over blocks is
// kept in fp32 registers, since the scales change from block to block:  acc += (xs[b][row] ws[o / 128][b]) * products.  That is a read of tensor
// memory and an FMA for each product of a block, 128 x BN of them on each SM under the next block's MMAs: 256 cycles on the FMA pipes of the
// 512 that the tensor core needs for N = 256.  Each SM holds half of the operands (128 rows of x, BN / 2 rows of w) in its shared memory: the
// pair reads a row of w once where two single SMs would read it twice.
//   * one warp per SM issues the tensor-map copies of its half; both halves' bytes are counted on the leader's barrier;
//   * one thread of the leader issues the MMAs of the pair; its commits go to both SMs;
//   * eight warps per SM sum: a quarter of the rows and half of the columns each.  They bring the scales in by 4-byte asynchronous copies,
//     eight blocks ahead, each thread its own (no barrier), and store through shared memory and tensor-map stores.
// Tiles are taken in turn (persistent blocks), eight row tiles at a time down the columns, so that what the SMs read at one time stays in L2.
// Every wait is bounded.
#define DLP_INLINE_WAITS
#include "scaled_ip.cuh"

namespace dlp {
namespace sip {
namespace {

constexpr int WARP_COPY = 0, WARP_MMA = 1, WARP_SUM0 = 4;
constexpr int NUM_THREADS = 384, SUM_WARPS = 8;
constexpr int REGS_LAUNCH = 168, REGS_ISSUE = 40, REGS_SUM = 232;
static_assert(REGS_ISSUE + 2 * REGS_SUM <= 3 * REGS_LAUNCH, "setmaxnreg draws on the launch's registers");
constexpr int MAX_STAGES = 8, MAX_ACC = 4;
constexpr int AHEAD = 8;                    // blocks of K whose scales are on their way
constexpr int STORE_BYTES = 4096;           // of a warp: 32 rows of 128 bytes
constexpr int ROW_GROUP = 8;                // row tiles that are taken together

struct Shared {
    unsigned long long full[MAX_STAGES], empty[MAX_STAGES], acc_full[MAX_ACC], acc_empty[MAX_ACC], drain;
    uint32_t tmem_base;
    int abort_flag;
};

struct Params {
    const float *x_scales, *w_scales, *bias;
    void *y;
    long long x_scale_stride, w_scale_stride, y_stride;
    int rows, outputs, kblocks, row_tiles, col_tiles, y_type, act, stages;
    int mapped;             // the result goes out by tensor-map stores
};

__device__ __forceinline__ void tma_load_pair(uint32_t dst, const void *tmap, int x, int y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const void *tmap, int x, int y, uint32_t src)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(tmap), "r"(x), "r"(y), "r"(src) : "memory");
}
// to this barrier in both blocks of the pair
__device__ __forceinline__ void commit_pair(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((unsigned short)3) : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t remote) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory"); }
__device__ __forceinline__ void scale_copy(uint32_t dst, const float *src, bool there)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}

struct Tile { int row, col; };
__device__ __forceinline__ Tile tile_at(int t, const Params &q)
{
    const int in_group = ROW_GROUP * q.col_tiles, g = t / in_group, height = min(ROW_GROUP, q.row_tiles - g * ROW_GROUP);
    t -= g * in_group;
    Tile w;
    w.col = t / height;
    w.row = g * ROW_GROUP + t - w.col * height;
    return w;
}

template<int BN>
__global__ void __launch_bounds__(NUM_THREADS, 1)
scaled_ip_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_y,
                      const Params q, int *status)
{
    extern __shared__ unsigned char smem_raw[];
    constexpr int ACC = 512 / BN;
    constexpr int X_BYTES = BM * BK, W_BYTES = BN / 2 * BK, STAGE_BYTES = X_BYTES + W_BYTES;
    constexpr int COLS = BN / 2;                             // of a summing warp
    unsigned char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    Shared *sh = reinterpret_cast<Shared *>(smem);
    const uint32_t store0 = smem_u32(smem) + 1024;                                  // a store box for each summing warp
    const uint32_t scales0 = store0 + SUM_WARPS * STORE_BYTES;                      // [block of K][thread]: scale of the row, scale of the columns
    const uint32_t ring0 = scales0 + AHEAD * SUM_WARPS * 32 * 8;
    static_assert(sizeof(Shared) <= 1024, "barrier block");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = q.stages, kblocks = q.kblocks;
    const uint32_t rank = cluster_rank();
    const int tiles = q.row_tiles * q.col_tiles, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    int *abort_flag = &sh->abort_flag;

    if(threadIdx.x == 0) {
        for(int s = 0; s < MAX_STAGES; s++) { mbar_init(&sh->full[s], 1); mbar_init(&sh->empty[s], 1); }
        for(int a = 0; a < MAX_ACC; a++) { mbar_init(&sh->acc_full[a], 1); mbar_init(&sh->acc_empty[a], 2 * SUM_WARPS); }
        mbar_init(&sh->drain, 1);
        sh->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if(warp == WARP_MMA) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh->tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                          // the other block's barriers are there
    tc_fence_after();
    const uint32_t tmem_base = *(volatile uint32_t *)&sh->tmem_base;
    pdl_wait();

    if(warp < WARP_SUM0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_ISSUE));
        if(warp == WARP_COPY && lane == 0) {
            uint32_t it = 0;
            bool live = true;
            for(int t = first; t < tiles && live; t += step) {
                const Tile w = tile_at(t, q);
                const int x_row = w.row * 2 * BM + int(rank) * BM, w_row = w.col * BN + int(rank) * (BN / 2);
                for(int kb = 0; kb < kblocks; kb++, it++) {
                    const int s = it % S;
                    if(!mbar_wait(&sh->empty[s], ((it / S) & 1) ^ 1, abort_flag, status, SIP_EMPTY)) { live = false; break; }
                    const uint32_t bar = place_in(smem_u32(&sh->full[s]), 0);
                    if(rank == 0) mbar_arrive_expect_tx(&sh->full[s], 2 * STAGE_BYTES);
                    tma_load_pair(ring0 + s * STAGE_BYTES, &tm_x, kb * BK, x_row, bar);
                    tma_load_pair(ring0 + s * STAGE_BYTES + X_BYTES, &tm_w, kb * BK, w_row, bar);
                }
            }
            // nothing may still be on its way into shared memory when the blocks end (the other block waits for this one below)
            if(rank == 0)
                for(uint32_t n = it > uint32_t(S) ? it - S : 0; n < it; n++) {
                    const long long t0 = global_ns();
                    while(!mbar_try_wait(&sh->full[n % S], (n / S) & 1)) {
                        __nanosleep(256);
                        if(global_ns() - t0 > WAIT_LIMIT_NS) { atomicCAS(status, 0, SIP_DRAIN); break; }
                    }
                }
        }
        else if(warp == WARP_MMA && lane == 0 && rank == 0) {
            constexpr uint32_t IDESC = (1u << 4) | (uint32_t(BN >> 3) << 17) | (uint32_t(2 * BM >> 4) << 24);     // fp32 sums of e4m3, K-major, M 256
            constexpr uint64_t DESC_HI = uint64_t((1024u >> 4) | (1u << 14) | (2u << 29)) << 32;   // 8-row groups 1024 bytes apart, version 1, SWIZZLE_128B
            uint32_t it = 0;
            bool live = true;
            for(int t = first; t < tiles && live; t += step)
                for(int kb = 0; kb < kblocks; kb++, it++) {
                    const int s = it % S, b = it % ACC;
                    if(!mbar_wait(&sh->acc_empty[b], ((it / ACC) & 1) ^ 1, abort_flag, status, SIP_ACC_EMPTY)) { live = false; break; }
                    if(!mbar_wait(&sh->full[s], (it / S) & 1, abort_flag, status, SIP_FULL)) { live = false; break; }
                    tc_fence_after();
                    const uint32_t base = (((ring0 + s * STAGE_BYTES) & 0x3FFFF) >> 4) | (1u << 16);
                    const uint64_t xd = DESC_HI | base, wd = DESC_HI | (base + (X_BYTES >> 4));
                    #pragma unroll
                    for(int j = 0; j < 4; j++)
                        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                                     "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                                     ::"r"(tmem_base + b * BN), "l"(xd + 2 * j), "l"(wd + 2 * j), "r"(IDESC), "r"(j) : "memory");
                    commit_pair(smem_u32(&sh->empty[s]));
                    commit_pair(smem_u32(&sh->acc_full[b]));
                }
        }
    }
    else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SUM));
        const int me = warp - WARP_SUM0, quad = warp & 3, half = me >> 2;
        const uint32_t my_scales = scales0 + (me * 32 + lane) * 8, my_store = store0 + me * STORE_BYTES;
        const uint32_t empty0 = place_in(smem_u32(&sh->acc_empty[0]), 0);
        const float2 clamp = act_clamp(q.act);
        const int oblocks = (q.outputs + SCALE_BLOCK - 1) / SCALE_BLOCK;
        uint32_t it = 0;
        bool live = true;
        // the scales of block kb of a tile: one group of asynchronous copies, empty beyond the last block
        const float *xs = q.x_scales, *ws = q.w_scales;
        bool xs_in = false, ws_in = false;
        auto aim = [&](int t) {
            const Tile w = tile_at(t, q);
            const int row = w.row * 2 * BM + int(rank) * BM + quad * 32 + lane, block = (w.col * BN + half * COLS) / SCALE_BLOCK;
            xs_in = row < q.rows;
            ws_in = block < oblocks;
            xs = q.x_scales + (xs_in ? row : 0);
            ws = q.w_scales + (ws_in ? block * q.w_scale_stride : 0);
        };
        auto ask = [&](int kb) {
            if(kb < kblocks) {
                const uint32_t dst = my_scales + (kb % AHEAD) * (SUM_WARPS * 32 * 8);
                scale_copy(dst, xs + kb * q.x_scale_stride, xs_in);
                scale_copy(dst + 4, ws + kb, ws_in);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        if(first < tiles) {
            aim(first);
            for(int kb = 0; kb < AHEAD; kb++) ask(kb);
        }
        for(int t = first; t < tiles && live; t += step) {
            float acc[COLS];
            #pragma unroll
            for(int j = 0; j < COLS; j++) acc[j] = 0.0f;
            #pragma unroll 1
            for(int kb = 0; kb < kblocks; kb++, it++) {
                const int b = it % ACC;
                asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
                float2 s2;
                asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(s2.x), "=f"(s2.y) : "r"(my_scales + (kb % AHEAD) * (SUM_WARPS * 32 * 8)) : "memory");
                // (written out: it keeps the copy into the same place, asked for below, behind the loads)
                float s;
                asm volatile("mul.f32 %0, %1, %2;" : "=f"(s) : "f"(s2.x), "f"(s2.y) : "memory");
                if(!warp_wait(&sh->acc_full[b], (it / ACC) & 1, abort_flag, status, SIP_ACC_FULL, lane)) { live = false; break; }
                ask(kb + AHEAD);
                tc_fence_after();
                const uint32_t taddr = tmem_base + (uint32_t(quad * 32) << 16) + b * BN + half * COLS;
                uint32_t v[2][32];
                tmem_ld(taddr, v[0]);
                #pragma unroll
                for(int g = 0; g < COLS / 32; g++) {
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if(g + 1 < COLS / 32) tmem_ld(taddr + (g + 1) * 32, v[(g + 1) & 1]);
                    else {
                        tc_fence_before();
                        __syncwarp();
                        if(lane == 0) arrive_at(empty0 + 8 * b);
                    }
                    #pragma unroll
                    for(int j = 0; j < 32; j++) acc[g * 32 + j] = fmaf(__uint_as_float(v[g & 1][j]), s, acc[g * 32 + j]);
                }
            }
            if(!live) break;
            const Tile w = tile_at(t, q);
            if(t + step < tiles) {                           // the next tile's first scales, under this one's way out
                aim(t + step);
                for(int kb = 0; kb < AHEAD; kb++) ask(kb);
            }
            // ---- bias, activation, out
            const int row0 = w.row * 2 * BM + int(rank) * BM + quad * 32, col0 = w.col * BN + half * COLS;
            if(row0 >= q.rows || col0 >= q.outputs) continue;
            #pragma unroll
            for(int g = 0; g < COLS / 32; g++) {
                float bias_g = 0.0f;
                if(q.bias) bias_g = col0 + g * 32 + lane < q.outputs ? ld_plain(q.bias + col0 + g * 32 + lane) : 0.0f;
                if(q.bias) {
                    #pragma unroll
                    for(int j = 0; j < 32; j++) acc[g * 32 + j] += __shfl_sync(0xffffffffu, bias_g, j);
                }
            }
            if(act_is_clamp(q.act)) {
                #pragma unroll
                for(int j = 0; j < COLS; j++) acc[j] = fminf(fmaxf(acc[j], clamp.x), clamp.y);
            }
            else {
                // through shared memory, so that the function is there once and not for every column
                if(lane == 0) bulk_wait_group_read<0>();
                __syncwarp();
                #pragma unroll
                for(int g = 0; g < COLS / 32; g++) {
                    const uint32_t mine = my_store + lane * 128;
                    #pragma unroll
                    for(int c = 0; c < 8; c++)
                        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mine + ((c ^ (lane & 7)) << 4)), "f"(acc[g * 32 + 4 * c]), "f"(acc[g * 32 + 4 * c + 1]),
                                     "f"(acc[g * 32 + 4 * c + 2]), "f"(acc[g * 32 + 4 * c + 3]) : "memory");
                    #pragma unroll 1
                    for(int c = 0; c < 8; c++) {
                        float4 f;
                        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(mine + (c << 4)) : "memory");
                        f.x = apply_act(f.x, q.act); f.y = apply_act(f.y, q.act); f.z = apply_act(f.z, q.act); f.w = apply_act(f.w, q.act);
                        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mine + (c << 4)), "f"(f.x), "f"(f.y), "f"(f.z), "f"(f.w) : "memory");
                    }
                    #pragma unroll
                    for(int c = 0; c < 8; c++)
                        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(acc[g * 32 + 4 * c]), "=f"(acc[g * 32 + 4 * c + 1]), "=f"(acc[g * 32 + 4 * c + 2]),
                                     "=f"(acc[g * 32 + 4 * c + 3]) : "r"(mine + ((c ^ (lane & 7)) << 4)) : "memory");
                }
            }
            // Boxes of 32 rows x 128 bytes in shared memory, swizzled as the map says.  A tensor-map store takes the box away; it leaves out rows and
            // columns beyond the result, but columns only by 16 bytes, so that a box which ends inside such a piece, and results that no map
            // describes, are stored by the warp, a row at a time.
            auto box = [&](const uint32_t (&v)[32], int col, int size) {
                if(col >= q.outputs) return;
                if(lane == 0) bulk_wait_group_read<0>();
                __syncwarp();
                #pragma unroll
                for(int c = 0; c < 8; c++)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(my_store + lane * 128 + ((c ^ (lane & 7)) << 4)), "r"(v[4 * c]), "r"(v[4 * c + 1]),
                                 "r"(v[4 * c + 2]), "r"(v[4 * c + 3]) : "memory");
                const int bytes = min(q.outputs - col, 128 / size) * size;
                if(q.mapped && bytes % 16 == 0) {
                    fence_proxy_async_shared();
                    __syncwarp();
                    if(lane == 0) {
                        tma_store_2d(&tm_y, col, row0, my_store);
                        bulk_commit_group();
                    }
                    return;
                }
                __syncwarp();
                char *at = static_cast<char *>(q.y) + ((long long)row0 * q.y_stride + col) * size + lane * 4;
                const int rows = min(32, q.rows - row0);
                #pragma unroll 1
                for(int r = 0; r < rows; r++, at += q.y_stride * size) {
                    uint32_t word;
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(word) : "r"(my_store + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) : "memory");
                    if(size == 4) {
                        if(lane * 4 < bytes) *reinterpret_cast<uint32_t *>(at) = word;
                    }
                    else {                                   // (a row may start on any element)
                        if(lane * 4 < bytes) *reinterpret_cast<unsigned short *>(at) = (unsigned short)word;
                        if(lane * 4 + 2 < bytes) *reinterpret_cast<unsigned short *>(at + 2) = (unsigned short)(word >> 16);
                    }
                }
                __syncwarp();
            };
            if(q.y_type == DLP_TYPE_F32) {
                #pragma unroll
                for(int g = 0; g < COLS / 32; g++) {
                    uint32_t v[32];
                    #pragma unroll
                    for(int j = 0; j < 32; j++) v[j] = __float_as_uint(acc[g * 32 + j]);
                    box(v, col0 + g * 32, 4);
                }
            }
            else {
                #pragma unroll
                for(int g = 0; g < COLS / 64; g++) {
                    uint32_t v[32];
                    #pragma unroll
                    for(int j = 0; j < 32; j++) {
                        const float lo = acc[g * 64 + 2 * j], hi = acc[g * 64 + 2 * j + 1];
                        if(q.y_type == DLP_TYPE_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v[j]) : "f"(hi), "f"(lo));
                        else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v[j]) : "f"(hi), "f"(lo));
                    }
                    box(v, col0 + g * 64, 2);
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if(lane == 0) bulk_wait_group<0>();
    }

    // ---------------------------------------------------------------------- teardown
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if(rank == 0 && *(volatile int *)abort_flag) {
        // a wait gave up: let the MMAs already issued retire (bounded) before tensor memory goes away
        if(warp == WARP_MMA && lane == 0) {
            asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&sh->drain)) : "memory");
            const long long t0 = global_ns();
            while(!mbar_try_wait(&sh->drain, 0)) {
                __nanosleep(256);
                if(global_ns() - t0 > WAIT_LIMIT_NS) { atomicCAS(status, 0, SIP_DRAIN); break; }
            }
        }
        __syncthreads();
    }
    cluster_sync();                                          // nobody leaves while the other block's copies, MMAs or arrivals may still come here
    if(warp == WARP_MMA) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
    }
}

template<int BN> dlp_status launch_bn(const Problem &p, cudaStream_t stream)
{
    dlp_status st = allow_shared<scaled_ip_pair_kernel<BN>>(SMEM_LIMIT);
    if(st != DLP_OK) return st;
    int *status = device_status_word();
    if(!status) return fail(DLP_CUDA_ERROR, "cannot resolve the device status word");
    Params q = {};
    q.x_scales = p.x_scales; q.w_scales = p.w_scales; q.bias = p.bias; q.y = p.y;
    q.x_scale_stride = p.x_scale_stride; q.w_scale_stride = p.w_scale_stride; q.y_stride = p.y_stride;
    q.rows = p.rows; q.outputs = p.outputs; q.kblocks = p.kblocks; q.y_type = p.y_type; q.act = p.act;
    q.row_tiles = ceil_div(p.rows, 2 * BM);
    q.col_tiles = ceil_div(p.outputs, BN);
    DLP_REQUIRE((long long)q.row_tiles * q.col_tiles < (1ll << 31) / std::max(1, p.kblocks), "too many tiles");
    const size_t size = type_size(p.y_type);
    q.mapped = aligned_to(p.y, 16) && p.y_stride * size % 16 == 0 && p.y_stride * size < (1ull << 40);
    CUtensorMap mx, mw, my = {};
    st = encode_operand(mx, p.x, p.x_stride, p.rows, p.inputs, BM);
    if(st == DLP_OK) st = encode_operand(mw, p.w, p.w_stride, p.outputs, p.inputs, BN / 2);
    if(st == DLP_OK && q.mapped) st = encode_result(my, p);
    if(st != DLP_OK) return st;
    const int fixed = 2048 + SUM_WARPS * STORE_BYTES + AHEAD * SUM_WARPS * 32 * 8, stage = (BM + BN / 2) * BK;
    q.stages = std::min(MAX_STAGES, (SMEM_LIMIT - fixed) / stage);
    const int tiles = q.row_tiles * q.col_tiles, pairs = std::min(tiles, sm_count() / 2);
    DLP_LAUNCH_PDL(launch_pdl_cluster(few_items(2 * tiles), 2, scaled_ip_pair_kernel<BN>, 2 * pairs, NUM_THREADS, fixed + q.stages * stage, stream, mx, mw, my, q,
                                      status), "scaled_ip_pair_kernel");
    return DLP_OK;
}

} // namespace

dlp_status launch_pair(const Problem &p, cudaStream_t stream)
{
    return launch_bn<256>(p, stream);
}

} // namespace sip
} // namespace dlp

// InnerProduct of 8-bit operands with block scales, many rows: pairs of SMs share a tile of 256 rows x BN outputs (tcgen05 cta_group::2).
//
// A block of K (128) is four tcgen05.mma (M 256, N 128, K 32) for each 128 outputs, into one of four accumulators in tensor memory; the sum over
// blocks is kept in fp32 registers, since the scales change from block to block:  acc += (xs[b][row] ws[o / 128][b]) * products.  That is a read of
// tensor memory and an FMA for each product of a block, 128 x BN of them on each SM under the next block's MMAs: 256 cycles on the FMA pipes of the
// 512 that the tensor core needs for 256 outputs.  Each SM holds half of the operands (128 rows of x, BN / 2 rows of w) in its shared memory: the
// pair reads a row of w once where two single SMs would read it twice.
//   * one warp per SM issues the tensor-map copies of its half; both halves' bytes are counted on the leader's barrier;
//   * one thread of the leader issues the MMAs of the pair; its commits go to both SMs;
//   * eight warps per SM sum: a quarter of the rows and half of the columns each, and store through shared memory and tensor-map stores;
//   * two warps per SM bring in the scales, eight blocks of K at a time, and leave their products in shared memory.
// Tiles are taken in turn (persistent blocks), eight row tiles at a time down the columns, so that what the SMs read at one time stays in L2.
// Every wait is bounded.
//
// What bounds it: an accumulator goes round by MMA, commit to both SMs, the read of tensor memory, an arrival at the leader and the next issue, and four
// of them do not hide all of that: a block of K of a tile of 256 outputs takes 820 cycles, of which its MMAs are 512.  8192 rows, 4096 -> 24576: 765 to 830 us (2.0 to
// 2.15 PFLOP/s) in short series, 945 (1.75) in long ones, where the clock falls to 1.57 GHz at 990 W.  What it came from, same product, us: 1736 with arrivals that released
// the thread's other memory operations, too; 841 without, 804 with the scales through shared memory; 812 to 922 with accumulators of 256 columns, two
// of them, measured in turn with this form.
#define DLP_INLINE_WAITS
#include "scaled_ip.cuh"
#include <algorithm>

namespace dlp {
namespace sip {
namespace {

constexpr int WARP_COPY = 0, WARP_MMA = 1, WARP_SCALE0 = 2, WARP_SUM0 = 4;
constexpr int NUM_THREADS = 384, SUM_WARPS = 8;
constexpr int REGS_LAUNCH = 168, REGS_ISSUE = 56, REGS_SUM = 224;
static_assert(REGS_ISSUE + 2 * REGS_SUM <= 3 * REGS_LAUNCH, "setmaxnreg draws on the launch's registers");
constexpr int MAX_STAGES = 8, MAX_ACC = 4, N = 128;        // N: columns of an MMA, and of an accumulator
constexpr int CHUNK = 8;                    // blocks of K whose scales are brought in together
constexpr int SCALE_BYTES = CHUNK * 2 * BM * 4;             // [block][half of the columns][row]
constexpr int STORE_BYTES = 2 * 4096;       // of a warp: two boxes of 32 rows of 128 bytes
constexpr int ROW_GROUP = 8;                // row tiles that are taken together

struct Shared {
    unsigned long long full[MAX_STAGES], empty[MAX_STAGES], acc_full[MAX_ACC], acc_empty[MAX_ACC], scale_full[2], scale_empty[2], drain;
    uint32_t tmem_base;
    int abort_flag;
};

struct Params {
    const float *x_scales, *w_scales, *bias;
    void *y;
    long long x_scale_stride, w_scale_stride, y_stride;
    int rows, outputs, kblocks, row_tiles, col_tiles, y_type, act;
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
// Relaxed: what it says is that tensor memory has been read, and that is complete: every lane has waited for its loads, and the tcgen05 fence and the warp's
// barrier come before it.  No other memory is handed over.  A release to the cluster is a fence of all that the thread did before, at each arrival: 8192 rows,
// 4096 -> 24576 1487 us with it, 765 without, 1024 rows 214 and 110.
__device__ __forceinline__ void arrive_at(bool mine, uint32_t remote)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n\t}" ::"r"(remote), "r"(uint32_t(mine)) : "memory");
}
constexpr int FIXED_BYTES = 2048 + SUM_WARPS * STORE_BYTES + 2 * SCALE_BYTES;       // alignment slack, barriers, store boxes, scales
constexpr int stages_for(int bn) { return std::min(MAX_STAGES, (SMEM_LIMIT - FIXED_BYTES) / ((BM + bn / 2) * BK)); }

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
    constexpr int H = BN / N, SETS = MAX_ACC / H;            // MMAs to a block of K; sets of as many accumulators in tensor memory
    constexpr int X_BYTES = BM * BK, W_BYTES = BN / 2 * BK, STAGE_BYTES = X_BYTES + W_BYTES;
    constexpr int COLS = BN / 2;                             // of a summing warp
    unsigned char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    Shared *sh = reinterpret_cast<Shared *>(smem);
    const uint32_t store0 = smem_u32(smem) + 1024;                                  // a store box for each summing warp
    const uint32_t scales0 = store0 + SUM_WARPS * STORE_BYTES, ring0 = scales0 + 2 * SCALE_BYTES;
    constexpr int S = stages_for(BN);
    static_assert(sizeof(Shared) <= 1024, "barrier block");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kblocks = q.kblocks;
    const uint32_t rank = cluster_rank();
    const int tiles = q.row_tiles * q.col_tiles, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    int *abort_flag = &sh->abort_flag;

    if(threadIdx.x == 0) {
        for(int s = 0; s < MAX_STAGES; s++) { mbar_init(&sh->full[s], 1); mbar_init(&sh->empty[s], 1); }
        for(int a = 0; a < MAX_ACC; a++) { mbar_init(&sh->acc_full[a], 1); mbar_init(&sh->acc_empty[a], 2 * SUM_WARPS / H); }
        for(int a = 0; a < 2; a++) { mbar_init(&sh->scale_full[a], 2); mbar_init(&sh->scale_empty[a], SUM_WARPS); }
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
        // (elected threads: see scaled_ip_few_kernel)
        if(warp == WARP_COPY) {
            if(elect_one()) {
                uint32_t s = 0, phase = 1, count = 0;
                bool live = true;
                const uint32_t full0 = place_in(smem_u32(&sh->full[0]), 0), empty0 = smem_u32(&sh->empty[0]);
                for(int t = first; t < tiles && live; t += step) {
                    const Tile w = tile_at(t, q);
                    const int x_row = w.row * 2 * BM + int(rank) * BM, w_row = w.col * BN + int(rank) * (N / 2);
                    #pragma unroll 1
                    for(int kb = 0; kb < kblocks; kb++) {
                        if(!wait_quietly(empty0 + 8 * s, phase, abort_flag, status, SIP_EMPTY)) { live = false; break; }
                        const uint32_t slot = ring0 + s * STAGE_BYTES, bar = full0 + 8 * s;
                        if(rank == 0) mbar_arrive_expect_tx(&sh->full[s], 2 * STAGE_BYTES);
                        tma_load_pair(slot, &tm_x, kb * BK, x_row, bar);
                        #pragma unroll
                        for(int h = 0; h < H; h++) tma_load_pair(slot + X_BYTES + h * (W_BYTES / H), &tm_w, kb * BK, w_row + h * N, bar);
                        count++;
                        if(++s == S) { s = 0; phase ^= 1; }
                    }
                }
                // nothing may still be on its way into shared memory when the blocks end (the other block waits for this one below)
                if(rank == 0)
                    for(uint32_t n = count > uint32_t(S) ? count - S : 0; n < count; n++) {
                        const long long t0 = global_ns();
                        while(!mbar_try_wait(&sh->full[n % S], (n / S) & 1)) {
                            __nanosleep(256);
                            if(global_ns() - t0 > WAIT_LIMIT_NS) { atomicCAS(status, 0, SIP_DRAIN); break; }
                        }
                    }
            }
            __syncwarp();
        }
        else if(warp == WARP_MMA) {
            if(rank == 0 && elect_one()) {
                constexpr uint32_t IDESC = (1u << 4) | (uint32_t(N >> 3) << 17) | (uint32_t(2 * BM >> 4) << 24);      // fp32 sums of e4m3, K-major, M 256
                constexpr uint64_t DESC_HI = uint64_t((1024u >> 4) | (1u << 14) | (2u << 29)) << 32;   // 8-row groups 1024 bytes apart, version 1, SWIZZLE_128B
                const uint32_t ring = ((ring0 & 0x3FFFF) >> 4) | (1u << 16);
                const uint32_t full0 = smem_u32(&sh->full[0]), empty0 = smem_u32(&sh->empty[0]), acc_full0 = smem_u32(&sh->acc_full[0]), acc_empty0 = smem_u32(&sh->acc_empty[0]);
                uint32_t s = 0, phase = 0, b = 0, b_phase = 1;
                bool live = true;
                const long long total = (long long)((tiles - first + step - 1) / step) * kblocks;
                #pragma unroll 1
                for(long long it = 0; it < total && live; it++) {
                    // (the operands have been there for a while; the accumulator is what is waited for)
                    if(!wait_quietly(full0 + 8 * s, phase, abort_flag, status, SIP_FULL)) break;
                    const uint32_t xd = ring + s * (STAGE_BYTES >> 4);
                    #pragma unroll
                    for(int h = 0; h < H; h++) {
                        const uint32_t wd = xd + ((X_BYTES + h * (W_BYTES / H)) >> 4), acc = b * H + h;
                        if(!wait_quietly(acc_empty0 + 8 * acc, b_phase, abort_flag, status, SIP_ACC_EMPTY)) { live = false; break; }
                        tc_fence_after();
                        #pragma unroll
                        for(int j = 0; j < 4; j++)
                            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                                         "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                                         ::"r"(tmem_base + acc * N), "l"(DESC_HI | (xd + 2 * j)), "l"(DESC_HI | (wd + 2 * j)), "r"(IDESC), "r"(j) : "memory");
                        commit_pair(acc_full0 + 8 * acc);
                    }
                    commit_pair(empty0 + 8 * s);
                    if(++s == S) { s = 0; phase ^= 1; }
                    if(++b == SETS) { b = 0; b_phase ^= 1; }
                }
            }
            __syncwarp();
        }
        else if(warp >= WARP_SCALE0) {
            // products of the two scales, a chunk of blocks of K at a time; a lane has two of the tile's rows
            const int r0 = (warp - WARP_SCALE0) * 64 + lane, oblocks = (q.outputs + SCALE_BLOCK - 1) / SCALE_BLOCK;
            uint32_t slot = 0, phase = 1;
            bool live = true;
            for(int t = first; t < tiles && live; t += step) {
                const Tile w = tile_at(t, q);
                const int row = w.row * 2 * BM + int(rank) * BM + r0, block0 = w.col * BN / SCALE_BLOCK, block1 = (w.col * BN + COLS) / SCALE_BLOCK;
                const bool in0 = row < q.rows, in1 = row + 32 < q.rows, cols0 = block0 < oblocks, cols1 = block1 < oblocks;
                const float *xs = q.x_scales + row, *ws0 = q.w_scales + block0 * q.w_scale_stride, *ws1 = q.w_scales + block1 * q.w_scale_stride;
                #pragma unroll 1
                for(int kb0 = 0; kb0 < kblocks; kb0 += CHUNK) {
                    warp_wait_quietly(smem_u32(&sh->scale_empty[slot]), phase, abort_flag, status, SIP_SCALE_EMPTY, lane == 0);
                    if(*(volatile int *)abort_flag) { live = false; break; }
                    #pragma unroll
                    for(int i0 = 0; i0 < CHUNK; i0 += 4) {
                        float x0[4], x1[4], w0[4], w1[4];
                        #pragma unroll
                        for(int i = 0; i < 4; i++) {
                            const int kb = kb0 + i0 + i;
                            const bool there = kb < kblocks;
                            x0[i] = there && in0 ? ld_plain(xs + kb * q.x_scale_stride) : 0.0f;
                            x1[i] = there && in1 ? ld_plain(xs + kb * q.x_scale_stride + 32) : 0.0f;
                            w0[i] = there && cols0 ? ld_plain(ws0 + kb) : 0.0f;
                            w1[i] = there && cols1 ? ld_plain(ws1 + kb) : 0.0f;
                        }
                        #pragma unroll
                        for(int i = 0; i < 4; i++) {
                            const uint32_t at = scales0 + slot * SCALE_BYTES + ((i0 + i) * 2 * BM + r0) * 4;
                            asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(x0[i] * w0[i]) : "memory");
                            asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + 128), "f"(x1[i] * w0[i]) : "memory");
                            asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + BM * 4), "f"(x0[i] * w1[i]) : "memory");
                            asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + BM * 4 + 128), "f"(x1[i] * w1[i]) : "memory");
                        }
                    }
                    __syncwarp();
                    if(lane == 0) mbar_arrive(&sh->scale_full[slot]);
                    slot ^= 1;
                    if(slot == 0) phase ^= 1;
                }
            }
        }
    }
    else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SUM));
        const int me = warp - WARP_SUM0, quad = warp & 3, half = me >> 2;
        const uint32_t my_store = store0 + me * STORE_BYTES;
        const uint32_t acc_empty0 = place_in(smem_u32(&sh->acc_empty[H == 1 ? 0 : half]), 0), acc_full0 = smem_u32(&sh->acc_full[H == 1 ? 0 : half]);
        const float2 clamp = act_clamp(q.act);
        const uint32_t my_scales = scales0 + (half * BM + quad * 32 + lane) * 4, scale_empty0 = smem_u32(&sh->scale_empty[0]), scale_full0 = smem_u32(&sh->scale_full[0]);
        const bool leader = lane == 0;
        uint32_t it = 0, slot = 1, s_phase = 1, store_at = my_store;
        bool live = true;
        for(int t = first; t < tiles && live; t += step) {
            float acc[COLS];
            #pragma unroll
            for(int j = 0; j < COLS; j++) acc[j] = 0.0f;
            // What a block of K costs beside its products -- waits, the trip to tensor memory -- runs under the last products of the block before:
            // begin() makes the scale ready, waits for the accumulator and asks for its first 32 columns.
            constexpr int G = COLS / 32;
            static_assert(G % 2 == 0, "the two buffers are taken in turn");
            uint32_t v[2][32];
            float s, s_next = 0.0f;
            uint32_t scale_at = 0, taddr = 0;
            auto begin = [&](int kb) {
                if(kb % CHUNK == 0) {
                    slot ^= 1;
                    if(slot == 0) s_phase ^= 1;
                    warp_wait_quietly(scale_full0 + 8 * slot, s_phase, abort_flag, status, SIP_SCALE_FULL, leader);
                    scale_at = my_scales + slot * SCALE_BYTES;
                }
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(s_next) : "r"(scale_at) : "memory");
                scale_at += 2 * BM * 4;
                const uint32_t b = it % SETS;
                warp_wait_quietly(acc_full0 + 8 * b * H, (it / SETS) & 1, abort_flag, status, SIP_ACC_FULL, leader);
                tc_fence_after();
                taddr = tmem_base + (uint32_t(quad * 32) << 16) + b * BN + half * COLS;
                tmem_ld(taddr, v[0]);
            };
            begin(0);
            #pragma unroll 1
            for(int kb = 0; kb < kblocks; kb++) {
                s = s_next;
                #pragma unroll
                for(int g = 0; g < G; g++) {
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if(g + 1 < G) tmem_ld(taddr + (g + 1) * 32, v[(g + 1) & 1]);
                    else {
                        tc_fence_before();
                        __syncwarp();
                        arrive_at(leader, acc_empty0 + 8 * (it % SETS) * H);
                        if(kb % CHUNK == CHUNK - 1 || kb + 1 == kblocks) arrive_if(leader, scale_empty0 + 8 * slot);
                        it++;
                        if(kb + 1 < kblocks) begin(kb + 1);
                    }
                    #pragma unroll
                    for(int j = 0; j < 32; j++) acc[g * 32 + j] = fmaf(__uint_as_float(v[g & 1][j]), s, acc[g * 32 + j]);
                }
                if(kb % CHUNK == 0 && *(volatile int *)abort_flag) {
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    break;
                }
            }
            live = live && !*(volatile int *)abort_flag;
            if(!live) break;
            const Tile w = tile_at(t, q);
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
            if(q.act == DLP_ACT_IDENTITY) {}
            else if(act_is_clamp(q.act)) {
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
                store_at = store_at == my_store ? my_store + 4096 : my_store;
                if(lane == 0) bulk_wait_group_read<1>();         // this box's last store is two back
                __syncwarp();
                #pragma unroll
                for(int c = 0; c < 8; c++)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(store_at + lane * 128 + ((c ^ (lane & 7)) << 4)), "r"(v[4 * c]), "r"(v[4 * c + 1]),
                                 "r"(v[4 * c + 2]), "r"(v[4 * c + 3]) : "memory");
                const int bytes = min(q.outputs - col, 128 / size) * size;
                if(q.mapped && bytes % 16 == 0) {
                    fence_proxy_async_shared();
                    __syncwarp();
                    if(lane == 0) {
                        tma_store_2d(&tm_y, col, row0, store_at);
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
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(word) : "r"(store_at + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) : "memory");
                    if(size == 4) {
                        if(lane * 4 < bytes) *reinterpret_cast<uint32_t *>(at) = word;
                    }
                    else {                                   // (a row may start on any element)
                        if(lane * 4 < bytes) *reinterpret_cast<unsigned short *>(at) = (unsigned short)word;
                        if(lane * 4 + 2 < bytes) *reinterpret_cast<unsigned short *>(at + 2) = (unsigned short)(word >> 16);
                    }
                }
                __syncwarp();
                if(lane == 0) bulk_commit_group();           // an empty one: the waits count boxes
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
        if(lane == 0) bulk_wait_group<0>();
    }

    // ---------------------------------------------------------------------- teardown
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if(rank == 0 && *(volatile int *)abort_flag) {
        // a wait gave up: let the MMAs already issued retire (bounded) before tensor memory goes away
        if(warp == WARP_MMA && elect_one()) {
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
    if(st == DLP_OK) st = encode_operand(mw, p.w, p.w_stride, p.outputs, p.inputs, N / 2);
    if(st == DLP_OK && q.mapped) st = encode_result(my, p);
    if(st != DLP_OK) return st;
    const int tiles = q.row_tiles * q.col_tiles, pairs = std::min(tiles, sm_count() / 2);
    DLP_LAUNCH_PDL(launch_pdl_cluster(few_items(2 * tiles), 2, scaled_ip_pair_kernel<BN>, 2 * pairs, NUM_THREADS, FIXED_BYTES + stages_for(BN) * (BM + BN / 2) * BK, stream, mx, mw, my, q,
                                      status), "scaled_ip_pair_kernel");
    return DLP_OK;
}

} // namespace

dlp_status launch_pair(const Problem &p, int bn, cudaStream_t stream)
{
    note_route("scaled_pair", bn, 1);
    return bn == 256 ? launch_bn<256>(p, stream) : launch_bn<128>(p, stream);
}

} // namespace sip
} // namespace dlp

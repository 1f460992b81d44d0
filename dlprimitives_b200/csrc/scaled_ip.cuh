// InnerProduct of 8-bit operands: what its kernels share (scaled_ip.cu has the entry point and the kernel for few rows, scaled_ip_pair.cu the
// one for many).
#pragma once
#include "block8.cuh"
#include "tc_device.cuh"
#include <cuda.h>

namespace dlp {
namespace sip {

using namespace tc;

constexpr int BM = 128, BK = 128;           // rows of an operand tile; a block of K, one 128-byte row of the swizzled operand tiles
constexpr int SMEM_LIMIT = 227 * 1024;
enum { SIP_EMPTY = 501, SIP_FULL = 502, SIP_ACC_EMPTY = 503, SIP_ACC_FULL = 504, SIP_DRAIN = 505, SIP_SCALE_EMPTY = 506, SIP_SCALE_FULL = 507 };

struct Problem {
    const void *x, *w;
    long long x_stride, w_stride;
    const float *x_scales, *w_scales, *bias;
    void *y;
    long long x_scale_stride, w_scale_stride, y_stride;
    int rows, inputs, outputs;
    int kblocks;            // of the whole K
    int y_type, act;
};

// an 8-bit matrix in boxes of 128 columns x box_rows rows, 128-byte swizzled
dlp_status encode_operand(CUtensorMap &map, const void *p, long long stride, int rows, int cols, int box_rows);
// the result in boxes of 128 bytes x 32 rows, 128-byte swizzled; its rows are on 16-byte boundaries
dlp_status encode_result(CUtensorMap &map, const Problem &p);
dlp_status launch_pair(const Problem &p, int bn, cudaStream_t stream);        // bn: 128 or 256 outputs to a tile

// Bounded wait, as mbar_wait, for kernels whose other warps need the issue slots: a try that may suspend the thread for 2 us costs none of them,
// where one that comes back at once, asked again and again, took a fifth.
__device__ __forceinline__ bool wait_quietly(uint32_t bar, uint32_t parity, int *abort_flag, int *status, int code)
{
    if(mbar_try_wait(bar, parity)) return true;
    const long long t0 = global_ns();
    #pragma unroll 1
    for(;;) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\t"
                     "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 2000;\n\t"
                     "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if(ok) return true;
        if(*(volatile int *)abort_flag) return false;
        if(global_ns() - t0 > WAIT_LIMIT_NS) {
            *(volatile int *)abort_flag = 1;
            atomicCAS(status, 0, code);
            return false;
        }
    }
}
// The same by one lane for its warp (leader: lane 0), for the innermost loops.  Straight-line code as long as the barrier is complete, and nobody
// votes: when the limit runs out the abort flag is raised, and the caller looks at it where it matters; what it reads until then means nothing.
__device__ __forceinline__ void warp_wait_quietly(uint32_t bar, uint32_t parity, int *abort_flag, int *status, int code, bool leader)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p, l;\n\t"
                 "setp.ne.u32 l, %3, 0;\n\t"
                 "setp.eq.u32 p, %3, 0;\n\t"
                 "@l mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity), "r"(uint32_t(leader)) : "memory");
    if(!ok) wait_quietly(bar, parity, abort_flag, status, code);
    __syncwarp();
}
// arrival of one lane, without a branch
__device__ __forceinline__ void arrive_if(bool mine, uint32_t bar)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar), "r"(uint32_t(mine)) : "memory");
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive;" ::: "memory");
    asm volatile("barrier.cluster.wait;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(r)); return r; }
// the same place of shared memory in another block of the cluster
__device__ __forceinline__ uint32_t place_in(uint32_t addr, uint32_t rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}

} // namespace sip
} // namespace dlp

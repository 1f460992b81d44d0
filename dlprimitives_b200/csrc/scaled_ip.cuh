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
dlp_status launch_pair(const Problem &p, cudaStream_t stream);

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

// Draw of a class from each row of logits with given random numbers: temperature, top-k, top-p and min-p.
//
// The classes of a row in the order of falling logits (equal ones in index order) have masses w_i = exp((x_i - max) / t).  top-k keeps
// the first k, top-p of these the shortest prefix with at least p of their mass, min-p of these the ones with w_i >= m (max: w = 1).  The
// class drawn is the first one in index order whose running mass over the kept ones exceeds u times their whole mass.
//
// Which class it is hangs on sums of up to a few hundred thousand masses, compared with a border.  Masses are whole numbers here,
// round(w 2^b) with 63 - log2(classes) bits: their sums are exact in any order, so the result depends neither on timing nor on how
// a row is shared out.  Nothing is sorted: a radix selection on the logits' bits finds where each prefix ends, eight bits a step.
#include "block8.cuh"

namespace dlp {
namespace {

typedef unsigned long long u64;

struct SampleArgs {
    const void *x;
    const float *temperature, *top_p, *min_p, *u;
    const int *top_k;
    int *tokens;
    long long stride;
    int classes, bits;      // bits of a mass of 1
};

constexpr int THREADS = 1024, WARPS = THREADS / 32;
constexpr unsigned MASKED = 0;                   // the key of -inf and of NaN

// Keys are ordered as the logits; 0 for classes that cannot be drawn.
__device__ __forceinline__ unsigned key_of(float v)
{
    const unsigned b = __float_as_uint(v);
    if(!(v > __int_as_float(0xff800000))) return MASKED;
    return v == 0.0f ? 0x80000000u : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

struct Row {
    double top, inverse_t, one;                  // largest logit; 1 / temperature; mass of 1
    unsigned top_key;
    __device__ __forceinline__ double weight(unsigned key) const
    {
        return key == top_key ? 1.0 : (key == MASKED ? 0.0 : exp((double(value_of(key)) - top) * inverse_t));
    }
    __device__ __forceinline__ u64 mass(unsigned key) const { return u64(__double2ll_rn(weight(key) * one)); }
};

// Where a prefix of the sorted row ends: all above `key` and the first `ties` of those equal to it.
struct Cut { unsigned key; unsigned ties; };

struct Shared {
    u64 mass[256];
    unsigned count[256];
    u64 warp_mass[WARPS];
    unsigned warp_count[WARPS], digit, rest;
    u64 above;
    int token;
};

template<typename T>
__global__ void __launch_bounds__(THREADS) sample_kernel(const SampleArgs a)
{
    pdl_wait();
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.classes;
    const long long row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.stride;
    auto key_at = [&](int i) { return key_of(to_float(ld_plain(x + i))); };

    unsigned top = MASKED;
    for(int i = tid; i < n; i += THREADS) top = max(top, key_at(i));
    top = __reduce_max_sync(0xffffffffu, top);
    if(lane == 0) sh.warp_count[warp] = top;
    __syncthreads();
    for(int i = 0; i < WARPS; i++) top = max(top, sh.warp_count[i]);
    if(top == MASKED) {                          // nothing to draw from
        if(tid == 0) a.tokens[row] = -1;
        return;
    }
    const float t = a.temperature ? ld_plain(a.temperature + row) : 1.0f;
    const bool greedy = !(t > 0.0f);
    Row r;
    r.top_key = top;
    r.top = double(value_of(top));
    r.inverse_t = greedy ? 1.0 : 1.0 / double(t);
    r.one = double(1ull << a.bits);
    const int k = greedy ? 1 : (a.top_k ? ld_plain(a.top_k + row) : 0);
    const float p = a.top_p ? ld_plain(a.top_p + row) : 1.0f, m = a.min_p ? ld_plain(a.min_p + row) : 0.0f, uf = ld_plain(a.u + row);

    // The end of the shortest prefix that holds `want` classes, or that much mass, of the classes that `limit` keeps; the mass above its key.
    auto select = [&](bool by_mass, u64 want, Cut limit, u64 &above) {
        unsigned prefix = 0;
        above = 0;
        u64 left = want;
        unsigned equal = 0;
        for(int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if(tid < 256) { sh.mass[tid] = 0; sh.count[tid] = 0; }
            __syncthreads();
            for(int i = tid; i < n; i += THREADS) {
                const unsigned key = key_at(i);
                if(key == MASKED || key < limit.key || (shift < 24 && (key ^ prefix) >> (shift + 8))) continue;
                const unsigned d = key >> shift & 255;
                atomicAdd(&sh.mass[d], r.mass(key));
                atomicAdd(&sh.count[d], 1u);
            }
            __syncthreads();
            if(tid == 0) {
                u64 more = 0;
                int d = 255;
                for(; d > 0; d--) {
                    u64 here = by_mass ? sh.mass[d] : sh.count[d];
                    // (of the limit's own key only the first ties count)
                    if(by_mass && shift == 0 && (prefix | d) == limit.key && limit.ties < sh.count[d]) here = limit.ties * r.mass(limit.key);
                    if(here >= left) break;
                    left -= here;
                    more += sh.mass[d];
                }
                sh.digit = d;
                sh.above = more;
                sh.rest = sh.count[d];
                sh.mass[0] = left;
            }
            __syncthreads();
            prefix |= sh.digit << shift;
            above += sh.above;
            left = sh.mass[0];
            equal = sh.rest;
        }
        Cut c;
        c.key = prefix;
        const u64 w = r.mass(prefix);
        const u64 need = by_mass ? (w ? (left + w - 1) / w : 1) : left;
        c.ties = unsigned(need < equal ? need : equal);
        if(c.key == limit.key && c.ties > limit.ties) c.ties = limit.ties;
        return c;
    };

    Cut cut = { 1u, 0xffffffffu };
    u64 whole = 0;
    bool known = false;                          // whole: the mass of what `cut` keeps
    if(k > 0 && k < n) {
        cut = select(false, u64(k), cut, whole);
        whole += cut.ties * r.mass(cut.key);
        known = true;
    }
    if(!greedy && p < 1.0f) {
        if(!known) {
            u64 mine = 0;
            for(int i = tid; i < n; i += THREADS) mine += r.mass(key_at(i));
            for(int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
            __syncthreads();
            if(lane == 0) sh.warp_mass[warp] = mine;
            __syncthreads();
            for(int i = 0; i < WARPS; i++) whole += sh.warp_mass[i];
        }
        // the least whole number that is no less than p * whole
        const u64 pf = p > 0.0f ? u64(double(p) * 18446744073709551616.0) : 0;
        u64 want = __umul64hi(pf, whole) + (pf * whole != 0);
        if(want == 0) want = 1;
        u64 above;
        cut = select(true, want, cut, above);
    }

    // Masses in index order: the whole of the kept ones first, then where the running sum passes u times that.
    const double least = m > 0.0f ? fmin(double(m), 1.0) : 0.0;
    u64 target = 0;
    for(int pass = 0; pass < 2; pass++) {
        u64 before = 0;
        unsigned ties_before = 0;
        if(pass == 1 && tid == 0) sh.token = n;
        for(int i0 = 0; i0 < n; i0 += THREADS) {
            const int i = i0 + tid;
            const unsigned key = i < n ? key_at(i) : MASKED;
            const bool tie = key == cut.key;
            const unsigned votes = __ballot_sync(0xffffffffu, tie);
            __syncthreads();
            if(lane == 0) sh.warp_count[warp] = __popc(votes);
            __syncthreads();
            unsigned ties = ties_before + __popc(votes & ((1u << lane) - 1));
            for(int j = 0; j < WARPS; j++) {
                if(j < warp) ties += sh.warp_count[j];
                ties_before += sh.warp_count[j];
            }
            u64 w = 0;
            if(key > cut.key || (tie && ties < cut.ties)) {
                const double f = r.weight(key);
                if(f >= least) w = u64(__double2ll_rn(f * r.one));
            }
            u64 run = w;
            for(int o = 1; o < 32; o <<= 1) {
                const u64 other = __shfl_up_sync(0xffffffffu, run, o);
                if(lane >= o) run += other;
            }
            if(lane == 31) sh.warp_mass[warp] = run;
            __syncthreads();
            run += before;
            for(int j = 0; j < WARPS; j++) {
                if(j < warp) run += sh.warp_mass[j];
                before += sh.warp_mass[j];
            }
            if(pass == 1 && w > 0 && run > target && run - w <= target) sh.token = i;
        }
        if(pass == 0) {
            const u64 uu = uf > 0.0f ? (uf < 1.0f ? u64(double(uf) * 18446744073709551616.0) : ~0ull) : 0;
            target = __umul64hi(uu, before);
        }
    }
    __syncthreads();
    if(tid == 0) a.tokens[row] = sh.token;
}

template<typename T> dlp_status launch_sample(const SampleArgs &a, int rows, cudaStream_t stream)
{
    DLP_LAUNCH_PDL(launch_pdl(one_wave(rows, THREADS), sample_kernel<T>, rows, THREADS, 0, stream, a), "sample_kernel");
    return DLP_OK;
}

} // namespace
} // namespace dlp

using namespace dlp;

extern "C" {

dlp_status dlp_sample_fwd(const void *logits, long long stride, int type, int rows, int classes, const float *temperature, const int *top_k,
                          const float *top_p, const float *min_p, const float *u, int *tokens, void *stream)
{
    DLP_REQUIRE(rows >= 0 && classes > 0 && classes <= DLP_SAMPLE_MAX_CLASSES, "bad shape");
    DLP_REQUIRE(is_real_type(type), "the logits' type must be fp32, fp16 or bf16");
    if(rows == 0) return DLP_OK;
    DLP_REQUIRE(logits && u && tokens, "null tensor");
    DLP_REQUIRE(rows <= 1 || stride >= classes, "rows overlap");
    DLP_REQUIRE(aligned_to(logits, type_size(type)) && aligned_to(u, 4) && aligned_to(tokens, 4) && aligned_to(temperature, 4) && aligned_to(top_k, 4) &&
                aligned_to(top_p, 4) && aligned_to(min_p, 4), "a tensor is not aligned to its elements");
    int log2 = 0;
    while((1ll << log2) < classes) log2++;
    const SampleArgs a = { logits, temperature, top_p, min_p, u, top_k, tokens, stride, classes, std::min(52, 63 - log2) };
    if(type == DLP_TYPE_F32) return launch_sample<float>(a, rows, (cudaStream_t)stream);
    if(type == DLP_TYPE_F16) return launch_sample<__half>(a, rows, (cudaStream_t)stream);
    return launch_sample<__nv_bfloat16>(a, rows, (cudaStream_t)stream);
}

} // extern "C"

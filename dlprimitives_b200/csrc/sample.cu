// Draw of a class from each row of logits with given random numbers: temperature, top-k, top-p and min-p.
//
// The classes of a row in the order of falling logits (equal ones in index order) have masses w_i = exp((x_i - max) / t).  top-k keeps
// the first k, top-p of these the shortest prefix with at least p of their mass, min-p of these the ones with w_i >= m (max: w = 1).  The
// class drawn is the first one in index order whose running mass over the kept ones exceeds u times their whole mass.
//
// Which class it is hangs on sums of up to a few hundred thousand masses, compared with a border.  Masses are whole numbers here,
// round(w 2^b), b = min(51, 63 - log2(classes) rounded up): their sums are exact in any order, so the result depends neither on timing nor on how
// a row is shared out.  A sum is off by up to half a unit, 2^-(b+1) of the largest mass, for each class in it; classes under half a unit
// have no mass.
//
// A row is read a few times, from memory once and then from L2, by a cluster of 1 to 8 blocks (so that few rows use the whole GPU); the
// blocks gather what each has found through distributed shared memory and all come to the same conclusions.
//   * First the largest logit, and the largest of each of 512 groups of classes.
//   * With a small k (up to 256): the k-th largest of the groups' maxima has at least k classes at or above it, and for classes in no
//     particular order only a few more (512 ln(512 / (512 - k)) of them are expected).  These are collected, and the rest is done on
//     them alone: two readings of the row, and masses of a few hundred classes.
//   * Otherwise the end of a prefix is found from sums over 2048 bins of falling logits: the bin it lies in is collected, and divided
//     further as long as it holds more than 512 classes.  Then the masses of the kept classes are summed by
//     segments of the row, and the one segment that the random number points into is gone through.
//
// Measured (captured): one row of 32000 with top-p and k of 50 9.5 us, of 200 15.7, of 300 (no small k any more) 44, top-p alone 25, neither 9.5, greedy 4.0; 64 rows of
// 128000 bf16 without settings 32, with top-p 75, 256 rows of 150001 fp32 with settings of their own 137.  Two blocks of 512 threads on an SM leave 64
// registers, under which some are spilled (16-bit logits 140 bytes stored and 268 loaded a thread, fp32 272 and 380).  Memory is not what bounds it (they are 128 KB, 16 MB and 154 MB): one row is a chain of barriers, short sorts and first
// fetches of code, 7500 cycles up to the k-th largest, 5500 to collect, 13000 for the list; many rows are masses (about 30 instructions to a
// class, 17000 cycles for 64000 on an SM) and sums over bins (two atomic additions to a class, 25000).  Tried: masses of fp32 pairs, within 2^-30, a tenth
// less on rows without settings, nothing on the others; halves of the bins in arrays of their own, and barriers that a block only waits for when it
// needs them: nothing.
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

constexpr int THREADS = 512, WARPS = THREADS / 32, MAX_PARTS = 8;
constexpr int BINS = 2048, CAP = THREADS;        // bins of a histogram; classes that are sorted at once
constexpr int SMALL_K = 256;
constexpr unsigned MASKED = 0;                   // the key of -inf and of NaN
constexpr unsigned LOWEST = 0x00800000u;         // the key of the lowest finite number

// Keys are ordered as the logits; 0 for classes that cannot be drawn.
__device__ __forceinline__ unsigned key_of(float v)
{
    const unsigned b = __float_as_uint(v);
    if(!(v > __int_as_float(0xff800000))) return MASKED;
    return v == 0.0f ? 0x80000000u : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
// Low bits that are the same in the keys of all numbers of one sign.
template<typename T> constexpr int grain_bits = sizeof(T) == 4 ? 0 : 13;
template<> constexpr int grain_bits<__nv_bfloat16> = 16;

struct Scratch {
    u64 all_mass[BINS];                          // sums over the row's classes,
    unsigned all_count[BINS];
    uint2 mass[BINS];                            // and over this block's, in two halves
    unsigned count[BINS];
    u64 cand[CAP], list[CAP], list_mass[CAP];    // classes as (key, ~index): this block's, and the row's with their masses
    u64 sorted[2][CAP];
    u64 seg_mass[WARPS];                         // kept masses of each warp's segment, and classes equal to the cut's key
    unsigned seg_ties[WARPS];
    u64 best[WARPS];
    unsigned group[THREADS];
    u64 warp_sum[2][WARPS];
    u64 found[3], rest[2];
    double table[1024];                          // of Masses
    unsigned cands;
};

// ---- distributed shared memory: the same place in another block of the cluster
__device__ __forceinline__ uint32_t place_in(const void *p, int rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ u64 peer(const u64 *p, int rank)
{
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(place_in(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ unsigned peer(const unsigned *p, int rank)
{
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(place_in(p, rank)) : "memory");
    return v;
}

// A mass of a class.  w = 2^-t with t = (max - x) log2(e) / temperature, in 64 bits: t = i + j / 1024 + r with whole i and j, |r| <= 1/2048, and
// 2^-r by the series of exp(-r ln 2), whose fourth term is under 2^-50.
constexpr int STEPS = 1024;
struct Masses {
    double top_t, factor, one;                   // factor: log2(e) / temperature; top_t: max times that; one: 2^bits
    float top;
    const double *table;                         // 2^(-j / STEPS)
    // No branches: a chain of dependent operations, of which several run side by side where several are asked for.
    __device__ __forceinline__ double weight(float x) const
    {
        const double v = double(x), magic = 6755399441055744.0 / STEPS, t = fma(-v, factor, top_t), z = t + magic, r = t - (z - magic);
        const int k = __double2loint(z);         // STEPS i + j
        constexpr double L = 0.69314718055994530942, C2 = L * L / 2, C3 = L * C2 / 3;
        const double e = fma(r, fma(r, fma(r, -C3, C2), -L), 1.0) * table[k & (STEPS - 1)];
        // for t < 1000: e is in (0.49, 1.01), k / STEPS under 1001, and the exponent stays normal.  (t is infinite or NaN for -inf and NaN, and where the
        // largest logit is infinite.)
        const double w = t < 1000.0 ? __hiloint2double(__double2hiint(e) - (k / STEPS << 20), __double2loint(e)) : 0.0;
        return x == top ? 1.0 : w;
    }
    // a whole number below 2^52 is the low part of itself + 2^52
    __device__ __forceinline__ u64 whole(double w) const { return u64(__double_as_longlong(fma(w, one, 4503599627370496.0)) & 0xfffffffffffffll); }
    __device__ __forceinline__ u64 mass(float x) const { return whole(weight(x)); }
    __device__ __forceinline__ u64 mass(unsigned key) const { return mass(value_of(key)); }
};

// Where a prefix of the sorted row ends: all above `key` and the first `ties` of those equal to it.
struct Cut { unsigned key, ties; };

// ---- over the block (every thread takes part)
// Sum up to and with this thread's value, and of all.  flip: changes from call to call, so that one barrier a call is enough.
__device__ __forceinline__ u64 scan(u64 v, Scratch &sh, int &flip, u64 &all)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    #pragma unroll
    for(int o = 1; o < 32; o <<= 1) {
        const u64 other = __shfl_up_sync(0xffffffffu, v, o);
        if(lane >= o) v += other;
    }
    flip ^= 1;
    if(lane == 31) sh.warp_sum[flip][warp] = v;
    __syncthreads();
    u64 sums = sh.warp_sum[flip][lane & (WARPS - 1)];
    #pragma unroll
    for(int o = 1; o < WARPS; o <<= 1) {
        const u64 other = __shfl_up_sync(0xffffffffu, sums, o);
        if((lane & (WARPS - 1)) >= o) sums += other;
    }
    all = __shfl_sync(0xffffffffu, sums, WARPS - 1);
    const u64 before = __shfl_sync(0xffffffffu, sums, warp > 0 ? warp - 1 : 0);
    return v + (warp > 0 ? before : 0);
}
// Sum over the block; flip: as in scan.
__device__ __forceinline__ u64 sum_all(u64 v, Scratch &sh, int &flip)
{
    const int lane = threadIdx.x & 31;
    #pragma unroll
    for(int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    flip ^= 1;
    if(lane == 0) sh.warp_sum[flip][threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh.warp_sum[flip][lane & (WARPS - 1)];
    #pragma unroll
    for(int o = WARPS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Lists of up to CAP classes in shared memory.  Short ones are gone through, each class against each, by `each` neighbouring threads (a power of two, at
// most 32) to a class that share the list: f(number, mass) for a thread's share.  Long ones are sorted.
constexpr int COUNTED = 256;
template<typename F> __device__ __forceinline__ void through(const Scratch &sh, int total, int each, F f)
{
    #pragma unroll 4
    for(int i = threadIdx.x & (each - 1); i < total; i += each) f(sh.list[i], sh.list_mass[i]);
}
__device__ __forceinline__ u64 sum_of(u64 v, int each)       // over the threads that share a class
{
    for(int o = 1; o < each; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sorts the threads' numbers, the largest first.
__device__ __forceinline__ u64 sort(u64 v, Scratch &sh)
{
    const int tid = threadIdx.x;
    int buf = 0;
    #pragma unroll 1
    for(int k = 2; k <= THREADS; k <<= 1)
        #pragma unroll 1
        for(int j = k >> 1; j > 0; j >>= 1) {
            u64 other;
            if(j >= 32) {
                sh.sorted[buf][tid] = v;
                __syncthreads();
                other = sh.sorted[buf][tid ^ j];
                buf ^= 1;
            }
            else other = __shfl_xor_sync(0xffffffffu, v, j);
            const bool larger = ((tid & j) == 0) == ((tid & k) == 0 || k == THREADS);
            v = larger == (v > other) ? v : other;
        }
    return v;
}

template<typename T>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const SampleArgs a)
{
    pdl_wait();
    extern __shared__ __align__(16) unsigned char smem[];
    Scratch &sh = *reinterpret_cast<Scratch *>(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.classes;
    int parts, part, flip = 0;
    asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(parts));
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(part));
    const long long row = blockIdx.x / parts;
    const T *x = static_cast<const T *>(a.x) + row * a.stride;
    auto everyone = [&] {
        if(parts > 1) {
            asm volatile("barrier.cluster.arrive;" ::: "memory");
            asm volatile("barrier.cluster.wait;" ::: "memory");
        }
        else __syncthreads();
    };

    // The row in pieces of 16 bytes on their boundaries; each warp of the cluster has a segment of consecutive ones.
    constexpr int V = 16 / sizeof(T);
    const int shift = int(reinterpret_cast<uintptr_t>(x) / sizeof(T) % V);
    const int pieces = (n + shift + V - 1) / V, per = ceil_div(pieces, parts * WARPS);
    const int piece0 = min(pieces, (part * WARPS + warp) * per), piece1 = min(pieces, piece0 + per);
    // f(logit, index) for the segment's classes, a piece at a time (f is there 4 V times: something short); a thread's come in index order
    auto each = [&](auto f) {
        constexpr int DEEP = 4;
        #pragma unroll 1
        for(int p = piece0 + lane; p < piece1; p += 32 * DEEP) {
            union { uint4 w; T e[V]; } u[DEEP];
            #pragma unroll
            for(int d = 0; d < DEEP; d++) {
                const int i0 = (p + d * 32) * V - shift;
                if(p + d * 32 < piece1 && i0 >= 0 && i0 + V <= n) u[d].w = ld_plain(reinterpret_cast<const uint4 *>(x + i0));
            }
            #pragma unroll
            for(int d = 0; d < DEEP; d++) {
                const int i0 = (p + d * 32) * V - shift;
                if(p + d * 32 >= piece1) break;
                if(i0 < 0 || i0 + V > n) {                   // the row's ends
                    #pragma unroll
                    for(int e = 0; e < V; e++) u[d].e[e] = i0 + e >= 0 && i0 + e < n ? ld_plain(x + i0 + e) : from_float<T>(__int_as_float(0xff800000));
                }
                #pragma unroll
                for(int e = 0; e < V; e++) f(to_float(u[d].e[e]), i0 + e);
            }
        }
    };
    // f(logits) for the segment's classes, BATCH a thread at a time (-inf: none): their masses are worked out side by side, under the load of the next piece
    constexpr int BATCH = 2;
    auto each_batch = [&](auto f) {
        union Piece { uint4 w; T e[V]; } u0, u1;
        auto ask = [&](int p, Piece &u) {
            const int i0 = p * V - shift;
            if(p < piece1 && i0 >= 0 && i0 + V <= n) u.w = ld_plain(reinterpret_cast<const uint4 *>(x + i0));
            else {
                #pragma unroll
                for(int e = 0; e < V; e++) u.e[e] = p < piece1 && i0 + e >= 0 && i0 + e < n ? ld_plain(x + i0 + e) : from_float<T>(__int_as_float(0xff800000));
            }
        };
        auto take = [&](const Piece &u) {
            #pragma unroll
            for(int e = 0; e < V; e += BATCH) {
                float v[BATCH];
                #pragma unroll
                for(int d = 0; d < BATCH; d++) v[d] = to_float(u.e[e + d]);
                f(v);
            }
        };
        int p = piece0 + lane;
        if(p >= piece1) return;
        ask(p, u0);
        #pragma unroll 1
        for(;; p += 64) {
            if(p + 32 < piece1) ask(p + 32, u1);
            take(u0);
            if(p + 32 >= piece1) break;
            if(p + 64 < piece1) ask(p + 64, u0);
            take(u1);
            if(p + 64 >= piece1) break;
        }
    };

    // (asked for early, all at once)
    const float t = a.temperature ? ld_plain(a.temperature + row) : 1.0f, p = a.top_p ? ld_plain(a.top_p + row) : 1.0f;
    const float m = a.min_p ? ld_plain(a.min_p + row) : 0.0f, uf = ld_plain(a.u + row);
    const int asked = a.top_k ? ld_plain(a.top_k + row) : 0, k = t > 0.0f ? asked : 1;

    // ---- the largest logit, its first place, and the groups' largest (a group: `parts` neighbouring threads)
    for(int i = tid; i < STEPS; i += THREADS) sh.table[i] = exp2(i * (-1.0 / STEPS));
    if(tid == 0) sh.cands = 0;
    float most = __int_as_float(0xff800000);
    int where = 0;
    each([&](float v, int i) {
        if(v > most) { most = v; where = i; }
    });
    unsigned group = key_of(most);
    u64 best = u64(group) << 32 | unsigned(~where);
    for(int o = 1; o < parts; o <<= 1) group = max(group, __shfl_xor_sync(0xffffffffu, group, o));
    if(tid % parts == 0) sh.group[tid / parts] = group;
    #pragma unroll
    for(int o = 16; o > 0; o >>= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if(lane == 0) sh.best[warp] = best;
    everyone();
    {
        const int per_part = THREADS / parts;
        group = parts > 1 ? peer(sh.group + tid % per_part, tid / per_part) : sh.group[tid];
    }
    for(int i = lane; i < parts * WARPS; i += 32) {
        const u64 other = parts > 1 ? peer(sh.best + i % WARPS, i / WARPS) : sh.best[i];
        best = other > best ? other : best;
    }
    #pragma unroll
    for(int o = 16; o > 0; o >>= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    const unsigned top = unsigned(best >> 32);
    if(top == MASKED || k == 1) {                // nothing to draw from, or one
        if(part == 0 && tid == 0) a.tokens[row] = top == MASKED ? -1 : int(~unsigned(best));
        everyone();                              // nobody leaves while its memory is being read
        return;
    }
    Masses f;
    f.top = value_of(top);
    f.factor = 1.4426950408889634074 / double(t);
    f.top_t = double(f.top) * f.factor;
    f.one = double(1ull << a.bits);
    f.table = sh.table;
    // min-p keeps the logits from `least_kept` on: the least one with exp((x - max) / t) >= m.  The estimate max + t ln m is right to a few units of
    // fp32, and the lanes try the numbers around it.  (Classes under it need no mass: 64 rows of 128000 33 -> 29 us, where each mass was compared before.)
    float least_kept = __int_as_float(0xff800000);
    if(m >= 1.0f) least_kept = f.top;
    else if(m > 0.0f && f.top < __int_as_float(0x7f800000)) {
        const float guess = float(double(f.top) + double(t) * log(double(m)));
        if(guess >= __int_as_float(0xff7fffff)) {            // (else all finite ones are kept)
            const unsigned key = key_of(guess) + lane - 16;
            const float x = value_of(key);
            const bool in = key >= top || (key >= LOWEST && f.weight(x) >= double(m));
            const unsigned yes = __ballot_sync(0xffffffffu, in);
            least_kept = fminf(__shfl_sync(0xffffffffu, x, yes ? __ffs(yes) - 1 : 31), f.top);
        }
    }
    // the least whole number that is no less than p times `whole`
    auto share_of = [&](u64 whole) {
        const u64 pf = p > 0.0f ? u64(double(p) * 18446744073709551616.0) : 0;
        const u64 want = __umul64hi(pf, whole) + (pf * whole != 0);
        return want > 0 ? want : 1;
    };
    auto point_in = [&](u64 whole) { return __umul64hi(uf > 0.0f ? (uf < 1.0f ? u64(double(uf) * 18446744073709551616.0) : ~0ull) : 0ull, whole); };

    // Collects the classes with lo <= key <= hi (lo > MASKED): their number, and in every block the list of them with their masses, in no order, if
    // there are at most CAP.  The second barrier comes after the last look into another block's memory.
    auto collect = [&](unsigned lo, unsigned hi) {
        const float low = value_of(lo), high = value_of(hi);
        each([&](float v, int i) {
            if(v >= low && v <= high) {
                const unsigned at = atomicAdd(&sh.cands, 1u);
                if(at < CAP) sh.cand[at] = u64(key_of(v)) << 32 | unsigned(~i);
            }
        });
        everyone();
        unsigned total = 0, place = 0;
        int from = 0;
        for(int q = 0; q < parts; q++) {
            const unsigned c = parts > 1 ? peer(&sh.cands, q) : sh.cands;
            if(unsigned(tid) >= total && unsigned(tid) < total + c) { from = q; place = tid - total; }
            total += c;
        }
        u64 mine = 0;
        if(total <= CAP && unsigned(tid) < total) mine = parts > 1 ? peer(sh.cand + place, from) : sh.cand[place];
        everyone();
        if(tid == 0) sh.cands = 0;
        if(mine) {
            sh.list[tid] = mine;
            sh.list_mass[tid] = f.mass(unsigned(mine >> 32));
        }
        __syncthreads();
        return int(min(total, CAP + 1u));
    };
    // threads to a class of a short list
    auto share = [](int total) {
        int e = 1;
        while(e < 32 && total * e * 2 <= THREADS) e <<= 1;
        return e;
    };
    // The list in order: a thread's class, its mass, its place, and the mass of what comes before it.  True for one thread of each class.
    auto arrange = [&](int total, u64 &mine, u64 &mass, u64 &place, u64 &above) {
        if(total <= COUNTED) {
            const int e = share(total), me = tid / e;
            const u64 id = me < total ? sh.list[me] : 0;
            u64 p = 0, m = 0;
            through(sh, total, e, [&](u64 c, u64 w) {
                if(c > id) { p++; m += w; }
            });
            mine = id;
            mass = me < total ? sh.list_mass[me] : 0;
            place = sum_of(p, e);
            above = sum_of(m, e);
            return me < total && (tid & (e - 1)) == 0;
        }
        mine = sort(tid < total ? sh.list[tid] : 0, sh);
        mass = tid < total ? f.mass(unsigned(mine >> 32)) : 0;
        u64 all;
        place = tid;
        above = scan(mass, sh, flip, all) - mass;
        return tid < total;
    };

    // ---- few classes are kept: all of them in one sorted list
    const bool few = k > 0 && k <= SMALL_K && k < n;
    if(few || n <= CAP) {
        unsigned floor_key = LOWEST;
        if(few) {
            // the k-th largest of the groups' maxima, from the top bit in which they differ down; done when exactly k of them are left (and but for the
            // last eight bits: a little lower is as good)
            const unsigned differ = __reduce_or_sync(0xffffffffu, group ^ top);
            if(lane == 0) sh.seg_ties[warp] = differ;        // (free yet; the groups' maxima may still be read by other blocks)
            __syncthreads();
            const unsigned any = __reduce_or_sync(0xffffffffu, sh.seg_ties[lane & (WARPS - 1)]);
            const int high = 31 - __clz(int(any | 1));
            unsigned at = high == 31 ? 0 : top >> (high + 1) << (high + 1);
            #pragma unroll 1
            for(int bit = high; bit >= 8; bit--) {
                const unsigned higher = at | 1u << bit;
                const int above = __syncthreads_count(group >= higher);
                if(above >= k) at = higher;
                if(above == k) break;
            }
            floor_key = max(at, LOWEST);
        }
        const int total = collect(floor_key, top);
        if(total <= CAP) {
            if(part != 0) return;
            u64 mine, mass, place, above;
            const bool one = arrange(total, mine, mass, place, above);
            bool kept = one && !(k > 0 && place >= u64(k));
            const u64 whole = sum_all(kept ? mass : 0, sh, flip);
            if(p < 1.0f && place > 0 && above >= share_of(whole)) kept = false;
            if(kept && value_of(unsigned(mine >> 32)) < least_kept) kept = false;
            const u64 kept_mass = kept ? mass : 0, target = point_in(sum_all(kept_mass, sh, flip));
            // and in index order: what has a larger ~index comes before
            u64 before = 0, here = kept_mass, id = mine;
            if(total <= COUNTED) {
                const int e = share(total);
                if(one) sh.list_mass[tid / e] = kept_mass;
                __syncthreads();
                through(sh, total, e, [&](u64 c, u64 w) {
                    if(unsigned(c) > unsigned(mine)) before += w;
                });
                before = sum_of(before, e);
            }
            else {
                sh.list_mass[tid] = kept_mass;
                __syncthreads();
                const u64 by_index = sort(kept_mass ? (mine & 0xffffffffull) << 32 | unsigned(tid) : 0, sh);
                here = by_index ? sh.list_mass[unsigned(by_index)] : 0;
                id = by_index >> 32;
                u64 all;
                before = scan(here, sh, flip, all) - here;
            }
            if(here && before <= target && before + here > target) a.tokens[row] = int(~unsigned(id));
            return;
        }
    }

    // ---- the ends of long prefixes
    const bool by_count = k > 0 && k < n, by_mass = p < 1.0f;
    // Bins for the logits down to RANGE temperatures under the largest one; what is further down is summed up without one.
    constexpr float RANGE = 20.0f;
    const float bin_scale = fminf(float(BINS) / (RANGE * t), 1e30f), top_value = value_of(top);
    // bin of a logit, 0 for the largest ones; BINS: none
    auto bin_of = [&](float v) { return v == top_value ? 0 : int(fminf((top_value - v) * bin_scale, float(BINS))); };
    // Sums over bins of the classes with lo <= key <= hi, the same in every block; bits < 0: bins of logits, else of (hi - key) >> bits.  A mass is
    // added in two 32-bit halves with a carry between them (64-bit additions in shared memory are loops).  rest_..: sums of what has no bin.
    u64 rest_mass = 0, rest_count = 0;
    auto histogram = [&](unsigned lo, unsigned hi, int bits) {
        __syncthreads();
        for(int i = tid; i < BINS; i += THREADS) { sh.mass[i] = make_uint2(0, 0); sh.count[i] = 0; }
        __syncthreads();
        u64 rest_m = 0, rest_c = 0;
        const float low = value_of(lo), high = value_of(hi);
        each_batch([&](const float (&v)[BATCH]) {
            u64 mass[BATCH];
            bool any = false;
            #pragma unroll
            for(int d = 0; d < BATCH; d++) any = any || (v[d] >= low && v[d] <= high);
            if(!any) return;
            #pragma unroll
            for(int d = 0; d < BATCH; d++) mass[d] = f.mass(v[d]);
            #pragma unroll
            for(int d = 0; d < BATCH; d++) {
                if(!(v[d] >= low && v[d] <= high)) continue;
                const int b = bits < 0 ? bin_of(v[d]) : int((hi - key_of(v[d])) >> bits);
                if(b >= BINS) {
                    rest_m += mass[d];
                    if(by_count) rest_c++;
                    continue;
                }
                const unsigned low32 = unsigned(mass[d]), was = atomicAdd(&sh.mass[b].x, low32), high32 = unsigned(mass[d] >> 32) + (was + low32 < low32);
                if(high32) atomicAdd(&sh.mass[b].y, high32);
                if(by_count) atomicAdd(&sh.count[b], 1u);
            }
        });
        rest_m = sum_all(rest_m, sh, flip);
        rest_c = sum_all(rest_c, sh, flip);
        if(tid == 0) { sh.rest[0] = rest_m; sh.rest[1] = rest_c; }
        everyone();
        rest_mass = rest_count = 0;
        for(int q = 0; q < parts; q++) {
            rest_mass += parts > 1 ? peer(sh.rest, q) : sh.rest[0];
            rest_count += parts > 1 ? peer(sh.rest + 1, q) : sh.rest[1];
        }
        #pragma unroll 2
        for(int i = tid; i < BINS; i += THREADS) {
            u64 s = 0;
            unsigned c = 0;
            for(int q = 0; q < parts; q++) {
                const u64 *from = reinterpret_cast<const u64 *>(sh.mass + i);
                s += parts > 1 ? peer(from, q) : *from;
                if(by_count) c += parts > 1 ? peer(sh.count + i, q) : sh.count[i];
            }
            sh.all_mass[i] = s;
            sh.all_count[i] = c;
        }
        everyone();
    };
    constexpr int MINE = BINS / THREADS;
    // The bin in which the running sum (of masses, or of numbers) reaches `want`: it, and the sums before it; BINS if that is in none.
    auto find_bin = [&](bool masses, u64 want, u64 &mass_before, u64 &count_before) {
        u64 ms = 0, cs = 0, all_m, all_c = 0;
        for(int i = 0; i < MINE; i++) { ms += sh.all_mass[MINE * tid + i]; cs += sh.all_count[MINE * tid + i]; }
        const u64 m_own = ms, c_own = cs;
        ms = scan(ms, sh, flip, all_m) - m_own;
        if(by_count) cs = scan(cs, sh, flip, all_c) - c_own;
        if((masses ? all_m : all_c) < want) {
            mass_before = all_m;
            count_before = all_c;
            return BINS;
        }
        if((masses ? ms : cs) < want && (masses ? ms + m_own : cs + c_own) >= want) {
            int b = MINE * tid;
            for(;; b++) {                                    // (ends in one of the thread's bins, by the condition above)
                const u64 mb = sh.all_mass[b], cb = sh.all_count[b];
                if((masses ? ms + mb : cs + cb) >= want) break;
                ms += mb;
                cs += cb;
            }
            sh.found[0] = b;
            sh.found[1] = ms;
            sh.found[2] = cs;
        }
        __syncthreads();
        mass_before = sh.found[1];
        count_before = sh.found[2];
        return int(sh.found[0]);
    };
    // The end of the shortest prefix with `want` classes, or that much mass, and its mass.  The sums over the bins of logits are in place.
    auto find_cut = [&](bool masses, u64 want, u64 &mass) {
        constexpr int G = grain_bits<T>;
        u64 mass_before, count_before;
        int b = find_bin(masses, want, mass_before, count_before);
        // the keys of that bin (or of what has none): from the least key with bin <= b up to the least one with bin < b
        // (a warp tries 32 keys at a time, least first: the bins fall as the keys rise)
        auto least_key = [&](unsigned from, int most) {      // the least key >= from whose bin is <= most; top's is
            unsigned l = from, size = top - from;            // it is in l .. l + size
            #pragma unroll 1
            while(size > 0) {
                const unsigned step = size / 32 + 1;
                const unsigned reach = lane * (unsigned long long)step < size ? l + lane * step : top;
                const unsigned yes = __ballot_sync(0xffffffffu, bin_of(value_of(reach)) <= most);
                const int at = __ffs(yes) - 1;               // the first lane that has one (the last ones stand for top)
                if(at == 0) return l;
                if(at < 0) {
                    l += 31 * step + 1;
                    size = top - l;
                    continue;
                }
                const unsigned end = min((unsigned long long)(at * (unsigned long long)step), (unsigned long long)size) + l;
                l += (at - 1) * step + 1;
                size = end - l;
            }
            return l;
        };
        unsigned low = least_key(LOWEST, b);
        unsigned hi = b > 0 ? least_key(low, b - 1) - 1 : top;
        mass = mass_before;
        u64 left = want - (masses ? mass_before : count_before);
        bool many = b == BINS;                               // more classes than a list takes: divided further
        Cut c;
        for(;;) {
            if(!many) {
                const int total = collect(low, min(hi, top));
                if(total <= CAP) {
                    u64 mine, w, place, above;
                    const bool one = arrange(total, mine, w, place, above);
                    __syncthreads();                         // (found has been read)
                    if(one && (masses ? above < left && above + w >= left : place + 1 == left)) {
                        sh.found[0] = place;
                        sh.found[1] = above + w;
                        sh.found[2] = mine >> 32;
                    }
                    __syncthreads();
                    c.key = unsigned(sh.found[2]);
                    c.ties = __syncthreads_count(one && unsigned(mine >> 32) == c.key && place <= sh.found[0]);
                    mass += sh.found[1];
                    return c;
                }
                if(low >> G == hi >> G) break;
            }
            // Bins end between numbers: of the 2^G keys with the same high bits the first is a number's if it is positive, the last if it is negative.
            // So hi goes up to the last of its 2^G, or, where that is a number and hi is not, down to the last before them: no number comes into the range,
            // and none leaves it.
            if(!(hi & 0x80000000u) && (~hi & ((1u << G) - 1))) hi -= 1u << G;
            hi |= (1u << G) - 1;
            int bits = G;
            while((hi - low) >> bits >= BINS) bits++;
            histogram(low, hi, bits);
            b = find_bin(masses, left, mass_before, count_before);
            mass += mass_before;
            left -= masses ? mass_before : count_before;
            hi -= unsigned(b) << bits;
            low = max(low, hi - ((1u << bits) - 1));
            many = false;
        }
        // more equal logits than a list takes
        c.key = hi & 0x80000000u ? hi >> G << G : hi | ((1u << G) - 1);
        const u64 w = f.mass(c.key), need = masses ? (left + w - 1) / w : left;
        c.ties = unsigned(need);
        mass += need * w;
        return c;
    };

    Cut cut = { MASKED, 0 };
    if(by_count || by_mass) {
        histogram(LOWEST, top, -1);
        u64 whole = 0, number = 0;
        for(int i = 0; i < MINE; i++) { whole += sh.all_mass[MINE * tid + i]; number += sh.all_count[MINE * tid + i]; }
        whole = sum_all(whole, sh, flip) + rest_mass;
        number = by_count ? sum_all(number, sh, flip) + rest_count : 0;
        bool fresh = true;                                   // the sums are those of all logits
        if(by_count && u64(k) < number) {
            cut = find_cut(false, u64(k), whole);
            fresh = false;
        }
        if(by_mass) {
            if(!fresh) histogram(LOWEST, top, -1);
            u64 mass;
            cut = find_cut(true, share_of(whole), mass);
        }
    }

    // ---- kept masses by segments
    {
        u64 sure = 0;
        unsigned ties = 0;
        const float at = cut.key == MASKED ? __int_as_float(0xff800000) : value_of(cut.key), least = fmaxf(at, least_kept);
        each_batch([&](const float (&v)[BATCH]) {
            bool any = false;
            #pragma unroll
            for(int d = 0; d < BATCH; d++) any = any || v[d] >= least;
            if(!any) return;
            #pragma unroll
            for(int d = 0; d < BATCH; d++) {
                const u64 mass = f.mass(v[d]);
                if(v[d] > at) sure += v[d] >= least_kept ? mass : 0;
                else if(v[d] == at && cut.key != MASKED) ties++;
            }
        });
        #pragma unroll
        for(int o = 16; o > 0; o >>= 1) sure += __shfl_xor_sync(0xffffffffu, sure, o);
        ties = __reduce_add_sync(0xffffffffu, ties);
        if(lane == 0) { sh.seg_mass[warp] = sure; sh.seg_ties[warp] = ties; }
    }
    everyone();
    u64 tie_mass = 0;
    if(cut.key != MASKED && value_of(cut.key) >= least_kept) tie_mass = f.mass(cut.key);
    const int segs = parts * WARPS;
    u64 seg = 0, seg_ties = 0;
    if(tid < segs) {
        seg = parts > 1 ? peer(sh.seg_mass + tid % WARPS, tid / WARPS) : sh.seg_mass[tid];
        seg_ties = parts > 1 ? peer(sh.seg_ties + tid % WARPS, tid / WARPS) : sh.seg_ties[tid];
    }
    everyone();
    u64 whole;
    const u64 ties_before = scan(seg_ties, sh, flip, whole) - seg_ties;
    if(seg_ties && ties_before < cut.ties) seg += tie_mass * min(seg_ties, cut.ties - ties_before);
    const u64 run = scan(seg, sh, flip, whole), target = point_in(whole);
    if(seg && run > target && run - seg <= target) { sh.found[0] = tid; sh.found[1] = run - seg; sh.found[2] = ties_before; }
    __syncthreads();
    const int seg_at = int(sh.found[0]);
    u64 before = sh.found[1], ties_seen = sh.found[2];
    if(seg_at / WARPS != part) return;

    // ---- the segment that the random number points into, a stretch of consecutive classes at a time
    const int from = max(0, seg_at * per * V - shift), to = int(min((long long)n, (long long)(seg_at + 1) * per * V - shift));
    #pragma unroll 1
    for(int i0 = from; i0 < to; i0 += THREADS) {
        const int i = i0 + tid;
        const unsigned key = i < to ? key_of(to_float(ld_plain(x + i))) : MASKED;
        const bool tie = key != MASKED && key == cut.key;
        u64 all_ties = 0, all;
        const u64 rank = cut.key != MASKED ? scan(tie ? 1 : 0, sh, flip, all_ties) : 0;
        u64 mass = 0;
        if(tie) mass = ties_seen + rank <= cut.ties ? tie_mass : 0;
        else if(key > cut.key && value_of(key) >= least_kept) mass = f.mass(key);
        const u64 to_here = before + scan(mass, sh, flip, all);
        if(mass && to_here > target && to_here - mass <= target) a.tokens[row] = i;
        before += all;
        ties_seen += all_ties;
        if(before > target) return;              // (the same in every thread)
    }
}

template<typename T> dlp_status launch_sample(const SampleArgs &a, int rows, cudaStream_t stream)
{
    const dlp_status st = allow_shared<sample_kernel<T>>(int(sizeof(Scratch)));
    if(st != DLP_OK) return st;
    // Blocks of a row: as many as there is room for (two on an SM), with 4096 classes or more to each; and with many classes to a row two or more
    // in any case: rows take very different times, and short blocks fill the gaps (256 rows of 150001 with settings of their own 321 -> 176 us when it came in).
    int parts = 1;
    while(parts < MAX_PARTS && (((long long)rows * parts <= sm_count() && a.classes / (parts * 2) >= 4096) || a.classes / (parts * 2) >= 32768)) parts *= 2;
    DLP_REQUIRE((long long)rows * parts < (1ll << 31), "too many rows");
    DLP_LAUNCH_PDL(launch_pdl_cluster(one_wave((long long)rows * parts, THREADS), parts, sample_kernel<T>, rows * parts, THREADS, sizeof(Scratch), stream, a),
                   "sample_kernel");
    return DLP_OK;
}

} // namespace
} // namespace dlp

using namespace dlp;

extern "C" {

dlp_status dlp_sample_fwd(const dlp_sample_args *args, void *stream)
{
    DLP_REQUIRE(args != nullptr, "null arguments");
    const auto [logits, temperature, top_k, top_p, min_p, u, tokens, stride, rows, classes, type] = *args;
    DLP_REQUIRE(rows >= 0 && classes > 0 && classes <= DLP_SAMPLE_MAX_CLASSES, "bad shape");
    DLP_REQUIRE(is_real_type(type), "the logits' type must be fp32, fp16 or bf16");
    if(rows == 0) return DLP_OK;
    DLP_REQUIRE(logits && u && tokens, "null tensor");
    DLP_REQUIRE(rows <= 1 || stride >= classes, "rows overlap");
    DLP_REQUIRE(aligned_to(logits, type_size(type)) && aligned_to(u, 4) && aligned_to(tokens, 4) && aligned_to(temperature, 4) && aligned_to(top_k, 4) &&
                aligned_to(top_p, 4) && aligned_to(min_p, 4), "a tensor is not aligned to its elements");
    int log2 = 0;
    while((1ll << log2) < classes) log2++;
    const SampleArgs a = { logits, temperature, top_p, min_p, u, top_k, tokens, stride, classes, std::min(51, 63 - log2) };
    if(type == DLP_TYPE_F32) return launch_sample<float>(a, rows, (cudaStream_t)stream);
    if(type == DLP_TYPE_F16) return launch_sample<__half>(a, rows, (cudaStream_t)stream);
    return launch_sample<__nv_bfloat16>(a, rows, (cudaStream_t)stream);
}

} // extern "C"

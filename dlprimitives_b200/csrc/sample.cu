// Draw of a class from each row of logits with given random numbers: temperature, top-k, top-p and min-p.
//
// The classes of a row in the order of falling logits (equal ones in index order) have masses w_i = exp((x_i - max) / t).  top-k keeps
// the first k, top-p of these the shortest prefix with at least p of their mass, min-p of these the ones with w_i >= m (max: w = 1).  The
// class drawn is the first one in index order whose running mass over the kept ones exceeds u times their whole mass.
//
// Which class it is hangs on sums of up to a few hundred thousand masses, compared with a border.  Masses are whole numbers here,
// round(w 2^b) with 63 - log2(classes) bits: their sums are exact in any order, so the result depends neither on timing nor on how
// a row is shared out.
//
// A row is read a few times, from memory once and then from L2, by a cluster of 1 to 8 blocks (so that few rows use the whole GPU); the
// blocks gather what each has found through distributed shared memory and all come to the same conclusions.
//   * First the largest logit, and the largest of each of 512 groups of classes.
//   * With a small k (up to 256): the k-th largest of the groups' maxima has at least k classes at or above it, and for classes in no
//     particular order only a few more (512 ln(512 / (512 - k)) of them are expected).  These are collected, sorted, and the rest is done on
//     them alone: two readings of the row, and masses of a few hundred classes.
//   * Otherwise the end of a prefix is found from sums over 4096 bins of falling logits: the bin it lies in is collected and sorted,
//     and divided further as long as it holds more than 512 classes.  Then the masses of the kept classes are summed by
//     segments of the row, and the one segment that the random number points into is gone through.
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
constexpr int BINS = 4096, CAP = THREADS;        // bins of a histogram; classes that are sorted at once
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
    unsigned mass_lo[BINS], mass_hi[BINS], count[BINS];     // and over this block's
    u64 cand[CAP], sorted[2][CAP];               // classes as (key, ~index)
    u64 seg_mass[WARPS];                         // kept masses of each warp's segment, and classes equal to the cut's key
    unsigned seg_ties[WARPS];
    u64 best[WARPS];
    unsigned group[THREADS];
    u64 warp_sum[2][WARPS];
    u64 found[3];
    double table[64];                            // 2^(-j / 64)
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

// A mass of a class.  w = 2^-t with t = (max - x) log2(e) / temperature, in 64 bits: t = i + j / 64 + r with whole i and j, |r| <= 1/128, and
// 2^-r by the series of exp(-r ln 2), whose sixth term is under 2^-53.
struct Masses {
    double top, factor, one, least;              // factor: log2(e) / temperature; one: 2^bits; least: w of min-p
    unsigned top_key;
    const double *table;
    __device__ __forceinline__ double weight(unsigned key) const
    {
        if(key == top_key) return 1.0;
        const double t = (top - double(value_of(key))) * factor;
        if(!(t < 1000.0)) return 0.0;            // (and an infinite logit's NaN)
        const double magic = 6755399441055744.0 / 64.0, z = t + magic, r = t - (z - magic);
        const int k = __double2loint(z);         // 64 i + j
        constexpr double L = 0.69314718055994530942, C2 = L * L / 2, C3 = L * C2 / 3, C4 = L * C3 / 4, C5 = L * C4 / 5;
        const double e = fma(r, fma(r, fma(r, fma(r, fma(r, -C5, C4), -C3), C2), -L), 1.0) * table[k & 63];
        const int i = k >> 6;
        return __hiloint2double(__double2hiint(e) - (i << 20), __double2loint(e));      // e is in (0.49, 1.01), i under 1001: the exponent stays normal
    }
    // a whole number below 2^52 is the low part of itself + 2^52
    __device__ __forceinline__ u64 whole(double w) const { return u64(__double_as_longlong(fma(w, one, 4503599627370496.0)) & 0xfffffffffffffll); }
    __device__ __forceinline__ u64 mass(unsigned key) const { return key == MASKED ? 0 : whole(weight(key)); }
};

// Where a prefix of the sorted row ends: all above `key` and the first `ties` of those equal to it.
struct Cut { unsigned key, ties; };

// ---- over the first `active` threads (a multiple of 32, THREADS: the whole block), all of which take part
__device__ __forceinline__ void sync(int active)
{
    if(active == THREADS) __syncthreads();
    else if(active == 32) __syncwarp();
    else asm volatile("bar.sync 1, %0;" ::"r"(active) : "memory");
}
// Sum up to and with this thread's value, and of all.  flip: changes from call to call, so that one barrier a call is enough.
__device__ __forceinline__ u64 scan(u64 v, Scratch &sh, int &flip, u64 &all, int active)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    #pragma unroll
    for(int o = 1; o < 32; o <<= 1) {
        const u64 other = __shfl_up_sync(0xffffffffu, v, o);
        if(lane >= o) v += other;
    }
    if(active == 32) {
        all = __shfl_sync(0xffffffffu, v, 31);
        return v;
    }
    flip ^= 1;
    if(lane == 31) sh.warp_sum[flip][warp] = v;
    sync(active);
    u64 sums = lane < active / 32 ? sh.warp_sum[flip][lane] : 0;
    #pragma unroll
    for(int o = 1; o < WARPS; o <<= 1) {
        const u64 other = __shfl_up_sync(0xffffffffu, sums, o);
        if(lane >= o) sums += other;
    }
    all = __shfl_sync(0xffffffffu, sums, WARPS - 1);
    const u64 before = __shfl_sync(0xffffffffu, sums, warp > 0 ? warp - 1 : 0);
    return v + (warp > 0 ? before : 0);
}
// Sorts the numbers of the first `size` threads (a power of two), the largest first; the others' are zeros.
__device__ __forceinline__ u64 sort(u64 v, int size, Scratch &sh, int active)
{
    const int tid = threadIdx.x;
    int buf = 0;
    #pragma unroll 1
    for(int k = 2; k <= size; k <<= 1)
        #pragma unroll 1
        for(int j = k >> 1; j > 0; j >>= 1) {
            u64 other;
            if(j >= 32) {
                sh.sorted[buf][tid] = v;
                sync(active);
                other = sh.sorted[buf][tid ^ j];
                buf ^= 1;
            }
            else other = __shfl_xor_sync(0xffffffffu, v, j);
            const bool larger = ((tid & j) == 0) == ((tid & k) == 0 || k == size);
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
    // f(key) for the segment's classes that can be drawn, one at a time (f is there four times)
    auto each_key = [&](auto f) {
        constexpr int DEEP = 4;
        const int from = max(0, piece0 * V - shift), to = min(n, piece1 * V - shift);
        #pragma unroll 1
        for(int i = from + lane; i < to; i += 32 * DEEP) {
            float v[DEEP];
            #pragma unroll
            for(int d = 0; d < DEEP; d++) v[d] = i + d * 32 < to ? to_float(ld_plain(x + i + d * 32)) : __int_as_float(0xff800000);
            #pragma unroll
            for(int d = 0; d < DEEP; d++) {
                const unsigned key = key_of(v[d]);
                if(key != MASKED) f(key);
            }
        }
    };

    // ---- the largest logit, its first place, and the groups' largest (a group: `parts` neighbouring threads)
    if(tid < 64) sh.table[tid] = exp2(tid * (-1.0 / 64));
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
    const float t = a.temperature ? ld_plain(a.temperature + row) : 1.0f;
    const bool greedy = !(t > 0.0f);
    const int k = greedy ? 1 : (a.top_k ? ld_plain(a.top_k + row) : 0);
    const float p = a.top_p ? ld_plain(a.top_p + row) : 1.0f, m = a.min_p ? ld_plain(a.min_p + row) : 0.0f, uf = ld_plain(a.u + row);
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
    f.top_key = top;
    f.top = double(value_of(top));
    f.factor = 1.4426950408889634074 / double(t);
    f.one = double(1ull << a.bits);
    f.least = m > 0.0f ? fmin(double(m), 1.0) : 0.0;
    f.table = sh.table;
    // the least whole number that is no less than p times `whole`
    auto share_of = [&](u64 whole) {
        const u64 pf = p > 0.0f ? u64(double(p) * 18446744073709551616.0) : 0;
        const u64 want = __umul64hi(pf, whole) + (pf * whole != 0);
        return want > 0 ? want : 1;
    };
    auto point_in = [&](u64 whole) { return __umul64hi(uf > 0.0f ? (uf < 1.0f ? u64(double(uf) * 18446744073709551616.0) : ~0ull) : 0ull, whole); };

    // Collects the classes with lo <= key <= hi (lo > MASKED): their number, and each thread's one of them, unsorted, if there are at most CAP.
    // Two barriers, the second after the last look into another block's memory.
    auto collect = [&](unsigned lo, unsigned hi, u64 &mine) {
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
        mine = 0;
        if(total <= CAP && unsigned(tid) < total) mine = parts > 1 ? peer(sh.cand + place, from) : sh.cand[place];
        everyone();
        if(tid == 0) sh.cands = 0;
        return total;
    };
    auto size_for = [](unsigned total) {
        int size = 32;
        while(size < int(total)) size <<= 1;
        return size;
    };

    // ---- few classes are kept: all of them in one sorted list
    const bool few = k > 0 && k <= SMALL_K && k < n;
    if(few || n <= CAP) {
        unsigned floor_key = LOWEST;
        if(few) {
            // the k-th largest of the groups' maxima, from the top bit down; done when exactly k of them are left (and but for the last eight bits:
            // a little lower is as good)
            unsigned at = 0;
            #pragma unroll 1
            for(int bit = 31; bit >= 8; bit--) {
                const unsigned higher = at | 1u << bit;
                const int above = __syncthreads_count(group >= higher);
                if(above >= k) at = higher;
                if(above == k) break;
            }
            floor_key = max(at, LOWEST);
        }
        u64 mine;
        const unsigned total = collect(floor_key, top, mine);
        if(total <= CAP) {
            const int size = size_for(total);
            if(part != 0 || tid >= size) return;
            const u64 got = sort(mine, size, sh, size);
            const unsigned key = unsigned(got >> 32);
            const int kept_k = k > 0 && k < int(total) ? k : int(total);
            const double w = tid < kept_k ? f.weight(key) : 0.0;
            u64 mass = tid < kept_k ? f.whole(w) : 0, whole, run = scan(mass, sh, flip, whole, size);
            if(p < 1.0f && run - mass >= share_of(whole)) mass = 0;
            if(w < f.least) mass = 0;
            // in index order: by ~index, the largest first, with the place of the mass
            sh.all_mass[tid] = mass;
            const u64 by_index = sort(mass ? (got & 0xffffffffull) << 32 | unsigned(tid) : 0, size, sh, size);
            sync(size);
            mass = by_index ? sh.all_mass[unsigned(by_index)] : 0;
            run = scan(mass, sh, flip, whole, size);
            const u64 target = point_in(whole);
            if(mass && run > target && run - mass <= target) a.tokens[row] = int(~unsigned(by_index >> 32));
            return;
        }
    }

    // ---- the ends of long prefixes
    const bool by_count = k > 0 && k < n, by_mass = p < 1.0f;
    const float bin_scale = fminf(float(BINS) / (30.0f * t), 1e30f), top_value = value_of(top);
    // bin of a key, 0 for the largest logits
    auto bin_of = [&](unsigned key) { return key == top ? 0 : int(fminf((top_value - value_of(key)) * bin_scale, float(BINS - 1))); };
    // Sums over bins of the classes with lo <= key <= hi, the same in every block; bits < 0: bins of logits, else of (hi - key) >> bits.  A mass is
    // added in two 32-bit halves with a carry between them (64-bit additions in shared memory are loops).
    auto histogram = [&](unsigned lo, unsigned hi, int bits) {
        __syncthreads();
        for(int i = tid; i < BINS; i += THREADS) sh.mass_lo[i] = sh.mass_hi[i] = sh.count[i] = 0;
        __syncthreads();
        each_key([&](unsigned key) {
            if(key < lo || key > hi) return;
            const int b = bits < 0 ? bin_of(key) : int((hi - key) >> bits);
            const u64 mass = f.mass(key);
            const unsigned low = unsigned(mass), was = atomicAdd(&sh.mass_lo[b], low), high = unsigned(mass >> 32) + (was + low < low);
            if(high) atomicAdd(&sh.mass_hi[b], high);
            atomicAdd(&sh.count[b], 1u);
        });
        everyone();
        for(int i = tid; i < BINS; i += THREADS) {
            u64 s = 0;
            unsigned c = 0;
            for(int q = 0; q < parts; q++) {
                s += parts > 1 ? u64(peer(sh.mass_hi + i, q)) << 32 : u64(sh.mass_hi[i]) << 32;
                s += parts > 1 ? peer(sh.mass_lo + i, q) : sh.mass_lo[i];
                c += parts > 1 ? peer(sh.count + i, q) : sh.count[i];
            }
            sh.all_mass[i] = s;
            sh.all_count[i] = c;
        }
        everyone();
    };
    constexpr int MINE = BINS / THREADS;
    // The bin in which the running sum (of masses, or of numbers) reaches `want`: it, and the sums before it.
    auto find_bin = [&](bool masses, u64 want, u64 &mass_before, u64 &count_before) {
        u64 ms = 0, cs = 0, whole;
        for(int i = 0; i < MINE; i++) { ms += sh.all_mass[MINE * tid + i]; cs += sh.all_count[MINE * tid + i]; }
        const u64 m_own = ms, c_own = cs;
        ms = scan(ms, sh, flip, whole, THREADS) - m_own;
        cs = scan(cs, sh, flip, whole, THREADS) - c_own;
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
    // The end of the shortest prefix with `want` classes, or that much mass, and its mass.  The sums over the bins of all logits are in place.
    auto find_cut = [&](bool masses, u64 want, u64 &mass) {
        constexpr int G = grain_bits<T>;
        Cut c;
        u64 mass_before, count_before;
        int b = find_bin(masses, want, mass_before, count_before);
        // the keys of that bin: from the least key with bin <= b up to the least one with bin < b
        unsigned lo, hi = top;
        {
            unsigned l = LOWEST - 1, h = top;
            #pragma unroll 1
            while(h - l > 1) { const unsigned mid = l + (h - l) / 2; if(bin_of(mid) <= b) h = mid; else l = mid; }
            lo = h;
            if(b > 0) {
                l = lo - 1; h = top;
                #pragma unroll 1
                while(h - l > 1) { const unsigned mid = l + (h - l) / 2; if(bin_of(mid) < b) h = mid; else l = mid; }
                hi = h - 1;
            }
        }
        mass = mass_before;
        u64 left = want - (masses ? mass_before : count_before);
        unsigned equal = sh.all_count[b];
        while(equal > CAP && lo >> G < hi >> G) {
            int bits = G;
            while((hi - lo) >> bits >= BINS) bits++;
            hi |= (1u << G) - 1;                             // (bins end between numbers)
            histogram(lo, hi, bits);
            b = find_bin(masses, left, mass_before, count_before);
            mass += mass_before;
            left -= masses ? mass_before : count_before;
            equal = sh.all_count[b];
            hi -= unsigned(b) << bits;
            lo = max(lo, hi - ((1u << bits) - 1));
        }
        if(equal > CAP) {                                    // more equal logits than are sorted at once
            c.key = hi & 0x80000000u ? hi >> G << G : hi | ((1u << G) - 1);
            const u64 w = f.mass(c.key), need = masses ? (left + w - 1) / w : left;
            c.ties = unsigned(need);
            mass += need * w;
            return c;
        }
        u64 mine;
        const unsigned total = collect(lo, min(hi, top), mine);
        const u64 got = sort(mine, size_for(total), sh, THREADS);
        const unsigned key = unsigned(got >> 32);
        const bool in = unsigned(tid) < total;
        u64 whole;
        const u64 w = in ? f.mass(key) : 0, run = scan(w, sh, flip, whole, THREADS);
        const bool last = in && (masses ? run >= left && run - w < left : u64(tid) + 1 == left);
        __syncthreads();
        if(last) { sh.found[0] = tid; sh.found[1] = run; sh.found[2] = key; }
        __syncthreads();
        const int at = int(sh.found[0]);
        mass += sh.found[1];
        c.key = unsigned(sh.found[2]);
        c.ties = __syncthreads_count(in && tid <= at && key == c.key);
        return c;
    };

    Cut cut = { MASKED, 0 };
    if(by_count || by_mass) {
        histogram(LOWEST, top, -1);
        u64 whole = 0, number = 0;
        for(int i = 0; i < MINE; i++) { whole += sh.all_mass[MINE * tid + i]; number += sh.all_count[MINE * tid + i]; }
        scan(whole, sh, flip, whole, THREADS);
        scan(number, sh, flip, number, THREADS);
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
        each_key([&](unsigned key) {
            if(key == cut.key) ties++;
            else if(key > cut.key) {
                const double w = f.weight(key);
                if(w >= f.least) sure += f.whole(w);
            }
        });
        #pragma unroll
        for(int o = 16; o > 0; o >>= 1) sure += __shfl_xor_sync(0xffffffffu, sure, o);
        ties = __reduce_add_sync(0xffffffffu, ties);
        if(lane == 0) { sh.seg_mass[warp] = sure; sh.seg_ties[warp] = ties; }
    }
    everyone();
    u64 tie_mass = 0;
    if(cut.key != MASKED) {
        const double w = f.weight(cut.key);
        if(w >= f.least) tie_mass = f.whole(w);
    }
    const int segs = parts * WARPS;
    u64 seg = 0, seg_ties = 0;
    if(tid < segs) {
        seg = parts > 1 ? peer(sh.seg_mass + tid % WARPS, tid / WARPS) : sh.seg_mass[tid];
        seg_ties = parts > 1 ? peer(sh.seg_ties + tid % WARPS, tid / WARPS) : sh.seg_ties[tid];
    }
    everyone();
    u64 whole;
    const u64 ties_before = scan(seg_ties, sh, flip, whole, THREADS) - seg_ties;
    if(seg_ties && ties_before < cut.ties) seg += tie_mass * min(seg_ties, cut.ties - ties_before);
    const u64 run = scan(seg, sh, flip, whole, THREADS), target = point_in(whole);
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
        const u64 rank = cut.key != MASKED ? scan(tie ? 1 : 0, sh, flip, all_ties, THREADS) : 0;
        u64 mass = 0;
        if(tie) mass = ties_seen + rank <= cut.ties ? tie_mass : 0;
        else if(key > cut.key) {
            const double w = f.weight(key);
            if(w >= f.least) mass = f.whole(w);
        }
        const u64 to_here = before + scan(mass, sh, flip, all, THREADS);
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
    // blocks of a row: as many as there is room for (two on an SM), with 4096 classes or more to each
    int parts = 1;
    while(parts < MAX_PARTS && (long long)rows * parts <= sm_count() && a.classes / (parts * 2) >= 4096) parts *= 2;
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

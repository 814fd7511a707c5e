// sample.cu -- the choice of a token from a row of logits by a given uniform
// number, with temperature, top-k, top-p and min-p (greedy rows: argmax).
//
//   w_i = 2^((l_i - max l) log2(e) / temperature)
//   in the order (l downwards, index upwards): keep the first k; of those, each
//   whose mass before it is below p times their total (the first always); of
//   those, w_i >= min_p.  The token is the first index whose running sum of the
//   kept w, in index order, exceeds u times their total.
//
// Every filter keeps a first part of one order, that of the keys
// (order-preserving bits of l, mask - index), which no two tokens share.
//
// Borders between tokens are sharp, so masses are whole numbers: w in units of
// 2^-44 from a 64-bit evaluation (1.3e-12 relative), which add up exactly and in
// any order.  fp32 weights would move the borders of a flat distribution over
// 32768 tokens by 1e-8 each, one row in some ten thousand.
//
// What bounds it: the logits come from HBM once and from L2 after that; a weight
// is 10 operations of 64 bits and 20 around them, so issue slots bound a pass over
// all weights (256 x 32768: 10 us against 5 for the first read), and the filters
// are arranged to need few of them.
//   A row's 512 groups of tokens (a thread's, or those of some threads of a
// cluster) have a maximum each: no fewer than k tokens lie at or above the k-th
// largest of these.  What does, a few tokens more than are kept, is listed, sorted
// and chosen from (256 x 32768 fp32, k = 50: 18 us).
//   Top-p, and top-k whose list would be too long, go by counts in 2048 bins of equal
// width below the maximum, which leave some bins in which the border can lie, and
// one pass over the weights (p = 0.9: 52 us).
//   What is left, top-p of a large top-k and rows of equal logits, goes by
// histograms of the masses and then by the leading bits of the keys.
//
// A row belongs to one CTA, or to a cluster of up to 8 where rows are few (a
// barrier of a cluster costs about 0.5 us: 256 x 32768 with k = 50 17 us in one CTA
// a row, 28 in two; 4 x 32768 with p = 0.9 in one 54, in four 19).
#include <cooperative_groups.h>

#include "mi_elem.cuh"

namespace mi {
namespace sample {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 512, LIST = THREADS, FINE = 2048, MAX_CLUSTER = 8,
              MAX_V = 262144, MAX_SEG = 131072;
constexpr int SCALE = 44;                      // weights are whole numbers of 2^-44
constexpr uint32_t LOWEST = 0x00800000u;       // key of -FLT_MAX
constexpr uint32_t INF = 0xff800000u;          // key of +inf; NaN above it

struct Args {
    const void* logits;
    int64_t ld;
    const float* u;
    const float* temperature;  // [rows] or NULL: the scalar
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    float temperature1, top_p1, min_p1;
    int top_k1;
    int64_t* token;
    float* prob;  // may be NULL
    int V, cs, seg;
};

__device__ __forceinline__ uint32_t key_of(float v) {  // of a v without -0
    if (v != v) return 0xffffffffu;
    const uint32_t b = __float_as_uint(v);
    return b ^ ((int32_t)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key ^ ((int32_t)key < 0 ? 0x80000000u : 0xffffffffu));
}

// What the row's weights depend on.
constexpr int ROOTS = 32;
struct Weights {
    double most, scale;   // ROOTS log2(e) / temperature
    const double* roots;  // 2^(i / ROOTS + SCALE), in shared memory
    float end;            // there are no weights below it
    __device__ __forceinline__ Weights() {}
    __device__ __forceinline__ Weights(float m, float temperature, const double* r)
        : most(m), scale(ROOTS * 1.4426950408889634 / (double)temperature), roots(r) {
        // 2^-(SCALE + 1) is half a unit; in front of -infinity even if the weights do not end
        end = fmaxf(-3.402823466e38f, __double2float_rd(most - (SCALE + 1) * ROOTS / scale));
    }
    __device__ __forceinline__ double power(float v) const { return ((double)v - most) * scale; }  // of the ROOTS-th root of 2
    // 2^(y / ROOTS) in units of 2^-SCALE, rounded to a whole one.  y = n + f with |f| <= 1/2: a root, a shift of the
    // exponent, and the power series of 2^(f / ROOTS) up to the fourth power, which leaves 1.3e-12.  Adding 1.5 2^52
    // rounds to a whole number, which the sum's low bits hold.
    __device__ __forceinline__ u64 mass(float v) const {
        constexpr double ROUND = 6755399441055744.0, L = 0.693147180559945309417 / ROOTS;
        constexpr double C2 = L * L / 2, C3 = C2 * L / 3, C4 = C3 * L / 4;
        const bool some = v >= end;  // no branch: neighbouring tokens' chains run side by side
        const double y = power(some ? v : end), r = __dadd_rn(y, ROUND), f = __dsub_rn(y, __dsub_rn(r, ROUND));
        double p = __fma_rn(C4, f, C3);
        p = __fma_rn(p, f, C2);
        p = __fma_rn(p, f, L);
        p = __fma_rn(p, f, 1.0);
        const int n = __double2loint(r);
        const double root = roots[n & (ROOTS - 1)];
        p = __fma_rn(p, __hiloint2double(__double2hiint(root) + ((n >> 5) << 20), __double2loint(root)), ROUND);
        return some ? (u64)(__double_as_longlong(p) - __double_as_longlong(ROUND)) : 0;
    }
    __device__ __forceinline__ float share(float v, u64 total) const {
        return (float)(exp2(power(v) * (1.0 / ROOTS) + SCALE) / (double)total);
    }
};
static_assert(ROOTS == 32, "the shift of n");

// Bins of equal width downwards from the maximum; falls monotonically as v rises.
template <int N>
struct Bins {
    float most, scale;
    // over the least of `range` and what the weights reach (they end SCALE powers of 2 below the maximum)
    __device__ __forceinline__ Bins(float most, float temperature, float range) : most(most) {
        scale = __fdiv_rn((float)N, fminf(range, __fmul_rn((SCALE + 2) * 0.6931472f, temperature)));
        if (!(scale < 3.0e38f)) scale = 0.0f;  // a row of one value
    }
    __device__ __forceinline__ float at(float v) const { return __fmul_rn(__fsub_rn(most, v), scale); }
    __device__ __forceinline__ int operator()(float v) const {
        const float x = at(v);
        return x < (float)(N - 1) ? (int)x : N - 1;
    }
};

struct Entry {
    u64 key, mass;
};
struct Shared {
    // what the CTAs of a row tell one another
    uint32_t most[MAX_CLUSTER][WARPS], at[MAX_CLUSTER][WARPS], listed_by[MAX_CLUSTER];
    u64 sums[MAX_CLUSTER][WARPS], above[MAX_CLUSTER][WARPS];
    uint32_t maxima[THREADS];
    Entry all[LIST];
    // this CTA's own
    Entry own[LIST];
    u64 swap[2][THREADS];
    union {
        struct {
            uint32_t count[2][BINS], limb[2][3][BINS];  // limbs of 15 bits, which MAX_SEG tokens do not overflow
        };
        struct {
            uint32_t fine[FINE], depth[FINE];  // tokens of a bin, and the sum of how far they lie in it, in 256ths
        };
    };
    double roots[ROOTS];
    u64 warp_low[WARPS];
    u64 warp_mass[WARPS];
    uint32_t warp_count[WARPS];
    uint32_t listed, bound;
    // a border's bin: what lies above it, what it holds
    u64 above_mass, in_mass, target, cut;
    uint32_t above_count, in_count, bin, edge[2], upto[2];
};

// The smallest key in (lo, hi] for which pred holds; it holds for hi, and from some key on.  By a whole warp.
template <typename P>
__device__ __forceinline__ uint32_t first_key(uint32_t lo, uint32_t hi, P pred) {
    const int lane = threadIdx.x & 31;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 31) / 32;  // >= 1
        const uint64_t at64 = (uint64_t)lo + (uint64_t)step * (lane + 1);
        const uint32_t at = at64 < hi ? (uint32_t)at64 : hi;
        const uint32_t yes = __ballot_sync(0xffffffffu, at == hi || pred(at));
        const int first = __ffs(yes) - 1;
        const uint64_t to = (uint64_t)lo + (uint64_t)step * (first + 1);
        lo += step * first;
        if (to < hi) hi = (uint32_t)to;
    }
    return hi;
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}
template <typename V>
__device__ __forceinline__ V warp_scan(V v) {  // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const V o = __shfl_up_sync(0xffffffffu, v, m);
        if (lane >= m) v += o;
    }
    return v;
}

// share of `total`, as the smallest whole number that is not below it, from 1 to total
__device__ __forceinline__ u64 part_of(u64 total, double share) {
    const double t = ceil(share * (double)total);
    return t >= (double)total ? total : t < 1.0 ? 1 : (u64)t;
}
// the number that a running sum has to exceed
__device__ __forceinline__ u64 target_of(u64 total, float u) {
    const double t = floor((double)u * (double)total);
    return !(t > 0.0) ? 0 : t >= (double)total ? total - 1 : (u64)t < total ? (u64)t : total - 1;
}

template <typename T>
struct Chooser {
    static constexpr int K = 16 / sizeof(T);
    const Args& a;
    Shared& sh;
    const T* from;            // this CTA's tokens: first .. first + n - 1 of the row
    int n, first, rank, cs, part;  // part: neighbouring tokens of a warp
    int tid, warp, lane;
    int bits;                 // of an index
    Weights weights;
    float temperature;
    uint32_t kmax;
    int level = 0;            // of the histograms, which alternate

    __device__ __forceinline__ u64 full_key(float v, int e) const {
        return (u64)key_of(v) << bits | (u64)((1u << bits) - 1 - (uint32_t)(first + e));
    }
    __device__ __forceinline__ float value(u64 key) const { return value_of((uint32_t)(key >> bits)); }
    __device__ __forceinline__ int index(u64 key) const { return (int)((1u << bits) - 1 - ((uint32_t)key & ((1u << bits) - 1))); }
    // v is at or above the cut, of which only equal values need the index
    __device__ __forceinline__ bool kept(float v, int e, float vcut, u64 cut) const {
        return v > vcut || (v == vcut && full_key(v, e) >= cut);
    }
    __device__ __forceinline__ void sync() {
        if (cs > 1)
            cg::this_cluster().sync();
        else
            __syncthreads();
    }
    __device__ __forceinline__ Shared& of(int r) { return cs > 1 ? *cg::this_cluster().map_shared_rank(&sh, r) : sh; }

    // f(v, e) for this warp's tokens e .. e + K - 1, by blocks of 16 bytes, U of them a lane at a time and the next U on
    // their way; beside the tokens a block may hold others' places, for which v is -infinity.
    template <int U, typename F>
    __device__ __forceinline__ void each(F f) const {
        const int begin = warp * part, end = min(begin + part, n);
        const int off = (int)((reinterpret_cast<uintptr_t>(from + begin) & 15) / sizeof(T));
        constexpr int STEP = U * 32 * K;
        Pack<T, K> v[U], next[U];
        auto load = [&](int e0) {
#pragma unroll
            for (int j = 0; j < U; j++) {
                const int e = e0 + j * 32 * K;
                if (e >= begin && e + K <= end) {
                    next[j] = *reinterpret_cast<const Pack<T, K>*>(from + e);
                } else {
#pragma unroll
                    for (int i = 0; i < K; i++)
                        next[j].v[i] = e + i >= begin && e + i < end ? from[e + i] : from_f<T>(-__int_as_float(0x7f800000));
                }
            }
        };
        int e0 = begin - off + lane * K;
        if (e0 < end) load(e0);
        for (; e0 < end; e0 += STEP) {
#pragma unroll
            for (int j = 0; j < U; j++) v[j] = next[j];
            if (e0 + STEP < end) load(e0 + STEP);
#pragma unroll
            for (int j = 0; j < U; j++) {
                float x[K];
#pragma unroll
                for (int i = 0; i < K; i++) x[i] = __fadd_rn(to_f(v[j].v[i]), 0.0f);  // no -0: it is as good as 0
                f(x, e0 + j * 32 * K);
            }
        }
    }

    // The warps' sums to all CTAs; the row's total.
    __device__ __forceinline__ u64 exchange_sums(u64 sum) {
        sum = warp_sum(sum);
        if (lane < cs) of(lane).sums[rank][warp] = sum;
        sync();
        const u64* sums = &sh.sums[0][0];
        u64 own = 0;
        for (int i = lane; i < cs * WARPS; i += 32) own += sums[i];
        return warp_sum(own);
    }

    // The sum over the CTA's threads before this one, and over all.
    __device__ __forceinline__ u64 block_before(u64 v, u64& all) {
        u64 upto = warp_scan(v);
        __syncthreads();  // the last sums were read
        if (lane == 31) sh.warp_mass[warp] = upto;
        __syncthreads();
        all = 0;
#pragma unroll
        for (int i = 0; i < WARPS; i++) {
            if (i == warp) upto += all;
            all += sh.warp_mass[i];
        }
        return upto - v;
    }

    // Sorts `size` values (a power of 2 from 32 to THREADS), one a thread, into falling order.
    template <typename V>
    __device__ __forceinline__ V sorted(V v, int size) {
        V(*swap)[THREADS] = reinterpret_cast<V(*)[THREADS]>(sh.swap);
        int set = 0;
        for (int k = 2; k <= size; k <<= 1) {
            for (int j = k >> 1; j; j >>= 1) {
                V o;
                if (j >= 32) {
                    swap[set][tid] = v;
                    __syncthreads();
                    o = swap[set][tid ^ j];
                    set ^= 1;
                } else {
                    o = __shfl_xor_sync(0xffffffffu, v, j);
                }
                const bool larger = ((tid & k) == 0) == ((tid & j) == 0);
                v = larger == (v > o) ? v : o;
            }
        }
        return v;
    }

    __device__ __forceinline__ void list_one(float v, int e) {
        const uint32_t i = atomicAdd(&sh.listed, 1u);
        if (i < LIST) sh.own[i].key = full_key(v, e);
    }
    // Brings the CTAs' listed tokens to CTA 0's sh.all.  Their number, or -1 if they are too many.
    __device__ __forceinline__ int gather() {
        __syncthreads();
        const int mine = min(sh.listed, (uint32_t)LIST + 1);
        if (tid < cs) of(tid).listed_by[rank] = mine;
        sync();
        int all = 0, before = 0;
        for (int r = 0; r < cs; r++) {
            if (r == rank) before = all;
            all += sh.listed_by[r];
        }
        if (all > LIST) return -1;
        if (tid < mine) of(0).all[before + tid].key = sh.own[tid].key;
        sync();
        return all;
    }
    __device__ __forceinline__ int size_of(int m) const {
        int size = 32;
        while (size < m) size *= 2;
        return size;
    }

    __device__ __forceinline__ int part_of_cta(int r) const {
        return cdiv(cdiv(max(0, min(a.seg, a.V - r * a.seg)), WARPS), 32) * 32;
    }

    // The choice, from the sums of the kept masses by the row's warps, in the order of the indices.  By the CTA whose
    // token it is, or by this one.
    template <typename F>
    __device__ __forceinline__ void finish(const u64* sums, float u, int64_t row, F kept, bool here) {
        // every warp adds up all of them, some neighbouring ones a lane
        const int all = cs * WARPS, some = cdiv(all, 32);
        u64 own = 0;
        for (int i = lane * some; i < (lane + 1) * some && i < all; i++) own += sums[i];
        const u64 to_lane = warp_scan(own), total = __shfl_sync(0xffffffffu, to_lane, 31);
        const u64 target = target_of(total, u);
        const int in = __ffs(__ballot_sync(0xffffffffu, to_lane > target)) - 1;
        u64 before = __shfl_sync(0xffffffffu, to_lane - own, in);
        int owner = in * some;
        for (; before + sums[owner] <= target; owner++) before += sums[owner];
        const int r = owner / WARPS, part = part_of_cta(r);
        if (!here && r != rank) return;
        // its tokens, some neighbouring ones a thread; e counts from this CTA's first on
        const int begin = (r - rank) * a.seg + owner % WARPS * part;
        const int end = min(begin + part, min((r + 1) * a.seg, a.V) - first);
        const int per = cdiv(part, THREADS), e0 = begin + tid * per;
        auto at = [&](int e) { return __fadd_rn(to_f(from[e]), 0.0f); };
        u64 mine = 0;
        for (int e = e0; e < e0 + per && e < end; e++) {
            const float v = at(e);
            if (kept(v, e)) mine += weights.mass(v);
        }
        u64 block;
        u64 sum = before + block_before(mine, block);
        if (sum <= target && target < sum + mine) {
            for (int e = e0; e < e0 + per && e < end; e++) {
                const float v = at(e);
                if (!kept(v, e)) continue;
                const u64 w = weights.mass(v);
                if (sum + w > target) {
                    a.token[row] = first + e;
                    if (a.prob) a.prob[row] = weights.share(v, total);
                    break;
                }
                sum += w;
            }
        }
    }

    // The filters and the choice on the listed tokens, which hold all that are kept.  By CTA 0.
    __device__ __forceinline__ void choose_listed(int m, bool by_k, int k, bool by_p, double p, u64 total, double least_power,
                                                  float u, int64_t row) {
        const int size = size_of(m);
        u64 q = sorted(tid < m ? sh.all[tid].key : 0, size);
        const bool some = tid < m;
        const float v = value(q);
        u64 mass = some ? weights.mass(v) : 0;
        bool keep = some && (!by_k || tid < k);
        if (by_p) {
            u64 all;
            const u64 before = block_before(keep ? mass : 0, all);
            keep = keep && (before < part_of(by_k ? all : total, p) || tid == 0);
        }
        if (keep && !(weights.power(v) >= least_power)) keep = false;
        __syncthreads();  // the sort before is over for all
        // now by index: the lowest comes first
        q = sorted(keep ? (u64)(0xffffffffu - index(q)) << 32 | key_of(v) : 0, size);
        const float chosen = value_of((uint32_t)q);
        mass = q ? weights.mass(chosen) : 0;
        const u64 before = block_before(mass, total), target = target_of(total, u);
        if (mass && before <= target && target < before + mass) {
            a.token[row] = 0xffffffffu - (uint32_t)(q >> 32);
            if (a.prob) a.prob[row] = weights.share(chosen, total);
        }
    }

    // The border of top-k, or of top-p of all tokens, by counts in fine bins, and the choice.  The counts give the bin of the
    // k-th token.  The mass of a bin's c tokens, which lie t_i into it (0 to 1) where weights fall by r, is the sum of
    // r^t_i: at least c r^mean(t), as r^t is convex, and at most c - (1 - r) sum(t), the chord's.  That bounds the masses
    // up to each bin from both sides, to 1e-4, and so the bins in which top-p's border can lie.
    // One pass over the weights then adds up what lies above those bins, by warps, and lists the tokens in them (or all
    // down to them, if they are few).  CTA 0 finds the border among these and has the sums of what is kept.  `least`: the
    // row's least finite value; `floor`: the least that min-p keeps.  False: too many tokens lie in those bins.
    __device__ __forceinline__ bool choose_by_bins(bool by_k, int k, double p, float least, float floor, double least_power, float u,
                                                   int64_t row) {
        const Bins<FINE> bins(value_of(kmax), temperature, __fsub_rn(value_of(kmax), least));
        for (int i = tid; i < FINE; i += THREADS) sh.fine[i] = sh.depth[i] = 0;
        __syncthreads();
        // what has no weight is never chosen, but counts for top-k
        const float end = by_k ? -3.402823466e38f : weights.end;
        each<2>([&](const float (&v)[K], int) {
            int b[K], t[K];
#pragma unroll
            for (int i = 0; i < K; i++) {
                b[i] = bins(v[i]);
                t[i] = (int)((bins.at(v[i]) - (float)b[i]) * 256.0f);
            }
#pragma unroll
            for (int i = 0; i < K; i++)
                if (v[i] >= end) {
                    atomicAdd(&sh.fine[b[i]], 1u);
                    if (!by_k) atomicAdd(&sh.depth[b[i]], (uint32_t)min(t[i], 255));
                }
        });
        sync();
        if (cs > 1) {  // each CTA adds up a part of the bins for all
            for (int i = rank * (FINE / cs) + tid; i < (rank + 1) * (FINE / cs); i += THREADS) {
                uint32_t all = 0, deep = 0;
                for (int r = 0; r < cs; r++) all += of(r).fine[i], deep += of(r).depth[i];
                for (int r = 0; r < cs; r++) of(r).fine[i] = all, of(r).depth[i] = deep;
            }
            sync();
        }
        constexpr int PER = FINE / THREADS;
        uint32_t c[PER], counts = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) c[i] = sh.fine[tid * PER + i];
        // in units of 2^-30; 3e-5 for the rounding of the weights and of (most - v) * scale.  Whole numbers again, so that
        // every thread of every CTA has the same sums.  A single bin and the last one are open downwards.
        u64 low[PER], high[PER], lows = 0, highs = 0;
        const bool one = !(bins.scale > 0.0f);
        const float width = one ? 0.0f : (float)(weights.scale * (1.0 / ROOTS) / (double)bins.scale);
        const float fall = 1.0f - exp2f(-width);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int b = tid * PER + i;
            const float n = (float)c[i], t = (float)sh.depth[b] * (1.0f / 256.0f), edge = exp2f(30.0f - (float)b * width);
            const bool open = one || b == FINE - 1;
            high[i] = (u64)(edge * (open ? n : n - fall * t) * (1 + 3e-5f)) + (c[i] > 0);
            low[i] = open || !c[i] ? 0 : (u64)(edge * n * exp2f(-width * (t / n + 1.0f / 256.0f)) * (1 - 3e-5f));
            lows += low[i], highs += high[i], counts += c[i];
        }
        u64 lup = warp_scan(lows), hup = warp_scan(highs);
        uint32_t cup = warp_scan(counts);
        if (lane == 31) sh.warp_low[warp] = lup, sh.warp_mass[warp] = hup, sh.warp_count[warp] = cup;
        __syncthreads();
        u64 lall = 0, hall = 0;
        for (int i = 0; i < WARPS; i++) {
            if (i == warp) lup += lall, hup += hall;
            if (i < warp) cup += sh.warp_count[i];
            lall += sh.warp_low[i], hall += sh.warp_mass[i];
        }
        lup -= lows, hup -= highs, cup -= counts;
        if (by_k) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                if (cup < k && (k <= cup + c[i] || tid * PER + i == FINE - 1))
                    sh.edge[0] = sh.edge[1] = tid * PER + i, sh.upto[0] = cup, sh.upto[1] = cup + c[i];
                cup += c[i];
            }
        } else {
            // the first bin whose upper sum reaches the least that is wanted, and the first whose lower sum reaches the most
            const u64 want_low = (u64)fmax(p * (double)lall * (1 - 1e-9), 0.0);
            const u64 want_high = (u64)(fmax(p, 0.0) * (double)hall * (1 + 1e-9)) + 1;
            bool below_low = tid == 0 || hup < want_low, below_high = tid == 0 || lup < want_high;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                hup += high[i], lup += low[i];
                if (below_low && hup >= want_low) sh.edge[0] = tid * PER + i, sh.upto[0] = cup;
                cup += c[i];
                if (below_high && (lup >= want_high || tid * PER + i == FINE - 1)) sh.edge[1] = tid * PER + i, sh.upto[1] = cup;
                below_low = hup < want_low, below_high = lup < want_high;
            }
        }
        __syncthreads();
        const int b0 = sh.edge[0], b1 = sh.edge[1], counted = sh.upto[0];
        const bool whole = sh.upto[1] <= LIST;
        if (!whole && sh.upto[1] - counted > LIST) return false;
        u64 sum = 0, above = 0;
        const int from_bin = whole ? 0 : b0;
        each<1>([&](const float (&v)[K], int e) {
            bool any = !by_k;
            int b[K];
#pragma unroll
            for (int i = 0; i < K; i++) b[i] = bins(v[i]), any = any || b[i] <= b1;
            if (!any) return;  // of top-k only what may be kept has to be weighed
            u64 w[K];
#pragma unroll
            for (int i = 0; i < K; i++) w[i] = weights.mass(v[i]);
#pragma unroll
            for (int i = 0; i < K; i++) {
                sum += w[i];
                above += b[i] < b0 && v[i] >= floor ? w[i] : 0;
            }
#pragma unroll
            for (int i = 0; i < K; i++)
                if (b[i] <= b1 && b[i] >= from_bin && v[i] >= end) list_one(v[i], e + i);
        });
        above = warp_sum(above);
        if (lane == 0) of(0).above[rank][warp] = above;
        const u64 total = exchange_sums(sum);
        const int m = gather();
        if (m < 0) return false;
        if (rank) return true;
        if (whole) {
            choose_listed(m, by_k, k, !by_k, p, total, least_power, u, row);
            return true;
        }
        u64* sums = &sh.above[0][0];
        u64 over = 0;
        for (int i = lane; i < cs * WARPS; i += 32) over += sums[i];
        over = warp_sum(over);
        const u64 q = sorted(tid < m ? sh.all[tid].key : 0, size_of(m));
        const float v = value(q);
        const u64 w = tid < m ? weights.mass(v) : 0;
        u64 all;
        const u64 before = block_before(w, all);  // behind its barriers `sums` is read by all
        bool keep = tid < m && v >= floor && weights.power(v) >= least_power;
        // min-p's floor only lowers `over` where the border lies below it, and then nothing listed is kept
        keep = keep && (by_k ? tid < k - counted : over + before < part_of(total, p));
        if (tid == 0) sh.cut = ~0ull;
        if (tid < cs * WARPS)
            for (int j = 0; j < 3; j++) sh.limb[0][j][tid] = 0;
        __syncthreads();
        if (keep) {
            const int at = index(q), r = at / a.seg, part = part_of_cta(r);
#pragma unroll
            for (int j = 0; j < 3; j++)
                atomicAdd(&sh.limb[0][j][r * WARPS + (at - r * a.seg) / part], (uint32_t)(w >> (15 * j)) & 0x7fffu);
        }
        const uint32_t some = __ballot_sync(0xffffffffu, keep);
        if (some && lane == 31 - __clz(some)) atomicMin(&sh.cut, q);  // the warp's last in the order
        __syncthreads();
        if (tid < cs * WARPS)
            for (int j = 0; j < 3; j++) sums[tid] += (u64)sh.limb[0][j][tid] << (15 * j);
        const u64 cut = sh.cut;
        __syncthreads();
        finish(sums, u, row, [&](float v, int e) { return v >= floor && (bins(v) < b0 || full_key(v, e) >= cut); }, true);
        return true;
    }

    // ----- by histograms -----
    __device__ __forceinline__ void clear(int set) {
        for (int i = tid; i < BINS; i += THREADS) {
            sh.count[set][i] = 0;
#pragma unroll
            for (int j = 0; j < 3; j++) sh.limb[set][j][i] = 0;
        }
    }
    template <bool MASS>
    __device__ __forceinline__ void add(int at, float v) {
        atomicAdd(&sh.count[level & 1][at], 1u);
        if (MASS) {
            const u64 w = weights.mass(v);
#pragma unroll
            for (int j = 0; j < 3; j++) atomicAdd(&sh.limb[level & 1][j][at], (uint32_t)(w >> (15 * j)) & 0x7fffu);
        }
    }

    // Adds up the row's histograms and finds the bin of the border: by count, the bin of the target-th
    // token; by mass, the bin in which the mass reaches the target, `share` of all if `share` is given.
    // false: there are no more than target tokens.
    template <bool MASS>
    __device__ __forceinline__ bool border(u64 target, const double* share) {
        const int k = level & 1;
        static_assert(BINS == THREADS, "a bin a thread");
        sync();
        uint32_t c = 0;
        u64 m = 0;
        for (int r = 0; r < cs; r++) {
            const Shared& with = of(r);
            c += with.count[k][tid];
            if (MASS) {
#pragma unroll
                for (int j = 0; j < 3; j++) m += (u64)with.limb[k][j][tid] << (15 * j);
            }
        }
        clear(k ^ 1);  // last read before this barrier
        uint32_t cup = warp_scan(c);
        u64 mup = MASS ? warp_scan(m) : 0;
        if (lane == 31) sh.warp_count[warp] = cup, sh.warp_mass[warp] = mup;
        if (tid == 0) sh.listed = 0;
        __syncthreads();
        uint32_t call = 0;
        u64 mall = 0;
        for (int i = 0; i < WARPS; i++) {
            if (i == warp) cup += call, mup += mall;
            call += sh.warp_count[i];
            mall += sh.warp_mass[i];
        }
        if (MASS && share) target = part_of(mall, *share);
        level++;
        if (!MASS && call <= target) return false;
        const uint32_t cb = cup - c;
        const u64 mb = mup - m;
        if (MASS ? mb < target && target <= mup : cb < target && target <= cup) {
            sh.bin = tid;
            sh.above_count = cb, sh.above_mass = mb, sh.in_count = c, sh.in_mass = m, sh.target = target;
        }
        __syncthreads();
        return true;
    }

    // Moves the cut to the border: by count, the target-th token's key, by mass, the key of the token with
    // which the mass reaches `share` of all that is kept.
    template <bool MASS>
    __device__ __forceinline__ void descend(uint32_t k, double share, u64& cut) {
        const float vcut = value(cut);
        const Bins<BINS> bins(value_of(kmax), temperature, __int_as_float(0x7f800000));
        each<1>([&](const float (&v)[K], int e) {
#pragma unroll
            for (int i = 0; i < K; i++)
                if (kept(v[i], e + i, vcut, cut)) add<MASS>(bins(v[i]), v[i]);
        });
        if (!border<MASS>(k, &share)) return;
        // the keys of the bin
        const int b = sh.bin;
        if (warp < 2) {
            const int last = b - warp;
            const uint32_t edge = last < 0 ? kmax + 1
                                  : last == BINS - 1
                                      ? LOWEST
                                      : first_key(LOWEST - 1, kmax, [&](uint32_t q) { return bins(value_of(q)) <= last; });
            if (lane == 0) sh.edge[warp] = edge;
        }
        __syncthreads();
        u64 lo = (u64)sh.edge[0] << bits, hi = ((u64)sh.edge[1] << bits) - 1;
        if (lo < cut) lo = cut;
        u64 target = sh.target;
        while (true) {
            const u64 left = target - (MASS ? sh.above_mass : sh.above_count);
            if (left == (MASS ? sh.in_mass : sh.in_count) || lo == hi) {  // the whole bin
                cut = lo;
                __syncthreads();
                return;
            }
            const float vlo = value(lo), vhi = value(hi);
            if (sh.in_count <= LIST) {
                each<1>([&](const float (&v)[K], int e) {
#pragma unroll
                    for (int j = 0; j < K; j++) {
                        if (!(v[j] >= vlo && v[j] <= vhi)) continue;
                        const u64 q = full_key(v[j], e + j);
                        if (q < lo || q > hi) continue;
                        const uint32_t i = atomicAdd(&sh.listed, 1u);
                        if (i < LIST) sh.own[i] = {q, MASS ? weights.mass(v[j]) : 1ull};
                    }
                });
                sync();
                uint32_t m = 0;
                for (int r = 0; r < cs; r++) {
                    const Shared& with = of(r);
                    const uint32_t some = with.listed;
                    if (tid < some && m + tid < LIST) sh.all[m + tid] = with.own[tid];
                    m += some;
                }
                if (m > LIST) m = LIST;
                __syncthreads();
                if (tid < m) {
                    const Entry mine = sh.all[tid];
                    u64 before = 0;
                    for (uint32_t i = 0; i < m; i++) before += sh.all[i].key > mine.key ? sh.all[i].mass : 0;
                    if (before < left && left <= before + mine.mass) sh.cut = mine.key;
                }
                __syncthreads();
                cut = sh.cut;
                return;
            }
            // too many for the list: by the leading bits of their keys
            int shift = 0;
            while (((hi - lo) >> shift) >= BINS) shift++;
            const u64 in_lo = lo, in_hi = hi;
            each<1>([&](const float (&v)[K], int e) {
#pragma unroll
                for (int i = 0; i < K; i++) {
                    if (!(v[i] >= vlo && v[i] <= vhi)) continue;
                    const u64 q = full_key(v[i], e + i);
                    if (q >= in_lo && q <= in_hi) add<MASS>((int)((in_hi - q) >> shift), v[i]);
                }
            });
            border<MASS>(left, nullptr);
            hi = in_hi - ((u64)sh.bin << shift);
            const u64 span = ((u64)1 << shift) - 1;
            lo = hi - in_lo > span ? hi - span : in_lo;
            target = sh.target;
        }
    }

    // The choice among the tokens from the cut on.  Tokens of a warp are neighbours: the sums by warp are in the
    // order of the indices.
    __device__ __forceinline__ void choose(float u, u64 cut, int64_t row) {
        const float vcut = value(cut);
        u64 sum = 0;
        each<1>([&](const float (&v)[K], int e) {
            bool in[K], any = false;
#pragma unroll
            for (int i = 0; i < K; i++) in[i] = kept(v[i], e + i, vcut, cut), any = any || in[i];
            if (!any) return;
            u64 w[K];
#pragma unroll
            for (int i = 0; i < K; i++) w[i] = weights.mass(v[i]);
#pragma unroll
            for (int i = 0; i < K; i++) sum += in[i] ? w[i] : 0;
        });
        sum = warp_sum(sum);
        if (lane < cs) of(lane).sums[rank][warp] = sum;
        sync();
        finish(&sh.sums[0][0], u, row, [&](float v, int e) { return kept(v, e, vcut, cut); }, false);
    }
};

template <typename T>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const __grid_constant__ Args a) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cs = a.cs, rank = blockIdx.x % cs;
    const int64_t row = blockIdx.x / cs;
    Chooser<T> c = {a, sh};
    c.first = rank * a.seg, c.n = max(0, min(a.seg, a.V - c.first));
    c.rank = rank, c.cs = cs, c.tid = tid, c.warp = warp, c.lane = lane;
    c.from = static_cast<const T*>(a.logits) + row * a.ld + c.first;
    c.bits = 32 - __clz(a.V - 1 | 1);
    c.part = c.part_of_cta(rank);
    if (cs > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");  // this CTA has started
    grid_dependency_sync();
    const float temperature = a.temperature ? a.temperature[row] : a.temperature1;
    const int k = a.top_k ? a.top_k[row] : a.top_k1;
    const float p = a.top_p ? a.top_p[row] : a.top_p1, min_p = a.min_p ? a.min_p[row] : a.min_p1;
    const bool greedy = !(temperature > 0.0f), by_k = k > 0 && k < a.V, by_p = p < 1.0f, by_m = min_p > 0.0f;
    if (tid == 0) sh.listed = 0;
    if (tid < ROOTS) sh.roots[tid] = exp2((double)tid / ROOTS + SCALE);
    const bool wide = a.V > LIST && by_k != by_p;  // bins down to the least value are likely
    float top = -__int_as_float(0x7f800000), low = __int_as_float(0x7f800000);
    constexpr int K = Chooser<T>::K;
    c.template each<2>([&](const float (&v)[K], int) {
#pragma unroll
        for (int i = 0; i < K; i++) {
            top = max_nan(top, v[i]);
            if (wide && v[i] > -__int_as_float(0x7f800000)) low = fminf(low, v[i]);
        }
    });
    {
        const uint32_t q = key_of(top), m = __reduce_max_sync(0xffffffffu, q);
        if (cs > 1) asm volatile("barrier.cluster.wait;" ::: "memory");
        const uint32_t l = __reduce_min_sync(0xffffffffu, key_of(low));
        if (lane < cs) c.of(lane).most[rank][warp] = m, c.of(lane).at[rank][warp] = l;
        if (by_k) {
            uint32_t g = q;
            for (int i = 1; i < cs; i <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, i));
            // cs neighbouring threads are a group, and each tells one CTA
            c.of(lane % cs).maxima[(rank * THREADS + tid) / cs] = g;
        }
    }
    c.sync();
    uint32_t most = 0, least = 0xffffffffu;
    for (int i = lane; i < cs * WARPS; i += 32)
        most = max(most, (&sh.most[0][0])[i]), least = min(least, (&sh.at[0][0])[i]);
    most = __reduce_max_sync(0xffffffffu, most);
    least = __reduce_min_sync(0xffffffffu, least);
    // greedy rows, and those whose maximum leaves no distribution: infinite, NaN, or nothing but -infinity
    if (greedy || most >= INF || most < LOWEST) {
        uint32_t at = 0xffffffffu;
        c.template each<2>([&](const float (&v)[K], int e) {
#pragma unroll
            for (int i = 0; i < K; i++)
                if (key_of(v[i]) == most) at = min(at, (uint32_t)(c.first + e + i));
        });
        at = __reduce_min_sync(0xffffffffu, at);
        c.sync();  // all have read the least values there
        if (lane == 0) c.of(0).at[rank][warp] = at;
        c.sync();
        if (rank || warp) return;
        at = 0xffffffffu;
        for (int i = lane; i < cs * WARPS; i += 32) at = min(at, (&sh.at[0][0])[i]);
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) {
            a.token[row] = at;
            if (a.prob) a.prob[row] = 1.0f;
        }
        return;
    }
    c.kmax = most;
    c.temperature = temperature;
    c.weights = Weights(value_of(most), temperature, sh.roots);
    // min-p as the power that a token has to reach, and as the least value that does
    const double least_power = !by_m ? -1e300 : min_p < 1.0f ? ROOTS * log2((double)min_p) : 0.0;
    float floor = -3.402823466e38f;
    if (by_m) {
        if (warp == 0) {
            const uint32_t q = first_key(LOWEST - 1, most, [&](uint32_t q) { return c.weights.power(value_of(q)) >= least_power; });
            if (lane == 0) sh.bound = q;
        }
        __syncthreads();
        floor = value_of(sh.bound);
        __syncthreads();
    }
    // a bound that all kept tokens reach
    bool bounded = (by_m && !(by_k && by_p)) || (a.V <= LIST && (by_k || by_p || by_m));
    float bound = by_m && !(by_k && by_p) ? floor : -3.402823466e38f;
    if (a.V > LIST && by_k && k <= (by_p ? THREADS : THREADS * 5 / 8)) {  // beyond, the list is likely to be too long
        const uint32_t q = c.sorted(sh.maxima[tid], THREADS);
        if (tid == k - 1) sh.bound = q;
        __syncthreads();
        if (sh.bound >= LOWEST) bounded = true, bound = fmaxf(bound, value_of(sh.bound));
    }
    if (bounded && (by_k || !by_p || a.V <= LIST)) {
        c.template each<2>([&](const float (&v)[K], int e) {
#pragma unroll
            for (int i = 0; i < K; i++)
                if (v[i] >= bound) c.list_one(v[i], e + i);
        });
        u64 total = 0;
        if (by_p && !by_k) {  // of a row as short as a list
            u64 sum = 0;
            c.template each<1>([&](const float (&v)[K], int) {
#pragma unroll
                for (int i = 0; i < K; i++) sum += c.weights.mass(v[i]);
            });
            total = c.exchange_sums(sum);
        }
        const int m = c.gather();
        if (m >= 0) {
            if (rank == 0) c.choose_listed(m, by_k, k, by_p, (double)p, total, least_power, a.u[row], row);
            return;
        }
        __syncthreads();
        if (tid == 0) sh.listed = 0;
    }
    if (wide && c.choose_by_bins(by_k, k, (double)p, value_of(least), floor, least_power, a.u[row], row)) return;
    u64 cut = (u64)LOWEST << c.bits;
    if (by_k || by_p) {
        c.sync();  // all have read what lies in the histograms' place
        c.clear(0);
        c.clear(1);
        if (tid == 0) sh.listed = 0;
        __syncthreads();
        if (by_k) c.template descend<false>(k, 0.0, cut);
        if (by_p) c.template descend<true>(0, (double)p, cut);
    }
    if (((u64)key_of(floor) << c.bits) > cut) cut = (u64)key_of(floor) << c.bits;
    c.choose(a.u[row], cut, row);
}

// CTAs of a row: doubled where rows leave SMs idle, down to 8192 tokens a CTA.
static inline int cluster_of(int rows, int V) {
    int cs = 1;
    while (cs < MAX_CLUSTER && (V > cs * MAX_SEG || ((int64_t)rows * cs * 2 <= 148 && V > cs * 8192))) cs *= 2;
    return cs;
}

}  // namespace sample
}  // namespace mi

extern "C" int mi_sample_rows(const void* logits, int64_t ld, const float* u, const float* temperature,
                              const int32_t* top_k, const float* top_p, const float* min_p, float temperature1, int top_k1,
                              float top_p1, float min_p1, int64_t* token, float* prob, int rows, int V, int dtype,
                              void* stream) {
    if (!logits || !u || !token || rows < 0 || V <= 0 || ld < 0) return MI_ERR_INVALID;
    if (V > mi::sample::MAX_V || rows > 1 << 27) return MI_ERR_UNSUPPORTED;
    mi::sample::Args a = {};
    a.logits = logits, a.ld = ld, a.u = u, a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p;
    a.temperature1 = temperature1, a.top_k1 = top_k1, a.top_p1 = top_p1, a.min_p1 = min_p1;
    a.token = token, a.prob = prob, a.V = V;
    a.cs = mi::sample::cluster_of(rows, V);
    a.seg = mi::cdiv(mi::cdiv(V, a.cs), 8) * 8;
    MI_DISPATCH_DTYPE(dtype, T, {
        if (rows == 0) return MI_OK;
        static std::atomic<uint64_t> allowed{0};
        auto kernel = mi::sample::sample_kernel<T>;
        if (!mi::allow_smem(kernel, sizeof(mi::sample::Shared), allowed)) return MI_ERR_CUDA;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(rows * a.cs);
        cfg.blockDim = dim3(mi::sample::THREADS);
        cfg.dynamicSmemBytes = sizeof(mi::sample::Shared);
        cfg.stream = (cudaStream_t)stream;
        cudaLaunchAttribute attr[2];
        int m = 0;
        if (a.cs > 1) {
            attr[m].id = cudaLaunchAttributeClusterDimension;
            attr[m].val.clusterDim.x = a.cs;
            attr[m].val.clusterDim.y = attr[m].val.clusterDim.z = 1;
            m++;
        }
        if (mi::pdl_enabled()) {
            attr[m].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[m].val.programmaticStreamSerializationAllowed = 1;
            m++;
        }
        cfg.attrs = attr;
        cfg.numAttrs = m;
        if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
            cudaGetLastError();
            return MI_ERR_CUDA;
        }
        return MI_OK;
    });
}

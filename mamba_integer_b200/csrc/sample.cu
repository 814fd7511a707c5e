// sample.cu -- the choice of a token from a row of logits by a given uniform
// number, with temperature, top-k, top-p and min-p (greedy rows: argmax).
//
//   w_i = 2^((l_i - max l) log2(e) / temperature)
//   in the order (l downwards, index upwards): keep the first k; of those, each
//   whose mass before it is below p times their total (the first always); of
//   those, w_i >= min_p.  The token is the first index whose running sum of the
//   kept w, in index order, exceeds u times their total.
//
// Every filter keeps a first part of one order, so all of them end in one
// number: a token's rank is key = (order-preserving bits of l, mask - index),
// which no two tokens share, and the kept ones are those with key >= cut.
//
// Borders between tokens are sharp, so masses are whole numbers: w in units of
// 2^-44 from a 64-bit evaluation (2^-42 relative), which add up exactly and in
// any order.  fp32 weights would move the borders of a flat distribution over
// 32768 tokens by 1e-8 each, one row in some ten thousand.
//
// A row lies in the shared memory of one CTA or of a cluster of up to 8, read
// once.  A border is found by a histogram over 1024 bins of equal width between
// the maximum and where the weights end, which leaves a bin of few tokens; these
// are listed and ranked against one another, or, where they are many (equal or
// nearly equal logits), divided again by the bits of their keys.
#include <cooperative_groups.h>

#include "mi_elem.cuh"

namespace mi {
namespace sample {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 1024, LIST = 256, MAX_CLUSTER = 8, MAX_SEG = 32768;
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
    int V, cs, seg, vec;
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
struct Weights {
    double most, scale;  // log2(e) / temperature
    __device__ __forceinline__ double power(float v) const { return ((double)v - most) * scale; }
    // 2^x times 2^SCALE: x = n + f, |f| <= 1/2; the power series of 2^f, ended behind (f ln 2)^10 / 10!,
    // leaves 2.2e-13.  Not rounded to a whole number; 0 where less than half of one is left.
    __device__ __forceinline__ static double scaled(double x) {
        if (!(x > -(SCALE + 1))) return 0.0;
        const double n = __dsub_rn(__dadd_rn(x, 6755399441055744.0), 6755399441055744.0), f = __dsub_rn(x, n);
        const double g = f * 0.693147180559945309417;
        double p = 1.0 / 3628800;
        p = __fma_rn(p, g, 1.0 / 362880);
        p = __fma_rn(p, g, 1.0 / 40320);
        p = __fma_rn(p, g, 1.0 / 5040);
        p = __fma_rn(p, g, 1.0 / 720);
        p = __fma_rn(p, g, 1.0 / 120);
        p = __fma_rn(p, g, 1.0 / 24);
        p = __fma_rn(p, g, 1.0 / 6);
        p = __fma_rn(p, g, 0.5);
        p = __fma_rn(p, g, 1.0);
        p = __fma_rn(p, g, 1.0);
        return p * __hiloint2double((1023 + SCALE + (int)n) << 20, 0);
    }
    __device__ __forceinline__ u64 mass(float v) const { return __double2ull_rn(scaled(power(v))); }
};

// Bins of equal width downwards from the maximum; falls monotonically as v rises.
struct Bins {
    float most, scale;
    __device__ __forceinline__ int operator()(float v) const {
        const float at = __fmul_rn(__fsub_rn(most, v), scale);
        return at < (float)(BINS - 1) ? (int)at : BINS - 1;
    }
};

struct Row {  // what the CTAs of a row tell one another
    uint32_t most[MAX_CLUSTER], at[MAX_CLUSTER], least[MAX_CLUSTER];
    u64 sums[MAX_CLUSTER][WARPS];
};
struct Entry {
    u64 key, mass;
};
struct Shared {
    u64 mass[2][BINS];
    Entry own[LIST], all[LIST];
    Row row;
    uint32_t count[2][BINS];
    u64 warp_mass[WARPS];
    uint32_t warp_count[WARPS], warp_low[WARPS];
    uint32_t listed;
    // a border's bin: what lies above it, what it holds
    u64 above_mass, in_mass, target;
    uint32_t above_count, in_count, bin, edge[2];
    u64 cut, floor;
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

template <typename T>
struct Chooser {
    const Args& a;
    Shared& sh;
    float* vals;
    int n, first, rank;  // this CTA's tokens: first .. first + n - 1
    int cs, bits;        // bits of an index
    Weights weights;
    Bins bins;
    uint32_t kmax;
    int level = 0;  // of the histograms, which alternate

    __device__ __forceinline__ u64 full_key(float v, int e) const {
        return (u64)key_of(v) << bits | (u64)((1u << bits) - 1 - (uint32_t)(first + e));
    }
    __device__ __forceinline__ void sync() {
        if (cs > 1)
            cg::this_cluster().sync();
        else
            __syncthreads();
    }

    // Adds up the row's histograms and finds the bin of the border: by count, the bin of the target-th
    // token; by mass, the bin in which the mass reaches the target, `share` of all if `share` is given.
    // false: there are no more than target tokens.
    template <bool MASS>
    __device__ __forceinline__ bool border(uint64_t target, const double* share) {
        const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, k = level & 1;
        constexpr int PER = BINS / THREADS;
        sync();
        uint32_t c[PER] = {}, ctot = 0;
        u64 m[PER] = {}, mtot = 0;
        for (int r = 0; r < cs; r++) {
            const Shared& from = cs > 1 ? *cg::this_cluster().map_shared_rank(&sh, r) : sh;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                c[i] += from.count[k][tid * PER + i];
                if (MASS) m[i] += from.mass[k][tid * PER + i];
            }
        }
#pragma unroll
        for (int i = 0; i < PER; i++) ctot += c[i], mtot += m[i];
        // the other set was last read before this barrier
        for (int i = tid; i < BINS; i += THREADS) sh.count[k ^ 1][i] = 0, sh.mass[k ^ 1][i] = 0;
        uint32_t cup = warp_scan(ctot);
        u64 mup = MASS ? warp_scan(mtot) : 0;
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
        if (MASS && share) {
            const double t = ceil(*share * (double)mall);
            target = t >= (double)mall ? mall : t < 1.0 ? 1 : (u64)t;
        }
        level++;
        if (!MASS && call <= target) return false;
        uint32_t cb = cup - ctot;
        u64 mb = mup - mtot;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const bool here = MASS ? mb < target && target <= mb + m[i] : cb < target && target <= cb + c[i];
            if (here) {
                sh.bin = tid * PER + i;
                sh.above_count = cb, sh.above_mass = mb, sh.in_count = c[i], sh.in_mass = m[i], sh.target = target;
            }
            cb += c[i], mb += m[i];
        }
        __syncthreads();
        return true;
    }

    // Moves the cut to the border: by count, the target-th token's key, by mass, the key of the token with
    // which the mass reaches `share` of all that is kept.
    template <bool MASS>
    __device__ __forceinline__ void descend(uint32_t k, double share, u64& cut) {
        const int tid = threadIdx.x, warp = tid >> 5;
        const float vcut = value_of((uint32_t)(cut >> bits));
        for (int e = tid; e < n; e += THREADS) {
            const float v = vals[e];
            if (!(v >= vcut) || full_key(v, e) < cut) continue;
            const int at = bins(v);
            atomicAdd(&sh.count[level & 1][at], 1u);
            if (MASS) atomicAdd(&sh.mass[level & 1][at], weights.mass(v));
        }
        if (!border<MASS>(k, &share)) return;
        // the keys of the bin
        const int b = sh.bin;
        if (warp < 2) {
            const int last = b - warp;
            const uint32_t edge = last < 0 ? kmax + 1
                                  : last == BINS - 1 ? LOWEST
                                                     : first_key(LOWEST - 1, kmax, [&](uint32_t q) { return bins(value_of(q)) <= last; });
            if ((tid & 31) == 0) sh.edge[warp] = edge;
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
            const float vlo = value_of((uint32_t)(lo >> bits)), vhi = value_of((uint32_t)(hi >> bits));
            if (sh.in_count <= LIST) {
                for (int e = tid; e < n; e += THREADS) {
                    const float v = vals[e];
                    if (!(v >= vlo && v <= vhi)) continue;
                    const u64 q = full_key(v, e);
                    if (q < lo || q > hi) continue;
                    const uint32_t i = atomicAdd(&sh.listed, 1u);
                    if (i < LIST) sh.own[i] = {q, MASS ? weights.mass(v) : 1ull};
                }
                sync();
                uint32_t m = 0;
                for (int r = 0; r < cs; r++) {
                    const Shared& from = cs > 1 ? *cg::this_cluster().map_shared_rank(&sh, r) : sh;
                    const uint32_t some = from.listed;
                    for (uint32_t i = tid; i < some && m + i < LIST; i += THREADS) sh.all[m + i] = from.own[i];
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
            const u64 next = left;
            for (int e = tid; e < n; e += THREADS) {
                const float v = vals[e];
                if (!(v >= vlo && v <= vhi)) continue;
                const u64 q = full_key(v, e);
                if (q < in_lo || q > in_hi) continue;
                const int at = (int)((in_hi - q) >> shift);
                atomicAdd(&sh.count[level & 1][at], 1u);
                if (MASS) atomicAdd(&sh.mass[level & 1][at], weights.mass(v));
            }
            border<MASS>(next, nullptr);
            const u64 b2 = sh.bin;
            hi = in_hi - (b2 << shift);
            const u64 span = ((u64)1 << shift) - 1;
            lo = hi - in_lo > span ? hi - span : in_lo;
            target = sh.target;
        }
    }

    // Tokens of a warp are neighbours: the sums by warp are in the order of the indices.
    __device__ __forceinline__ void choose(float u, u64 cut, int64_t row) {
        const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
        const int part = cdiv(cdiv(n, WARPS), 32) * 32;  // tokens a warp
        const float vcut = value_of((uint32_t)(cut >> bits));
        u64 sum = 0;
        for (int e = warp * part + lane; e < (warp + 1) * part && e < n; e += 32) {
            const float v = vals[e];
            if (v >= vcut && full_key(v, e) >= cut) sum += weights.mass(v);
        }
        sum = warp_sum(sum);
        if (lane < cs) {
            Row& to = cs > 1 ? *cg::this_cluster().map_shared_rank(&sh.row, lane) : sh.row;
            to.sums[rank][warp] = sum;
        }
        sync();
        // every warp adds up all of them, some neighbouring ones a lane
        const u64* sums = &sh.row.sums[0][0];
        const int all = cs * WARPS, some = cdiv(all, 32);
        u64 own = 0;
        for (int i = lane * some; i < (lane + 1) * some && i < all; i++) own += sums[i];
        u64 to_lane = warp_scan(own);
        const u64 total = __shfl_sync(0xffffffffu, to_lane, 31);
        // the token whose sum is the first above `target`
        const double t = floor((double)u * (double)total);
        const u64 target = !(t > 0.0) ? 0 : t >= (double)total ? total - 1 : (u64)t < total ? (u64)t : total - 1;
        const int in = __ffs(__ballot_sync(0xffffffffu, to_lane > target)) - 1;
        u64 before = __shfl_sync(0xffffffffu, to_lane - own, in);
        int owner = in * some;
        for (; before + sums[owner] <= target; owner++) before += sums[owner];
        if (owner / WARPS != rank) return;
        const int begin = owner % WARPS * part, end = min(begin + part, n);
        const int each = cdiv(part, THREADS), e0 = begin + tid * each;
        u64 mine = 0;
        for (int e = e0; e < e0 + each && e < end; e++) {
            const float v = vals[e];
            if (v >= vcut && full_key(v, e) >= cut) mine += weights.mass(v);
        }
        u64 upto = warp_scan(mine);
        if (lane == 31) sh.warp_mass[warp] = upto;
        __syncthreads();
        for (int i = 0; i < warp; i++) upto += sh.warp_mass[i];
        upto += before;
        if (upto - mine <= target && target < upto) {
            u64 at = upto - mine;
            for (int e = e0; e < e0 + each && e < end; e++) {
                const float v = vals[e];
                if (!(v >= vcut) || full_key(v, e) < cut) continue;
                const u64 w = weights.mass(v);
                if (at + w > target) {
                    a.token[row] = first + e;
                    if (a.prob) a.prob[row] = (float)(Weights::scaled(weights.power(v)) / (double)total);
                    break;
                }
                at += w;
            }
        }
    }
};

template <typename T>
__global__ void __launch_bounds__(THREADS) sample_kernel(const Args a) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    float* vals = reinterpret_cast<float*>(smem + sizeof(Shared));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cs = a.cs, rank = blockIdx.x % cs;
    const int64_t row = blockIdx.x / cs;
    const int first = rank * a.seg, n = max(0, min(a.seg, a.V - first));
    const T* from = static_cast<const T*>(a.logits) + row * a.ld + first;
    grid_dependency_sync();
    for (int i = tid; i < 2 * BINS; i += THREADS) sh.count[0][i] = 0, sh.mass[0][i] = 0;
    // the row's part into shared memory; its first maximum (NaN above all) and its least finite value
    uint32_t most = 0, at = 0xffffffffu, least = 0xffffffffu;
    auto take = [&](float v, int e) {
        v = __fadd_rn(v, 0.0f);  // no -0: it is as good as 0
        vals[e] = v;
        const uint32_t q = key_of(v);
        if (q > most) most = q, at = first + e;
        if (q >= LOWEST && q < least) least = q;
    };
    constexpr int K = 16 / sizeof(T);
    if (a.vec) {
        int e = tid * K;
#pragma unroll 4
        for (; e + K <= n; e += THREADS * K) {
            const Pack<T, K> p = *reinterpret_cast<const Pack<T, K>*>(from + e);
#pragma unroll
            for (int i = 0; i < K; i++) take(to_f(p.v[i]), e + i);
        }
        for (int i = n / K * K + tid; i < n; i += THREADS) take(to_f(from[i]), i);
    } else {
#pragma unroll 4
        for (int e = tid; e < n; e += THREADS) take(to_f(from[e]), e);
    }
    {
        const uint32_t m = __reduce_max_sync(0xffffffffu, most);
        at = __reduce_min_sync(0xffffffffu, most == m ? at : 0xffffffffu);
        least = __reduce_min_sync(0xffffffffu, least);
        if (lane == 0) sh.warp_count[warp] = m, sh.warp_low[warp] = least, sh.edge[0] = 0, sh.warp_mass[warp] = at;
    }
    if (cs > 1)
        cg::this_cluster().sync();  // the others have started
    else
        __syncthreads();
    if (warp == 0) {
        most = lane < WARPS ? sh.warp_count[lane] : 0;
        at = lane < WARPS ? (uint32_t)sh.warp_mass[lane] : 0xffffffffu;
        least = lane < WARPS ? sh.warp_low[lane] : 0xffffffffu;
        const uint32_t m = __reduce_max_sync(0xffffffffu, most);
        at = __reduce_min_sync(0xffffffffu, most == m ? at : 0xffffffffu);
        least = __reduce_min_sync(0xffffffffu, least);
        if (lane < cs) {
            Row& to = cs > 1 ? *cg::this_cluster().map_shared_rank(&sh.row, lane) : sh.row;
            to.most[rank] = m, to.at[rank] = at, to.least[rank] = least;
        }
    }
    if (cs > 1)
        cg::this_cluster().sync();
    else
        __syncthreads();
    most = 0, at = 0xffffffffu, least = 0xffffffffu;
    for (int i = 0; i < cs; i++) {
        const uint32_t m = sh.row.most[i];
        if (m > most) most = m, at = sh.row.at[i];
        if (sh.row.least[i] < least) least = sh.row.least[i];
    }
    const float temperature = a.temperature ? a.temperature[row] : a.temperature1;
    // greedy rows, and those whose maximum leaves no distribution: infinite, NaN, or nothing but -infinity
    if (!(temperature > 0.0f) || most >= INF || most < LOWEST) {
        if (rank == 0 && tid == 0) {
            a.token[row] = at;
            if (a.prob) a.prob[row] = 1.0f;
        }
        return;
    }
    const int k = a.top_k ? a.top_k[row] : a.top_k1;
    const float p = a.top_p ? a.top_p[row] : a.top_p1, min_p = a.min_p ? a.min_p[row] : a.min_p1;
    Chooser<T> c = {a, sh, vals, n, first, rank, cs, 32 - __clz(a.V - 1 | 1)};
    c.kmax = most;
    c.weights.most = (double)value_of(most);
    c.weights.scale = 1.4426950408889634 / (double)temperature;
    c.bins.most = value_of(most);
    // the weights end SCALE powers of 2 below the maximum; the row may end before
    const float range = fminf(__fsub_rn(c.bins.most, value_of(least)), __fmul_rn((SCALE + 2) * 0.6931472f, temperature));
    const float scale = __fdiv_rn((float)BINS, range);
    c.bins.scale = scale < 3.0e38f ? scale : 0.0f;  // rows of one value
    u64 cut = (u64)LOWEST << c.bits;
    if (k > 0 && k < a.V) c.template descend<false>(k, 0.0, cut);
    if (p < 1.0f) c.template descend<true>(0, (double)p, cut);
    if (min_p > 0.0f) {
        if (warp == 0) {
            const double least_power = min_p < 1.0f ? log2((double)min_p) : 0.0;
            const uint32_t q = first_key(LOWEST - 1, most, [&](uint32_t q) { return c.weights.power(value_of(q)) >= least_power; });
            if (lane == 0) sh.floor = (u64)q << c.bits;
        }
        __syncthreads();
        if (sh.floor > cut) cut = sh.floor;
    }
    c.choose(a.u[row], cut, row);
}

// CTAs of a row: as many as its shared memory needs, and more where the rows leave SMs idle, down to 4096 tokens a CTA.
static inline int cluster_of(int rows, int V) {
    int cs = 1;
    while (cs < MAX_CLUSTER && ((int64_t)cs * MAX_SEG < V || ((int64_t)rows * cs * 2 <= 148 * 2 && V > cs * 4096))) cs *= 2;
    return cs;
}

}  // namespace sample
}  // namespace mi

extern "C" int mi_sample_rows(const void* logits, int64_t ld, const float* u, const float* temperature,
                              const int32_t* top_k, const float* top_p, const float* min_p, float temperature1, int top_k1,
                              float top_p1, float min_p1, int64_t* token, float* prob, int rows, int V, int dtype,
                              void* stream) {
    if (!logits || !u || !token || rows < 0 || V <= 0 || ld < 0) return MI_ERR_INVALID;
    if (V > mi::sample::MAX_CLUSTER * mi::sample::MAX_SEG) return MI_ERR_UNSUPPORTED;
    if (rows > 1 << 27) return MI_ERR_UNSUPPORTED;
    mi::sample::Args a = {};
    a.logits = logits, a.ld = ld, a.u = u, a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p;
    a.temperature1 = temperature1, a.top_k1 = top_k1, a.top_p1 = top_p1, a.min_p1 = min_p1;
    a.token = token, a.prob = prob, a.V = V;
    a.cs = mi::sample::cluster_of(rows, V);
    a.seg = mi::cdiv(mi::cdiv(V, a.cs), 8) * 8;
    const size_t smem = sizeof(mi::sample::Shared) + sizeof(float) * a.seg;
    MI_DISPATCH_DTYPE(dtype, T, {
        a.vec = mi::aligned16(logits) && ld % (16 / sizeof(T)) == 0;
        if (rows == 0) return MI_OK;
        static std::atomic<uint64_t> allowed{0};
        auto kernel = mi::sample::sample_kernel<T>;
        if (!mi::allow_smem(kernel, sizeof(mi::sample::Shared) + sizeof(float) * mi::sample::MAX_SEG, allowed)) return MI_ERR_CUDA;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(rows * a.cs);
        cfg.blockDim = dim3(mi::sample::THREADS);
        cfg.dynamicSmemBytes = smem;
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

// recurrence.cu -- the gated linear recurrence of a float layer, its backward
// pass and its form for one new token.
//
//   f' = f + bias;  a = sigmoid(f');  c = 1 - a = sigmoid(-f') (convex) or 1
//   h[t] = a[t] h[t-1] + c[t] x[t],  h[-1] = h0          per channel
//   y[t] = h[t] * z sigmoid(z)  (h[t] without z; 0 from the length on)
//
// and, with g the gradient of h, running backwards:
//   ds = dy z sigmoid(z);  g[t] = ds[t] + G[t+1],  G[t] = a[t] g[t]
//   dx = c g;  df = g (h[t-1] - x) a (1 - a)  (without x where not convex)
//   dz = dy h (z sigmoid(z))';  dh0 = G[0]
//
// A position and channel move 3 elements forward (4 with z) and meet 2 (4)
// special-function results, so HBM bounds it as long as enough loads are in
// flight: the recurrence must not wait for them, nor a long sequence for its
// few channels.
//
// Layout: a CTA has 64 channels, two a lane, and walks the sequence in tiles;
// a warp has SUB neighbouring positions of a tile, which asynchronous copies
// bring into slots of its own one tile ahead.  A stretch of positions acts on
// the state as h -> P h + H; the warps fold theirs through shared memory, once
// a tile, and then run their own positions again from the state they start
// from, with a and c x still in registers.  Where the channels leave SMs idle,
// a cluster of up to 8 CTAs shares the tiles of a round and folds over
// distributed shared memory; nothing is read twice.
//
// Gates never reach 0: e^-|f| is at least 2^-126, so that an infinite state
// stays infinite and an infinite input reaches it, whether or not a stretch is
// folded; and a fold adds to an infinite state, as a P that underflowed to 0
// would make a NaN of it.
#include <cooperative_groups.h>

#include "mi_elem.cuh"

namespace mi {
namespace rec {

constexpr int WARPS = 8, THREADS = WARPS * 32, CB = 64;  // channels a CTA
constexpr int CK = 8;          // positions between the states kept for the backward pass
constexpr int MAX_CLUSTER = 8;
constexpr int STAGES = 2;

struct Seq {  // a [batch, L, D] operand with unit last stride
    const void* p;
    int64_t sb, sl;
};

struct Args {
    Seq x, f, z, dy;
    const float* bias;   // [D] or NULL
    const float* h0;     // [batch, D] or NULL
    const float* dhT;    // gradient of the final state or NULL
    const int* lengths;  // [batch] or NULL
    void* y;             // [batch, L, D]
    float* hT;           // [batch, D] or NULL
    float* ckpt;         // [batch, cdiv(L, CK), D] or NULL
    void *dx, *df, *dz;
    float* dh0;          // [batch, D] or NULL
    float* part;         // [batch * cluster, D]: the CTAs' sums of df, or NULL
    int batch, L, D;
    int vec;             // inputs' rows start on 16 bytes
    int ovec;            // outputs' rows start on a lane's two elements' alignment
    int cs;              // CTAs of a cluster
};

__device__ __forceinline__ int length_of(const Args& a, int b) {
    if (!a.lengths) return a.L;
    const int n = a.lengths[b];
    return n < 0 ? 0 : (n < a.L ? n : a.L);
}

// sigmoid(v) and sigmoid(-v), neither taken from 1 minus the other.  e^-|v| to
// 2 ulp and the argument's rounding, |v| 2^-24 of it, are far below half a step
// of 16 bits; fp32 values take expf and a Newton step for the reciprocal.
template <typename T>
__device__ __forceinline__ void sigmoids(float v, float& up, float& down) {
    float e, r;
    if constexpr (sizeof(T) == 4) {
        e = max_nan(expf(-fabsf(v)), 1.17549435e-38f);
        const float d = __fadd_rn(1.0f, e);
        r = rcp_fast(d);
        r = __fmaf_rn(r, __fmaf_rn(-d, r, 1.0f), r);
    } else {
        e = max_nan(exp2_fast(__fmul_rn(fabsf(v), -LOG2E)), 1.17549435e-38f);
        r = rcp_fast(__fadd_rn(1.0f, e));
    }
    const float s = __fmul_rn(e, r);
    up = v < 0.0f ? s : r;
    down = v < 0.0f ? r : s;
}

// z sigmoid(z) and, from the same sigmoid, its derivative
template <typename T>
__device__ __forceinline__ float silu(float z, float& slope) {
    float s, n;
    sigmoids<T>(z, s, n);
    slope = __fmaf_rn(__fmul_rn(z, s), n, s);
    return __fmul_rn(z, s);
}
template <typename T>
__device__ __forceinline__ float silu(float z) {
    if constexpr (sizeof(T) == 4) {
        float s;
        return silu<T>(z, s);
    } else {
        return __fmul_rn(z, sigmoid(z));
    }
}

template <typename T>
__device__ __forceinline__ float2 pair(const T* p) {
    const Pack<T, 2> v = *reinterpret_cast<const Pack<T, 2>*>(p);
    return make_float2(to_f(v.v[0]), to_f(v.v[1]));
}
template <typename T>
__device__ __forceinline__ void put(T* p, float2 v, int valid, bool vec) {
    const float o[2] = {v.x, v.y};
    store_pack<2>(p, o, valid, vec);
}
__device__ __forceinline__ float2 load2(const float* p, int valid) {
    return make_float2(valid > 0 ? p[0] : 0.0f, valid > 1 ? p[1] : 0.0f);
}
__device__ __forceinline__ void store2(float* p, float2 v, int valid) {
    if (valid > 0) p[0] = v.x;
    if (valid > 1) p[1] = v.y;
}

// what a stretch of positions does to the state of two channels: s -> p s + q
struct Fold {
    float2 p, q;
};
__device__ __forceinline__ float fold1(float s, float p, float q) {
    return fabsf(s) == __int_as_float(0x7f800000) ? __fadd_rn(s, q) : __fmaf_rn(p, s, q);
}
__device__ __forceinline__ float2 fold(float2 s, const Fold& f) {
    return make_float2(fold1(s.x, f.p.x, f.q.x), fold1(s.y, f.p.y, f.q.y));
}
__device__ __forceinline__ Fold join(const Fold& a, const Fold& b) {  // a, then b
    return {__fmul2_rn(a.p, b.p), make_float2(fold1(a.q.x, b.p.x, b.q.x), fold1(a.q.y, b.p.y, b.q.y))};
}

// A warp's rows of one operand in shared memory, SUB rows of CB channels.
template <typename T, int SUB>
struct Rows {
    alignas(16) T v[SUB][CB];
};

// Starts the copies of the operand's rows t0 .. t0 + SUB - 1 of sequence b,
// channels c0 on, into this warp's slot; rows from `end` on and channels from D
// on become zeros.
template <typename T, int SUB>
__device__ __forceinline__ void fetch_rows(Rows<T, SUB>& to, const Seq& s, int b, int t0, int end, int c0, int D, int vec) {
    constexpr int K = 16 / sizeof(T), PER = CB / K;
    const int lane = threadIdx.x & 31;
    const T* base = static_cast<const T*>(s.p) + (int64_t)b * s.sb + c0;
    if (vec) {
#pragma unroll
        for (int i = 0; i < SUB * PER / 32; i++) {
            const int at = i * 32 + lane, row = at / PER, col = at % PER * K;
            const int valid = t0 + row < end ? D - c0 - col : 0;
            fetch_pack<K>(&to.v[row][col], base + (int64_t)(t0 + row) * s.sl + col, s.p, valid, true);
        }
    } else {
#pragma unroll 4
        for (int row = 0; row < SUB; row++) {
            const T* p = base + (int64_t)(t0 + row) * s.sl;
#pragma unroll
            for (int col = 0; col < CB; col += 32)
                to.v[row][col + lane] = t0 + row < end && c0 + col + lane < D ? p[col + lane] : from_f<T>(0.0f);
        }
    }
}

// The folds of a round, in order: `mine` is this warp's, `s` the state that the
// round starts from.  Returns the state that this warp starts from; s becomes
// the state after the round.  Rounds alternate between two sets of slots, so one
// barrier a round is enough.
struct Exchange {
    Fold warp[2][WARPS][32];
    Fold cta[2][MAX_CLUSTER][32];
};
template <bool CLUSTER>
__device__ __forceinline__ float2 exchange(Exchange& ex, int round, int cs, const Fold& mine, float2& s) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, k = round & 1;
    ex.warp[k][warp][lane] = mine;
    __syncthreads();
    float2 from = s;
    if constexpr (!CLUSTER) {
#pragma unroll
        for (int i = 0; i < WARPS; i++) {
            if (i == warp) from = s;
            s = fold(s, ex.warp[k][i][lane]);
        }
    } else {
        namespace cg = cooperative_groups;
        cg::cluster_group cluster = cg::this_cluster();
        const int rank = cluster.block_rank();
        if (warp < cs) {  // warp i tells CTA i
            Fold all = ex.warp[k][0][lane];
#pragma unroll
            for (int i = 1; i < WARPS; i++) all = join(all, ex.warp[k][i][lane]);
            *cluster.map_shared_rank(&ex.cta[k][rank][lane], warp) = all;
        }
        cluster.sync();
        for (int i = 0; i < cs; i++) {
            if (i == rank) from = s;
            s = fold(s, ex.cta[k][i][lane]);
        }
        for (int i = 0; i < warp; i++) from = fold(from, ex.warp[k][i][lane]);
    }
    return from;
}

template <typename T>
constexpr int SUB_FWD = 32 / sizeof(T);  // 16 positions of 16 bits, 8 of fp32: slots of 2 KB

template <typename T, bool GATE>
struct FwdSlots {
    Rows<T, SUB_FWD<T>> x[STAGES][WARPS], f[STAGES][WARPS], z[GATE ? STAGES : 1][GATE ? WARPS : 1];
};

template <typename T, bool CONVEX, bool GATE, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, 2) fwd_kernel(const Args a) {
    constexpr int SUB = SUB_FWD<T>, TT = SUB * WARPS;
    extern __shared__ __align__(16) unsigned char smem[];
    FwdSlots<T, GATE>& slots = *reinterpret_cast<FwdSlots<T, GATE>*>(smem);
    Exchange& ex = *reinterpret_cast<Exchange*>(smem + sizeof(FwdSlots<T, GATE>));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cs = CLUSTER ? a.cs : 1;
    const int b = blockIdx.y, c0 = blockIdx.x / cs * CB, rank = blockIdx.x % cs;
    const int c = c0 + 2 * lane, valid = a.D - c;
    grid_dependency_sync();
    const int len = length_of(a, b);
    const int rounds = cdiv(len, TT * cs);
    const float2 bias = a.bias ? load2(a.bias + c, valid) : make_float2(0.0f, 0.0f);
    float2 s = a.h0 ? load2(a.h0 + (int64_t)b * a.D + c, valid) : make_float2(0.0f, 0.0f);
    auto start = [&](int round) { return (round * cs + rank) * TT + warp * SUB; };
    auto fetch = [&](int round) {
        if (round < rounds) {
            const int t0 = start(round), k = round % STAGES;
            fetch_rows<T, SUB>(slots.x[k][warp], a.x, b, t0, len, c0, a.D, a.vec);
            fetch_rows<T, SUB>(slots.f[k][warp], a.f, b, t0, len, c0, a.D, a.vec);
            if (GATE) fetch_rows<T, SUB>(slots.z[k][warp], a.z, b, t0, len, c0, a.D, a.vec);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES; i++) fetch(i);
    if (CLUSTER) cooperative_groups::this_cluster().sync();  // the other CTAs' shared memory is there from here on
    for (int round = 0; round < rounds; round++) {
        const int t0 = start(round), k = round % STAGES;
        const int n = len - t0;  // positions of this stretch that exist
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        float2 av[SUB], uv[SUB];
#pragma unroll
        for (int i = 0; i < SUB; i++) {
            const float2 f = __fadd2_rn(pair(&slots.f[k][warp].v[i][2 * lane]), bias);
            const float2 x = pair(&slots.x[k][warp].v[i][2 * lane]);
            float2 w;
            sigmoids<T>(f.x, av[i].x, w.x);
            sigmoids<T>(f.y, av[i].y, w.y);
            uv[i] = CONVEX ? __fmul2_rn(w, x) : x;
        }
        if (n < SUB) {
#pragma unroll
            for (int i = 0; i < SUB; i++)
                if (i >= n) av[i] = make_float2(1.0f, 1.0f), uv[i] = make_float2(0.0f, 0.0f);
        }
        Fold mine = {av[0], uv[0]};
#pragma unroll
        for (int i = 1; i < SUB; i++) {
            mine.p = __fmul2_rn(mine.p, av[i]);
            mine.q = __ffma2_rn(av[i], mine.q, uv[i]);
        }
        float2 h = exchange<CLUSTER>(ex, round, cs, mine, s);
        if (n > 0) {
            T* y = static_cast<T*>(a.y) + ((int64_t)b * a.L + t0) * a.D + c;
            float* ck = a.ckpt ? a.ckpt + ((int64_t)b * cdiv(a.L, CK) + t0 / CK) * a.D + c : nullptr;
#pragma unroll
            for (int i = 0; i < SUB; i++) {
                if (i % CK == 0 && ck && i < n) put(ck + (int64_t)(i / CK) * a.D, h, valid, a.D % 2 == 0);
                h = __ffma2_rn(av[i], h, uv[i]);
                float2 o = h;
                if (GATE) {
                    const float2 z = pair(&slots.z[k][warp].v[i][2 * lane]);
                    o = __fmul2_rn(o, make_float2(silu<T>(z.x), silu<T>(z.y)));
                }
                if (i < n) put(y + (int64_t)i * a.D, o, valid, a.ovec);
            }
        }
        __syncwarp();
        fetch(round + STAGES);
    }
    cp_async_wait();
    if (a.hT && rank == 0 && warp == 0) store2(a.hT + (int64_t)b * a.D + c, s, valid);
    for (int t = len + rank * WARPS + warp; t < a.L; t += cs * WARPS)
        put(static_cast<T*>(a.y) + ((int64_t)b * a.L + t) * a.D + c, make_float2(0.0f, 0.0f), valid, a.ovec);
}

template <typename T, bool GATE>
struct BwdSlots {
    Rows<T, CK> x[STAGES][WARPS], f[STAGES][WARPS], dy[STAGES][WARPS], z[GATE ? STAGES : 1][GATE ? WARPS : 1];
};

// The tiles in reverse: warp 0 of CTA 0 has a round's last positions.  A stretch
// is as long as the distance between the kept states, so each warp has its own.
template <typename T, bool CONVEX, bool GATE, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, 2) bwd_kernel(const Args a) {
    constexpr int SUB = CK, TT = SUB * WARPS;
    extern __shared__ __align__(16) unsigned char smem[];
    BwdSlots<T, GATE>& slots = *reinterpret_cast<BwdSlots<T, GATE>*>(smem);
    Exchange& ex = *reinterpret_cast<Exchange*>(smem + sizeof(BwdSlots<T, GATE>));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cs = CLUSTER ? a.cs : 1;
    const int b = blockIdx.y, c0 = blockIdx.x / cs * CB, rank = blockIdx.x % cs;
    const int c = c0 + 2 * lane, valid = a.D - c;
    const int len = length_of(a, b);
    const int stretches = cdiv(len, SUB), rounds = cdiv(stretches, WARPS * cs);
    const float2 bias = a.bias ? load2(a.bias + c, valid) : make_float2(0.0f, 0.0f);
    float2 s = a.dhT ? load2(a.dhT + (int64_t)b * a.D + c, valid) : make_float2(0.0f, 0.0f);
    float2 dbias = make_float2(0.0f, 0.0f), next_h = make_float2(0.0f, 0.0f);
    auto stretch = [&](int round) { return stretches - 1 - ((round * cs + rank) * WARPS + warp); };  // < 0: none
    auto fetch = [&](int round) {
        const int j = round < rounds ? stretch(round) : -1;
        if (j >= 0) {
            const int t0 = j * SUB, k = round % STAGES;
            fetch_rows<T, SUB>(slots.x[k][warp], a.x, b, t0, len, c0, a.D, a.vec);
            fetch_rows<T, SUB>(slots.f[k][warp], a.f, b, t0, len, c0, a.D, a.vec);
            fetch_rows<T, SUB>(slots.dy[k][warp], a.dy, b, t0, len, c0, a.D, a.vec);
            if (GATE) fetch_rows<T, SUB>(slots.z[k][warp], a.z, b, t0, len, c0, a.D, a.vec);
        }
        cp_async_commit();
    };
    auto fetch_h = [&](int round) {
        const int j = round < rounds ? stretch(round) : -1;
        if (j >= 0) next_h = load2(a.ckpt + ((int64_t)b * cdiv(a.L, CK) + j) * a.D + c, valid);
    };
#pragma unroll
    for (int i = 0; i < STAGES; i++) fetch(i);
    fetch_h(0);
    if (CLUSTER) cooperative_groups::this_cluster().sync();
    for (int round = 0; round < rounds; round++) {
        const int j = stretch(round), t0 = j * SUB, k = round % STAGES;
        const int n = j >= 0 ? len - t0 : 0;
        const int64_t at = ((int64_t)b * a.L + t0) * a.D + c;
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        float2 av[SUB], wv[SUB], hv[SUB], dv[SUB];  // a, 1 - a, h[t-1], ds
        Fold mine = {make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
        if (j >= 0) {
            float2 h = next_h;
            fetch_h(round + 1);
#pragma unroll
            for (int i = 0; i < SUB; i++) {
                const float2 f = __fadd2_rn(pair(&slots.f[k][warp].v[i][2 * lane]), bias);
                const float2 x = pair(&slots.x[k][warp].v[i][2 * lane]);
                dv[i] = pair(&slots.dy[k][warp].v[i][2 * lane]);
                sigmoids<T>(f.x, av[i].x, wv[i].x);
                sigmoids<T>(f.y, av[i].y, wv[i].y);
                hv[i] = h;
                h = __ffma2_rn(av[i], h, CONVEX ? __fmul2_rn(wv[i], x) : x);
                if (GATE) {
                    const float2 z = pair(&slots.z[k][warp].v[i][2 * lane]);
                    float2 gate, slope;
                    gate.x = silu<T>(z.x, slope.x);
                    gate.y = silu<T>(z.y, slope.y);
                    if (i < n)
                        put(static_cast<T*>(a.dz) + at + (int64_t)i * a.D, __fmul2_rn(__fmul2_rn(dv[i], h), slope), valid,
                            a.ovec);
                    dv[i] = __fmul2_rn(dv[i], gate);
                }
            }
            if (n < SUB) {
#pragma unroll
                for (int i = 0; i < SUB; i++)
                    if (i >= n) av[i] = make_float2(1.0f, 1.0f), dv[i] = make_float2(0.0f, 0.0f);
            }
            mine = {av[SUB - 1], __fmul2_rn(av[SUB - 1], dv[SUB - 1])};
#pragma unroll
            for (int i = SUB - 2; i >= 0; i--) {
                mine.p = __fmul2_rn(mine.p, av[i]);
                mine.q = __fmul2_rn(av[i], __fadd2_rn(dv[i], mine.q));
            }
        }
        float2 G = exchange<CLUSTER>(ex, round, cs, mine, s);
        if (j >= 0) {
#pragma unroll
            for (int i = SUB - 1; i >= 0; i--) {
                const float2 g = __fadd2_rn(dv[i], G);
                G = __fmul2_rn(av[i], g);
                if (i < n) {
                    float2 d = hv[i];
                    if (CONVEX) {
                        const float2 x = pair(&slots.x[k][warp].v[i][2 * lane]);
                        d = make_float2(__fsub_rn(d.x, x.x), __fsub_rn(d.y, x.y));
                    }
                    const float2 df = __fmul2_rn(__fmul2_rn(G, wv[i]), d);
                    dbias = make_float2(__fadd_rn(dbias.x, df.x), __fadd_rn(dbias.y, df.y));
                    put(static_cast<T*>(a.df) + at + (int64_t)i * a.D, df, valid, a.ovec);
                    put(static_cast<T*>(a.dx) + at + (int64_t)i * a.D, CONVEX ? __fmul2_rn(wv[i], g) : g, valid, a.ovec);
                }
            }
        }
        __syncwarp();
        fetch(round + STAGES);
    }
    cp_async_wait();
    if (a.dh0 && rank == 0 && warp == 0) store2(a.dh0 + (int64_t)b * a.D + c, s, valid);
    for (int t = len + rank * WARPS + warp; t < a.L; t += cs * WARPS) {
        const int64_t at = ((int64_t)b * a.L + t) * a.D + c;
        const float2 zero = make_float2(0.0f, 0.0f);
        put(static_cast<T*>(a.dx) + at, zero, valid, a.ovec);
        put(static_cast<T*>(a.df) + at, zero, valid, a.ovec);
        if (GATE) put(static_cast<T*>(a.dz) + at, zero, valid, a.ovec);
    }
    if (!a.part) return;
    float2* sums = reinterpret_cast<float2*>(smem);  // [WARPS][32], in the place of the slots
    __syncthreads();
    sums[threadIdx.x] = dbias;
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (int i = 1; i < WARPS; i++) dbias = __fadd2_rn(dbias, sums[i * 32 + lane]);
        store2(a.part + ((int64_t)b * cs + rank) * a.D + c, dbias, valid);
    }
}

// One position: 4 channels a thread.
template <typename T, bool CONVEX, bool GATE>
__global__ void __launch_bounds__(128) step_kernel(const T* __restrict__ x, int64_t sx, const T* __restrict__ f, int64_t sf,
                                                   const T* __restrict__ z, int64_t sz, const float* __restrict__ bias,
                                                   float* __restrict__ h, T* __restrict__ y, int D, int vec) {
    const int c = (blockIdx.x * 128 + threadIdx.x) * 4;
    const int64_t b = blockIdx.y;
    grid_dependency_sync();
    if (c >= D) return;
    const int valid = D - c;
    float* ph = h + b * D + c;
    const Pack<T, 4> px = load_pack<4>(x + b * sx + c, valid, vec), pf = load_pack<4>(f + b * sf + c, valid, vec);
    Pack<T, 4> pz;
    if (GATE) pz = load_pack<4>(z + b * sz + c, valid, vec);
    const Pack<float, 4> hp = load_pack<4>(ph, valid, vec);
    Pack<float, 4> pb = {};
    if (bias) pb = load_pack<4>(bias + c, valid, vec);
    float hn[4], o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float up, down;
        sigmoids<T>(__fadd_rn(to_f(pf.v[i]), pb.v[i]), up, down);
        hn[i] = __fmaf_rn(up, hp.v[i], CONVEX ? __fmul_rn(down, to_f(px.v[i])) : to_f(px.v[i]));
        o[i] = GATE ? __fmul_rn(hn[i], silu<T>(to_f(pz.v[i]))) : hn[i];
    }
    store_pack<4>(ph, hn, valid, vec);
    store_pack<4>(y + b * D + c, o, valid, vec);
}

// CTAs of a cluster: as many as it takes to give every SM two CTAs, and no more
// than the sequence has tiles.
static inline int cluster_of(int batch, int L, int D, int tile) {
    int cs = 1;
    while (cs < MAX_CLUSTER && (int64_t)batch * cdiv(D, CB) * cs < 148 * 2 && cs * tile < L) cs *= 2;
    return cs;
}

template <typename T, bool CONVEX, bool GATE, bool CLUSTER, bool BWD>
static int launch(const Args& a, cudaStream_t s) {
    constexpr size_t smem = (BWD ? sizeof(BwdSlots<T, GATE>) : sizeof(FwdSlots<T, GATE>)) + sizeof(Exchange);
    static std::atomic<uint64_t> allowed{0};
    void (*kernel)(const Args);
    if constexpr (BWD)
        kernel = bwd_kernel<T, CONVEX, GATE, CLUSTER>;
    else
        kernel = fwd_kernel<T, CONVEX, GATE, CLUSTER>;
    if (!allow_smem(kernel, smem, allowed)) return MI_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cdiv(a.D, CB) * a.cs, a.batch);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (CLUSTER) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = a.cs;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        n++;
    }
    if (!BWD && pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        n++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
        cudaGetLastError();
        return MI_ERR_CUDA;
    }
    return MI_OK;
}

template <typename T, bool BWD>
static int dispatch(const Args& a, bool convex, cudaStream_t s) {
#define MI_REC(CONVEX, GATE) \
    return a.cs > 1 ? launch<T, CONVEX, GATE, true, BWD>(a, s) : launch<T, CONVEX, GATE, false, BWD>(a, s)
    if (convex) {
        if (a.z.p) MI_REC(true, true);
        MI_REC(true, false);
    }
    if (a.z.p) MI_REC(false, true);
    MI_REC(false, false);
#undef MI_REC
}

static inline int elem_size(int dtype) { return dtype == MI_DT_F32 ? 4 : 2; }
static inline bool rows_vec(const Seq& s, int dtype) {
    const int k = 16 / elem_size(dtype);
    return !s.p || (s.sb % k == 0 && s.sl % k == 0 && aligned16(s.p));
}

}  // namespace rec
}  // namespace mi

static int mi_rec_check(const mi::rec::Seq& x, const mi::rec::Seq& f, const mi::rec::Seq& z, int batch, int L, int D,
                        int dtype) {
    if (!x.p || !f.p || batch < 0 || L <= 0 || D <= 0 || dtype < 0 || dtype > 2) return MI_ERR_INVALID;
    for (const mi::rec::Seq* s : {&x, &f, &z})
        if (s->p && (s->sb < 0 || s->sl < 0)) return MI_ERR_INVALID;
    if (batch > 65535 || L > 1 << 30 || D > 1 << 24) return MI_ERR_UNSUPPORTED;
    return MI_OK;
}

extern "C" int64_t mi_gated_recurrence_checkpoints(int batch, int L, int D) {
    if (batch <= 0 || L <= 0 || D <= 0) return 0;
    return (int64_t)batch * mi::cdiv(L, mi::rec::CK) * D;
}

extern "C" int mi_gated_recurrence(const void* x, int64_t x_batch, int64_t x_row, const void* f, int64_t f_batch,
                                   int64_t f_row, const void* z, int64_t z_batch, int64_t z_row, const float* bias,
                                   const float* h0, const int32_t* lengths, void* y, float* h_out, float* checkpoints,
                                   int batch, int L, int D, int convex, int dtype, void* stream) {
    mi::rec::Args a = {};
    a.x = {x, x_batch, x_row}, a.f = {f, f_batch, f_row}, a.z = {z, z_batch, z_row};
    const int rc = mi_rec_check(a.x, a.f, a.z, batch, L, D, dtype);
    if (rc != MI_OK) return rc;
    if (!y) return MI_ERR_INVALID;
    if (batch == 0) return MI_OK;
    a.bias = bias, a.h0 = h0, a.lengths = lengths, a.y = y, a.hT = h_out, a.ckpt = checkpoints;
    a.batch = batch, a.L = L, a.D = D;
    const int e = mi::rec::elem_size(dtype);
    a.ovec = D % 2 == 0 && reinterpret_cast<uintptr_t>(y) % (2 * e) == 0;
    a.vec = D % (16 / e) == 0 && mi::rec::rows_vec(a.x, dtype) && mi::rec::rows_vec(a.f, dtype) &&
            mi::rec::rows_vec(a.z, dtype);
    MI_DISPATCH_DTYPE(dtype, T, {
        a.cs = mi::rec::cluster_of(batch, L, D, mi::rec::SUB_FWD<T> * mi::rec::WARPS);
        return (mi::rec::dispatch<T, false>(a, convex, (cudaStream_t)stream));
    });
}

extern "C" int64_t mi_gated_recurrence_backward_workspace(int batch, int L, int D) {
    if (batch <= 0 || L <= 0 || D <= 0) return 0;
    return (int64_t)sizeof(float) * batch * D * mi::rec::cluster_of(batch, L, D, mi::rec::CK * mi::rec::WARPS);
}

extern "C" int mi_gated_recurrence_backward(const void* dy, int64_t dy_batch, int64_t dy_row, const float* dh_out,
                                            const void* x, int64_t x_batch, int64_t x_row, const void* f, int64_t f_batch,
                                            int64_t f_row, const void* z, int64_t z_batch, int64_t z_row, const float* bias,
                                            const int32_t* lengths, const float* checkpoints, void* dx, void* df, void* dz,
                                            float* dbias, float* dh0, void* workspace, int batch, int L, int D, int convex,
                                            int dtype, void* stream) {
    mi::rec::Args a = {};
    a.x = {x, x_batch, x_row}, a.f = {f, f_batch, f_row}, a.z = {z, z_batch, z_row}, a.dy = {dy, dy_batch, dy_row};
    const int rc = mi_rec_check(a.x, a.f, a.z, batch, L, D, dtype);
    if (rc != MI_OK) return rc;
    if (!dy || dy_batch < 0 || dy_row < 0 || !checkpoints || !dx || !df || (z && !dz) || (dbias && !workspace))
        return MI_ERR_INVALID;
    cudaStream_t s = (cudaStream_t)stream;
    if (batch == 0) {
        if (dbias && cudaMemsetAsync(dbias, 0, sizeof(float) * D, s) != cudaSuccess) return MI_ERR_CUDA;
        return MI_OK;
    }
    a.bias = bias, a.dhT = dh_out, a.lengths = lengths, a.ckpt = const_cast<float*>(checkpoints);
    a.dx = dx, a.df = df, a.dz = dz, a.dh0 = dh0, a.part = dbias ? static_cast<float*>(workspace) : nullptr;
    a.batch = batch, a.L = L, a.D = D;
    const int e = mi::rec::elem_size(dtype);
    a.ovec = D % 2 == 0;
    for (const void* p : {dx, df, z ? dz : nullptr}) a.ovec = a.ovec && reinterpret_cast<uintptr_t>(p) % (2 * e) == 0;
    a.vec = D % (16 / e) == 0 && mi::rec::rows_vec(a.x, dtype) && mi::rec::rows_vec(a.f, dtype) &&
            mi::rec::rows_vec(a.z, dtype) && mi::rec::rows_vec(a.dy, dtype);
    a.cs = mi::rec::cluster_of(batch, L, D, mi::rec::CK * mi::rec::WARPS);
    int rc2 = MI_ERR_INVALID;
    MI_DISPATCH_DTYPE(dtype, T, (rc2 = mi::rec::dispatch<T, true>(a, convex, s)););
    if (rc2 != MI_OK || !dbias) return rc2;
    mi::column_sum_kernel<<<mi::cdiv(D, 32), 1024, 0, s>>>(a.part, dbias, batch * a.cs, D);
    MI_CHECK_LAUNCH();
    return MI_OK;
}

extern "C" int mi_gated_recurrence_step(const void* x, int64_t x_batch, const void* f, int64_t f_batch, const void* z,
                                        int64_t z_batch, const float* bias, float* h, void* y, int batch, int D,
                                        int convex, int dtype, void* stream) {
    const mi::rec::Seq sx = {x, x_batch, 0}, sf = {f, f_batch, 0}, sz = {z, z_batch, 0};
    const int rc = mi_rec_check(sx, sf, sz, batch, 1, D, dtype);
    if (rc != MI_OK) return rc;
    if (!h || !y) return MI_ERR_INVALID;
    if (batch == 0) return MI_OK;
    const int e = mi::rec::elem_size(dtype);
    int vec = D % 4 == 0 && mi::aligned16(h) && (!bias || mi::aligned16(bias)) && reinterpret_cast<uintptr_t>(y) % (4 * e) == 0;
    for (const mi::rec::Seq* q : {&sx, &sf, &sz})
        vec = vec && (!q->p || (q->sb % 4 == 0 && reinterpret_cast<uintptr_t>(q->p) % (4 * e) == 0));
    const dim3 grid(mi::cdiv(mi::cdiv(D, 4), 128), batch);
#define MI_REC_STEP(CONVEX, GATE)                                                                                          \
    MI_LAUNCH_DEPENDENT(mi::rec::step_kernel<T, CONVEX, GATE>, grid, 128, 0, (cudaStream_t)stream,                         \
                        static_cast<const T*>(x), x_batch, static_cast<const T*>(f), f_batch, static_cast<const T*>(z),     \
                        z_batch, bias, h, static_cast<T*>(y), D, vec)
    MI_DISPATCH_DTYPE(dtype, T, {
        if (convex && z)
            MI_REC_STEP(true, true);
        else if (convex)
            MI_REC_STEP(true, false);
        else if (z)
            MI_REC_STEP(false, true);
        else
            MI_REC_STEP(false, false);
    });
#undef MI_REC_STEP
    return MI_OK;
}

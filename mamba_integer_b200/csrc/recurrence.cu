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
// flight and the instructions are few (33 a channel and position with z, of
// which 4 are special functions; 57 backward).  32 x 512 x 1536 bf16 with z: forward 47 us
// (201 MB, 4.3 TB/s), 36 without the arithmetic; backward 82 (352 MB, 4.3 TB/s),
// 78 without: what is left is two CTAs of 128 registers a thread an SM, whose
// warps load, wait for the fold and store by turns.
//
// Layout: a CTA has 64 channels, two a lane in f32x2 arithmetic, and walks the
// sequence in tiles; a warp has SUB neighbouring positions of a tile, whose rows
// asynchronous copies bring into slots of its own one tile ahead.  A stretch of
// positions acts on the state as h -> P h + H; the warps fold theirs through
// shared memory, once a tile, and then run their own positions again from the
// state they start from, with a and c x still in registers.  Where the channels
// leave SMs idle, a cluster of up to 16 CTAs shares the tiles of a round: each
// sends its fold to the others' shared memory, counted by their mbarriers;
// nothing is read twice.  Long sequences of few channels are cut into chunks,
// whose folds a pass in front takes.
//
// Gates and folds never reach 0: gate logits count as at least -87, and a stretch's
// P is at least 2^-126, so that an infinite state stays infinite, whether or not a
// stretch is folded.  (A state of 1e38 leaves up to 1 of itself behind a stretch that
// forgets it.)  An input's weight does reach 0, where it would be below 2^-126: what a
// gate keeps out counts for nothing, the type's lowest value included.
#include <type_traits>

#include "mi_elem.cuh"
#include "mi_folds.cuh"

namespace mi {
namespace rec {

constexpr int CB = 64;         // channels a CTA
constexpr int CK = 8;          // positions between the states kept for the backward pass

struct Seq {  // a [batch, L, D] operand with unit last stride
    const void* p;
    int64_t sb, sl;
};

enum { X, F, Z, DY };  // operands that are read by rows

struct Args {
    Seq in[4];
    const float* bias;   // [D] or NULL
    const float* h0;     // [batch, D] or NULL
    const float* dhT;    // gradient of the final state or NULL
    const int* lengths;  // [batch] or NULL
    void* y;             // [batch, L, D]
    float* hT;           // [batch, D] or NULL
    float* ckpt;         // [batch, cdiv(L, CK), D] or NULL
    void *dx, *df, *dz;
    float* dh0;          // [batch, D] or NULL
    float* part;         // [batch * chunks * cluster, D]: the CTAs' sums of df, or NULL
    float* folds;        // with chunks > 1: [batch, chunks, 2, D], what each chunk does to the state
    int batch, L, D;
    int ovec;            // outputs' rows start on a lane's two elements' alignment
    int cs;              // CTAs of a cluster
    int chunks, span;    // chunks of a sequence, positions of a chunk
};

__device__ __forceinline__ int length_of(const Args& a, int b) {
    if (!a.lengths) return a.L;
    const int n = a.lengths[b];
    return n < 0 ? 0 : (n < a.L ? n : a.L);
}

// sigmoid(v), at least e^-87, and sigmoid(-v), 0 from v = 87.4 on, neither taken from
// 1 minus the other (a NaN stays one).  The product with log2(e) is
// carried on in two parts, which keeps the power to 2 ulp where |v| is large, and
// a Newton step makes the reciprocal right to its last bit: where a is near 1, a
// state has its error as often as its memory is long.
__device__ __forceinline__ void sigmoids(float2 v, float2& up, float2& down) {
    v.x = max_nan(min_nan(v.x, 127.0f), -87.0f);
    v.y = max_nan(min_nan(v.y, 127.0f), -87.0f);
    const float2 t = __fmul2_rn(v, dup(-LOG2E));
    const float2 r = __ffma2_rn(v, dup(1.92596299e-8f), __ffma2_rn(v, dup(LOG2E), t));  // t is too large by this
    float2 e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
    e = __ffma2_rn(__fmul2_rn(e, dup(-LN2)), r, e);
    const float2 d = __ffma2_rn(e, dup(-1.0f), dup(-1.0f));  // -(1 + e)
    const float2 q = make_float2(rcp_fast(-d.x), rcp_fast(-d.y));
    up = __ffma2_rn(q, __ffma2_rn(d, q, dup(1.0f)), q);
    down = __fmul2_rn(e, up);
}

// z sigmoid(z), and its derivative.  Unlike a state's gate an output gate reaches 0:
// a sigmoid below e^-87 counts as 0 (2^-126 in 16 bits), so that at the types' lowest
// values both are 0 and not the smallest gate times z.  In 16 bits without
// sigmoids()' care: |z| 2^-24 of the power is far below half a step.  Sigmoids that
// fall on below e^-87 in fp32 cost 3 us of 78 (forward, 8 x 2048 x 1536).
template <typename T>
__device__ __forceinline__ float2 silu(float2 z, float2& slope) {
    float2 s, n;
    if constexpr (sizeof(T) == 4) {
        sigmoids(z, s, n);
        s = make_float2(z.x < -87.0f ? 0.0f : s.x, z.y < -87.0f ? 0.0f : s.y);
    } else {
        const float2 t = __fmul2_rn(z, dup(-LOG2E));
        const float2 e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
        const float2 d = __fadd2_rn(e, dup(1.0f));
        s = make_float2(rcp_fast(d.x), rcp_fast(d.y));
        // where s is 0, so that infinity times it is not a NaN
        n = __fmul2_rn(make_float2(min_nan(e.x, 8.5070592e37f), min_nan(e.y, 8.5070592e37f)), s);  // 2^126
    }
    const float2 zs = __fmul2_rn(z, s);
    slope = __ffma2_rn(zs, n, s);
    return zs;
}
template <typename T>
__device__ __forceinline__ float2 silu(float2 z) {
    if constexpr (sizeof(T) == 4) {
        float2 s, n;
        sigmoids(z, s, n);
        return __fmul2_rn(z, make_float2(z.x < -87.0f ? 0.0f : s.x, z.y < -87.0f ? 0.0f : s.y));
    } else {
        const float2 t = __fmul2_rn(z, dup(-LOG2E));
        const float2 d = __fadd2_rn(make_float2(exp2_fast(t.x), exp2_fast(t.y)), dup(1.0f));
        return __fmul2_rn(z, make_float2(rcp_fast(d.x), rcp_fast(d.y)));
    }
}

__device__ __forceinline__ float2 load2(const float* p, int valid) {
    return make_float2(valid > 0 ? p[0] : 0.0f, valid > 1 ? p[1] : 0.0f);
}
__device__ __forceinline__ void store2(float* p, float2 v, int valid) {
    if (valid > 0) p[0] = v.x;
    if (valid > 1) p[1] = v.y;
}
// FAST: both exist, aligned
template <bool FAST, typename T>
__device__ __forceinline__ void put(T* p, float2 v, int valid, bool vec) {
    if (FAST) {
        Pack<T, 2> o;
        o.v[0] = from_f<T>(v.x), o.v[1] = from_f<T>(v.y);
        *reinterpret_cast<Pack<T, 2>*>(p) = o;
    } else {
        const float o[2] = {v.x, v.y};
        store_pack<2>(p, o, valid, vec);
    }
}

// ---------------------------------------------------------------------------
// rows of the operands in shared memory
// ---------------------------------------------------------------------------
// A warp's rows of N operands: SUB rows of CB channels each.  Where rows start
// off 16 bytes (not VEC), the 16-byte blocks that hold a row's channels are
// copied whole, and the row starts inside the first one.
template <typename T, int N, int SUB, bool VEC>
struct Rows {
    static constexpr int K = 16 / sizeof(T), PITCH = VEC ? CB : CB + K;
    alignas(16) T v[N][SUB][PITCH];
};

// The copies of a warp's rows, 16 bytes each, dealt to its lanes.
template <typename T, int N, int SUB, bool VEC>
struct Fetch {
    static constexpr int K = 16 / sizeof(T), PER = CB / K, STEP = 32 / PER;  // blocks a row, rows a turn of the warp
    const char* base[N];  // VEC: this lane's block of the first row it copies; else row 0 of the sequence
    int size;             // VEC: bytes of the lane's block that exist, 0 or 16; else bytes of a row's channels

    template <typename... W>
    __device__ __forceinline__ void init(const Args& a, int b, int c0, W... which) {
        const int lane = threadIdx.x & 31, col = lane % PER * K;
        const int w[N] = {which...};
        size = VEC ? (c0 + col < a.D ? 16 : 0) : (a.D - c0 < CB ? a.D - c0 : CB) * (int)sizeof(T);
#pragma unroll
        for (int k = 0; k < N; k++) {
            const Seq& s = a.in[w[k]];
            int64_t at = (int64_t)b * s.sb;
            if (!VEC) at += c0;
            if (VEC && size) at += c0 + col + lane / PER * s.sl;
            base[k] = static_cast<const char*>(s.p) + at * (int64_t)sizeof(T);
        }
    }
    // rows t0 .. t0 + n - 1, n > 0
    template <typename... W>
    __device__ __forceinline__ void start(const Args& a, Rows<T, N, SUB, VEC>& to, int t0, int n, W... which) const {
        const int lane = threadIdx.x & 31;
        const int w[N] = {which...};
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int64_t row = a.in[w[k]].sl * (int64_t)sizeof(T);
            const char* from = base[k] + t0 * row;
            if (VEC) {
                char* slot = reinterpret_cast<char*>(&to.v[k][0][0]) + lane * 16;
                if (n >= SUB) {
#pragma unroll
                    for (int i = 0; i < SUB / STEP; i++) {
                        cp_async<16>(slot + i * 512, from, size);
                        from += STEP * row;
                    }
                } else {
                    for (int i = 0; i * STEP + lane / PER < n; i++) {
                        cp_async<16>(slot + i * 512, from, size);
                        from += STEP * row;
                    }
                }
            } else {
                // whole blocks of 16 bytes: what lies before a row in its first block is read and not used
                for (int at = lane; at < SUB * (PER + 1); at += 32) {
                    const int r = at / (PER + 1), col = at % (PER + 1);
                    const char* p = from + r * row;
                    const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15), left = off + size - col * 16;
                    if (r < n && left > 0) cp_async<16>(&to.v[k][r][col * K], p - off + col * 16, left < 16 ? left : 16);
                }
            }
        }
    }
};

// A lane's two channels of a row; `off`: where a row off 16 bytes starts.
template <bool VEC, typename T>
__device__ __forceinline__ float2 pair(const T* row, uint32_t off) {
    const int lane = threadIdx.x & 31;
    if (VEC) {
        const Pack<T, 2> v = *reinterpret_cast<const Pack<T, 2>*>(row + 2 * lane);
        return make_float2(to_f(v.v[0]), to_f(v.v[1]));
    }
    return make_float2(to_f(row[off + 2 * lane]), to_f(row[off + 2 * lane + 1]));
}
template <bool VEC, typename T>
__device__ __forceinline__ uint32_t off16(const Seq& s, int b, int t, int c0) {
    if (VEC) return 0;
    return (uint32_t)((reinterpret_cast<uintptr_t>(s.p) / sizeof(T) + (int64_t)b * s.sb + (int64_t)t * s.sl + c0) %
                      (16 / sizeof(T)));
}

// Slots a warp: as many as leave room for two CTAs an SM.
template <typename R>
constexpr int STAGES = sizeof(R) * WARPS * 2 + sizeof(Exchange) + 8 * CTA_FOLDS <= 113 * 1024 ? 2 : 1;

// A chunk's place in its sequence of `len` positions.
struct Chunk {
    int b, ch, org, end;  // its positions: org .. end - 1 (those that exist)
    __device__ __forceinline__ Chunk(const Args& a, int y) {
        b = a.chunks == 1 ? y : y / a.chunks, ch = a.chunks == 1 ? 0 : y - b * a.chunks;
        org = ch * a.span;
        end = min(length_of(a, b), a.L - org > a.span ? org + a.span : a.L);
    }
};

// The state in front of a chunk (behind it, backwards): `s` from the sequence's end on through the other chunks between.
// The warps fold some each.
template <bool BWD>
__device__ __forceinline__ float2 through_chunks(const Args& a, const Chunk& k, int c, int valid, Fold (*slots)[32], float2 s) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = BWD ? a.chunks - 1 - k.ch : k.ch;
    if (n == 0) return s;
    const int each = cdiv(n, WARPS), to = min((warp + 1) * each, n);
    Fold mine = {dup(1.0f), dup(0.0f)};
#pragma unroll 4
    for (int i = warp * each; i < to; i++) {
        const float* p = a.folds + ((int64_t)k.b * a.chunks + (BWD ? a.chunks - 1 - i : i)) * 2 * a.D + c;
        mine = join(mine, {load2(p, valid), load2(p + a.D, valid)});
    }
    slots[warp][lane] = mine;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WARPS; i++) s = fold(s, slots[i][lane]);
    __syncthreads();
    return s;
}

template <typename T>
constexpr int SUB_FWD = sizeof(T) == 2 ? 16 : 8;

template <typename T, bool CONVEX, bool GATE, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) fwd_kernel(const __grid_constant__ Args a) {
    constexpr int SUB = SUB_FWD<T>, TT = SUB * WARPS, N = GATE ? 3 : 2;
    using R = Rows<T, N, SUB, VEC>;
    constexpr int ST = STAGES<R>;
    extern __shared__ __align__(16) unsigned char smem[];
    Exchange& ex = *reinterpret_cast<Exchange*>(smem);
    R(*slots)[WARPS] = reinterpret_cast<R(*)[WARPS]>(smem + sizeof(Exchange));
    Fold* folds = reinterpret_cast<Fold*>(smem + sizeof(Exchange) + sizeof(R) * ST * WARPS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cs = a.cs, c0 = blockIdx.x / cs * CB, rank = blockIdx.x % cs;
    const int c = c0 + 2 * lane, valid = a.D - c;
    begin(ex, cs);
    grid_dependency_sync();
    const Chunk chunk(a, blockIdx.y);
    const int b = chunk.b, len = chunk.end;
    const int rounds = len > chunk.org ? cdiv(len - chunk.org, TT * cs) : 0;
    const float2 bias = a.bias ? load2(a.bias + c, valid) : dup(0.0f);
    float2 s = a.h0 ? load2(a.h0 + (int64_t)b * a.D + c, valid) : dup(0.0f);
    Fetch<T, N, SUB, VEC> fetch;
    if constexpr (GATE)
        fetch.init(a, b, c0, X, F, Z);
    else
        fetch.init(a, b, c0, X, F);
    auto start = [&](int round) { return chunk.org + (round * cs + rank) * TT + warp * SUB; };
    auto load = [&](int round) {
        const int t0 = start(round);
        if (round < rounds && t0 < len) {
            if constexpr (GATE)
                fetch.start(a, slots[round % ST][warp], t0, len - t0, X, F, Z);
            else
                fetch.start(a, slots[round % ST][warp], t0, len - t0, X, F);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < ST; i++) load(i);
    if (a.chunks > 1) s = through_chunks<false>(a, chunk, c, valid, ex.warp[0], s);
    for (int round = 0; round < rounds; round++) {
        const int t0 = start(round), k = round % ST;
        const int n = len - t0;  // positions of this stretch that exist
        R& rows = slots[k][warp];
        cp_async_wait<ST - 1>();
        __syncwarp();
        float2 av[SUB], uv[SUB];
        Fold mine = {dup(1.0f), dup(0.0f)};
        if (n > 0) {
#pragma unroll
            for (int i = 0; i < SUB; i++) {
                const float2 f = __fadd2_rn(pair<VEC>(rows.v[1][i], off16<VEC, T>(a.in[F], b, t0 + i, c0)), bias);
                const float2 x = pair<VEC>(rows.v[0][i], off16<VEC, T>(a.in[X], b, t0 + i, c0));
                float2 w;
                sigmoids(f, av[i], w);
                uv[i] = CONVEX ? __fmul2_rn(w, x) : x;
            }
            if (n < SUB) {
#pragma unroll
                for (int i = 0; i < SUB; i++)
                    if (i >= n) av[i] = dup(1.0f), uv[i] = dup(0.0f);
            }
            mine = {av[0], uv[0]};
#pragma unroll
            for (int i = 1; i < SUB; i++) {
                mine.p = __fmul2_rn(mine.p, av[i]);
                mine.q = __ffma2_rn(av[i], mine.q, uv[i]);
            }
        }
        float2 h = exchange(ex, folds, round, cs, rank, mine, s);
        if (n > 0) {
            T* y = static_cast<T*>(a.y) + ((int64_t)b * a.L + t0) * a.D + c;
            float* ck = a.ckpt ? a.ckpt + ((int64_t)b * cdiv(a.L, CK) + t0 / CK) * a.D + c : nullptr;
            auto finish = [&](auto fast) {
                constexpr bool FAST = decltype(fast)::value;
#pragma unroll
                for (int i = 0; i < SUB; i++) {
                    if (i % CK == 0 && ck && (FAST || i < n)) put<FAST>(ck + (int64_t)(i / CK) * a.D, h, valid, a.D % 2 == 0);
                    h = __ffma2_rn(av[i], h, uv[i]);
                    float2 o = h;
                    if (GATE) o = __fmul2_rn(o, silu<T>(pair<VEC>(rows.v[N - 1][i], off16<VEC, T>(a.in[Z], b, t0 + i, c0))));
                    if (FAST || i < n) put<FAST>(y + (int64_t)i * a.D, o, valid, a.ovec);
                }
            };
            if (a.ovec && n >= SUB && c0 + CB <= a.D)
                finish(std::true_type());
            else
                finish(std::false_type());
        }
        __syncwarp();
        load(round + ST);
    }
    cp_async_wait();
    if (a.hT && rank == 0 && warp == 0 && chunk.ch == a.chunks - 1) store2(a.hT + (int64_t)b * a.D + c, s, valid);
    const int last = min(a.L - chunk.org, a.span) + chunk.org;
    for (int t = max(len, chunk.org) + rank * WARPS + warp; t < last; t += cs * WARPS)
        put<false>(static_cast<T*>(a.y) + ((int64_t)b * a.L + t) * a.D + c, dup(0.0f), valid, a.ovec);
    if (cs > 1) cooperative_groups::this_cluster().sync();  // none leaves before the others are done with its memory
}

// The tiles in reverse: warp 0 of CTA 0 has a round's last positions.  A stretch
// is as long as the distance between the kept states, so each warp has its own.
template <typename T, bool CONVEX, bool GATE, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) bwd_kernel(const __grid_constant__ Args a) {
    constexpr int SUB = CK, N = GATE ? 4 : 3;
    using R = Rows<T, N, SUB, VEC>;
    constexpr int ST = STAGES<R>;
    extern __shared__ __align__(16) unsigned char smem[];
    Exchange& ex = *reinterpret_cast<Exchange*>(smem);
    R(*slots)[WARPS] = reinterpret_cast<R(*)[WARPS]>(smem + sizeof(Exchange));
    Fold* folds = reinterpret_cast<Fold*>(smem + sizeof(Exchange) + sizeof(R) * ST * WARPS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cs = a.cs, c0 = blockIdx.x / cs * CB, rank = blockIdx.x % cs;
    const int c = c0 + 2 * lane, valid = a.D - c;
    begin(ex, cs);
    const Chunk chunk(a, blockIdx.y);
    const int b = chunk.b, len = chunk.end;
    const int stretches = len > chunk.org ? cdiv(len - chunk.org, SUB) : 0, rounds = cdiv(stretches, WARPS * cs);
    const float2 bias = a.bias ? load2(a.bias + c, valid) : dup(0.0f);
    float2 s = a.dhT ? load2(a.dhT + (int64_t)b * a.D + c, valid) : dup(0.0f);
    float2 dbias = dup(0.0f), next_h = dup(0.0f);
    Fetch<T, N, SUB, VEC> fetch;
    if constexpr (GATE)
        fetch.init(a, b, c0, X, F, DY, Z);
    else
        fetch.init(a, b, c0, X, F, DY);
    auto stretch = [&](int round) { return stretches - 1 - ((round * cs + rank) * WARPS + warp); };  // < 0: none
    auto load = [&](int round) {
        const int j = stretch(round);
        if (j >= 0) {
            const int t0 = chunk.org + j * SUB;
            if constexpr (GATE)
                fetch.start(a, slots[round % ST][warp], t0, len - t0, X, F, DY, Z);
            else
                fetch.start(a, slots[round % ST][warp], t0, len - t0, X, F, DY);
        }
        cp_async_commit();
    };
    auto load_h = [&](int round) {
        const int j = stretch(round);
        if (j >= 0) next_h = load2(a.ckpt + ((int64_t)b * cdiv(a.L, CK) + chunk.org / CK + j) * a.D + c, valid);
    };
#pragma unroll
    for (int i = 0; i < ST; i++) load(i);
    load_h(0);
    if (a.chunks > 1) s = through_chunks<true>(a, chunk, c, valid, ex.warp[0], s);
    for (int round = 0; round < rounds; round++) {
        const int j = stretch(round), t0 = chunk.org + j * SUB, k = round % ST;
        const int n = j >= 0 ? len - t0 : 0;
        const int64_t at = ((int64_t)b * a.L + t0) * a.D + c;
        const bool fast = a.ovec && n >= SUB && c0 + CB <= a.D;
        R& rows = slots[k][warp];
        cp_async_wait<ST - 1>();
        __syncwarp();
        float2 av[SUB], wv[SUB], mv[SUB], dv[SUB];  // a, 1 - a, dh[t]/df, ds
        Fold mine = {dup(1.0f), dup(0.0f)};
        if (n > 0) {
            float2 h = next_h;
            load_h(round + 1);
            auto enter = [&](auto quick) {
                constexpr bool FAST = decltype(quick)::value;
#pragma unroll
                for (int i = 0; i < SUB; i++) {
                    const float2 f = __fadd2_rn(pair<VEC>(rows.v[1][i], off16<VEC, T>(a.in[F], b, t0 + i, c0)), bias);
                    const float2 x = pair<VEC>(rows.v[0][i], off16<VEC, T>(a.in[X], b, t0 + i, c0));
                    dv[i] = pair<VEC>(rows.v[2][i], off16<VEC, T>(a.in[DY], b, t0 + i, c0));
                    sigmoids(f, av[i], wv[i]);
                    mv[i] = __fmul2_rn(__fmul2_rn(av[i], wv[i]), CONVEX ? __ffma2_rn(x, dup(-1.0f), h) : h);
                    h = __ffma2_rn(av[i], h, CONVEX ? __fmul2_rn(wv[i], x) : x);
                    if (GATE) {
                        float2 slope;
                        const float2 gate = silu<T>(pair<VEC>(rows.v[N - 1][i], off16<VEC, T>(a.in[Z], b, t0 + i, c0)), slope);
                        if (FAST || i < n)
                            put<FAST>(static_cast<T*>(a.dz) + at + (int64_t)i * a.D, __fmul2_rn(__fmul2_rn(dv[i], h), slope),
                                      valid, a.ovec);
                        dv[i] = __fmul2_rn(dv[i], gate);
                    }
                }
            };
            if (fast) {
                enter(std::true_type());
            } else {
                enter(std::false_type());
#pragma unroll
                for (int i = 0; i < SUB; i++)
                    if (i >= n) av[i] = dup(1.0f), dv[i] = dup(0.0f);
            }
            mine = {av[SUB - 1], __fmul2_rn(av[SUB - 1], dv[SUB - 1])};
#pragma unroll
            for (int i = SUB - 2; i >= 0; i--) {
                mine.p = __fmul2_rn(mine.p, av[i]);
                mine.q = __fmul2_rn(av[i], __fadd2_rn(dv[i], mine.q));
            }
        }
        float2 G = exchange(ex, folds, round, cs, rank, mine, s);
        if (n > 0) {
            auto leave = [&](auto quick) {
                constexpr bool FAST = decltype(quick)::value;
#pragma unroll
                for (int i = SUB - 1; i >= 0; i--) {
                    const float2 g = __fadd2_rn(dv[i], G);
                    G = __fmul2_rn(av[i], g);
                    if (FAST || i < n) {
                        const float2 df = __fmul2_rn(g, mv[i]);
                        dbias = __fadd2_rn(dbias, df);
                        put<FAST>(static_cast<T*>(a.df) + at + (int64_t)i * a.D, df, valid, a.ovec);
                        put<FAST>(static_cast<T*>(a.dx) + at + (int64_t)i * a.D, CONVEX ? __fmul2_rn(wv[i], g) : g, valid, a.ovec);
                    }
                }
            };
            if (fast)
                leave(std::true_type());
            else
                leave(std::false_type());
        }
        __syncwarp();
        load(round + ST);
    }
    cp_async_wait();
    if (a.dh0 && rank == 0 && warp == 0 && chunk.ch == 0) store2(a.dh0 + (int64_t)b * a.D + c, s, valid);
    const int last = min(a.L - chunk.org, a.span) + chunk.org;
    for (int t = max(len, chunk.org) + rank * WARPS + warp; t < last; t += cs * WARPS) {
        const int64_t at = ((int64_t)b * a.L + t) * a.D + c;
        put<false>(static_cast<T*>(a.dx) + at, dup(0.0f), valid, a.ovec);
        put<false>(static_cast<T*>(a.df) + at, dup(0.0f), valid, a.ovec);
        if (GATE) put<false>(static_cast<T*>(a.dz) + at, dup(0.0f), valid, a.ovec);
    }
    if (a.part) {
        float2(*sums)[32] = reinterpret_cast<float2(*)[32]>(slots);  // every copy into them has arrived
        __syncthreads();
        sums[warp][lane] = dbias;
        __syncthreads();
        if (warp == 0) {
#pragma unroll
            for (int i = 1; i < WARPS; i++) dbias = __fadd2_rn(dbias, sums[i][lane]);
            store2(a.part + ((int64_t)blockIdx.y * cs + rank) * a.D + c, dbias, valid);
        }
    }
    if (cs > 1) cooperative_groups::this_cluster().sync();
}

// What a chunk does to the state (backwards: to its gradient), for long sequences
// of few channels.  Each warp walks positions of its own, without a barrier.
template <typename T, bool CONVEX, bool GATE, bool VEC, bool BWD>
__global__ void __launch_bounds__(THREADS, 2) chunk_kernel(const __grid_constant__ Args a) {
    constexpr int SUB = BWD ? CK : SUB_FWD<T>, N = BWD && GATE ? 3 : 2, ST = 2;
    using R = Rows<T, N, SUB, VEC>;
    extern __shared__ __align__(16) unsigned char smem[];
    R(*slots)[WARPS] = reinterpret_cast<R(*)[WARPS]>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c0 = blockIdx.x * CB, c = c0 + 2 * lane, valid = a.D - c;
    grid_dependency_sync();
    const Chunk chunk(a, blockIdx.y);
    if (chunk.ch == (BWD ? 0 : a.chunks - 1)) return;  // nothing lies behind it
    const int b = chunk.b;
    const float2 bias = a.bias ? load2(a.bias + c, valid) : dup(0.0f);
    Fetch<T, N, SUB, VEC> fetch;
    // a warp's stretches, in the order in which they are passed
    const int part = a.span / WARPS, first = chunk.org + warp * part, end = min(first + part, chunk.end);
    const int stretches = end > first ? cdiv(end - first, SUB) : 0;
    auto start = [&](int i) { return first + (BWD ? stretches - 1 - i : i) * SUB; };
    auto load = [&](int i) {
        if (i < stretches) {
            const int t0 = start(i);
            if constexpr (BWD && GATE)
                fetch.start(a, slots[i % ST][warp], t0, end - t0, F, DY, Z);
            else if constexpr (BWD)
                fetch.start(a, slots[i % ST][warp], t0, end - t0, F, DY);
            else
                fetch.start(a, slots[i % ST][warp], t0, end - t0, F, X);
        }
        cp_async_commit();
    };
    if constexpr (BWD && GATE)
        fetch.init(a, b, c0, F, DY, Z);
    else if constexpr (BWD)
        fetch.init(a, b, c0, F, DY);
    else
        fetch.init(a, b, c0, F, X);
    load(0), load(1);
    Fold all = {dup(1.0f), dup(0.0f)};
    for (int k = 0; k < stretches; k++) {
        const int t0 = start(k), n = end - t0;
        R& rows = slots[k % ST][warp];
        cp_async_wait<ST - 1>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < SUB; j++) {
            const int i = BWD ? SUB - 1 - j : j;
            const float2 f = __fadd2_rn(pair<VEC>(rows.v[0][i], off16<VEC, T>(a.in[F], b, t0 + i, c0)), bias);
            float2 in = pair<VEC>(rows.v[1][i], off16<VEC, T>(a.in[BWD ? DY : X], b, t0 + i, c0));
            float2 up, down;
            sigmoids(f, up, down);
            if (BWD && GATE) in = __fmul2_rn(in, silu<T>(pair<VEC>(rows.v[N - 1][i], off16<VEC, T>(a.in[Z], b, t0 + i, c0))));
            if (!BWD && CONVEX) in = __fmul2_rn(down, in);
            if (i < n) {
                all.p = __fmul2_rn(all.p, up);
                all.q = BWD ? __fmul2_rn(up, __fadd2_rn(in, all.q)) : __ffma2_rn(up, all.q, in);
            }
        }
        all.p = some(all.p);
        __syncwarp();
        load(k + ST);
    }
    cp_async_wait();
    Fold(*sums)[32] = reinterpret_cast<Fold(*)[32]>(smem);
    __syncthreads();
    sums[warp][lane] = all;
    __syncthreads();
    if (warp == 0) {
        Fold f = sums[BWD ? WARPS - 1 : 0][lane];
#pragma unroll
        for (int i = 1; i < WARPS; i++) f = join(f, sums[BWD ? WARPS - 1 - i : i][lane]);
        float* to = a.folds + (int64_t)blockIdx.y * 2 * a.D + c;
        store2(to, f.p, valid);
        store2(to + a.D, f.q, valid);
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
    for (int i = 0; i < 4; i += 2) {
        const float2 x = make_float2(to_f(px.v[i]), to_f(px.v[i + 1]));
        float2 up, down;
        sigmoids(make_float2(__fadd_rn(to_f(pf.v[i]), pb.v[i]), __fadd_rn(to_f(pf.v[i + 1]), pb.v[i + 1])), up, down);
        const float2 hh = __ffma2_rn(up, make_float2(hp.v[i], hp.v[i + 1]), CONVEX ? __fmul2_rn(down, x) : x);
        const float2 oo = GATE ? __fmul2_rn(hh, silu<T>(make_float2(to_f(pz.v[i]), to_f(pz.v[i + 1])))) : hh;
        hn[i] = hh.x, hn[i + 1] = hh.y, o[i] = oo.x, o[i + 1] = oo.y;
    }
    store_pack<4>(ph, hn, valid, vec);
    store_pack<4>(y + b * D + c, o, valid, vec);
}

// How a call's positions are shared out: CTAs of a cluster, or, for long sequences of
// few channels, chunks, with a pass for each chunk's fold in front (which reads 2
// operands, 3 backwards, a first time).  By an estimate of the time, in tiles that a
// CTA passes one after the other (and `start` for its first, `pass` for the chunks'):
//   tile     what one costs by CTAs of a cluster, whose folds go through the cluster;
//            `twice` in a chunk, whose operands are read twice
//   waves    so many CTAs run at once, or alone on an SM, where one takes `alone` of
//            the time.  Clusters of 4 and more do not find places on every SM: above
//            33, 15, 7 of 4, 8, 16 CTAs they share SMs, and above 66, 33, 14 they take
//            turns.
// Widths off 16 bytes, whose tiles cost more, have figures of their own.  Fitted to
// 1405 sizes each (1 to 400 CTAs without sharing, 100 to 32768 positions, bf16 and fp32,
// both directions), where the choice takes 0.5 % (0.3 %) more than the best plan on
// average and up to 20 % (fp32 1 x 300 x 2112, 7.1 us for 5.9).  us of a gated call,
// 1 x L x 64 base, in clusters of 16 (8 from base 16 on) and in chunks:
//             L =   4096         6144         8192         16384
//   base 2, bf16     8.1 10.2    11.1 10.8    14.0 10.8    26 16
//     backward       16 18       22 18        27 18        50 21
//   base 4, bf16     8.3 10.5    11.2 13.9    14.2 16.0    27 20
//     fp32           12.1 13.4   17.6 18.7    22.6 20.1    43 23
//   base 16, bf16    20 19       28 25        37 30        70 52
//     backward       35 28       49 36        63 45        120 77
//   base 33, bf16    24 30       34 41        43 52        82 94
//   base 34, bf16    32 30       44 41        58 52        110 94
// By CTAs of a cluster, 1, 2, 4, 8, forward and backward in bf16: 8 x 2048 x 1536 63
// 55 58 71, 104 113 97 115; 4 x 2048 x 1536 39 37 30 38, 70 59 60 61; 8 x 2048 x 2048
// 62 72 77 92, 105 117 127 150; 1 x 2048 x 512 of 8 and 16: 7.3 9.9, 14.3 12.7.
// By CTAs of a cluster, off 16 bytes, forward: 8 x 2048 x 1531 bf16 114 104 96 106,
// 1 x 2048 x 763 of 8 and 16 13.1 9.9.
struct Plan {
    int cs, chunks, span;
};
struct Costs {
    double alone, start, tile[5], twice, pass;
};
static inline Plan plan_of(int batch, int L, int D, int tile, bool backward, bool off16) {
    static constexpr Costs COSTS[2][2] = {{{0.7, 0.84, {1, 1.07, 1.12, 1.21, 1.57}, 1.36, 1.83},
                                           {0.85, 0.84, {1, 1.07, 1.12, 1.21, 1.57}, 1.35, 1.83}},
                                          {{0.9, 0.55, {1, 1.08, 1.1, 1.17, 1.27}, 1.66, 1.29},
                                           {0.82, 0.55, {1, 1.08, 1.1, 1.17, 1.27}, 1.46, 1.29}}};
    static constexpr int APART[5] = {148, 148, 132, 120, 112}, AT_ONCE[5] = {296, 296, 264, 264, 224};
    const Costs& cost = COSTS[off16][backward];
    const int64_t base = (int64_t)batch * cdiv(D, CB);
    const auto waves = [&](int64_t ctas, int log_cs) {
        const int64_t rest = ctas % AT_ONCE[log_cs];
        return (double)(ctas / AT_ONCE[log_cs]) + (rest == 0 ? 0.0 : rest > APART[log_cs] ? 1.0 : cost.alone);
    };
    Plan p = {1, 1, L};
    double least = 0;
    for (int i = 0; i < 5; i++) {
        const int cs = 1 << i;
        const double time = (cdiv(L, cs * tile) + cost.start) * cost.tile[i] * waves(base * cs, i);
        if (i == 0 || time < least) least = time, p.cs = cs;
        if (cs * tile >= L) break;
    }
    if (L >= 2048 && base <= 49) {  // chunks of at least 256 positions, at least 6 of them where the length allows
        const int64_t room = 148 * 2 / base, most = L / 256;
        const int span = cdiv(cdiv(L, (int)(room < most ? room : most)), tile) * tile, chunks = cdiv(L, span);
        const double time = (span / tile + cost.start) * cost.twice * waves(base * chunks, 0) + cost.pass;
        if (chunks > 1 && time < least) p = {1, chunks, span};
    }
    return p;
}

// Clusters of more than 8 CTAs are not portable: whether this device takes them, asked once (by two bits a device).
static bool allow_wide_clusters(void (*kernel)(const Args), size_t smem, std::atomic<uint64_t>& known) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 32) return false;
    const uint64_t have = known.load(std::memory_order_relaxed) >> (2 * dev) & 3;
    if (have) return have == 3;
    bool yes = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
    if (yes) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(MAX_CLUSTER);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = MAX_CLUSTER;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int fit = 0;
        yes = cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg) == cudaSuccess && fit > 0;
    }
    cudaGetLastError();
    known.fetch_or((uint64_t)(yes ? 3 : 1) << (2 * dev), std::memory_order_relaxed);
    return yes;
}

template <typename T, bool CONVEX, bool GATE, bool VEC, bool BWD>
static int launch(Args& a, cudaStream_t s) {
    constexpr int N = (GATE ? 3 : 2) + BWD, SUB = BWD ? CK : SUB_FWD<T>;
    using R = Rows<T, N, SUB, VEC>;
    constexpr size_t alone = sizeof(R) * STAGES<R> * WARPS + sizeof(Exchange);
    static std::atomic<uint64_t> allowed{0}, wide{0};
    void (*kernel)(const Args);
    if constexpr (BWD)
        kernel = bwd_kernel<T, CONVEX, GATE, VEC>;
    else
        kernel = fwd_kernel<T, CONVEX, GATE, VEC>;
    if (!allow_smem(kernel, alone + MAX_CLUSTER * CTA_FOLDS, allowed)) return MI_ERR_CUDA;
    if (a.chunks > 1) {
        constexpr size_t bytes = sizeof(Rows<T, BWD && GATE ? 3 : 2, SUB, VEC>) * 2 * WARPS;
        static std::atomic<uint64_t> let{0};
        if (!allow_smem(chunk_kernel<T, CONVEX, GATE, VEC, BWD>, bytes, let)) return MI_ERR_CUDA;
        const dim3 grid(cdiv(a.D, CB), a.batch * a.chunks);
        if (BWD) {
            chunk_kernel<T, CONVEX, GATE, VEC, BWD><<<grid, THREADS, bytes, s>>>(a);
            MI_CHECK_LAUNCH();
        } else {
            MI_LAUNCH_DEPENDENT(chunk_kernel<T, CONVEX, GATE, VEC, BWD>, grid, THREADS, bytes, s, a);
        }
    }
    if (a.cs > 8 && !allow_wide_clusters(kernel, alone + MAX_CLUSTER * CTA_FOLDS, wide)) a.cs = 8;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cdiv(a.D, CB) * a.cs, a.batch * a.chunks);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = alone + (a.cs > 1 ? a.cs * CTA_FOLDS : 0);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (a.cs > 1) {
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
static int dispatch(Args& a, bool convex, bool vec, cudaStream_t s) {
    const Plan p = plan_of(a.batch, a.L, a.D, (BWD ? CK : SUB_FWD<T>)*WARPS, BWD, (int64_t)a.D * sizeof(T) % 16 != 0);
    a.cs = p.cs, a.chunks = p.chunks, a.span = p.span;
    if (a.chunks > 1 && !a.folds) return MI_ERR_INVALID;
#define MI_REC(CONVEX, GATE) return vec ? launch<T, CONVEX, GATE, true, BWD>(a, s) : launch<T, CONVEX, GATE, false, BWD>(a, s)
    if (convex) {
        if (a.in[Z].p) MI_REC(true, true);
        MI_REC(true, false);
    }
    if (a.in[Z].p) MI_REC(false, true);
    MI_REC(false, false);
#undef MI_REC
}

static inline int elem_size(int dtype) { return dtype == MI_DT_F32 ? 4 : 2; }
static inline bool width_off16(int D, int dtype) { return (int64_t)D * elem_size(dtype) % 16 != 0; }
static inline bool rows_vec(const Args& a, int D, int dtype) {
    const int k = 16 / elem_size(dtype);
    for (const Seq& s : a.in)
        if (s.p && (s.sb % k != 0 || s.sl % k != 0 || !aligned16(s.p))) return false;
    return D % k == 0;
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

namespace mi {
namespace rec {
static inline int64_t fold_bytes(const Plan& p, int batch, int D) {
    return p.chunks > 1 ? (int64_t)sizeof(float) * batch * p.chunks * 2 * D : 0;
}
}  // namespace rec
}  // namespace mi

extern "C" int64_t mi_gated_recurrence_workspace(int batch, int L, int D, int backward, int dtype) {
    if (batch <= 0 || L <= 0 || D <= 0 || dtype < 0 || dtype > 2) return 0;
    const int sub = backward ? mi::rec::CK : dtype == MI_DT_F32 ? mi::rec::SUB_FWD<float> : mi::rec::SUB_FWD<__half>;
    const mi::rec::Plan p = mi::rec::plan_of(batch, L, D, sub * mi::rec::WARPS, backward, mi::rec::width_off16(D, dtype));
    return mi::rec::fold_bytes(p, batch, D) + (backward ? (int64_t)sizeof(float) * batch * p.chunks * p.cs * D : 0);
}

extern "C" int mi_gated_recurrence(const void* x, int64_t x_batch, int64_t x_row, const void* f, int64_t f_batch,
                                   int64_t f_row, const void* z, int64_t z_batch, int64_t z_row, const float* bias,
                                   const float* h0, const int32_t* lengths, void* y, float* h_out, float* checkpoints,
                                   void* workspace, int batch, int L, int D, int convex, int dtype, void* stream) {
    mi::rec::Args a = {};
    a.in[mi::rec::X] = {x, x_batch, x_row}, a.in[mi::rec::F] = {f, f_batch, f_row}, a.in[mi::rec::Z] = {z, z_batch, z_row};
    const int rc = mi_rec_check(a.in[0], a.in[1], a.in[2], batch, L, D, dtype);
    if (rc != MI_OK) return rc;
    if (!y || (reinterpret_cast<uintptr_t>(checkpoints) & 7)) return MI_ERR_INVALID;
    if (batch == 0) return MI_OK;
    a.bias = bias, a.h0 = h0, a.lengths = lengths, a.y = y, a.hT = h_out, a.ckpt = checkpoints;
    a.folds = static_cast<float*>(workspace);
    a.batch = batch, a.L = L, a.D = D;
    const int e = mi::rec::elem_size(dtype);
    a.ovec = D % 2 == 0 && reinterpret_cast<uintptr_t>(y) % (2 * e) == 0;
    const bool vec = mi::rec::rows_vec(a, D, dtype);
    MI_DISPATCH_DTYPE(dtype, T, return (mi::rec::dispatch<T, false>(a, convex, vec, (cudaStream_t)stream)););
}

extern "C" int mi_gated_recurrence_backward(const void* dy, int64_t dy_batch, int64_t dy_row, const float* dh_out,
                                            const void* x, int64_t x_batch, int64_t x_row, const void* f, int64_t f_batch,
                                            int64_t f_row, const void* z, int64_t z_batch, int64_t z_row, const float* bias,
                                            const int32_t* lengths, const float* checkpoints, void* dx, void* df, void* dz,
                                            float* dbias, float* dh0, void* workspace, int batch, int L, int D, int convex,
                                            int dtype, void* stream) {
    mi::rec::Args a = {};
    a.in[mi::rec::X] = {x, x_batch, x_row}, a.in[mi::rec::F] = {f, f_batch, f_row}, a.in[mi::rec::Z] = {z, z_batch, z_row};
    a.in[mi::rec::DY] = {dy, dy_batch, dy_row};
    const int rc = mi_rec_check(a.in[0], a.in[1], a.in[2], batch, L, D, dtype);
    if (rc != MI_OK) return rc;
    if (!dy || dy_batch < 0 || dy_row < 0 || !checkpoints || !dx || !df || (z && !dz) || (dbias && !workspace))
        return MI_ERR_INVALID;
    cudaStream_t s = (cudaStream_t)stream;
    if (batch == 0) {
        if (dbias && cudaMemsetAsync(dbias, 0, sizeof(float) * D, s) != cudaSuccess) return MI_ERR_CUDA;
        return MI_OK;
    }
    a.bias = bias, a.dhT = dh_out, a.lengths = lengths, a.ckpt = const_cast<float*>(checkpoints);
    a.dx = dx, a.df = df, a.dz = dz, a.dh0 = dh0;
    a.batch = batch, a.L = L, a.D = D;
    const mi::rec::Plan p = mi::rec::plan_of(batch, L, D, mi::rec::CK * mi::rec::WARPS, true, mi::rec::width_off16(D, dtype));
    a.folds = static_cast<float*>(workspace);
    if (dbias) a.part = a.folds + mi::rec::fold_bytes(p, batch, D) / (int64_t)sizeof(float);
    const int e = mi::rec::elem_size(dtype);
    a.ovec = D % 2 == 0;
    for (const void* p : {dx, df, z ? dz : nullptr}) a.ovec = a.ovec && reinterpret_cast<uintptr_t>(p) % (2 * e) == 0;
    const bool vec = mi::rec::rows_vec(a, D, dtype);
    int rc2 = MI_ERR_INVALID;
    MI_DISPATCH_DTYPE(dtype, T, (rc2 = mi::rec::dispatch<T, true>(a, convex, vec, s)););
    if (rc2 != MI_OK || !dbias) return rc2;
    mi::column_sum_kernel<<<mi::cdiv(D, 32), 1024, 0, s>>>(a.part, dbias, batch * a.chunks * a.cs, D);
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

// selective.cu -- the selective scan of a float Mamba layer (exponential
// decays), its backward pass and its form for one new token.
//
//   dt = softplus(delta + delta_bias)  (or delta + delta_bias)
//   h[t] = exp(dt A) h[t-1] + dt B[t] u,   h[-1] = h0        per (channel, state)
//   s[t] = sum_n C[t] h[t] + D u;   y = s * z sigmoid(z)     (0 from the length on)
//
// and, with g the gradient of h, running backwards:
//   ds = dy z sigmoid(z);   g[t] = C[t] ds[t] + a[t+1] g[t+1],  a = exp(dt A)
//   dC = sum_d ds h;  dB = sum_d g dt u;  S1 = sum_n g B;  w = g a[t] h[t-1]
//   du = dt S1 + D ds;  d(dt) = u S1 + sum_n w A;  dA = sum_t w dt
//   ddelta = d(dt) sigmoid(delta + bias);  dz = dy s (z sigmoid(z))'
//
// What bounds it: with N states a position and channel move 4 elements and
// need N exponentials.  The special-function unit makes 16 a cycle and SM,
// 4.7e12 a second on the chip, so from N = 8 on it is slower than HBM: 16
// states, 8 x 2048 x 1536 positions and channels, are 86 us of exponentials
// against 31 us of 16-bit loads and stores.
//
// Layout: LN lanes share a channel and hold 4 states each (N <= 4 LN), so a warp
// spans 32 / LN channels.  States beyond N have A = B = C = 0, and where there
// are any (PAD) they are put back to 0 after each step: the channel's step size
// and input reach them too, and 0 times an infinite one is not 0.  12 states,
// 8 x 2048 x 1536 bf16, take 247 us forward and 1036 in training, and took 236
// and 995 without; kernels of their own keep that from the full lanes.
// Tiles of TT positions by CB channels are staged in shared memory as
// (dt, dt u); positions from the length on are staged with dt = 0, B = C = 0,
// where the recurrence leaves the state as it is.
#include <type_traits>

#include "mi_elem.cuh"

namespace mi {
namespace sscan {

constexpr int THREADS = 128;
constexpr int CK = 16;      // positions between the states that the forward pass keeps for the backward pass
constexpr int MAX_N = 64;

struct Seq {  // a [batch, L, *] operand with unit last stride
    const void* p;
    int64_t sb, sl;  // batch and row strides in elements
    int vec;         // rows start on 8 elements' alignment (4 for B and C)
};

struct Args {
    Seq u, delta, z, B, C, dy;
    const float* A;     // [D, N]
    const float* Dskip; // [D] or NULL
    const float* bias;  // [D] or NULL
    const float* h0;    // [batch, D, N] or NULL
    const float* dhT;   // gradient of the final state or NULL
    const int* lengths; // [batch] or NULL
    void* y;            // [batch, L, D]
    float* hT;          // [batch, D, N] or NULL
    float* ckpt;        // [batch, cdiv(L, CK), D, NP] or NULL
    // with chunks > 1: each chunk's own end state / the state it starts from, and its sum of dt
    float* cst;  // [batch, chunks, D, NP]
    float* cdt;  // [batch, chunks, D]
    void *du, *ddelta, *dz;
    float* part_bc;  // [channel blocks, batch, L, 2 NP]
    float* part_a;   // [batch * chunks, D, NP]
    float* part_d;   // [batch * chunks, 2, D]: dD and dbias
    float* dh0;      // [batch, D, N] or NULL
    int batch, L, D, N;
    int softplus;
    int chunks, span;  // positions a chunk (a multiple of 32)
    int ovec;          // outputs' rows start on 8 elements' alignment
};

__device__ __forceinline__ int length_of(const Args& a, int b) {
    if (!a.lengths) return a.L;
    const int n = a.lengths[b];
    return n < 0 ? 0 : (n < a.L ? n : a.L);
}

template <typename T>
__device__ __forceinline__ const T* row_of(const Seq& s, int b, int t) {
    return static_cast<const T*>(s.p) + (int64_t)b * s.sb + (int64_t)t * s.sl;
}

// 4 states n0 .. n0 + 3 of a row of N
__device__ __forceinline__ float4 load4(const float* p, int n0, int N) {
    if ((N & 3) == 0) return n0 < N ? *reinterpret_cast<const float4*>(p + n0) : make_float4(0, 0, 0, 0);
    float4 v;
    v.x = n0 + 0 < N ? p[n0 + 0] : 0.0f;
    v.y = n0 + 1 < N ? p[n0 + 1] : 0.0f;
    v.z = n0 + 2 < N ? p[n0 + 2] : 0.0f;
    v.w = n0 + 3 < N ? p[n0 + 3] : 0.0f;
    return v;
}
__device__ __forceinline__ void store4(float* p, int n0, int N, float4 v) {
    if ((N & 3) == 0) {
        if (n0 < N) *reinterpret_cast<float4*>(p + n0) = v;
        return;
    }
    if (n0 + 0 < N) p[n0 + 0] = v.x;
    if (n0 + 1 < N) p[n0 + 1] = v.y;
    if (n0 + 2 < N) p[n0 + 2] = v.z;
    if (n0 + 3 < N) p[n0 + 3] = v.w;
}

struct St {  // 4 states in two f32x2 pairs
    float2 a, b;
};
__device__ __forceinline__ St st(float4 v) { return {make_float2(v.x, v.y), make_float2(v.z, v.w)}; }
__device__ __forceinline__ float4 f4(St s) { return make_float4(s.a.x, s.a.y, s.b.x, s.b.y); }
__device__ __forceinline__ float2 dup(float v) { return make_float2(v, v); }
__device__ __forceinline__ St mul(St x, float v) { return {__fmul2_rn(x.a, dup(v)), __fmul2_rn(x.b, dup(v))}; }
__device__ __forceinline__ St mul(St x, St y) { return {__fmul2_rn(x.a, y.a), __fmul2_rn(x.b, y.b)}; }
__device__ __forceinline__ St fma(St x, St y, St z) { return {__ffma2_rn(x.a, y.a, z.a), __ffma2_rn(x.b, y.b, z.b)}; }
__device__ __forceinline__ St mul(St x, float2 v) { return {__fmul2_rn(x.a, v), __fmul2_rn(x.b, v)}; }
__device__ __forceinline__ St fma(St x, float2 v, St z) { return {__ffma2_rn(x.a, v, z.a), __ffma2_rn(x.b, v, z.b)}; }
__device__ __forceinline__ float dot(St x, St y) {
    const float2 p = __ffma2_rn(x.b, y.b, __fmul2_rn(x.a, y.a));
    return __fadd_rn(p.x, p.y);
}
// Which of a lane's 4 states n0 .. n0 + 3 (lane order `perm`: n0 + (i ^ perm)) there are.
template <bool PAD>
__device__ __forceinline__ uint4 within(int n0, int N, int perm = 0) {
    if (!PAD) return make_uint4(~0u, ~0u, ~0u, ~0u);
    return make_uint4(n0 + perm < N ? ~0u : 0u, n0 + (1 ^ perm) < N ? ~0u : 0u, n0 + (2 ^ perm) < N ? ~0u : 0u,
                      n0 + (3 ^ perm) < N ? ~0u : 0u);
}
__device__ __forceinline__ float2 masked(float2 v, uint32_t x, uint32_t y) {
    return make_float2(__uint_as_float(__float_as_uint(v.x) & x), __uint_as_float(__float_as_uint(v.y) & y));
}
template <bool PAD>
__device__ __forceinline__ St only(St s, uint4 m) {
    return PAD ? St{masked(s.a, m.x, m.y), masked(s.b, m.z, m.w)} : s;
}
// A row of A for base 2.  An infinite A becomes a large one: it forgets the
// state at once all the same, and a position of dt = 0 behind a length, which
// must leave the state alone, stays clear of 0 times infinity.
__device__ __forceinline__ float finite(float v) { return fabsf(v) > 1e20f ? copysignf(1e20f, v) : v; }
__device__ __forceinline__ St scaled(float4 A) {
    return {make_float2(finite(__fmul_rn(A.x, LOG2E)), finite(__fmul_rn(A.y, LOG2E))),
            make_float2(finite(__fmul_rn(A.z, LOG2E)), finite(__fmul_rn(A.w, LOG2E)))};
}
__device__ __forceinline__ St exp2s(St x) {
    return {make_float2(exp2_fast(x.a.x), exp2_fast(x.a.y)), make_float2(exp2_fast(x.b.x), exp2_fast(x.b.y))};
}

// 2^(A dt) of two positions on the FMA pipe: with x = A dt and n = x rounded,
// 2^x = 2^n 2^r, r = x - n in [-1/2, 1/2], and 2^r = 1 + r q(r), q of degree 5
// by Remez's exchange.  With its coefficients in fp32 the polynomial is off by
// up to 2^-26.1 of 2^r, and evaluated in fp32 by 2^-23.6.  A dt is at least
// -126, where the decay is 2^-126 and no more than rounding, and at most
// 128, where the largest fp32 number or infinity comes out (behind 128 the sum
// of the exponents would be a NaN): `limits` keeps dt there.
__device__ __forceinline__ float2 exp2_poly(float A, float2 dt) {
    const float magic = 12582912.0f;  // 1.5 2^23: adding it rounds to whole numbers and leaves them in the low bits
    const float2 t = __ffma2_rn(dup(A), dt, dup(magic));
    const float2 r = __ffma2_rn(dup(A), dt, __ffma2_rn(t, dup(-1.0f), dup(magic)));
    float2 p = __ffma2_rn(dup(1.5469732170458883e-4f), r, dup(1.3410000829026103e-3f));
    p = __ffma2_rn(p, r, dup(9.618030861020088e-3f));
    p = __ffma2_rn(p, r, dup(5.550297349691391e-2f));
    p = __ffma2_rn(p, r, dup(2.4022650718688965e-1f));
    p = __ffma2_rn(p, r, dup(6.931472420692444e-1f));
    p = __ffma2_rn(p, r, dup(1.0f));
    return make_float2(__int_as_float((__float_as_int(t.x) << 23) + __float_as_int(p.x)),
                       __int_as_float((__float_as_int(t.y) << 23) + __float_as_int(p.y)));
}

// 2^x of two states by the same polynomial, twice 2^r times 2^(n - 1): the
// product keeps a NaN, is infinite from 2^128 on, and 0 below 2^-125.5, where
// 2^(n - 1) has left the normal range.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
    x = make_float2(min_nan(max_nan(x.x, -126.0f), 128.0f), min_nan(max_nan(x.y, -126.0f), 128.0f));
    const float magic = 12582912.0f;
    const float2 t = __fadd2_rn(x, dup(magic));
    const float2 r = __fadd2_rn(x, __ffma2_rn(t, dup(-1.0f), dup(magic)));
    float2 p = __ffma2_rn(dup(2 * 1.5469732170458883e-4f), r, dup(2 * 1.3410000829026103e-3f));
    p = __ffma2_rn(p, r, dup(2 * 9.618030861020088e-3f));
    p = __ffma2_rn(p, r, dup(2 * 5.550297349691391e-2f));
    p = __ffma2_rn(p, r, dup(2 * 2.4022650718688965e-1f));
    p = __ffma2_rn(p, r, dup(2 * 6.931472420692444e-1f));
    p = __ffma2_rn(p, r, dup(2.0f));
    return __fmul2_rn(p, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f000000),
                                     __int_as_float((__float_as_int(t.y) << 23) + 0x3f000000)));
}

// The decays of 4 positions: one state of a lane's four goes through the FMA
// pipe, the others through the special-function unit.  The polynomial is the
// exacter of the two near 1, where a decay's error adds up over the longest
// memory; A usually begins with its slowest state, so it is the first of the
// four: dA's error against 64 bits is 6e-7 with it and 1.6e-6 without (8 x 2048
// x 1536), and the special-function unit, the slower of the two, has a quarter
// less to do.  `lim`: the limits of the first state's step sizes.  SIGNED: they
// may be negative (they are not from softplus).
template <bool SIGNED>
__device__ __forceinline__ void decays(const St& A2, float2 lim, const float (&dt)[4], St (&e)[4]) {
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
        float2 d = make_float2(fminf(dt[k], lim.y), fminf(dt[k + 1], lim.y));
        if (SIGNED) d = make_float2(fmaxf(d.x, lim.x), fmaxf(d.y, lim.x));
        const float2 p = exp2_poly(A2.a.x, d);
        e[k].a.x = p.x, e[k + 1].a.x = p.y;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float2 x = __fmul2_rn(A2.b, dup(dt[k]));
        e[k].a.y = exp2_fast(__fmul_rn(A2.a.y, dt[k]));
        e[k].b = make_float2(exp2_fast(x.x), exp2_fast(x.y));
    }
}
// The backward pass's, whose lanes hold the states in different orders: all
// by the special-function unit, which has time beside that pass's many
// multiply-adds; with EXACT (fp32 gradients) all by the polynomial.
template <bool EXACT>
__device__ __forceinline__ void decays(const St& A2, const float (&dt)[4], St (&e)[4]) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const St x = mul(A2, dup(dt[k]));
        e[k] = EXACT ? St{exp2_poly(x.a), exp2_poly(x.b)} : exp2s(x);
    }
}

// v[0 .. M): after the call the first M / 2 hold the sums over lanes that
// differ in bit `mask`; lanes with the bit clear keep the first half, with it
// set the second.
template <int M>
__device__ __forceinline__ void halve(float* v, int mask) {
    const bool up = (threadIdx.x & mask) != 0;
#pragma unroll
    for (int i = 0; i < M / 2; i++) {
        const float send = up ? v[i] : v[i + M / 2];
        const float keep = up ? v[i + M / 2] : v[i];
        v[i] = __fadd_rn(keep, __shfl_xor_sync(0xffffffffu, send, mask));
    }
}

// Sums of 4 positions' values over a channel's LN lanes: lane nl keeps position
// nl % 4 (LN = 2: positions 2 nl and 2 nl + 1).
template <int LN>
__device__ __forceinline__ void over_states(float (&y)[4]) {
    if constexpr (LN == 2) {
        halve<4>(y, 1);
    } else {
        halve<4>(y, 2);
        halve<2>(y, 1);
#pragma unroll
        for (int m = 4; m < LN; m *= 2) y[0] = __fadd_rn(y[0], __shfl_xor_sync(0xffffffffu, y[0], m));
    }
}
template <int LN, int STRIDE>
__device__ __forceinline__ void store_positions(float* col, const float* y, int nl) {
    if constexpr (LN == 2) {
        col[(2 * nl) * STRIDE] = y[0];
        col[(2 * nl + 1) * STRIDE] = y[1];
    } else {
        if (nl < 4) col[nl * STRIDE] = y[0];
    }
}

// Where the channels 2 u and 2 u + 1 of position t lie in its row of staged
// (dt, dt u): a thread stages 4 such pairs, 16 bytes each, and the rotation
// puts what 8 threads store at once into 8 different bank groups.
__device__ __forceinline__ int place(int u, int t) { return u ^ (((u >> 3) ^ ((t & 1) << 1)) & 3); }

// (dt, dt u) of a lane's channels c .. c + CPL - 1 at a position
template <int CPL>
__device__ __forceinline__ void staged(const float4* row, int c, int t, float (&dt)[CPL], float (&v)[CPL]) {
    if constexpr (CPL == 1) {
        const float2 x = reinterpret_cast<const float2*>(row + place(c >> 1, t))[c & 1];
        dt[0] = x.x, v[0] = x.y;
    } else {
#pragma unroll
        for (int j = 0; j < CPL; j += 2) {
            const float4 x = row[place((c + j) >> 1, t)];
            dt[j] = x.x, v[j] = x.y, dt[j + 1] = x.z, v[j + 1] = x.w;
        }
    }
}
// a thread's 8 (K) channels from c on
template <int K>
__device__ __forceinline__ void stage_steps(float4* row, int c, int t, const float (&dt)[K], const float (&v)[K]) {
#pragma unroll
    for (int k = 0; k < K; k += 2) row[place((c + k) >> 1, t)] = make_float4(dt[k], v[k], dt[k + 1], v[k + 1]);
}

// The least and the largest step size with -126 <= A dt <= 128, A of a lane's
// first state; a NaN in it, which the polynomial would lose, is put into the state.
__device__ __forceinline__ float2 limits(const St& A2, St& h) {
    if (isnan(A2.a.x)) h.a.x = A2.a.x;
    const float A = fmaxf(fabsf(A2.a.x), 1e-30f), decay = __fdiv_rn(126.0f, A), growth = __fdiv_rd(128.0f, A);
    return A2.a.x > 0.0f ? make_float2(-decay, growth) : make_float2(-growth, decay);
}

// The forward kernels' CTA: 4 warps that carry the recurrence, 4 that stage
// its tiles and finish its outputs.  CPL: channels a lane.
constexpr int WORKERS = 128, STAGERS = 128, CTA = WORKERS + STAGERS;
template <typename T, int LN, int CPL_>
struct Cfg {
    static constexpr int NP = 4 * LN;                    // padded states
    static constexpr int CL = 32 / LN;                   // channel lanes of a warp
    static constexpr int CPL = CPL_;
    static constexpr int CB = 4 * CL * CPL;              // channels a CTA: 64 or 32
    static constexpr int TT = 1024 / CB, E = TT * CB / STAGERS;  // positions a tile: 16 or 32; a stager's channels
    static constexpr int VPR = CB / E;                   // stagers a row
    static constexpr int QUADS = TT * LN;                // packs of 4 states of a tile, of each of B and C
    static constexpr int YS = CB + 8;  // the 4 positions that a step of the loop stores lie in different banks
    template <bool SCAN>
    struct Smem {
        float4 sd[2][TT][CB / 2];  // (dt, dt u) of two channels (chunk_kernel backwards: (dt, ds))
        float B[2][TT][NP];        // B (C)
        float C[SCAN ? 2 : 0][TT][NP];
        float y[SCAN ? 2 : 0][TT][YS];
        float bias[CB], skip[CB];
        // by stager, as they come: u (dy) and z until a tile is finished, the rest until it is staged
        alignas(16) T raw_u[4][STAGERS * E];
        alignas(16) T raw_z[4][STAGERS * E];
        alignas(16) T raw_d[2][STAGERS * E];
        alignas(16) T raw_bc[2][SCAN ? 2 : 1][QUADS * 4];
    };
};

// setmaxnreg: the workers' registers come from what the stagers give up.  The
// launch gives each of the 256 threads 128 (two CTAs an SM), 32768 in all:
// 128 x 176 + 128 x 80.  Three CTAs with 96 and 64 measured 210 us against 229
// at 8 x 2048 x 1536, but 62 against 53 for ragged prompts of 6 x 777 x 2048.
constexpr int CTA_REGS = 128;
__device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 176;\n"); }
__device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 80;\n"); }
__device__ __forceinline__ void cta_barrier() { asm volatile("bar.sync 1, 256;\n" ::: "memory"); }

template <int K, typename T>
__device__ __forceinline__ Pack<T, K> slot_pack(const T* slot) {
    return *reinterpret_cast<const Pack<T, K>*>(slot);
}

// The CTA's channels of a parameter (zeros without one, and beyond the last channel)
template <int CB>
__device__ __forceinline__ void stage_param(float (&to)[CB], const float* p, int d0, int D) {
    for (int c = threadIdx.x; c < CB; c += blockDim.x) to[c] = p && d0 + c < D ? p[d0 + c] : 0.0f;
}

template <int K>
__device__ __forceinline__ void getk(const float* p, float (&v)[K]) {
    const Pack<float, K> r = *reinterpret_cast<const Pack<float, K>*>(p);
#pragma unroll
    for (int i = 0; i < K; i++) v[i] = r.v[i];
}
template <int K>
__device__ __forceinline__ void setk(float* p, const float (&v)[K]) {
    Pack<float, K> r;
#pragma unroll
    for (int i = 0; i < K; i++) r.v[i] = v[i];
    *reinterpret_cast<Pack<float, K>*>(p) = r;
}

__device__ __forceinline__ float4 quad(const Pack<float, 4>& p) { return make_float4(p.v[0], p.v[1], p.v[2], p.v[3]); }
template <typename T>
__device__ __forceinline__ float4 quad(const Pack<T, 4>& p) {
    return make_float4(to_f(p.v[0]), to_f(p.v[1]), to_f(p.v[2]), to_f(p.v[3]));
}

// ---------------------------------------------------------------------------
// What the stagers of a forward kernel do: while the workers are at tile i,
// tile i + 2's inputs are on their way, tile i + 1 is staged and tile i - 1's
// outputs are gated and stored.  MODE: SCAN, or a chunk's own end state
// (CHUNK), or that of the gradient, backwards (RCHUNK: dy, z and C in the
// place of u, delta's neighbour, and B).
enum { SCAN, CHUNK, RCHUNK };
template <typename T, int LN, int CPL, int MODE>
__device__ __forceinline__ void stagers(const Args& a, typename Cfg<T, LN, CPL>::template Smem<MODE == SCAN>& sm, int d0, int b,
                                        int tb, int te, int end, int tiles) {
    using F = Cfg<T, LN, CPL>;
    constexpr int TT = F::TT, E = F::E, PER = (F::QUADS + STAGERS - 1) / STAGERS;
    constexpr bool REV = MODE == RCHUNK, GATED = MODE != CHUNK;
    const int tid = threadIdx.x - WORKERS;
    const int lt = tid / F::VPR, lc = E * (tid % F::VPR), d = d0 + lc, have = a.D - d;
    const int first = tb + (REV ? (tiles - 1) * TT : 0), rows = REV ? -TT : TT;
    const int nq = 4 * (tid % LN), tq = tid / LN;  // this thread's first pack of B and C
    const Seq &su = REV ? a.dy : a.u, &sB = REV ? a.C : a.B;
    const T *wu = row_of<T>(su, b, first + lt) + d, *wd = row_of<T>(a.delta, b, first + lt) + d;
    const T* wz = row_of<T>(a.z, b, first + lt) + d;
    const T *wB = row_of<T>(sB, b, first + tq) + nq, *wC = row_of<T>(a.C, b, first + tq) + nq;
    T* yp = MODE == SCAN ? static_cast<T*>(a.y) + ((int64_t)b * a.L + tb + lt) * a.D + d : nullptr;
    auto load = [&](int i) {
        if (i < tiles) {
            const int t0 = first + i * rows, valid = t0 + lt < end ? have : 0;
            fetch_pack<E>(&sm.raw_u[i & 3][E * tid], wu, su.p, valid, su.vec);
            fetch_pack<E>(&sm.raw_d[i & 1][E * tid], wd, a.delta.p, valid, a.delta.vec);
            if (GATED && a.z.p) fetch_pack<E>(&sm.raw_z[i & 3][E * tid], wz, a.z.p, valid, a.z.vec);
#pragma unroll
            for (int q = 0; q < PER; q++) {
                const int e = tid + q * STAGERS, r = tq + q * (STAGERS / LN), valid4 = t0 + r < end ? a.N - nq : 0;
                if (e >= F::QUADS) break;
                fetch_pack<4>(&sm.raw_bc[i & 1][0][4 * e], wB + q * (STAGERS / LN) * sB.sl, sB.p, valid4, sB.vec);
                if (MODE == SCAN)
                    fetch_pack<4>(&sm.raw_bc[i & 1][MODE == SCAN][4 * e], wC + q * (STAGERS / LN) * a.C.sl, a.C.p, valid4,
                                  a.C.vec);
            }
            wu += rows * su.sl, wd += rows * a.delta.sl, wz += rows * a.z.sl, wB += rows * sB.sl, wC += rows * a.C.sl;
        }
        cp_async_commit();
    };
    auto stage = [&](int i) {
        float dt[E], v[E];
        if (first + i * rows + lt < end) {
            const Pack<T, E> pu = slot_pack<E>(&sm.raw_u[i & 3][E * tid]), pd = slot_pack<E>(&sm.raw_d[i & 1][E * tid]);
            getk<E>(&sm.bias[lc], dt);
#pragma unroll
            for (int k = 0; k < E; k++) {
                dt[k] = __fadd_rn(to_f(pd.v[k]), dt[k]);
                if (a.softplus) dt[k] = softplus(dt[k]);
                v[k] = to_f(pu.v[k]);
                if (!REV) v[k] = __fmul_rn(dt[k], v[k]);
            }
            if (REV && a.z.p) {
                const Pack<T, E> pz = slot_pack<E>(&sm.raw_z[i & 3][E * tid]);
#pragma unroll
                for (int k = 0; k < E; k++) {
                    const float z = to_f(pz.v[k]);
                    v[k] = __fmul_rn(v[k], __fmul_rn(z, sigmoid(z)));
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < E; k++) dt[k] = v[k] = 0.0f;
        }
        stage_steps<E>(sm.sd[i & 1][lt], lc, lt, dt, v);
#pragma unroll
        for (int q = 0; q < PER; q++) {
            const int e = tid + q * STAGERS, r = tq + q * (STAGERS / LN);
            if (e >= F::QUADS) break;
            *reinterpret_cast<float4*>(&sm.B[i & 1][r][nq]) = quad(slot_pack<4>(&sm.raw_bc[i & 1][0][4 * e]));
            if (MODE == SCAN)
                *reinterpret_cast<float4*>(&sm.C[i & 1][r][nq]) = quad(slot_pack<4>(&sm.raw_bc[i & 1][MODE == SCAN][4 * e]));
        }
    };
    auto finish = [&](int i) {
        const int t = tb + i * TT + lt;
        if (t < te && have > 0) {
            float o[E];
            getk<E>(&sm.y[i & 1][lt][lc], o);
            if (a.Dskip) {
                const Pack<T, E> eu = slot_pack<E>(&sm.raw_u[i & 3][E * tid]);
                float skip[E];
                getk<E>(&sm.skip[lc], skip);
#pragma unroll
                for (int k = 0; k < E; k++) o[k] = __fmaf_rn(skip[k], to_f(eu.v[k]), o[k]);
            }
            if (a.z.p) {
                const Pack<T, E> ez = slot_pack<E>(&sm.raw_z[i & 3][E * tid]);
#pragma unroll
                for (int k = 0; k < E; k++) {
                    const float z = to_f(ez.v[k]);
                    o[k] = __fmul_rn(o[k], __fmul_rn(z, sigmoid(z)));
                }
            }
            if (t >= end) {
#pragma unroll
                for (int k = 0; k < E; k++) o[k] = 0.0f;
            }
            store_pack<E>(yp, o, have, a.ovec);
        }
        yp += (int64_t)TT * a.D;
    };
    load(0), load(1);
    cp_async_wait<1>();
    if (tiles > 0) stage(0);
    cta_barrier();
#pragma unroll 1
    for (int i = 0; i < tiles; i++) {
        load(i + 2);
        if (MODE == SCAN && i > 0) finish(i - 1);
        cp_async_wait<1>();
        if (i + 1 < tiles) stage(i + 1);
        cta_barrier();
    }
    if (MODE == SCAN) {
        if (tiles > 0) finish(tiles - 1);
        if (have > 0) {  // behind the length
            float zero[E];
#pragma unroll
            for (int k = 0; k < E; k++) zero[k] = 0.0f;
            for (int t = tb + tiles * TT + lt; t < te; t += TT, yp += (int64_t)TT * a.D)
                store_pack<E>(yp, zero, have, a.ovec);
        }
    }
}

// A chunk's own end state, from a zero start (REV = false), or the gradient
// that a chunk passes to the one before it, from a zero one behind it (REV =
// true; dy, z and C in the place of u, delta and B), and the sum of its dt.
// Only chunks > 1 need it: one more exponential for each state.
template <typename T, int LN, int CPL, bool REV, bool PAD>
__global__ void __launch_bounds__(CTA, 2) chunk_kernel(const Args a) {
    using F = Cfg<T, LN, CPL>;
    constexpr int CB = F::CB, TT = F::TT;
    using Smem = typename F::template Smem<false>;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const int d0 = blockIdx.x * CB, b = blockIdx.y, ck = blockIdx.z + (REV ? 1 : 0);
    const int len = length_of(a, b);
    const int tb = ck * a.span, te = tb + a.span < a.L ? tb + a.span : a.L;
    const int end = te < len ? te : len;  // past it nothing changes the state
    const int tiles = end > tb ? cdiv(end - tb, TT) : 0;
    stage_param(sm.bias, a.bias, d0, a.D);
    __syncthreads();
    if (threadIdx.x >= WORKERS) {
        give_registers();
        stagers<T, LN, CPL, REV ? RCHUNK : CHUNK>(a, sm, d0, b, tb, te, end, tiles);
        return;
    }
    take_registers();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nl = lane % LN, cl = lane / LN, n0 = 4 * nl;
    const int c0 = warp * F::CL * CPL + cl * CPL;
    const uint4 there = within<PAD>(n0, a.N);
    St A2[CPL], h[CPL];
    float sum[CPL];
    float2 lim[CPL];
#pragma unroll
    for (int j = 0; j < CPL; j++) {
        const int c = d0 + c0 + j;
        A2[j] = scaled(c < a.D ? load4(a.A + (int64_t)c * a.N, n0, a.N) : make_float4(0, 0, 0, 0));
        h[j] = st(make_float4(0, 0, 0, 0));
        lim[j] = limits(A2[j], h[j]);
        sum[j] = 0.0f;
    }
    auto run = [&](auto signed_steps) {
#pragma unroll 1
        for (int i = 0; i < tiles; i++) {
            const int buf = i & 1;
#pragma unroll 2
            for (int q4 = 0; q4 < TT; q4 += 4) {
                const int r4 = REV ? TT - 4 - q4 : q4;
                St m[4];
                float dt[4][CPL], v[4][CPL];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    m[k] = st(*reinterpret_cast<const float4*>(&sm.B[buf][r4 + k][n0]));
                    staged<CPL>(sm.sd[buf][r4 + k], c0, k, dt[k], v[k]);
                }
#pragma unroll
                for (int j = 0; j < CPL; j++) {
                    const float dj[4] = {dt[0][j], dt[1][j], dt[2][j], dt[3][j]};
                    St e[4];
                    decays<decltype(signed_steps)::value>(A2[j], lim[j], dj, e);
                    sum[j] = __fadd_rn(sum[j], __fadd_rn(__fadd_rn(dj[0], dj[1]), __fadd_rn(dj[2], dj[3])));
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int r = REV ? 3 - k : k;
                        h[j] = REV ? mul(e[r], fma(m[r], dup(v[r][j]), h[j])) : fma(e[r], h[j], mul(m[r], dup(v[r][j])));
                        h[j] = only<PAD>(h[j], there);
                    }
                }
            }
            cta_barrier();
        }
    };
    cta_barrier();
    if (!PAD && a.softplus)  // with PAD one loop takes steps of either sign
        run(std::bool_constant<PAD>());
    else
        run(std::true_type());
#pragma unroll
    for (int j = 0; j < CPL; j++) {
        const int c = d0 + c0 + j;
        if (c >= a.D) continue;
        const int64_t row = ((int64_t)b * a.chunks + ck) * a.D + c;
        *reinterpret_cast<float4*>(a.cst + row * F::NP + n0) = f4(h[j]);
        if (nl == 0) a.cdt[row] = sum[j];
    }
}

// 2^x h + own, x of a whole chunk: not 0 below 2^-126, so that an infinite state
// stays one, and not infinite where the state is 0, as the product of a growing
// state's factors is not.
__device__ __forceinline__ float over_chunk(float x, float h, float own) {
    const float e = exp2_fast(max_nan(x, -126.0f));
    return h == 0.0f && isinf(e) ? own : __fmaf_rn(e, h, own);
}
__device__ __forceinline__ St over_chunk(St x, St h, St own) {
    return {make_float2(over_chunk(x.a.x, h.a.x, own.a.x), over_chunk(x.a.y, h.a.y, own.a.y)),
            make_float2(over_chunk(x.b.x, h.b.x, own.b.x), over_chunk(x.b.y, h.b.y, own.b.y))};
}

// Turns each chunk's own end state into the state it starts from: a walk along
// the chunks, h <- exp(A sum dt) h + own.  REV: from the last chunk to the
// first, turning what each chunk passes on into what it receives from behind.
template <int LN, bool REV>
__global__ void __launch_bounds__(THREADS) join_kernel(const Args a) {
    constexpr int NP = 4 * LN;
    const int64_t item = (int64_t)blockIdx.x * THREADS + threadIdx.x;
    if (item >= (int64_t)a.batch * a.D * LN) return;
    const int n0 = 4 * (int)(item % LN), d = (int)(item / LN % a.D), b = (int)(item / LN / a.D);
    const St A2 = scaled(load4(a.A + (int64_t)d * a.N, n0, a.N));
    const float* init = REV ? a.dhT : a.h0;
    St h = st(init ? load4(init + ((int64_t)b * a.D + d) * a.N, n0, a.N) : make_float4(0, 0, 0, 0));
    const int last = REV ? 0 : a.chunks - 1;  // its own part is not needed
#pragma unroll 4
    for (int i = 0; i < a.chunks; i++) {
        const int ck = REV ? a.chunks - 1 - i : i;
        const int64_t row = ((int64_t)b * a.chunks + ck) * a.D + d;
        float4* p = reinterpret_cast<float4*>(a.cst + row * NP + n0);
        St own = st(make_float4(0, 0, 0, 0));
        float sum = 0.0f;
        if (ck != last) own = st(*p), sum = a.cdt[row];
        *p = f4(h);
        h = over_chunk(mul(A2, sum), h, own);
    }
}

// ---------------------------------------------------------------------------
// The scan of one chunk (the whole sequence with chunks = 1).  16 states, bf16,
// 8 x 2048 x 1536: 233 us, 1.7e12 decays a second, the issue slots 61 % busy, the
// special-function unit 45 %: 384 CTAs in two rounds of 296, the second one a
// third full.
template <typename T, int LN, int CPL, bool PAD>
__global__ void __launch_bounds__(CTA, 2) scan_kernel(const Args a) {
    using F = Cfg<T, LN, CPL>;
    constexpr int NP = F::NP, CB = F::CB, TT = F::TT;
    using Smem = typename F::template Smem<true>;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const int d0 = blockIdx.x * CB, b = blockIdx.y, ck = blockIdx.z;
    const int len = length_of(a, b);
    const int tb = ck * a.span, te = tb + a.span < a.L ? tb + a.span : a.L;
    const int end = te < len ? te : len;
    const int tiles = end > tb ? cdiv(end - tb, TT) : 0;  // tiles behind the length only get their zeros
    stage_param(sm.bias, a.bias, d0, a.D);
    stage_param(sm.skip, a.Dskip, d0, a.D);
    __syncthreads();
    if (threadIdx.x >= WORKERS) {
        give_registers();
        stagers<T, LN, CPL, SCAN>(a, sm, d0, b, tb, te, end, tiles);
        return;
    }
    take_registers();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nl = lane % LN, cl = lane / LN, n0 = 4 * nl;
    const int c0 = warp * F::CL * CPL + cl * CPL;
    const uint4 there = within<PAD>(n0, a.N);
    St A2[CPL], h[CPL];
    float2 lim[CPL];
#pragma unroll
    for (int j = 0; j < CPL; j++) {
        const int c = d0 + c0 + j;
        const bool in = c < a.D;
        A2[j] = scaled(in ? load4(a.A + (int64_t)c * a.N, n0, a.N) : make_float4(0, 0, 0, 0));
        float4 v = make_float4(0, 0, 0, 0);
        if (in && a.chunks > 1)
            v = *reinterpret_cast<const float4*>(a.cst + (((int64_t)b * a.chunks + ck) * a.D + c) * NP + n0);
        else if (in && a.h0)
            v = load4(a.h0 + ((int64_t)b * a.D + c) * a.N, n0, a.N);
        h[j] = st(v);
        St none = h[j];
        lim[j] = limits(A2[j], tiles > 0 ? h[j] : none);
    }
    float* keep = a.ckpt + (((int64_t)b * cdiv(a.L, CK) + tb / CK) * a.D + d0 + c0) * NP + n0;
    auto run = [&](auto signed_steps) {
#pragma unroll 1
        for (int i = 0; i < tiles; i++) {
            const int buf = i & 1, t0 = tb + i * TT;
#pragma unroll 1
            for (int r16 = 0; r16 < TT; r16 += CK) {
                if (a.ckpt && t0 + r16 < a.L) {
#pragma unroll
                    for (int j = 0; j < CPL; j++)
                        if (d0 + c0 + j < a.D) *reinterpret_cast<float4*>(keep + j * NP) = f4(h[j]);
                    keep += (int64_t)a.D * NP;
                }
                // 16 positions without a store in between, which would hold back the loads behind it
                constexpr int KEEP = LN == 2 ? 2 : 1;
                float out[CPL][4][KEEP];
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const int r4 = r16 + 4 * g;
                    St Bv[4], Cv[4];
                    float dt[4][CPL], v[4][CPL];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        Bv[k] = st(*reinterpret_cast<const float4*>(&sm.B[buf][r4 + k][n0]));
                        Cv[k] = st(*reinterpret_cast<const float4*>(&sm.C[buf][r4 + k][n0]));
                        staged<CPL>(sm.sd[buf][r4 + k], c0, k, dt[k], v[k]);
                    }
#pragma unroll
                    for (int j = 0; j < CPL; j++) {
                        const float dj[4] = {dt[0][j], dt[1][j], dt[2][j], dt[3][j]};
                        St e[4];
                        float y[4];
                        decays<decltype(signed_steps)::value>(A2[j], lim[j], dj, e);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            h[j] = only<PAD>(fma(e[k], h[j], mul(Bv[k], dup(v[k][j]))), there);
                            y[k] = dot(h[j], Cv[k]);
                        }
                        over_states<LN>(y);
#pragma unroll
                        for (int m = 0; m < KEEP; m++) out[j][g][m] = y[m];
                    }
                }
#pragma unroll
                for (int j = 0; j < CPL; j++)
#pragma unroll
                    for (int g = 0; g < 4; g++) store_positions<LN, F::YS>(&sm.y[buf][r16 + 4 * g][c0 + j], out[j][g], nl);
            }
            cta_barrier();
        }
    };
    cta_barrier();
    if (!PAD && a.softplus)  // with PAD one loop takes steps of either sign
        run(std::bool_constant<PAD>());
    else
        run(std::true_type());
    if (a.hT && ck == a.chunks - 1) {
#pragma unroll
        for (int j = 0; j < CPL; j++)
            if (d0 + c0 + j < a.D) store4(a.hT + ((int64_t)b * a.D + d0 + c0 + j) * a.N, n0, a.N, f4(h[j]));
    }
}

// ---------------------------------------------------------------------------
// Backward of one chunk.  Tiles of 16 positions, from the last to the first.
// From the state that the forward pass kept at a tile's start, 12 positions
// are run to find the states at positions 4, 8 and 12; then each block of 4,
// from the last, is run again with its decays and states held in registers,
// and walked backwards.  dB and dC are added over a lane's channels (where it
// has more than one), across the warp's channel lanes, and once a tile across
// the warps; sum_kernel adds the channel blocks.  PAD: also where lanes have
// channels beyond the last, which take no part in those sums (their zeros times
// an infinite B or C are none): 8 x 2048 x 1528 1010 us in training, 994 without.
//
// Across the channel lanes, a lane sends the half of its states that it does
// not keep.  Lanes hold their 4 states in an order of their own (state
// i ^ perm), so that what is kept always lies in the first registers and
// nothing has to be selected; B and C are staged once for each order.
//
// 16 states, 8 x 2048 x 1536 bf16, three chunks: 625 us.  255 registers a
// thread allow 8 warps an SM, and their latency bounds it: the issue slots are
// 43 % busy, and what a warp waits for is its own results and shared memory, by
// the counters hardly ever its loads, although a tile's have only the end of
// the tile before to arrive in.  The forward kernels' split of the warps, with
// the registers it leaves each, took longer.
template <typename T, int LN>
struct BCfg {
    static constexpr int NP = 4 * LN, CL = 32 / LN;
    static constexpr int CPL = LN == 2 ? 1 : LN == 16 ? 4 : 2, CB = 4 * CL * CPL;  // channels a lane, a CTA
    static constexpr int TT = CK, E = TT * CB / THREADS, VPR = CB / E;  // positions a tile; a thread stages E channels
    static constexpr int QUADS = (TT * LN + THREADS - 1) / THREADS;
    static constexpr int PERMS = CL < 4 ? CL : 4;  // orders of the states
    static constexpr int OS = CB + 8, BS = 2 * NP + 8;
    struct Smem {
        float4 sd[TT][CB / 2];                   // (dt, dt u) of two channels
        float ds[TT][CB];                        // dy z sigmoid(z)
        float B[PERMS][TT][NP], C[PERMS][TT][NP];
        float S[3][TT][OS];                      // sum_n g B, sum_n w A log2(e), sum_n C h
        float4 mid[4][CPL][3][32];               // by lane: the states at positions 4, 8 and 12
        float bc[4][TT][BS];                     // a warp's dB | dC
        float bias[CB], skip[CB];
        float4 kept[CPL][THREADS];               // by thread: the kept states of the next tile
        alignas(16) T raw[4][THREADS * E];       // by thread: u, delta, dy and z as they come
        alignas(16) T raw_bc[2][QUADS][THREADS * 4];
    };
};

__device__ __forceinline__ float2 swap(float2 v) { return make_float2(v.y, v.x); }
template <int PERMS>
__device__ __forceinline__ St permute(St s, int p) {
    if (p & 1) s.a = swap(s.a), s.b = swap(s.b);
    if (PERMS == 4 && (p & 2)) {
        const float2 t = s.a;
        s.a = s.b, s.b = t;
    }
    return s;
}
__device__ __forceinline__ float take(float keep, float send, int mask) {
    return __fadd_rn(keep, __shfl_xor_sync(0xffffffffu, send, mask));
}

template <typename T, int LN, bool PAD>
__global__ void __launch_bounds__(THREADS, 2) bwd_kernel(const Args a) {
    using F = BCfg<T, LN>;
    constexpr int NP = F::NP, CB = F::CB, CPL = F::CPL, TT = F::TT, CL = F::CL, PERMS = F::PERMS, E = F::E;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    typename F::Smem& sm = *reinterpret_cast<typename F::Smem*>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nl = lane % LN, cl = lane / LN, n0 = 4 * nl, perm = cl & (PERMS - 1);
    const int d0 = blockIdx.x * CB, b = blockIdx.y, ck = blockIdx.z;
    const int len = length_of(a, b);
    const int tb = ck * a.span, te = tb + a.span < a.L ? tb + a.span : a.L;
    const int end = te < len ? te : len;
    const int tiles = te > tb ? cdiv(te - tb, TT) : 0;
    const int active = end > tb ? cdiv(end - tb, TT) : 0;  // tiles behind the length change nothing
    const int lt = tid / F::VPR, lc = E * (tid % F::VPR), d = d0 + lc, have = a.D - d;
    const int c0 = warp * CL * CPL + cl * CPL;  // this lane's first channel in the CTA
    const uint4 there = within<PAD>(n0, a.N, perm);

    St A2[CPL], gc[CPL], dA[CPL];
#pragma unroll
    for (int j = 0; j < CPL; j++) {
        const int c = d0 + c0 + j;
        A2[j] = gc[j] = dA[j] = st(make_float4(0, 0, 0, 0));
        if (c < a.D) {
            A2[j] = permute<PERMS>(scaled(load4(a.A + (int64_t)c * a.N, n0, a.N)), perm);
            if (a.chunks > 1)
                gc[j] = st(*reinterpret_cast<const float4*>(a.cst + (((int64_t)b * a.chunks + ck) * a.D + c) * NP + n0));
            else if (a.dhT)
                gc[j] = st(load4(a.dhT + ((int64_t)b * a.D + c) * a.N, n0, a.N));
            gc[j] = permute<PERMS>(gc[j], perm);
        }
    }
    constexpr int AK = E / 4;  // dD and dbias of a quarter of this thread's channels, over 4 positions of each tile
    float accD[AK], accb[AK];
#pragma unroll
    for (int k = 0; k < AK; k++) accD[k] = accb[k] = 0.0f;

    // this thread's packs of 4 of a tile's dB | dC
    constexpr int PACKS = TT * 2 * NP / 4, PER = (PACKS + THREADS - 1) / THREADS, ROW4 = 2 * NP / 4;
    auto put_bc = [&](int t0, bool zero) {
        float* p = a.part_bc + (((int64_t)blockIdx.x * a.batch + b) * a.L + t0) * (2 * NP) + 4 * tid;
#pragma unroll
        for (int m = 0; m < PER; m++) {
            const int e = tid + m * THREADS, r = e / ROW4, k = 4 * (e % ROW4);
            if (e >= PACKS || t0 + r >= te) break;
            float4 x = make_float4(0, 0, 0, 0);
            if (!zero && t0 + r < end) {
                const float4 v0 = *reinterpret_cast<const float4*>(&sm.bc[0][r][k]);
                const float4 v1 = *reinterpret_cast<const float4*>(&sm.bc[1][r][k]);
                const float4 v2 = *reinterpret_cast<const float4*>(&sm.bc[2][r][k]);
                const float4 v3 = *reinterpret_cast<const float4*>(&sm.bc[3][r][k]);
                x.x = __fadd_rn(__fadd_rn(v0.x, v1.x), __fadd_rn(v2.x, v3.x));
                x.y = __fadd_rn(__fadd_rn(v0.y, v1.y), __fadd_rn(v2.y, v3.y));
                x.z = __fadd_rn(__fadd_rn(v0.z, v1.z), __fadd_rn(v2.z, v3.z));
                x.w = __fadd_rn(__fadd_rn(v0.w, v1.w), __fadd_rn(v2.w, v3.w));
            }
            *reinterpret_cast<float4*>(p + m * (4 * THREADS)) = x;
        }
    };
    auto put = [&](int t, const float (&du)[E], const float (&dd)[E], const float (&dz)[E]) {
        const int64_t o = ((int64_t)b * a.L + t) * a.D + d;
        store_pack<E>(static_cast<T*>(a.du) + o, du, have, a.ovec);
        store_pack<E>(static_cast<T*>(a.ddelta) + o, dd, have, a.ovec);
        if (a.z.p) store_pack<E>(static_cast<T*>(a.dz) + o, dz, have, a.ovec);
    };
    for (int i = active; i < tiles; i++) {
        float zero[E];
#pragma unroll
        for (int k = 0; k < E; k++) zero[k] = 0.0f;
        if (tb + i * TT + lt < te && have > 0) put(tb + i * TT + lt, zero, zero, zero);
        put_bc(tb + i * TT, true);
    }

    const int nq = 4 * (tid % LN), tq = tid / LN;
    stage_param(sm.bias, a.bias, d0, a.D);
    stage_param(sm.skip, a.Dskip, d0, a.D);
    __syncthreads();
    const int first = tb + (active - 1) * TT;
    const T *wu = row_of<T>(a.u, b, first + lt) + d, *wd = row_of<T>(a.delta, b, first + lt) + d;
    const T *wg = row_of<T>(a.dy, b, first + lt) + d, *wz = row_of<T>(a.z, b, first + lt) + d;
    const T *wB = row_of<T>(a.B, b, first + tq) + nq, *wC = row_of<T>(a.C, b, first + tq) + nq;
    const float* kp = a.ckpt + (((int64_t)b * cdiv(a.L, CK) + tb / CK + active - 1) * a.D + d0 + c0) * NP + n0;
    // a tile's inputs, into the slots that the tile behind it has left
    auto load = [&](int i) {
        const int t0 = tb + i * TT, valid = t0 + lt < end ? have : 0;
        fetch_pack<E>(&sm.raw[0][E * tid], wu, a.u.p, valid, a.u.vec);
        fetch_pack<E>(&sm.raw[1][E * tid], wd, a.delta.p, valid, a.delta.vec);
        fetch_pack<E>(&sm.raw[2][E * tid], wg, a.dy.p, valid, a.dy.vec);
        if (a.z.p) fetch_pack<E>(&sm.raw[3][E * tid], wz, a.z.p, valid, a.z.vec);
#pragma unroll
        for (int q = 0; q < F::QUADS; q++) {
            const int r = tq + q * (THREADS / LN), valid4 = t0 + r < end ? a.N - nq : 0;
            if (r >= TT) break;
            fetch_pack<4>(&sm.raw_bc[0][q][4 * tid], wB + q * (THREADS / LN) * a.B.sl, a.B.p, valid4, a.B.vec);
            fetch_pack<4>(&sm.raw_bc[1][q][4 * tid], wC + q * (THREADS / LN) * a.C.sl, a.C.p, valid4, a.C.vec);
        }
#pragma unroll
        for (int j = 0; j < CPL; j++) {
            const bool exists = d0 + c0 + j < a.D;
            cp_async<16>(&sm.kept[j][tid], exists ? kp + j * NP : a.ckpt, exists ? 16 : 0);
        }
        cp_async_commit();
        wu -= TT * a.u.sl, wd -= TT * a.delta.sl, wg -= TT * a.dy.sl, wz -= TT * a.z.sl;
        wB -= TT * a.B.sl, wC -= TT * a.C.sl, kp -= (int64_t)a.D * NP;
    };
    if (active > 0) load(active - 1);
    for (int i = active - 1; i >= 0; i--) {
        const int t0 = tb + i * TT, t = t0 + lt;
        const bool in = t < end;
        cp_async_wait();
        {
            const Pack<T, E> eu = slot_pack<E>(&sm.raw[0][E * tid]), ed = slot_pack<E>(&sm.raw[1][E * tid]);
            const Pack<T, E> eg = slot_pack<E>(&sm.raw[2][E * tid]), ez = slot_pack<E>(&sm.raw[3][E * tid]);
            float dt[E], v[E], g[E];
            getk<E>(&sm.bias[lc], dt);
#pragma unroll
            for (int k = 0; k < E; k++) {
                dt[k] = __fadd_rn(to_f(ed.v[k]), dt[k]);
                if (a.softplus) dt[k] = softplus(dt[k]);
                if (!in) dt[k] = 0.0f;
                v[k] = __fmul_rn(dt[k], to_f(eu.v[k]));
                g[k] = to_f(eg.v[k]);
                if (a.z.p) {
                    const float z = to_f(ez.v[k]);
                    g[k] = __fmul_rn(g[k], __fmul_rn(z, sigmoid(z)));
                }
            }
            stage_steps<E>(sm.sd[lt], lc, lt, dt, v);
            setk<E>(&sm.ds[lt][lc], g);
        }
#pragma unroll
        for (int q = 0; q < F::QUADS; q++) {
            const int r = tq + q * (THREADS / LN);
            if (r >= TT) break;
            const St sB = st(quad(slot_pack<4>(&sm.raw_bc[0][q][4 * tid])));
            const St sC = st(quad(slot_pack<4>(&sm.raw_bc[1][q][4 * tid])));
#pragma unroll
            for (int p = 0; p < PERMS; p++) {
                *reinterpret_cast<float4*>(&sm.B[p][r][nq]) = f4(permute<PERMS>(sB, p));
                *reinterpret_cast<float4*>(&sm.C[p][r][nq]) = f4(permute<PERMS>(sC, p));
            }
        }
        __syncthreads();
        {
            St h[CPL], mid[3][CPL];
#pragma unroll
            for (int j = 0; j < CPL; j++) h[j] = permute<PERMS>(st(sm.kept[j][tid]), perm);
#pragma unroll
            for (int q = 0; q < 3; q++) {
                St Bv[4];
                float dt[4][CPL], v[4][CPL];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    Bv[k] = st(*reinterpret_cast<const float4*>(&sm.B[perm][4 * q + k][n0]));
                    staged<CPL>(sm.sd[4 * q + k], c0, k, dt[k], v[k]);
                }
#pragma unroll
                for (int j = 0; j < CPL; j++) {
                    const float dj[4] = {dt[0][j], dt[1][j], dt[2][j], dt[3][j]};
                    St e[4];
                    decays<sizeof(T) == 4>(A2[j], dj, e);
#pragma unroll
                    for (int k = 0; k < 4; k++) h[j] = only<PAD>(fma(e[k], h[j], mul(Bv[k], dup(v[k][j]))), there);
                    mid[q][j] = h[j];
                }
            }
#pragma unroll
            for (int q = 0; q < 3; q++)
#pragma unroll
                for (int j = 0; j < CPL; j++) sm.mid[warp][j][q][lane] = f4(mid[q][j]);
        }
#pragma unroll 1
        for (int q = 3; q >= 0; q--) {
            St Bv[4], Cv[4], vB[4], vC[4];
            float dt[4][CPL], v[4][CPL], ds[4][CPL];
            const int inside = end - (t0 + 4 * q);  // behind the end dt is 0, which an infinite state times it is not
#pragma unroll
            for (int k = 0; k < 4; k++) {
                Bv[k] = st(*reinterpret_cast<const float4*>(&sm.B[perm][4 * q + k][n0]));
                Cv[k] = st(*reinterpret_cast<const float4*>(&sm.C[perm][4 * q + k][n0]));
                staged<CPL>(sm.sd[4 * q + k], c0, k, dt[k], v[k]);
                getk<CPL>(&sm.ds[4 * q + k][c0], ds[k]);
            }
            float out[3][CPL][4];
#pragma unroll
            for (int j = 0; j < CPL; j++) {
                const float dj[4] = {dt[0][j], dt[1][j], dt[2][j], dt[3][j]};
                const St h0 = q ? st(sm.mid[warp][j][q ? q - 1 : 0][lane]) : permute<PERMS>(st(sm.kept[j][tid]), perm);
                St e[4], h[4];
                decays<sizeof(T) == 4>(A2[j], dj, e);
#pragma unroll
                for (int k = 0; k < 4; k++)
                    h[k] = only<PAD>(fma(e[k], k ? h[k ? k - 1 : 0] : h0, mul(Bv[k], dup(v[k][j]))), there);
#pragma unroll
                for (int k = 3; k >= 0; k--) {
                    const float2 dsk = dup(ds[k][j]);
                    const St g = only<PAD>(fma(Cv[k], dsk, gc[j]), there);
                    if constexpr (PAD) {
                        if (!j) vB[k] = vC[k] = st(make_float4(0, 0, 0, 0));
                        if (d0 + c0 + j < a.D) vB[k] = fma(g, dup(v[k][j]), vB[k]), vC[k] = fma(h[k], dsk, vC[k]);
                    } else {
                        vB[k] = j ? fma(g, dup(v[k][j]), vB[k]) : mul(g, dup(v[k][j]));
                        vC[k] = j ? fma(h[k], dsk, vC[k]) : mul(h[k], dsk);
                    }
                    out[0][j][k] = dot(g, Bv[k]);
                    gc[j] = only<PAD>(mul(e[k], g), there);
                    const St w = mul(gc[j], k ? h[k ? k - 1 : 0] : h0);
                    out[1][j][k] = dot(w, A2[j]);
                    out[2][j][k] = dot(h[k], Cv[k]);
                    if (k < inside) dA[j] = fma(w, dup(dj[k]), dA[j]);
                }
#pragma unroll
                for (int m = 0; m < 3; m++) over_states<LN>(out[m][j]);
            }
            // over the warp's channel lanes
            float f[16];
            int pos = 0;
            if constexpr (PERMS == 4) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    f[2 * k] = take(take(vB[k].a.x, vB[k].b.x, 2 * LN), take(vB[k].a.y, vB[k].b.y, 2 * LN), LN);
                    f[2 * k + 1] = take(take(vC[k].a.x, vC[k].b.x, 2 * LN), take(vC[k].a.y, vC[k].b.y, 2 * LN), LN);
                }
                if constexpr (CL >= 8) halve<8>(f, 4 * LN), pos = ((cl >> 2) & 1) * 2;
                if constexpr (CL == 16) halve<4>(f, 8 * LN), pos += (cl >> 3) & 1;
            } else {  // two channel lanes: each keeps two states
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    f[4 * k] = take(vB[k].a.x, vB[k].a.y, LN), f[4 * k + 1] = take(vB[k].b.x, vB[k].b.y, LN);
                    f[4 * k + 2] = take(vC[k].a.x, vC[k].a.y, LN), f[4 * k + 3] = take(vC[k].b.x, vC[k].b.y, LN);
                }
            }
#pragma unroll
            for (int m = 0; m < 3; m++)
#pragma unroll
                for (int j = 0; j < CPL; j++) store_positions<LN, F::OS>(&sm.S[m][4 * q][c0 + j], out[m][j], nl);
            if constexpr (PERMS == 4) {
#pragma unroll
                for (int k = 0; k < 16 / CL && k < 4; k++) {
                    sm.bc[warp][4 * q + pos + k][n0 + perm] = f[2 * k];
                    sm.bc[warp][4 * q + pos + k][NP + n0 + perm] = f[2 * k + 1];
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    float* row = sm.bc[warp][4 * q + k] + n0 + perm;
                    row[0] = f[4 * k], row[2] = f[4 * k + 1], row[NP] = f[4 * k + 2], row[NP + 2] = f[4 * k + 3];
                }
            }
        }
        __syncthreads();
        float pD[E], pb[E];  // this position's terms of dD and dbias
#pragma unroll
        for (int k = 0; k < E; k++) pD[k] = pb[k] = 0.0f;
        if (t < te && have > 0) {
            const Pack<T, E> eu = slot_pack<E>(&sm.raw[0][E * tid]), ed = slot_pack<E>(&sm.raw[1][E * tid]);
            const Pack<T, E> eg = slot_pack<E>(&sm.raw[2][E * tid]), ez = slot_pack<E>(&sm.raw[3][E * tid]);
            float du[E], dd[E], dz[E], s1[E], ds[E], sc[E], skip[E], bias[E];
            getk<E>(&sm.S[0][lt][lc], s1);
            getk<E>(&sm.S[1][lt][lc], dd);
            getk<E>(&sm.S[2][lt][lc], sc);
            getk<E>(&sm.ds[lt][lc], ds);
            getk<E>(&sm.skip[lc], skip);
            getk<E>(&sm.bias[lc], bias);
#pragma unroll
            for (int k = 0; k < E; k += 2) {
                const float4 x = sm.sd[lt][place((lc + k) >> 1, lt)];
                du[k] = __fmul_rn(x.x, s1[k]), du[k + 1] = __fmul_rn(x.z, s1[k + 1]);
            }
#pragma unroll
            for (int k = 0; k < E; k++) {
                const float u = to_f(eu.v[k]);
                dd[k] = __fmaf_rn(u, s1[k], __fmul_rn(dd[k], LN2));
                if (a.Dskip) {
                    du[k] = __fmaf_rn(skip[k], ds[k], du[k]);
                    sc[k] = __fmaf_rn(skip[k], u, sc[k]);
                }
                if (a.softplus) dd[k] = __fmul_rn(dd[k], sigmoid(__fadd_rn(to_f(ed.v[k]), bias[k])));
                dz[k] = 0.0f;
                if (a.z.p) {
                    const float z = to_f(ez.v[k]), sg = sigmoid(z);
                    dz[k] = __fmul_rn(__fmul_rn(to_f(eg.v[k]), sc[k]),
                                      __fmul_rn(sg, __fmaf_rn(z, __fsub_rn(1.0f, sg), 1.0f)));
                }
                if (!in) du[k] = dd[k] = dz[k] = 0.0f;
                pD[k] = in ? __fmul_rn(ds[k], u) : 0.0f;
                pb[k] = dd[k];
            }
            put(t, du, dd, dz);
        }
        if (i > 0) load(i - 1);
        put_bc(t0, false);
        // over the warp's positions: lanes VPR (and 2 VPR) apart
        static_assert(F::VPR == 8, "4 positions a warp");
        halve<E>(pD, 8), halve<E>(pb, 8);
        halve<E / 2>(pD, 16), halve<E / 2>(pb, 16);
#pragma unroll
        for (int k = 0; k < AK; k++) accD[k] = __fadd_rn(accD[k], pD[k]), accb[k] = __fadd_rn(accb[k], pb[k]);
        __syncthreads();
    }
    const int64_t bk = (int64_t)b * a.chunks + ck;
#pragma unroll
    for (int j = 0; j < CPL; j++) {
        const int c = d0 + c0 + j;
        if (c >= a.D) break;
        *reinterpret_cast<float4*>(a.part_a + (bk * a.D + c) * NP + n0) = f4(permute<PERMS>(dA[j], perm));
        if (ck == 0 && a.dh0)
            store4(a.dh0 + ((int64_t)b * a.D + c) * a.N, n0, a.N, f4(permute<PERMS>(gc[j], perm)));
    }
    // what the halvings left with this thread
    const int off = ((lane >> 3) & 1) * (E / 2) + (lane >> 4) * (E / 4);
#pragma unroll
    for (int k = 0; k < AK; k++) sm.S[0][warp][lc + off + k] = accD[k], sm.S[1][warp][lc + off + k] = accb[k];
    __syncthreads();
    for (int e = tid; e < 2 * CB; e += THREADS) {
        const int c = e % CB, k = e / CB;
        if (d0 + c >= a.D) continue;
        float x = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; r++) x = __fadd_rn(x, sm.S[k][r][c]);
        a.part_d[(bk * 2 + k) * a.D + d0 + c] = x;
    }
}

// The partial sums, added in order.  The first `bc` blocks: dB and dC, over the
// channel blocks; the others: dA, dD and dbias, over the sequences and chunks.
struct Sums {
    const float *part_bc, *part_a, *part_d;
    void *dB, *dC;
    float *dA, *dD, *db;
    int64_t rows;
    int blocks, bc, P, D, N, NP;
};
__device__ __forceinline__ float strands(const float* p, int64_t step, int n) {
    float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    int i = 0;
    for (; i + 7 < n; i += 8)
#pragma unroll
        for (int j = 0; j < 8; j++) s[j] = __fadd_rn(s[j], p[(i + j) * step]);
    for (int j = 0; i < n; i++, j++) s[0] = __fadd_rn(s[0], p[i * step]);
    return __fadd_rn(__fadd_rn(__fadd_rn(s[0], s[1]), __fadd_rn(s[2], s[3])),
                     __fadd_rn(__fadd_rn(s[4], s[5]), __fadd_rn(s[6], s[7])));
}
template <typename T>
__global__ void __launch_bounds__(256) sum_kernel(const Sums a) {
    if ((int)blockIdx.x < a.bc) {
        const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
        const int k = (int)(e % (2 * a.NP)), n = k % a.NP;
        T* o = static_cast<T*>(k < a.NP ? a.dB : a.dC);
        if (e >= a.rows * 2 * a.NP || n >= a.N || !o) return;
        o[e / (2 * a.NP) * a.N + n] = from_f<T>(strands(a.part_bc + e, a.rows * 2 * a.NP, a.blocks));
        return;
    }
    const int64_t e = (int64_t)(blockIdx.x - a.bc) * 256 + threadIdx.x, DN = (int64_t)a.D * a.NP;
    if (e < DN) {
        const int n = (int)(e % a.NP);
        if (n < a.N && a.dA) a.dA[e / a.NP * a.N + n] = strands(a.part_a + e, DN, a.P);
    } else if (e < DN + 2 * a.D) {
        const int64_t f = e - DN;
        float* o = f < a.D ? a.dD : a.db;
        if (o) o[f % a.D] = strands(a.part_d + f, 2 * a.D, a.P);
    }
}

// ---------------------------------------------------------------------------
// One new token a stream: the state is read and written once, 8 bytes a state,
// which bounds it: 16 states, 256 x 2048 bf16, 18.2 us
// for 71 MB.  LN lanes a channel as above; a thread takes ROWS streams
// of its channel, so that A and the channel's parameters are read once for
// them and all their loads are on their way together.  VEC: N is a multiple
// of 4 and B and C are aligned, so that nothing is loaded behind a branch.
template <typename T, int LN, int ROWS, bool VEC>
__global__ void __launch_bounds__(THREADS) step_kernel(const Args a) {
    const int64_t item = ((int64_t)blockIdx.x * THREADS + threadIdx.x) / LN;
    const int n0 = 4 * (threadIdx.x % LN);
    grid_dependency_sync();
    const int d = (int)(item % a.D), b0 = (int)(item / a.D) * ROWS;
    const bool quad_in = n0 < a.N;
    const int nc = quad_in ? n0 : 0;
    float4 hv[ROWS], Av;
    Pack<T, 4> pB[ROWS], pC[ROWS];
    T tu[ROWS], td[ROWS], tz[ROWS];
    // streams beyond the last and states beyond the last quad read others' values, and use none
    Av = VEC ? *reinterpret_cast<const float4*>(a.A + (int64_t)d * a.N + nc) : load4(a.A + (int64_t)d * a.N, n0, a.N);
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const int b = b0 + r < a.batch ? b0 + r : a.batch - 1;
        const float* hp = a.hT + ((int64_t)b * a.D + d) * a.N;
        if (VEC) {
            hv[r] = *reinterpret_cast<const float4*>(hp + nc);
            pB[r] = *reinterpret_cast<const Pack<T, 4>*>(row_of<T>(a.B, b, 0) + nc);
            pC[r] = *reinterpret_cast<const Pack<T, 4>*>(row_of<T>(a.C, b, 0) + nc);
        } else {
            hv[r] = load4(hp, n0, a.N);
            pB[r] = load_pack<4>(row_of<T>(a.B, b, 0) + n0, a.N - n0, a.B.vec);
            pC[r] = load_pack<4>(row_of<T>(a.C, b, 0) + n0, a.N - n0, a.C.vec);
        }
        tu[r] = row_of<T>(a.u, b, 0)[d];
        td[r] = row_of<T>(a.delta, b, 0)[d];
        tz[r] = (a.z.p ? row_of<T>(a.z, b, 0) : row_of<T>(a.u, b, 0))[d];
    }
    const float bias = a.bias ? a.bias[d] : 0.0f, skip = a.Dskip ? a.Dskip[d] : 0.0f;
    if (VEC && !quad_in) {
        Av = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            hv[r] = Av;
#pragma unroll
            for (int i = 0; i < 4; i++) pB[r].v[i] = pC[r].v[i] = from_f<T>(0.0f);
        }
    }
    const St A2 = scaled(Av);
    const uint4 there = within<true>(n0, a.N);
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const int b = b0 + r;
        const bool live = b < a.batch;
        const float u = to_f(tu[r]);
        float t = __fadd_rn(to_f(td[r]), bias);
        if (a.softplus) t = softplus(t);
        const St h = only<true>(fma(exp2s(mul(A2, dup(t))), st(hv[r]), mul(st(quad(pB[r])), dup(__fmul_rn(t, u)))), there);
        if (live) store4(a.hT + ((int64_t)b * a.D + d) * a.N, n0, a.N, f4(h));
        float y = dot(h, st(quad(pC[r])));
#pragma unroll
        for (int m = 1; m < LN; m *= 2) y = __fadd_rn(y, __shfl_xor_sync(0xffffffffu, y, m));
        if (live && n0 == 0) {
            y = __fmaf_rn(skip, u, y);
            if (a.z.p) {
                const float z = to_f(tz[r]);
                y = __fmul_rn(y, __fmul_rn(z, sigmoid(z)));
            }
            static_cast<T*>(a.y)[(int64_t)b * a.D + d] = from_f<T>(y);
        }
    }
}

// ---------------------------------------------------------------------------
static inline int lanes_of(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

static inline int bwd_channels(int N) { return lanes_of(N) <= 4 ? BCfg<float, 4>::CB : BCfg<float, 8>::CB; }
static_assert(BCfg<float, 2>::CB == BCfg<float, 4>::CB && BCfg<float, 8>::CB == BCfg<float, 16>::CB, "bwd_channels");

// Channels a lane of the forward kernels.  Two share their loads of B and C,
// but make CTAs of 64 channels: with fewer than 4 of those an SM, the SMs with
// one more than the others cost more than the loads.  16 states, two against
// one: 64 x 512 x 2048 474 us and 505; 8 x 2048 x 1536 271 and 234; ragged
// prompts of 6 x 777 x 2048 85 and 55.
static inline int fwd_cpl(int batch, int D, int N) {
    const int LN = lanes_of(N);
    if (LN == 4) return (int64_t)batch * cdiv(D, 64) >= 148 * 4 ? 2 : 1;
    return LN == 2 ? 1 : LN == 8 ? 2 : 4;
}
static inline int fwd_channels(int batch, int D, int N) { return 4 * (32 / lanes_of(N)) * fwd_cpl(batch, D, N); }

// Chunks of the sequence, of 64 positions at least.  The chunks' states cost a
// pass of their own over all but one of them, which makes each exponential
// once more.
struct Plan {
    int chunks, span;
};
static inline Plan plan_of(int L, int64_t n) {
    Plan p = {1, cdiv(L, 32) * 32};
    if (n * 64 > L) n = L / 64;
    if (n < 2) return p;
    p.span = cdiv(cdiv(L, (int)n), 32) * 32;
    p.chunks = cdiv(L, p.span);
    return p;
}
// Forward: only where the channels alone leave SMs idle, and then as many as
// bring 2 CTAs to each.  With 384 CTAs (8 x 2048 x 1536) one chunk took 229 us,
// three 194 and 104 for their states; with 48 (one sequence of it) one took
// 98, six 29 and 24 for their states.
static inline Plan forward_plan(int batch, int L, int D, int N) {
    const int64_t ctas = (int64_t)batch * cdiv(D, fwd_channels(batch, D, N));
    return plan_of(L, ctas >= 148 || ctas == 0 ? 1 : 2 * 148 / ctas);
}
// Backward: 2 CTAs an SM at once, in rounds of 296 that take as long for one
// CTA on an SM as for two.  The number of least rounds / chunks +
// (chunks - 1) / 4 chunks, a quarter being what the pass for all chunks'
// states takes of the kernel's time: 8 x 2048 x 1536, 192 CTAs, 923 us in one
// chunk and 617 in three, with 104 for their states.
static inline Plan backward_plan(int batch, int L, int D, int N) {
    const int64_t ctas = (int64_t)batch * cdiv(D, bwd_channels(N));
    Plan best = {1, cdiv(L, 32) * 32};
    double least = 1e30;
    for (int n = 1; n <= 16 && (n == 1 || n * 64 <= L); n++) {
        const Plan p = plan_of(L, n);
        const double cost = (double)((ctas * p.chunks + 295) / 296) * p.span / L + 0.25 * (p.chunks - 1) / p.chunks;
        if (cost < least) least = cost, best = p;
    }
    return best;
}

static inline int64_t align16(int64_t floats) { return (floats + 3) & ~(int64_t)3; }

struct Ws {  // floats from the workspace's start
    int64_t cst, cdt, part_bc, part_a, part_d, total;
};
static inline Ws ws_of(int batch, int L, int D, int N, bool backward) {
    const int LN = lanes_of(N), NP = 4 * LN;
    const Plan p = backward ? backward_plan(batch, L, D, N) : forward_plan(batch, L, D, N);
    Ws w = {};
    int64_t at = 0;
    auto take = [&](int64_t n) {
        const int64_t o = at;
        at += align16(n);
        return o;
    };
    if (p.chunks > 1) {
        w.cst = take((int64_t)batch * p.chunks * D * NP);
        w.cdt = take((int64_t)batch * p.chunks * D);
    }
    if (backward) {
        w.part_bc = take((int64_t)cdiv(D, bwd_channels(N)) * batch * L * 2 * NP);
        w.part_a = take((int64_t)batch * p.chunks * D * NP);
        w.part_d = take((int64_t)batch * p.chunks * 2 * D);
    }
    w.total = at;
    return w;
}

// `unit` elements of `size` bytes are read at once (in pieces of 16 bytes at most)
static inline Seq seq(const void* p, int64_t sb, int64_t sl, int unit, int size) {
    Seq s = {p, sb, sl, 0};
    const int bytes = unit * size < 16 ? unit * size : 16;
    s.vec = reinterpret_cast<uintptr_t>(p) % bytes == 0 && sb * size % bytes == 0 && sl * size % bytes == 0;
    return s;
}

static int check(int batch, int L, int D, int N, int dtype) {
    if (batch < 0 || L < 0 || D <= 0 || N <= 0) return MI_ERR_INVALID;
    if (dtype != MI_DT_F32 && dtype != MI_DT_BF16 && dtype != MI_DT_F16) return MI_ERR_INVALID;
    if (N > MAX_N || batch > 65535) return MI_ERR_UNSUPPORTED;
    return MI_OK;
}

// the chunks' starting states (REV: what they receive from behind), in a.cst
template <typename T, int LN, int CPL, bool REV, bool PAD>
static int start_chunks(const Args& a, cudaStream_t s) {
    using F = Cfg<T, LN, CPL>;
    constexpr size_t smem = sizeof(typename F::template Smem<false>);
    static std::atomic<uint64_t> allowed{0};
    if (!allow_smem(chunk_kernel<T, LN, CPL, REV, PAD>, smem, allowed, CTA_REGS)) return MI_ERR_CUDA;
    chunk_kernel<T, LN, CPL, REV, PAD><<<dim3(cdiv(a.D, F::CB), a.batch, a.chunks - 1), CTA, smem, s>>>(a);
    MI_CHECK_LAUNCH();
    const int64_t items = (int64_t)a.batch * a.D * LN;
    join_kernel<LN, REV><<<(unsigned)((items + THREADS - 1) / THREADS), THREADS, 0, s>>>(a);
    MI_CHECK_LAUNCH();
    return MI_OK;
}

template <typename T, int LN, int CPL, bool PAD>
static int forward_cpl(Args& a, float* ws, cudaStream_t s) {
    using F = Cfg<T, LN, CPL>;
    const Plan p = forward_plan(a.batch, a.L, a.D, a.N);
    a.chunks = p.chunks, a.span = p.span;
    if constexpr (LN != 4 || CPL != 2) {  // two channels a lane come with 592 CTAs, and those with one chunk
        if (p.chunks > 1) {
            const Ws w = ws_of(a.batch, a.L, a.D, a.N, false);
            a.cst = ws + w.cst, a.cdt = ws + w.cdt;
            const int rc = start_chunks<T, LN, CPL, false, PAD>(a, s);
            if (rc != MI_OK) return rc;
        }
    }
    constexpr size_t smem = sizeof(typename F::template Smem<true>);
    static std::atomic<uint64_t> allowed{0};
    if (!allow_smem(scan_kernel<T, LN, CPL, PAD>, smem, allowed, CTA_REGS)) return MI_ERR_CUDA;
    scan_kernel<T, LN, CPL, PAD><<<dim3(cdiv(a.D, F::CB), a.batch, p.chunks), CTA, smem, s>>>(a);
    MI_CHECK_LAUNCH();
    return MI_OK;
}

template <typename T, int LN, bool PAD>
static int forward_pad(Args& a, float* ws, cudaStream_t s) {
    if constexpr (LN == 4) {
        if (fwd_cpl(a.batch, a.D, a.N) == 2) return forward_cpl<T, 4, 2, PAD>(a, ws, s);
        return forward_cpl<T, 4, 1, PAD>(a, ws, s);
    } else {
        return forward_cpl<T, LN, LN == 2 ? 1 : LN == 8 ? 2 : 4, PAD>(a, ws, s);
    }
}
template <typename T, int LN>
static int forward(Args& a, float* ws, cudaStream_t s) {
    return a.N < 4 * LN ? forward_pad<T, LN, true>(a, ws, s) : forward_pad<T, LN, false>(a, ws, s);
}

template <typename T, int LN, int ROWS, bool VEC>
static int step_rows(Args& a, cudaStream_t s) {
    const int64_t threads = (int64_t)cdiv(a.batch, ROWS) * a.D * LN;
    MI_LAUNCH_DEPENDENT(step_kernel<T, LN, ROWS, VEC>, (unsigned)((threads + THREADS - 1) / THREADS), THREADS, 0, s, a);
    return MI_OK;
}

// 4 streams a thread where that leaves every SM its 1024 threads (256 x 2048
// bf16: 18.2 us against 22.3 with 1; 2 take 18.3, 8 take 24); 1 elsewhere (4 x
// 512: 2.0 us against 2.7).
template <typename T, int LN>
static int step(Args& a, float*, cudaStream_t s) {
    if (a.N % 4 || !a.B.vec || !a.C.vec) return step_rows<T, LN, 1, false>(a, s);
    if ((int64_t)a.batch * a.D * LN >= 148 * 1024 * 4) return step_rows<T, LN, 4, true>(a, s);
    return step_rows<T, LN, 1, true>(a, s);
}

template <typename T, int LN, bool PAD>
static int backward_pad(Args& a, float* ws, cudaStream_t s) {
    using F = BCfg<T, LN>;
    const Plan p = backward_plan(a.batch, a.L, a.D, a.N);
    a.chunks = p.chunks, a.span = p.span;
    const Ws w = ws_of(a.batch, a.L, a.D, a.N, true);
    a.part_bc = ws + w.part_bc, a.part_a = ws + w.part_a, a.part_d = ws + w.part_d;
    if (p.chunks > 1) {
        a.cst = ws + w.cst, a.cdt = ws + w.cdt;
        constexpr int CPL = LN == 2 ? 1 : LN == 16 ? 4 : LN == 8 ? 2 : 1;
        const int rc = a.N < 4 * LN ? start_chunks<T, LN, CPL, true, true>(a, s) : start_chunks<T, LN, CPL, true, false>(a, s);
        if (rc != MI_OK) return rc;
    }
    constexpr size_t smem = sizeof(typename F::Smem);
    static std::atomic<uint64_t> allowed{0};
    if (!allow_smem(bwd_kernel<T, LN, PAD>, smem, allowed)) return MI_ERR_CUDA;
    bwd_kernel<T, LN, PAD><<<dim3(cdiv(a.D, F::CB), a.batch, p.chunks), THREADS, smem, s>>>(a);
    MI_CHECK_LAUNCH();
    return MI_OK;
}
template <typename T, int LN>
static int backward(Args& a, float* ws, cudaStream_t s) {
    return a.N < 4 * LN || a.D % BCfg<T, LN>::CB ? backward_pad<T, LN, true>(a, ws, s) : backward_pad<T, LN, false>(a, ws, s);
}

}  // namespace sscan
}  // namespace mi

#define MI_SSCAN_STATES(N, FN, T, ...)                            \
    do {                                                          \
        const int ln_ = mi::sscan::lanes_of(N);                   \
        if (ln_ == 2) return mi::sscan::FN<T, 2>(__VA_ARGS__);    \
        if (ln_ == 4) return mi::sscan::FN<T, 4>(__VA_ARGS__);    \
        if (ln_ == 8) return mi::sscan::FN<T, 8>(__VA_ARGS__);    \
        return mi::sscan::FN<T, 16>(__VA_ARGS__);                 \
    } while (0)

template <typename T>
static int mi_sscan_backward_states(mi::sscan::Args& a, float* ws, cudaStream_t s) {
    MI_SSCAN_STATES(a.N, backward, T, a, ws, s);
}

extern "C" int64_t mi_selective_scan_checkpoints(int batch, int L, int D, int N) {
    if (mi::sscan::check(batch, L, D, N, MI_DT_F32) != MI_OK) return 0;
    return (int64_t)batch * mi::cdiv(L, mi::sscan::CK) * D * 4 * mi::sscan::lanes_of(N);
}

extern "C" int64_t mi_selective_scan_workspace(int batch, int L, int D, int N, int backward) {
    if (mi::sscan::check(batch, L, D, N, MI_DT_F32) != MI_OK || batch == 0 || L == 0) return 0;
    return (int64_t)sizeof(float) * mi::sscan::ws_of(batch, L, D, N, backward != 0).total;
}

extern "C" int mi_selective_scan(const void* u, int64_t u_batch, int64_t u_row, const void* delta, int64_t delta_batch,
                                 int64_t delta_row, const float* A, const void* B, int64_t B_batch, int64_t B_row,
                                 const void* C, int64_t C_batch, int64_t C_row, const float* D, const void* z,
                                 int64_t z_batch, int64_t z_row, const float* delta_bias, const float* h0,
                                 const int32_t* lengths, void* y, float* h_out, float* checkpoints, void* workspace,
                                 int batch, int L, int Dm, int N, int softplus, int dtype, void* stream) {
    using namespace mi::sscan;
    const int rc = check(batch, L, Dm, N, dtype);
    if (rc != MI_OK) return rc;
    if (batch == 0) return MI_OK;
    if (L == 0) return MI_ERR_INVALID;  // nothing to scan: the caller's state is the initial one
    if (!u || !delta || !A || !B || !C || !y) return MI_ERR_INVALID;
    if (!workspace && ws_of(batch, L, Dm, N, false).total) return MI_ERR_INVALID;
    if (!mi::aligned16(A) || !mi::aligned16(h0) || !mi::aligned16(h_out) || !mi::aligned16(checkpoints) ||
        !mi::aligned16(workspace))
        return MI_ERR_INVALID;
    Args a = {};
    const int size = dtype == MI_DT_F32 ? 4 : 2;
    a.u = seq(u, u_batch, u_row, 8, size), a.delta = seq(delta, delta_batch, delta_row, 8, size);
    a.z = seq(z, z_batch, z_row, 8, size), a.B = seq(B, B_batch, B_row, 4, size), a.C = seq(C, C_batch, C_row, 4, size);
    a.A = A, a.Dskip = D, a.bias = delta_bias, a.h0 = h0, a.lengths = lengths;
    a.y = y, a.hT = h_out, a.ckpt = checkpoints;
    a.batch = batch, a.L = L, a.D = Dm, a.N = N, a.softplus = softplus;
    a.ovec = Dm % 8 == 0 && mi::aligned16(y);
    float* ws = static_cast<float*>(workspace);
    MI_DISPATCH_DTYPE(dtype, T, MI_SSCAN_STATES(N, forward, T, a, ws, (cudaStream_t)stream));
    return MI_ERR_INVALID;
}

extern "C" int mi_selective_scan_step(const void* u, int64_t u_batch, const void* delta, int64_t delta_batch,
                                      const float* A, const void* B, int64_t B_batch, const void* C, int64_t C_batch,
                                      const float* D, const void* z, int64_t z_batch, const float* delta_bias,
                                      float* h, void* y, int batch, int Dm, int N, int softplus, int dtype,
                                      void* stream) {
    using namespace mi::sscan;
    const int rc = check(batch < 0 ? -1 : 0, 1, Dm, N, dtype);
    if (rc != MI_OK) return rc;
    if (batch == 0) return MI_OK;
    if (!u || !delta || !A || !B || !C || !h || !y) return MI_ERR_INVALID;
    if (!mi::aligned16(A) || !mi::aligned16(h)) return MI_ERR_INVALID;
    Args a = {};
    const int size = dtype == MI_DT_F32 ? 4 : 2;
    a.u = seq(u, u_batch, 0, 8, size), a.delta = seq(delta, delta_batch, 0, 8, size), a.z = seq(z, z_batch, 0, 8, size);
    a.B = seq(B, B_batch, 0, 4, size), a.C = seq(C, C_batch, 0, 4, size);
    a.A = A, a.Dskip = D, a.bias = delta_bias, a.hT = h, a.y = y;
    a.batch = batch, a.L = 1, a.D = Dm, a.N = N, a.softplus = softplus;
    MI_DISPATCH_DTYPE(dtype, T, MI_SSCAN_STATES(N, step, T, a, nullptr, (cudaStream_t)stream));
    return MI_ERR_INVALID;
}

extern "C" int mi_selective_scan_backward(
    const void* dy, int64_t dy_batch, int64_t dy_row, const float* dh_out, const void* u, int64_t u_batch,
    int64_t u_row, const void* delta, int64_t delta_batch, int64_t delta_row, const float* A, const void* B,
    int64_t B_batch, int64_t B_row, const void* C, int64_t C_batch, int64_t C_row, const float* D, const void* z,
    int64_t z_batch, int64_t z_row, const float* delta_bias, const int32_t* lengths, const float* checkpoints,
    void* du, void* ddelta, float* dA, void* dB, void* dC, float* dD, void* dz, float* ddelta_bias, float* dh0,
    void* workspace, int batch, int L, int Dm, int N, int softplus, int dtype, void* stream) {
    using namespace mi::sscan;
    const int rc = check(batch, L, Dm, N, dtype);
    if (rc != MI_OK) return rc;
    if (batch == 0 || L == 0) return MI_ERR_INVALID;
    if (!dy || !u || !delta || !A || !B || !C || !checkpoints || !du || !ddelta || !workspace || (z && !dz))
        return MI_ERR_INVALID;
    if (!mi::aligned16(A) || !mi::aligned16(dh_out) || !mi::aligned16(dh0) || !mi::aligned16(checkpoints) ||
        !mi::aligned16(workspace))
        return MI_ERR_INVALID;
    Args a = {};
    const int size = dtype == MI_DT_F32 ? 4 : 2;
    a.u = seq(u, u_batch, u_row, 8, size), a.delta = seq(delta, delta_batch, delta_row, 8, size);
    a.z = seq(z, z_batch, z_row, 8, size), a.B = seq(B, B_batch, B_row, 4, size), a.C = seq(C, C_batch, C_row, 4, size);
    a.dy = seq(dy, dy_batch, dy_row, 8, size);
    a.A = A, a.Dskip = D, a.bias = delta_bias, a.lengths = lengths, a.dhT = dh_out;
    a.ckpt = const_cast<float*>(checkpoints);
    a.du = du, a.ddelta = ddelta, a.dz = dz, a.dh0 = dh0;
    a.batch = batch, a.L = L, a.D = Dm, a.N = N, a.softplus = softplus;
    a.ovec = Dm % 8 == 0 && mi::aligned16(du) && mi::aligned16(ddelta) && mi::aligned16(dz);
    float* ws = static_cast<float*>(workspace);
    cudaStream_t s = (cudaStream_t)stream;
    int rc2 = MI_OK;
    MI_DISPATCH_DTYPE(dtype, T, rc2 = mi_sscan_backward_states<T>(a, ws, s));
    if (rc2 != MI_OK) return rc2;
    Sums t = {};
    t.part_bc = a.part_bc, t.part_a = a.part_a, t.part_d = a.part_d;
    t.dB = dB, t.dC = dC, t.dA = dA, t.dD = dD, t.db = ddelta_bias;
    t.rows = (int64_t)batch * L, t.blocks = mi::cdiv(Dm, bwd_channels(N));
    t.P = batch * a.chunks, t.D = Dm, t.N = N, t.NP = 4 * lanes_of(N);
    t.bc = dB || dC ? (int)((t.rows * 2 * t.NP + 255) / 256) : 0;
    const int params = dA || dD || ddelta_bias ? (int)(((int64_t)Dm * (t.NP + 2) + 255) / 256) : 0;
    if (t.bc + params) {
        MI_DISPATCH_DTYPE(dtype, T, sum_kernel<T><<<t.bc + params, 256, 0, s>>>(t));
        MI_CHECK_LAUNCH();
    }
    return MI_OK;
}

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
// Layout: LN lanes share a channel and hold 4 states each (N <= 4 LN; states
// beyond N have A = B = C = 0 and stay 0), so a warp spans 32 / LN channels.
// Tiles of TT positions by CB channels are staged in shared memory as
// (dt, dt u); positions from the length on are staged with dt = 0, B = C = 0,
// where the recurrence leaves the state as it is.
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
__device__ __forceinline__ St fma(St x, float v, St z) {
    return {__ffma2_rn(x.a, dup(v), z.a), __ffma2_rn(x.b, dup(v), z.b)};
}
__device__ __forceinline__ float dot(St x, St y) {
    const float2 p = __ffma2_rn(x.b, y.b, __fmul2_rn(x.a, y.a));
    return __fadd_rn(p.x, p.y);
}
__device__ __forceinline__ St exp2s(St x) {
    return {make_float2(exp2_fast(x.a.x), exp2_fast(x.a.y)), make_float2(exp2_fast(x.b.x), exp2_fast(x.b.y))};
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

template <int LN>
struct Cfg {
    static constexpr int NP = 4 * LN;                    // padded states
    static constexpr int CL = 32 / LN;                   // channel lanes of a warp
    static constexpr int CPL = LN <= 4 ? 1 : LN / 4;     // channels a lane, forward
    static constexpr int CB = 4 * CL * CPL;              // channels a CTA: 64 (LN = 2) or 32
    static constexpr int TT = 8 * THREADS / CB;          // positions a tile: 16 or 32
    static constexpr int VPR = CB / 8;                   // packs of 8 channels a row
    static constexpr int QUADS = (TT * LN + THREADS - 1) / THREADS;  // packs of 4 states a thread, of each of B and C
};

// One thread's part of a tile's loads: 8 channels of one position of u, delta
// and z (or dy), and QUADS packs of B and C.
template <typename T, int QUADS>
struct Raw {
    Pack<T, 8> u, d, z;
    Pack<T, 4> B[QUADS], C[QUADS];
};

// ---------------------------------------------------------------------------
// A chunk's own end state, from a zero start (forward: REV = false), or the
// gradient that a chunk passes to the one before it, from a zero one behind it
// (REV = true; dy, z and C in the place of u, delta and B), and the sum of its
// dt.  Only chunks > 1 need it: one more exponential for each state.
template <typename T, int LN, bool REV>
__global__ void __launch_bounds__(THREADS) chunk_kernel(const Args a) {
    using F = Cfg<LN>;
    __shared__ __align__(16) float2 sd[F::TT][F::CB];  // (dt, dt u) or (dt, ds)
    __shared__ __align__(16) float sm[F::TT][F::NP];   // B or C
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nl = lane % LN, cl = lane / LN, n0 = 4 * nl;
    const int d0 = blockIdx.x * F::CB, b = blockIdx.y, ck = blockIdx.z + (REV ? 1 : 0);
    const int len = length_of(a, b);
    const int tb = ck * a.span, te = tb + a.span < a.L ? tb + a.span : a.L;
    const int end = te < len ? te : len;  // past it nothing changes the state
    const int lt = tid / F::VPR, lv = tid % F::VPR;  // this thread's row and pack of the loads
    const int ldd = d0 + 8 * lv;
    int ch[F::CPL];
    St A2[F::CPL], h[F::CPL];
    float sum[F::CPL];
#pragma unroll
    for (int j = 0; j < F::CPL; j++) {
        ch[j] = warp * F::CL * F::CPL + cl * F::CPL + j;
        const int d = d0 + ch[j];
        A2[j] = st(d < a.D ? load4(a.A + (int64_t)d * a.N, n0, a.N) : make_float4(0, 0, 0, 0));
        A2[j] = mul(A2[j], LOG2E);
        h[j] = st(make_float4(0, 0, 0, 0));
        sum[j] = 0.0f;
    }
    const int tiles = end > tb ? cdiv(end - tb, F::TT) : 0;
    for (int i = 0; i < tiles; i++) {
        const int t0 = tb + (REV ? tiles - 1 - i : i) * F::TT;
        const int t = t0 + lt;
        const bool in = t < end;
        {
            const int valid = in ? a.D - ldd : 0;
            const Pack<T, 8> pd = load_pack<8>(row_of<T>(a.delta, b, t) + ldd, valid, a.delta.vec);
            const Pack<T, 8> pu = REV ? load_pack<8>(row_of<T>(a.dy, b, t) + ldd, valid, a.dy.vec)
                                      : load_pack<8>(row_of<T>(a.u, b, t) + ldd, valid, a.u.vec);
            Pack<T, 8> pz;
            if (REV && a.z.p) pz = load_pack<8>(row_of<T>(a.z, b, t) + ldd, valid, a.z.vec);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                float dt = to_f(pd.v[k]);
                if (a.bias && ldd + k < a.D) dt = __fadd_rn(dt, a.bias[ldd + k]);
                if (a.softplus) dt = softplus(dt);
                if (!in || ldd + k >= a.D) dt = 0.0f;
                float v = to_f(pu.v[k]);
                if (!REV)
                    v = __fmul_rn(dt, v);
                else if (a.z.p) {
                    const float z = to_f(pz.v[k]);
                    v = __fmul_rn(v, __fmul_rn(z, sigmoid(z)));
                }
                sd[lt][8 * lv + k] = make_float2(dt, in ? v : 0.0f);
            }
        }
#pragma unroll
        for (int q = 0; q < F::QUADS; q++) {
            const int e = tid + q * THREADS, tq = t0 + e / LN, nq = 4 * (e % LN);
            if (e >= F::TT * LN) break;
            const Seq& s = REV ? a.C : a.B;
            const Pack<T, 4> p = load_pack<4>(row_of<T>(s, b, tq) + nq, tq < end ? a.N - nq : 0, s.vec);
            *reinterpret_cast<float4*>(&sm[e / LN][nq]) =
                make_float4(to_f(p.v[0]), to_f(p.v[1]), to_f(p.v[2]), to_f(p.v[3]));
        }
        __syncthreads();
#pragma unroll 4
        for (int k = 0; k < F::TT; k++) {
            const int r = REV ? F::TT - 1 - k : k;
            const St m = st(*reinterpret_cast<const float4*>(&sm[r][n0]));
#pragma unroll
            for (int j = 0; j < F::CPL; j++) {
                const float2 dd = sd[r][ch[j]];
                const St e = exp2s(mul(A2[j], dd.x));
                h[j] = REV ? mul(e, fma(m, dd.y, h[j])) : fma(e, h[j], mul(m, dd.y));
                sum[j] = __fadd_rn(sum[j], dd.x);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < F::CPL; j++) {
        const int d = d0 + ch[j];
        if (d >= a.D) continue;
        const int64_t row = ((int64_t)b * a.chunks + ck) * a.D + d;
        *reinterpret_cast<float4*>(a.cst + row * F::NP + n0) = f4(h[j]);
        if (nl == 0) a.cdt[row] = sum[j];
    }
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
    const St A2 = mul(st(load4(a.A + (int64_t)d * a.N, n0, a.N)), LOG2E);
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
        h = fma(exp2s(mul(A2, sum)), h, own);
    }
}

// ---------------------------------------------------------------------------
// The scan of one chunk (the whole sequence with chunks = 1).
template <typename T, int LN>
__global__ void __launch_bounds__(THREADS) fwd_kernel(const Args a) {
    using F = Cfg<LN>;
    constexpr int NP = F::NP, CB = F::CB, TT = F::TT, CPL = F::CPL;
    constexpr int YS = CB + 8;  // the 4 positions that a step of the loop stores lie in different banks
    __shared__ __align__(16) float2 sd[TT][CB];
    __shared__ __align__(16) float sB[TT][NP], sC[TT][NP];
    __shared__ __align__(16) float sy[TT][YS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nl = lane % LN, cl = lane / LN, n0 = 4 * nl;
    const int d0 = blockIdx.x * CB, b = blockIdx.y, ck = blockIdx.z;
    const int len = length_of(a, b);
    const int tb = ck * a.span, te = tb + a.span < a.L ? tb + a.span : a.L;
    const int end = te < len ? te : len;
    const int lt = tid / F::VPR, lv = tid % F::VPR, ldd = d0 + 8 * lv;
    int ch[CPL];
    St A2[CPL], h[CPL];
#pragma unroll
    for (int j = 0; j < CPL; j++) {
        ch[j] = warp * F::CL * CPL + cl * CPL + j;
        const int d = d0 + ch[j];
        const bool in = d < a.D;
        A2[j] = mul(st(in ? load4(a.A + (int64_t)d * a.N, n0, a.N) : make_float4(0, 0, 0, 0)), LOG2E);
        float4 v = make_float4(0, 0, 0, 0);
        if (in && a.chunks > 1)
            v = *reinterpret_cast<const float4*>(a.cst + (((int64_t)b * a.chunks + ck) * a.D + d) * NP + n0);
        else if (in && a.h0)
            v = load4(a.h0 + ((int64_t)b * a.D + d) * a.N, n0, a.N);
        h[j] = st(v);
    }
    float bias[8], skip[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        bias[k] = a.bias && ldd + k < a.D ? a.bias[ldd + k] : 0.0f;
        skip[k] = a.Dskip && ldd + k < a.D ? a.Dskip[ldd + k] : 0.0f;
    }
    const int tiles = te > tb ? cdiv(te - tb, TT) : 0;
    Raw<T, F::QUADS> raw;
    auto load = [&](int t0) {
        const int t = t0 + lt;
        const int valid = t < end ? a.D - ldd : 0;
        raw.u = load_pack<8>(row_of<T>(a.u, b, t) + ldd, valid, a.u.vec);
        raw.d = load_pack<8>(row_of<T>(a.delta, b, t) + ldd, valid, a.delta.vec);
        if (a.z.p) raw.z = load_pack<8>(row_of<T>(a.z, b, t) + ldd, valid, a.z.vec);
#pragma unroll
        for (int q = 0; q < F::QUADS; q++) {
            const int e = tid + q * THREADS, tq = t0 + e / LN, nq = 4 * (e % LN);
            const int have = tq < end && e < TT * LN ? a.N - nq : 0;
            raw.B[q] = load_pack<4>(row_of<T>(a.B, b, tq) + nq, have, a.B.vec);
            raw.C[q] = load_pack<4>(row_of<T>(a.C, b, tq) + nq, have, a.C.vec);
        }
    };
    load(tb);
    for (int i = 0; i < tiles; i++) {
        const int t0 = tb + i * TT, t = t0 + lt;
        const bool in = t < end;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            float dt = __fadd_rn(to_f(raw.d.v[k]), bias[k]);
            if (a.softplus) dt = softplus(dt);
            if (!in || ldd + k >= a.D) dt = 0.0f;
            sd[lt][8 * lv + k] = make_float2(dt, __fmul_rn(dt, to_f(raw.u.v[k])));
        }
#pragma unroll
        for (int q = 0; q < F::QUADS; q++) {
            const int e = tid + q * THREADS;
            if (e >= TT * LN) break;
            float4 v = make_float4(to_f(raw.B[q].v[0]), to_f(raw.B[q].v[1]), to_f(raw.B[q].v[2]), to_f(raw.B[q].v[3]));
            *reinterpret_cast<float4*>(&sB[e / LN][4 * (e % LN)]) = v;
            v = make_float4(to_f(raw.C[q].v[0]), to_f(raw.C[q].v[1]), to_f(raw.C[q].v[2]), to_f(raw.C[q].v[3]));
            *reinterpret_cast<float4*>(&sC[e / LN][4 * (e % LN)]) = v;
        }
        __syncthreads();
        const Pack<T, 8> ru = raw.u, rz = raw.z;
        if (i + 1 < tiles) load(t0 + TT);
        if (t0 < end) {
#pragma unroll 1
            for (int r4 = 0; r4 < TT; r4 += 4) {
                if (a.ckpt && (t0 + r4) % CK == 0 && t0 + r4 < a.L) {
#pragma unroll
                    for (int j = 0; j < CPL; j++)
                        if (d0 + ch[j] < a.D)
                            *reinterpret_cast<float4*>(
                                a.ckpt + (((int64_t)b * cdiv(a.L, CK) + (t0 + r4) / CK) * a.D + d0 + ch[j]) * NP + n0) =
                                f4(h[j]);
                }
                float y[CPL][4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const St Bv = st(*reinterpret_cast<const float4*>(&sB[r4 + k][n0]));
                    const St Cv = st(*reinterpret_cast<const float4*>(&sC[r4 + k][n0]));
#pragma unroll
                    for (int j = 0; j < CPL; j++) {
                        const float2 dd = sd[r4 + k][ch[j]];
                        h[j] = fma(exp2s(mul(A2[j], dd.x)), h[j], mul(Bv, dd.y));
                        y[j][k] = dot(h[j], Cv);
                    }
                }
                // sums over the channel's lanes: of 4 positions, each lane keeps one (LN = 2: two)
#pragma unroll
                for (int j = 0; j < CPL; j++) {
                    if constexpr (LN == 2) {
                        halve<4>(y[j], 1);
                        sy[r4 + 2 * nl][ch[j]] = y[j][0];
                        sy[r4 + 2 * nl + 1][ch[j]] = y[j][1];
                    } else {
                        halve<4>(y[j], 2);
                        halve<2>(y[j], 1);
#pragma unroll
                        for (int m = 4; m < LN; m *= 2)
                            y[j][0] = __fadd_rn(y[j][0], __shfl_xor_sync(0xffffffffu, y[j][0], m));
                        if (nl < 4) sy[r4 + nl][ch[j]] = y[j][0];
                    }
                }
            }
        }
        __syncthreads();
        if (t < te && ldd < a.D) {
            float o[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                float v = __fmaf_rn(skip[k], to_f(ru.v[k]), sy[lt][8 * lv + k]);
                if (a.z.p) {
                    const float z = to_f(rz.v[k]);
                    v = __fmul_rn(v, __fmul_rn(z, sigmoid(z)));
                }
                o[k] = in ? v : 0.0f;
            }
            store_pack<8>(static_cast<T*>(a.y) + ((int64_t)b * a.L + t) * a.D + ldd, o, a.D - ldd, a.ovec);
        }
    }
    if (a.hT && ck == a.chunks - 1) {
#pragma unroll
        for (int j = 0; j < CPL; j++)
            if (d0 + ch[j] < a.D) store4(a.hT + ((int64_t)b * a.D + d0 + ch[j]) * a.N, n0, a.N, f4(h[j]));
    }
}

// ---------------------------------------------------------------------------
// Backward of one chunk.  Tiles of 16 positions, from the last to the first.
// From the state that the forward pass kept at a tile's start, each half of 8
// positions is run again (the first half twice: once on the way to the
// second), with its decays and states held in registers, and then walked
// backwards.  A lane goes through its CPL channels one after the other, so
// that the terms of dB and dC add up over them in registers before they are
// added across the lanes, and once a tile across the warps; sum_bc_kernel adds
// the channel blocks.
template <int LN>
struct BCfg {
    static constexpr int NP = 4 * LN, CL = 32 / LN;
    static constexpr int CB = 64, CPL = CB / (4 * CL);  // channels a CTA, a lane
    static constexpr int TT = CK, VPR = CB / 8;
    static constexpr int QUADS = (TT * LN + THREADS - 1) / THREADS;
    static constexpr int OS = CB + 8;
    struct Smem {
        float2 sd[TT][CB];             // dt, dt u
        float ds[TT][CB];              // dy z sigmoid(z)
        float B[TT][NP], C[TT][NP];
        float S[3][TT][OS];            // sum_n g B, sum_n w A log2(e), sum_n C h
        float4 own[4][CPL][3][32];     // by lane: A log2(e), the gradient's carry, dA
        float bc[4][TT][2 * NP];       // a warp's dB | dC
        float acc[2][TT][CB];          // dD and dbias, by position of the tile
    };
};

template <typename T, int LN>
__global__ void __launch_bounds__(THREADS) bwd_kernel(const Args a) {
    using F = BCfg<LN>;
    constexpr int NP = F::NP, CB = F::CB, CPL = F::CPL, TT = F::TT, CL = F::CL;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    typename F::Smem& sm = *reinterpret_cast<typename F::Smem*>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nl = lane % LN, cl = lane / LN, n0 = 4 * nl;
    const int d0 = blockIdx.x * CB, b = blockIdx.y, ck = blockIdx.z;
    const int len = length_of(a, b);
    const int tb = ck * a.span, te = tb + a.span < a.L ? tb + a.span : a.L;
    const int end = te < len ? te : len;
    const int lt = tid / F::VPR, lv = tid % F::VPR, ldd = d0 + 8 * lv;
    const int nck = cdiv(a.L, CK);
    for (int j = 0; j < CPL; j++) {
        const int d = d0 + warp * CL * CPL + cl * CPL + j;
        const bool in = d < a.D;
        float4 A = make_float4(0, 0, 0, 0), g = A;
        if (in) {
            A = f4(mul(st(load4(a.A + (int64_t)d * a.N, n0, a.N)), LOG2E));
            if (a.chunks > 1)
                g = *reinterpret_cast<const float4*>(a.cst + (((int64_t)b * a.chunks + ck) * a.D + d) * NP + n0);
            else if (a.dhT)
                g = load4(a.dhT + ((int64_t)b * a.D + d) * a.N, n0, a.N);
        }
        sm.own[warp][j][0][lane] = A;
        sm.own[warp][j][1][lane] = g;
        sm.own[warp][j][2][lane] = make_float4(0, 0, 0, 0);
    }
    float bias[8], skip[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        bias[k] = a.bias && ldd + k < a.D ? a.bias[ldd + k] : 0.0f;
        skip[k] = a.Dskip && ldd + k < a.D ? a.Dskip[ldd + k] : 0.0f;
        sm.acc[0][lt][8 * lv + k] = 0.0f;
        sm.acc[1][lt][8 * lv + k] = 0.0f;
    }
    const int tiles = te > tb ? cdiv(te - tb, TT) : 0;
    for (int i = tiles - 1; i >= 0; i--) {
        const int t0 = tb + i * TT, t = t0 + lt;
        const bool in = t < end;
        const int valid = in ? a.D - ldd : 0;
        float u[8], sg[8], dyz[8], dsk[8];  // u; d dt / d delta; dy (z sigmoid(z))'; ds
        {
            const Pack<T, 8> pu = load_pack<8>(row_of<T>(a.u, b, t) + ldd, valid, a.u.vec);
            const Pack<T, 8> pd = load_pack<8>(row_of<T>(a.delta, b, t) + ldd, valid, a.delta.vec);
            const Pack<T, 8> pg = load_pack<8>(row_of<T>(a.dy, b, t) + ldd, valid, a.dy.vec);
            Pack<T, 8> pz;
            if (a.z.p) pz = load_pack<8>(row_of<T>(a.z, b, t) + ldd, valid, a.z.vec);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                u[k] = to_f(pu.v[k]);
                const float x = __fadd_rn(to_f(pd.v[k]), bias[k]);
                float dt = x;
                sg[k] = 1.0f;
                if (a.softplus) dt = softplus(x), sg[k] = sigmoid(x);
                if (!in || ldd + k >= a.D) dt = 0.0f;
                sm.sd[lt][8 * lv + k] = make_float2(dt, __fmul_rn(dt, u[k]));
                const float dy = to_f(pg.v[k]);
                dsk[k] = dy, dyz[k] = 0.0f;
                if (a.z.p) {
                    const float z = to_f(pz.v[k]), s = sigmoid(z);
                    dsk[k] = __fmul_rn(dy, __fmul_rn(z, s));
                    dyz[k] = __fmul_rn(dy, __fmul_rn(s, __fmaf_rn(z, __fsub_rn(1.0f, s), 1.0f)));
                }
                sm.ds[lt][8 * lv + k] = dsk[k];
            }
        }
#pragma unroll
        for (int q = 0; q < F::QUADS; q++) {
            const int e = tid + q * THREADS, tq = t0 + e / LN, nq = 4 * (e % LN);
            if (e < TT * LN) {
                const int have = tq < end ? a.N - nq : 0;
                const Pack<T, 4> pB = load_pack<4>(row_of<T>(a.B, b, tq) + nq, have, a.B.vec);
                const Pack<T, 4> pC = load_pack<4>(row_of<T>(a.C, b, tq) + nq, have, a.C.vec);
                *reinterpret_cast<float4*>(&sm.B[e / LN][nq]) =
                    make_float4(to_f(pB.v[0]), to_f(pB.v[1]), to_f(pB.v[2]), to_f(pB.v[3]));
                *reinterpret_cast<float4*>(&sm.C[e / LN][nq]) =
                    make_float4(to_f(pC.v[0]), to_f(pC.v[1]), to_f(pC.v[2]), to_f(pC.v[3]));
            }
        }
        __syncthreads();
        if (t0 < end) {  // a tile behind the length changes nothing
#pragma unroll 1
            for (int half = 1; half >= 0; half--) {
                float v[8][8];  // by position: 4 states' dB and dC
#pragma unroll
                for (int k = 0; k < 8; k++)
#pragma unroll
                    for (int m = 0; m < 8; m++) v[k][m] = 0.0f;
#pragma unroll 1
                for (int j = 0; j < CPL; j++) {
                    const int c = warp * CL * CPL + cl * CPL + j;
                    float4* mine = &sm.own[warp][j][0][lane];
                    const St A2 = st(mine[0]);
                    St h0 = st(make_float4(0, 0, 0, 0));
                    if (d0 + c < a.D)
                        h0 = st(*reinterpret_cast<const float4*>(
                            a.ckpt + (((int64_t)b * nck + t0 / CK) * a.D + d0 + c) * NP + n0));
                    if (half == 1) {
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const float2 dd = sm.sd[k][c];
                            const St Bv = st(*reinterpret_cast<const float4*>(&sm.B[k][n0]));
                            h0 = fma(exp2s(mul(A2, dd.x)), h0, mul(Bv, dd.y));
                        }
                    }
                    St e[8], h[8];
                    {
                        St x = h0;
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const float2 dd = sm.sd[8 * half + k][c];
                            const St Bv = st(*reinterpret_cast<const float4*>(&sm.B[8 * half + k][n0]));
                            e[k] = exp2s(mul(A2, dd.x));
                            x = fma(e[k], x, mul(Bv, dd.y));
                            h[k] = x;
                        }
                    }
                    St gc = st(mine[32]), dA = st(mine[64]);
                    float s[3][8];
#pragma unroll
                    for (int k = 7; k >= 0; k--) {
                        const int r = 8 * half + k;
                        const float2 dd = sm.sd[r][c];
                        const float ds = sm.ds[r][c];
                        const St Bv = st(*reinterpret_cast<const float4*>(&sm.B[r][n0]));
                        const St Cv = st(*reinterpret_cast<const float4*>(&sm.C[r][n0]));
                        const St g = fma(Cv, ds, gc);
                        const float4 fg = f4(g), fh = f4(h[k]);
                        v[k][0] = __fmaf_rn(fg.x, dd.y, v[k][0]);
                        v[k][1] = __fmaf_rn(fg.y, dd.y, v[k][1]);
                        v[k][2] = __fmaf_rn(fg.z, dd.y, v[k][2]);
                        v[k][3] = __fmaf_rn(fg.w, dd.y, v[k][3]);
                        v[k][4] = __fmaf_rn(fh.x, ds, v[k][4]);
                        v[k][5] = __fmaf_rn(fh.y, ds, v[k][5]);
                        v[k][6] = __fmaf_rn(fh.z, ds, v[k][6]);
                        v[k][7] = __fmaf_rn(fh.w, ds, v[k][7]);
                        s[0][k] = dot(g, Bv);
                        gc = mul(e[k], g);
                        const St w = mul(gc, k ? h[k ? k - 1 : 0] : h0);
                        s[1][k] = dot(w, A2);
                        s[2][k] = dot(h[k], Cv);
                        dA = fma(w, dd.x, dA);
                    }
                    mine[32] = f4(gc);
                    mine[64] = f4(dA);
                    // over the channel's lanes; each keeps 8 / LN of the 8 positions
#pragma unroll
                    for (int m = 0; m < 3; m++) {
                        constexpr int KEEP = LN >= 8 ? 1 : 8 / LN;
                        int pos = 0;
                        if constexpr (LN >= 8) {
                            halve<8>(s[m], 4), halve<4>(s[m], 2), halve<2>(s[m], 1);
                            pos = nl & 7;
                            if constexpr (LN == 16)
                                s[m][0] = __fadd_rn(s[m][0], __shfl_xor_sync(0xffffffffu, s[m][0], 8));
                        } else if constexpr (LN == 4) {
                            halve<8>(s[m], 2), halve<4>(s[m], 1);
                            pos = 2 * nl;
                        } else {
                            halve<8>(s[m], 1);
                            pos = 4 * nl;
                        }
                        if (LN < 16 || nl < 8) {
#pragma unroll
                            for (int k = 0; k < KEEP; k++) sm.S[m][8 * half + pos + k][c] = s[m][k];
                        }
                    }
                }
                // over the warp's channel lanes: first by position, then dB from dC
                float* f = &v[0][0];
                int pos = 0, cnt = 8;
                if constexpr (CL >= 2) halve<64>(f, LN), pos = (cl & 1) * 4, cnt = 4;
                if constexpr (CL >= 4) halve<32>(f, 2 * LN), pos += ((cl >> 1) & 1) * 2, cnt = 2;
                if constexpr (CL >= 8) halve<16>(f, 4 * LN), pos += (cl >> 2) & 1, cnt = 1;
                if constexpr (CL == 16) {
                    halve<8>(f, 8 * LN);
                    *reinterpret_cast<float4*>(&sm.bc[warp][8 * half + pos][((cl >> 3) & 1) * NP + n0]) =
                        make_float4(f[0], f[1], f[2], f[3]);
                } else {
#pragma unroll
                    for (int k = 0; k < (CL >= 8 ? 1 : 8 / CL); k++) {
                        float* row = sm.bc[warp][8 * half + pos + k];
                        *reinterpret_cast<float4*>(row + n0) = make_float4(f[8 * k], f[8 * k + 1], f[8 * k + 2], f[8 * k + 3]);
                        *reinterpret_cast<float4*>(row + NP + n0) =
                            make_float4(f[8 * k + 4], f[8 * k + 5], f[8 * k + 6], f[8 * k + 7]);
                    }
                }
            }
        }
        __syncthreads();
        for (int e = tid; e < TT * 2 * NP; e += THREADS) {
            const int r = e / (2 * NP), k = e % (2 * NP);
            if (t0 + r >= te) break;
            float x = 0.0f;
            if (t0 + r < end)
                x = __fadd_rn(__fadd_rn(sm.bc[0][r][k], sm.bc[1][r][k]), __fadd_rn(sm.bc[2][r][k], sm.bc[3][r][k]));
            a.part_bc[(((int64_t)blockIdx.x * a.batch + b) * a.L + t0 + r) * (2 * NP) + k] = x;
        }
        if (t < te && ldd < a.D) {
            float du[8], dd[8], dz[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int c = 8 * lv + k;
                const float dt = sm.sd[lt][c].x;
                const float s1 = sm.S[0][lt][c], s2 = __fmul_rn(sm.S[1][lt][c], LN2);
                const float sc = __fmaf_rn(skip[k], u[k], sm.S[2][lt][c]);
                du[k] = in ? __fmaf_rn(dt, s1, __fmul_rn(skip[k], dsk[k])) : 0.0f;
                dd[k] = in ? __fmul_rn(__fmaf_rn(u[k], s1, s2), sg[k]) : 0.0f;
                dz[k] = in ? __fmul_rn(dyz[k], sc) : 0.0f;
                if (in) {
                    sm.acc[0][lt][c] = __fmaf_rn(dsk[k], u[k], sm.acc[0][lt][c]);
                    sm.acc[1][lt][c] = __fadd_rn(sm.acc[1][lt][c], dd[k]);
                }
            }
            const int64_t o = ((int64_t)b * a.L + t) * a.D + ldd;
            store_pack<8>(static_cast<T*>(a.du) + o, du, a.D - ldd, a.ovec);
            store_pack<8>(static_cast<T*>(a.ddelta) + o, dd, a.D - ldd, a.ovec);
            if (a.z.p) store_pack<8>(static_cast<T*>(a.dz) + o, dz, a.D - ldd, a.ovec);
        }
        __syncthreads();
    }
    const int64_t bk = (int64_t)b * a.chunks + ck;
    for (int j = 0; j < CPL; j++) {
        const int d = d0 + warp * CL * CPL + cl * CPL + j;
        if (d >= a.D) continue;
        *reinterpret_cast<float4*>(a.part_a + (bk * a.D + d) * NP + n0) = sm.own[warp][j][2][lane];
        if (ck == 0 && a.dh0) store4(a.dh0 + ((int64_t)b * a.D + d) * a.N, n0, a.N, sm.own[warp][j][1][lane]);
    }
    __syncthreads();
    for (int e = tid; e < 2 * CB; e += THREADS) {
        const int c = e % CB, k = e / CB;
        if (d0 + c >= a.D) continue;
        float x = 0.0f;
        for (int r = 0; r < TT; r++) x = __fadd_rn(x, sm.acc[k][r][c]);
        a.part_d[(bk * 2 + k) * a.D + d0 + c] = x;
    }
}

// dB and dC: the channel blocks' partial sums, added in order
template <typename T>
__global__ void __launch_bounds__(256) sum_bc_kernel(const float* __restrict__ part, T* __restrict__ dB,
                                                     T* __restrict__ dC, int blocks, int64_t rows, int N, int NP) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= rows * 2 * NP) return;
    const int k = (int)(e % (2 * NP));
    const int64_t row = e / (2 * NP);
    const int n = k % NP;
    if (n >= N) return;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    int p = 0;
    for (; p + 3 < blocks; p += 4)
#pragma unroll
        for (int j = 0; j < 4; j++) s[j] = __fadd_rn(s[j], part[(p + j) * rows * 2 * NP + e]);
    for (; p < blocks; p++) s[0] = __fadd_rn(s[0], part[p * rows * 2 * NP + e]);
    const float x = __fadd_rn(__fadd_rn(s[0], s[1]), __fadd_rn(s[2], s[3]));
    T* o = k < NP ? dB : dC;
    if (o) o[row * N + n] = from_f<T>(x);
}

// dA, dD and dbias: the partial sums of P sequences and chunks, added in order
__global__ void __launch_bounds__(256) sum_params_kernel(const float* __restrict__ pa, const float* __restrict__ pd,
                                                         float* __restrict__ dA, float* __restrict__ dD,
                                                         float* __restrict__ db, int P, int D, int N, int NP) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e < (int64_t)D * NP) {
        const int n = (int)(e % NP);
        if (n >= N || !dA) return;
        float s = 0.0f;
        for (int p = 0; p < P; p++) s = __fadd_rn(s, pa[(int64_t)p * D * NP + e]);
        dA[e / NP * N + n] = s;
    } else if (e < (int64_t)D * (NP + 2)) {
        const int64_t f = e - (int64_t)D * NP;
        float s = 0.0f;
        for (int p = 0; p < P; p++) s = __fadd_rn(s, pd[(int64_t)p * 2 * D + f]);
        float* o = f < D ? dD : db;
        if (o) o[f % D] = s;
    }
}

// ---------------------------------------------------------------------------
// One new token a stream: the state is read and written once, 8 bytes a state,
// which bounds it.  LN lanes a channel as above.
template <typename T, int LN>
__global__ void __launch_bounds__(THREADS) step_kernel(const Args a) {
    const int64_t item = ((int64_t)blockIdx.x * THREADS + threadIdx.x) / LN;
    const int n0 = 4 * (threadIdx.x % LN);
    grid_dependency_sync();
    const bool live = item < (int64_t)a.batch * a.D;
    const int d = live ? (int)(item % a.D) : 0, b = live ? (int)(item / a.D) : 0;
    float* hp = a.hT + ((int64_t)b * a.D + d) * a.N;
    float y = 0.0f, u = 0.0f;
    if (live) {
        const float4 hv = load4(hp, n0, a.N), Av = load4(a.A + (int64_t)d * a.N, n0, a.N);
        const Pack<T, 4> pB = load_pack<4>(row_of<T>(a.B, b, 0) + n0, a.N - n0, a.B.vec);
        const Pack<T, 4> pC = load_pack<4>(row_of<T>(a.C, b, 0) + n0, a.N - n0, a.C.vec);
        u = to_f(row_of<T>(a.u, b, 0)[d]);
        float dt = to_f(row_of<T>(a.delta, b, 0)[d]);
        if (a.bias) dt = __fadd_rn(dt, a.bias[d]);
        if (a.softplus) dt = softplus(dt);
        const St Bv = st(make_float4(to_f(pB.v[0]), to_f(pB.v[1]), to_f(pB.v[2]), to_f(pB.v[3])));
        const St Cv = st(make_float4(to_f(pC.v[0]), to_f(pC.v[1]), to_f(pC.v[2]), to_f(pC.v[3])));
        const St e = exp2s(mul(mul(st(Av), LOG2E), dt));
        const St h = fma(e, st(hv), mul(Bv, __fmul_rn(dt, u)));
        store4(hp, n0, a.N, f4(h));
        y = dot(h, Cv);
    }
#pragma unroll
    for (int m = 1; m < LN; m *= 2) y = __fadd_rn(y, __shfl_xor_sync(0xffffffffu, y, m));
    if (live && n0 == 0) {
        if (a.Dskip) y = __fmaf_rn(a.Dskip[d], u, y);
        if (a.z.p) {
            const float z = to_f(row_of<T>(a.z, b, 0)[d]);
            y = __fmul_rn(y, __fmul_rn(z, sigmoid(z)));
        }
        static_cast<T*>(a.y)[(int64_t)b * a.D + d] = from_f<T>(y);
    }
}

// ---------------------------------------------------------------------------
static inline int lanes_of(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

// Chunks of the sequence: one where the channels alone give every SM 2 CTAs;
// else as many as bring it there, of 64 positions at least (a chunked scan
// makes each exponential twice).
struct Plan {
    int chunks, span;
};
static inline Plan plan_of(int batch, int L, int D, int channels) {
    const int64_t ctas = (int64_t)batch * cdiv(D, channels);
    Plan p = {1, cdiv(L, 32) * 32};
    const int64_t want = 148 * 2;
    if (ctas >= want || L < 128) return p;
    int64_t n = (want + ctas - 1) / ctas;
    if (n > L / 64) n = L / 64;
    p.span = cdiv(cdiv(L, (int)n), 32) * 32;
    p.chunks = cdiv(L, p.span);
    return p;
}

static inline int64_t align16(int64_t floats) { return (floats + 3) & ~(int64_t)3; }

struct Ws {  // floats from the workspace's start
    int64_t cst, cdt, part_bc, part_a, part_d, total;
};
static inline Ws ws_of(int batch, int L, int D, int N, bool backward) {
    const int LN = lanes_of(N), NP = 4 * LN;
    const Plan p = plan_of(batch, L, D, backward ? 64 : LN == 2 ? 64 : 32);
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
        w.part_bc = take((int64_t)cdiv(D, 64) * batch * L * 2 * NP);
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

template <typename T, int LN>
static int forward(Args& a, float* ws, cudaStream_t s) {
    using F = Cfg<LN>;
    const Plan p = plan_of(a.batch, a.L, a.D, F::CB);
    a.chunks = p.chunks, a.span = p.span;
    const int blocks = cdiv(a.D, F::CB);
    if (p.chunks > 1) {
        const Ws w = ws_of(a.batch, a.L, a.D, a.N, false);
        a.cst = ws + w.cst, a.cdt = ws + w.cdt;
        chunk_kernel<T, LN, false><<<dim3(blocks, a.batch, p.chunks - 1), THREADS, 0, s>>>(a);
        MI_CHECK_LAUNCH();
        const int64_t items = (int64_t)a.batch * a.D * LN;
        join_kernel<LN, false><<<(unsigned)((items + THREADS - 1) / THREADS), THREADS, 0, s>>>(a);
        MI_CHECK_LAUNCH();
    }
    fwd_kernel<T, LN><<<dim3(blocks, a.batch, p.chunks), THREADS, 0, s>>>(a);
    MI_CHECK_LAUNCH();
    return MI_OK;
}

template <typename T, int LN>
static int step(Args& a, float*, cudaStream_t s) {
    const int64_t threads = (int64_t)a.batch * a.D * LN;
    MI_LAUNCH_DEPENDENT(step_kernel<T, LN>, (unsigned)((threads + THREADS - 1) / THREADS), THREADS, 0, s, a);
    return MI_OK;
}

template <typename T, int LN>
static int backward(Args& a, float* ws, cudaStream_t s) {
    using F = BCfg<LN>;
    const Plan p = plan_of(a.batch, a.L, a.D, F::CB);
    a.chunks = p.chunks, a.span = p.span;
    const Ws w = ws_of(a.batch, a.L, a.D, a.N, true);
    a.part_bc = ws + w.part_bc, a.part_a = ws + w.part_a, a.part_d = ws + w.part_d;
    if (p.chunks > 1) {
        a.cst = ws + w.cst, a.cdt = ws + w.cdt;
        chunk_kernel<T, LN, true><<<dim3(cdiv(a.D, Cfg<LN>::CB), a.batch, p.chunks - 1), THREADS, 0, s>>>(a);
        MI_CHECK_LAUNCH();
        const int64_t items = (int64_t)a.batch * a.D * LN;
        join_kernel<LN, true><<<(unsigned)((items + THREADS - 1) / THREADS), THREADS, 0, s>>>(a);
        MI_CHECK_LAUNCH();
    }
    constexpr int smem = (int)sizeof(typename F::Smem);
    if (cudaFuncSetAttribute(bwd_kernel<T, LN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return MI_ERR_CUDA;
    bwd_kernel<T, LN><<<dim3(cdiv(a.D, F::CB), a.batch, p.chunks), THREADS, smem, s>>>(a);
    MI_CHECK_LAUNCH();
    return MI_OK;
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
    const int rc = check(batch, 1, Dm, N, dtype);
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
    const int NP = 4 * lanes_of(N), blocks = mi::cdiv(Dm, 64);
    const int64_t rows = (int64_t)batch * L;
    if (dB || dC) {
        const int64_t n = rows * 2 * NP;
        MI_DISPATCH_DTYPE(dtype, T,
                          sum_bc_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(
                              a.part_bc, static_cast<T*>(dB), static_cast<T*>(dC), blocks, rows, N, NP));
        MI_CHECK_LAUNCH();
    }
    if (dA || dD || ddelta_bias) {
        const int64_t n = (int64_t)Dm * (NP + 2);
        sum_params_kernel<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a.part_a, a.part_d, dA, dD, ddelta_bias,
                                                                      batch * a.chunks, Dm, N, NP);
        MI_CHECK_LAUNCH();
    }
    return MI_OK;
}

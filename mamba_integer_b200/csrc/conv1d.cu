// conv1d.cu -- the short causal depthwise convolution of a float Mamba layer
// (2 to 4 taps, optional bias and SiLU), its backward pass, and its form for
// one new token.
//
//   c[t] = bias + sum_k w[k] x[t - W + 1 + k]     (x before 0: the window, or 0)
//   y[t] = c[t] sigmoid(c[t])  or  c[t]           (0 from the sequence's length on)
//   win' = the last W - 1 inputs before the sequence's length
//   dc[t] = dy[t] silu'(c[t]);  dx[t] = sum_k w[k] dc[t + W - 1 - k]
//   dw[k] = sum_t dc[t] x[t - W + 1 + k];  dbias = sum_t dc[t]
//
// Bound by HBM: x is read and y written once.  A thread owns K neighbouring
// channels over a run of positions and slides the taps along in registers, so
// only the W - 1 rows in front of a run are read again, from L2.
#include "mi_elem.cuh"

namespace mi {
namespace conv1d {

constexpr int MAXW = 4;

struct Args {
    const void* x;
    const void* win;     // [batch, W-1, D], may be NULL
    const float* w;      // [D, W]
    const float* bias;   // may be NULL
    const int* lengths;  // may be NULL
    void* y;
    void* win_out;  // may be NULL
    const void* dy;
    const void* dwin_out;  // gradient of win_out, may be NULL
    void* dx;              // may be NULL
    void* dwin;            // gradient of win, may be NULL
    float* part;           // [parts, D, W + 1]
    int64_t xb, xl;        // strides of x in elements
    int64_t gb, gl;        // of dy
    int batch, L, D;
    int silu;
    int vec;
    int run;               // positions a thread, forward: 8, 16, 32 or 64
};

__device__ __forceinline__ int length_of(const int* lengths, int b, int L) {
    if (!lengths) return L;
    const int n = lengths[b];
    return n < 0 ? 0 : (n < L ? n : L);
}

// x at position t of sequence b: the window's rows at t < 0 (zero without one)
template <int W, int K, typename T>
__device__ __forceinline__ Pack<T, K> load_x(const Args& a, int b, int t, int c, bool vec) {
    const int valid = a.D - c;
    if (t >= 0) return load_pack<K>(static_cast<const T*>(a.x) + b * a.xb + t * a.xl + c, valid, vec);
    if (a.win)
        return load_pack<K>(static_cast<const T*>(a.win) + ((int64_t)b * (W - 1) + (t + W - 1)) * a.D + c, valid, vec);
    Pack<T, K> z;
#pragma unroll
    for (int i = 0; i < K; i++) z.v[i] = from_f<T>(0.0f);
    return z;
}

template <int W, int K>
__device__ __forceinline__ void load_w(const Args& a, int c, float (&w)[W][K], float (&bias)[K]) {
    if (W == 4 && a.vec) {  // a channel's taps at once
#pragma unroll
        for (int i = 0; i < K; i++) {
            const float4 t = reinterpret_cast<const float4*>(a.w)[c + i];
            w[0][i] = t.x, w[1][i] = t.y, w[W - 2][i] = t.z, w[W - 1][i] = t.w;
        }
        Pack<float, K> t;
#pragma unroll
        for (int i = 0; i < K; i++) t.v[i] = 0.0f;
        if (a.bias) t = *reinterpret_cast<const Pack<float, K>*>(a.bias + c);
#pragma unroll
        for (int i = 0; i < K; i++) bias[i] = t.v[i];
        return;
    }
#pragma unroll
    for (int i = 0; i < K; i++) {
        const bool in = c + i < a.D;
#pragma unroll
        for (int k = 0; k < W; k++) w[k][i] = in ? a.w[(int64_t)(c + i) * W + k] : 0.0f;
        bias[i] = in && a.bias ? a.bias[c + i] : 0.0f;
    }
}

// K channels of a row that exists, as they lie: no branch and no conversion,
// behind either of which a warp would wait for each load by itself.  Channels
// beyond the last read the row's first ones; nothing comes of them.
template <bool VEC, int K, typename T>
__device__ __forceinline__ Pack<T, K> raw_row(const T* p, int have) {
    if constexpr (VEC) {
        return *reinterpret_cast<const Pack<T, K>*>(p);
    } else {
        Pack<T, K> r;
#pragma unroll
        for (int i = 0; i < K; i++) r.v[i] = p[i < have ? i : 0];
        return r;
    }
}

// The W - 1 inputs in front of position t0 (a run's first)
template <int W, int K, bool VEC, typename T>
__device__ __forceinline__ void rows_before(const Args& a, int b, int t0, int len, int c, float (&x)[W - 1][K]) {
    const int have = a.D - c;
    Pack<T, K> p[W - 1];
    if (t0 > 0) {  // runs are longer than W - 1
#pragma unroll
        for (int k = 0; k < W - 1; k++)
            p[k] = raw_row<VEC, K>(static_cast<const T*>(a.x) + b * a.xb + (t0 - (W - 1) + k) * a.xl + c, have);
    } else if (a.win) {
#pragma unroll
        for (int k = 0; k < W - 1; k++)
            p[k] = raw_row<VEC, K>(static_cast<const T*>(a.win) + ((int64_t)b * (W - 1) + k) * a.D + c, have);
    }
    const bool some = t0 > 0 || a.win;
#pragma unroll
    for (int k = 0; k < W - 1; k++)
#pragma unroll
        for (int i = 0; i < K; i++) x[k][i] = some && t0 - (W - 1) + k < len ? to_f(p[k].v[i]) : 0.0f;
}

// A thread's run, 4 positions at a time, with the next 4 rows on their way;
// rows behind the sequence's length are named by its last one, and not used.
template <typename T, int W, int K, bool VEC>
__global__ void __launch_bounds__(128, 5) fwd_kernel(const Args a) {
    using P = Pack<T, K>;
    const int vecs = cdiv(a.D, K);
    const int runs = a.L > 0 ? cdiv(a.L, a.run) : 1;  // an empty sequence still passes its window on
    const int64_t item = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (item >= (int64_t)vecs * runs * a.batch) return;
    const int c = (int)(item % vecs) * K, have = a.D - c;
    const int run = (int)(item / vecs % runs), b = (int)(item / vecs / runs);
    const int len = length_of(a.lengths, b, a.L);
    const int t0 = run * a.run, t1 = t0 + a.run < a.L ? t0 + a.run : a.L;
    if (t0 < t1) {
        const T* xb = static_cast<const T*>(a.x) + b * a.xb + c;
        const int last = len > 0 ? len - 1 : 0;
        P p[4];
        auto fetch = [&](int t) {
#pragma unroll
            for (int j = 0; j < 4; j++) p[j] = raw_row<VEC, K>(xb + (int64_t)(t + j < last ? t + j : last) * a.xl, have);
        };
        fetch(t0);
        float x[W + 3][K], w[W][K], bias[K];
        rows_before<W, K, VEC, T>(a, b, t0, len, c, reinterpret_cast<float(&)[W - 1][K]>(x));
        load_w<W, K>(a, c, w, bias);
        T* y = static_cast<T*>(a.y) + ((int64_t)b * a.L + t0) * a.D + c;
#pragma unroll 1
        for (int t = t0; t < t1; t += 4) {
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < K; i++) x[W - 1 + j][i] = to_f(p[j].v[i]);
            fetch(t + 4);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float o[K];
#pragma unroll
                for (int i = 0; i < K; i++) {
                    float s = bias[i];
#pragma unroll
                    for (int k = 0; k < W; k++) s = __fmaf_rn(w[k][i], x[j + k][i], s);
                    if (a.silu) s = __fmul_rn(s, sigmoid(s));
                    o[i] = t + j < len ? s : 0.0f;
                }
                if (t + j < t1) store_pack<K>(y, o, have, VEC);
                y += a.D;
            }
#pragma unroll
            for (int j = 0; j < W - 1; j++)
#pragma unroll
                for (int i = 0; i < K; i++) x[j][i] = x[j + 4][i];
        }
    }
    // the window that leaves: inputs len - W + 1 .. len - 1, by the first run
    if (run == 0 && a.win_out) {
#pragma unroll
        for (int k = 0; k < W - 1; k++) {
            const P p = load_x<W, K, T>(a, b, len - (W - 1) + k, c, VEC);
            float o[K];
#pragma unroll
            for (int i = 0; i < K; i++) o[i] = to_f(p.v[i]);
            store_pack<K>(static_cast<T*>(a.win_out) + ((int64_t)b * (W - 1) + k) * a.D + c, o, have, VEC);
        }
    }
}

// Backward.  A CTA is 32 pairs of channels by 8 runs of one sequence, a run to
// a warp.  A thread walks its run forward, 4 positions at a time: dc[t] needs x
// up to t, dx[t] needs dc up to t + W - 1, so it goes W - 1 positions past its
// run, and dx comes out W - 1 positions late.  Its own positions' terms of dw
// and dbias stay in registers; the CTA adds its 8 runs in shared memory, in
// order, and writes one partial row, which sum_kernel adds.
//
// A position of x and dy is 128 bytes of each for a warp (16-bit types), too
// little to cover HBM's latency with the rows that registers can hold, and a
// copy for each pair costs as many instructions as the arithmetic: asynchronous
// copies of 16 bytes a lane bring the next DEPTH - 1 groups of 4 positions into
// the warp's ring (zeros behind the sequence's length).  Rows off 16 bytes
// (VEC = false) go through registers, one group ahead.  8 x 2048 x 1536 bf16:
// 53 us (150 MB, 2.8 TB/s), the issue slots 69 % busy; 74 with each
// lane's rows in registers, 80 with a copy for each pair, 56 with 4 CTAs an SM,
// whose 64 registers spill.
constexpr int BWD_RUNS = 8, DEPTH = 4, PAIR = 2;

template <int W>
constexpr int BWD_SUMS = BWD_RUNS * 32 * ((W + 1) * PAIR + 1) * (int)sizeof(float);
template <typename T, int W, bool VEC>
constexpr int bwd_smem() {
    constexpr int ring = DEPTH * 8 * 256 * PAIR * (int)sizeof(T);
    return VEC && ring > BWD_SUMS<W> ? ring : BWD_SUMS<W>;
}
template <typename T>
__device__ __forceinline__ float2 pair(const Pack<T, PAIR>& p) { return make_float2(to_f(p.v[0]), to_f(p.v[1])); }

template <typename T, int W, bool VEC>
__global__ void __launch_bounds__(256, VEC ? 3 : 2) bwd_kernel(const Args a) {
    constexpr int K = PAIR;
    using P = Pack<T, K>;
    constexpr int S = (W + 1) * K;
    extern __shared__ __align__(16) unsigned char smem[];
    const int cx = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int c0 = blockIdx.x * 32 * K, have = a.D - c0 - cx * K;
    const int c = have > 0 ? c0 + cx * K : c0;  // lanes beyond the last channel copy along and store nothing
    const int b = blockIdx.z;
    const int t0 = (blockIdx.y * BWD_RUNS + g) * a.run, t1 = t0 + a.run < a.L ? t0 + a.run : a.L;
    const int len = length_of(a.lengths, b, a.L);
    const float2 zero = make_float2(0.0f, 0.0f);
    float2 dw[W], db = zero;
#pragma unroll
    for (int k = 0; k < W; k++) dw[k] = zero;
    if (t0 < a.L && (VEC || have > 0)) {
        const T* xb = static_cast<const T*>(a.x) + b * a.xb;
        const T* gb = static_cast<const T*>(a.dy) + b * a.gb;
        const T* gwin = static_cast<const T*>(a.dwin_out);
        T* dxb = static_cast<T*>(a.dx);
        if (dxb) dxb += (int64_t)b * a.L * a.D + c;
        const int last = len > 0 ? len - 1 : 0;
        // VEC: the ring [DEPTH][x, dy][4][64 channels]; a lane's part of a group is pack q of row r, or of rows r and r + 2
        constexpr int PACK = 16 / (int)sizeof(T), ROW = 32 * K, PER = ROW / PACK, PARTS = 4 * PER / 32;
        T* ring = reinterpret_cast<T*>(smem) + g * (DEPTH * 8 * ROW);
        const int q = cx % PER, r0 = cx / PER;
        const bool exists = c0 + q * PACK < a.D;
        const T *xq = xb + (exists ? c0 + q * PACK : 0), *gq = gb + (exists ? c0 + q * PACK : 0);
        P nx[4], ng[4];
        auto fetch = [&](int t, int slot) {
            if constexpr (VEC) {
#pragma unroll
                for (int i = 0; i < PARTS; i++) {
                    const int r = r0 + i * (32 / PER), bytes = exists && t + r < len ? 16 : 0;
                    const int64_t row = t + r < last ? t + r : last;
                    T* to = ring + (slot * 8 + r) * ROW + q * PACK;
                    cp_async<16>(to, xq + row * a.xl, bytes);
                    cp_async<16>(to + 4 * ROW, gq + row * a.gl, bytes);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int64_t row = t + j < last ? t + j : last;
                    nx[j] = raw_row<VEC, K>(xb + row * a.xl + c, have);
                    ng[j] = raw_row<VEC, K>(gb + row * a.gl + c, have);
                }
            }
        };
        const int te = t1 + W - 1;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < DEPTH - 1; i++) {
                if (t0 + 4 * i < te) fetch(t0 + 4 * i, i);
                cp_async_commit();
            }
        } else {
            fetch(t0, 0);
        }
        float2 x[W + 3], dc[W + 3], w[W], bias;  // inputs and dc from W - 1 positions before a group to its end
        {
            float xf[W - 1][K], wf[W][K], bf[K];
            rows_before<W, K, VEC, T>(a, b, t0, len, c, xf);
            load_w<W, K>(a, c, wf, bf);
#pragma unroll
            for (int k = 0; k < W - 1; k++) x[k] = make_float2(xf[k][0], xf[k][1]), dc[k] = zero;
#pragma unroll
            for (int k = 0; k < W; k++) w[k] = make_float2(wf[k][0], wf[k][1]);
            bias = make_float2(bf[0], bf[1]);
        }
        int slot = 0;
#pragma unroll 1
        for (int t = t0; t < te; t += 4) {
            if constexpr (VEC) {
                cp_async_wait<DEPTH - 2>();
                __syncwarp();  // every lane's part has come, and the slot behind this one has been read
                if (t + 4 * (DEPTH - 1) < te) fetch(t + 4 * (DEPTH - 1), (slot + DEPTH - 1) % DEPTH);
                cp_async_commit();
                const P* at = reinterpret_cast<const P*>(ring + slot * 8 * ROW) + cx;
#pragma unroll
                for (int j = 0; j < 4; j++) x[W - 1 + j] = pair(at[j * 32]), dc[W - 1 + j] = pair(at[(4 + j) * 32]);
                slot = (slot + 1) % DEPTH;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[W - 1 + j] = t + j < len ? pair(nx[j]) : zero;
                    dc[W - 1 + j] = t + j < len ? pair(ng[j]) : zero;
                }
                fetch(t + 4, 0);
            }
            if (a.silu) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float2 s = bias;
#pragma unroll
                    for (int k = 0; k < W; k++) s = __ffma2_rn(w[k], x[j + k], s);
                    const float2 sg = make_float2(sigmoid(s.x), sigmoid(s.y));
                    const float2 rest = __fadd2_rn(make_float2(1.0f, 1.0f), make_float2(-sg.x, -sg.y));
                    const float2 f = __fmul2_rn(sg, __ffma2_rn(s, rest, make_float2(1.0f, 1.0f)));
                    dc[W - 1 + j] = __fmul2_rn(dc[W - 1 + j], f);
                }
                if (t + 4 > len) {  // 0 whatever f is
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (t + j >= len) dc[W - 1 + j] = zero;
                }
            }
            if (t < t1) {  // the run's own positions that there are (an infinite input times the others' 0 is not 0)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (t + j >= len) continue;
                    db = __fadd2_rn(db, dc[W - 1 + j]);
#pragma unroll
                    for (int k = 0; k < W; k++) dw[k] = __ffma2_rn(dc[W - 1 + j], x[j + k], dw[k]);
                }
            }
            // dx of the positions W - 1 earlier
            float2 o[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                o[j] = __fmul2_rn(w[0], dc[j + W - 1]);
#pragma unroll
                for (int k = 1; k < W; k++) o[j] = __ffma2_rn(w[k], dc[j + W - 1 - k], o[j]);
            }
            const int td0 = t - (W - 1);
            if (t > t0 && t + 4 <= len && td0 + 4 <= t1) {  // inside, and in front of the window that leaves
                if (dxb && have > 0) {
                    T* to = dxb + (int64_t)td0 * a.D;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float v[K] = {o[j].x, o[j].y};
                        store_pack<K>(to + (int64_t)j * a.D, v, have, VEC);
                    }
                }
            } else if (t > t0 && td0 >= len && td0 + 4 <= t1) {  // behind the length
                if (dxb && have > 0) {
                    const float none[K] = {};
                    T* to = dxb + (int64_t)td0 * a.D;
#pragma unroll
                    for (int j = 0; j < 4; j++) store_pack<K>(to + (int64_t)j * a.D, none, have, VEC);
                }
            } else if (have > 0) {
                if (t == 0 || t + 4 > len) {  // of the positions that there are: 0 times an infinite weight is not 0
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        o[j] = zero;
#pragma unroll
                        for (int k = 0; k < W; k++) {
                            const int of = td0 + j + W - 1 - k;
                            if (of >= 0 && of < len) o[j] = __ffma2_rn(w[k], dc[j + W - 1 - k], o[j]);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int td = td0 + j;
                    // the run that begins the sequence also makes the window's gradients, dx at t = -(W-1) .. -1
                    if ((t0 > 0 && td < t0) || td >= t1) continue;
                    // this input's place in the window that leaves, if it has one
                    const int kw = td - (len - (W - 1));
                    if (gwin && kw >= 0 && kw < W - 1)
                        o[j] = __fadd2_rn(o[j],
                                          pair(raw_row<VEC, K>(gwin + ((int64_t)b * (W - 1) + kw) * a.D + c, have)));
                    const float v[K] = {o[j].x, o[j].y};
                    T* dwin = static_cast<T*>(a.dwin);
                    if (td >= 0 ? dxb != nullptr : dwin != nullptr)
                        store_pack<K>(td >= 0 ? dxb + (int64_t)td * a.D
                                              : dwin + ((int64_t)b * (W - 1) + td + W - 1) * a.D + c,
                                      v, have, VEC);
                }
            }
#pragma unroll
            for (int j = 0; j < W - 1; j++) x[j] = x[j + 4], dc[j] = dc[j + 4];
        }
    }
    if (!a.part) return;
    if constexpr (VEC) {
        cp_async_wait();
        __syncthreads();  // the slots are done with
    }
    float(*sh)[32][S + 1] = reinterpret_cast<float(*)[32][S + 1]>(smem);
#pragma unroll
    for (int k = 0; k < W; k++) sh[g][cx][k] = dw[k].x, sh[g][cx][W + 1 + k] = dw[k].y;
    sh[g][cx][W] = db.x, sh[g][cx][2 * W + 1] = db.y;
    __syncthreads();
    float* part = a.part + ((int64_t)b * gridDim.y + blockIdx.y) * a.D * (W + 1);
    for (int e = threadIdx.x; e < 32 * S; e += 256) {
        const int64_t o = (int64_t)blockIdx.x * 32 * S + e;
        if (o >= (int64_t)a.D * (W + 1)) break;
        float v = sh[0][e / S][e % S];
#pragma unroll
        for (int r = 1; r < BWD_RUNS; r++) v = __fadd_rn(v, sh[r][e / S][e % S]);
        part[o] = v;
    }
}

// dw [D, W] and dbias [D] from the partial rows [P, D, W + 1], added in order
// within four strands of each of 8 groups
__global__ void __launch_bounds__(256) sum_kernel(const float* __restrict__ part, float* __restrict__ dw,
                                                  float* __restrict__ db, int P, int D, int W) {
    __shared__ float sh[8][33];
    const int64_t cols = (int64_t)D * (W + 1);
    const int64_t e = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int g = threadIdx.x >> 5;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (e < cols) {
        int p = g;
        for (; p + 24 < P; p += 32)
#pragma unroll
            for (int j = 0; j < 4; j++) s[j] = __fadd_rn(s[j], part[(p + 8 * j) * cols + e]);
        for (; p < P; p += 8) s[0] = __fadd_rn(s[0], part[p * cols + e]);
    }
    sh[g][threadIdx.x & 31] = __fadd_rn(__fadd_rn(s[0], s[1]), __fadd_rn(s[2], s[3]));
    __syncthreads();
    if (g == 0 && e < cols) {
        float v = sh[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < 8; i++) v = __fadd_rn(v, sh[i][threadIdx.x]);
        const int c = (int)(e / (W + 1)), k = (int)(e % (W + 1));
        if (k < W) {
            if (dw) dw[(int64_t)c * W + k] = v;
        } else if (db) {
            db[c] = v;
        }
    }
}

// One new position a stream: y, and the window moved on in place.
template <typename T, int W, int K>
__global__ void __launch_bounds__(128) step_kernel(const Args a) {
    const int vecs = cdiv(a.D, K);
    const int64_t item = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    grid_dependency_sync();
    if (item >= (int64_t)vecs * a.batch) return;
    const int c = (int)(item % vecs) * K;
    const int b = (int)(item / vecs);
    const int valid = a.D - c;
    const bool vec = a.vec != 0;
    float w[W][K], bias[K];
    load_w<W, K>(a, c, w, bias);
    T* win = static_cast<T*>(a.win_out) + (int64_t)b * (W - 1) * a.D + c;
    float row[W][K];
    Pack<T, K> p[W];
#pragma unroll
    for (int k = 0; k < W - 1; k++) p[k] = load_pack<K>(win + (int64_t)k * a.D, valid, vec);
    p[W - 1] = load_pack<K>(static_cast<const T*>(a.x) + b * a.xb + c, valid, vec);
    float o[K];
#pragma unroll
    for (int i = 0; i < K; i++) {
        float s = bias[i];
#pragma unroll
        for (int k = 0; k < W; k++) {
            row[k][i] = to_f(p[k].v[i]);
            s = __fmaf_rn(w[k][i], row[k][i], s);
        }
        o[i] = a.silu ? __fmul_rn(s, sigmoid(s)) : s;
    }
    store_pack<K>(static_cast<T*>(a.y) + (int64_t)b * a.D + c, o, valid, vec);
#pragma unroll
    for (int k = 0; k < W - 1; k++) store_pack<K>(win + (int64_t)k * a.D, row[k + 1], valid, vec);
}

// Channels a thread of the forward kernels.  Wider packs need fewer loads, but
// what a thread holds for each channel (4 taps, 7 inputs) costs registers, and
// occupancy is worth more than the loads: 8 x 2048 x 1536 bf16 took 41 us with
// 8 channels (209 registers) and 37 with 4; with the loads off their branches
// 27 us (100 MB, 3.7 TB/s).  fp32 with 4 taps spills 32 bytes at the 96
// registers that 5 CTAs an SM leave: 46 us (201 MB, 4.4 TB/s).
constexpr int KF = 4;

template <typename T, int W>
static int forward(Args& a, cudaStream_t s) {
    // long runs read fewer rows twice and their taps once; short ones where they are what fills the GPU (148 x 768 threads)
    const int64_t lanes = (int64_t)cdiv(a.D, KF) * a.batch;
    a.run = 64;
    while (a.run > 8 && lanes * cdiv(a.L, a.run) < 148 * 768) a.run /= 2;
    const int64_t items = lanes * (a.L > 0 ? cdiv(a.L, a.run) : 1);
    const unsigned grid = (unsigned)((items + 127) / 128);
    if (a.vec)
        fwd_kernel<T, W, KF, true><<<grid, 128, 0, s>>>(a);
    else
        fwd_kernel<T, W, KF, false><<<grid, 128, 0, s>>>(a);
    MI_CHECK_LAUNCH();
    return MI_OK;
}

template <typename T, int W>
static int step(const Args& a, cudaStream_t s) {
    const int64_t items = (int64_t)cdiv(a.D, KF) * a.batch;
    MI_LAUNCH_DEPENDENT(step_kernel<T, W, KF>, (unsigned)((items + 127) / 128), 128, 0, s, a);
    return MI_OK;
}

// Positions a thread: of 16, 32 and 64 the one with the least rounds of 3 CTAs
// an SM times what a run walks, 4 positions beyond its own.  8 x 2048 x 1536:
// 52 us with 64 (2 rounds), 61 with 32 (4 rounds).
static inline int bwd_run(int batch, int L, int D) {
    int64_t best = 16, least = INT64_MAX;
    for (int run = 64; run >= 16; run /= 2) {
        const int64_t ctas = (int64_t)cdiv(D, 32 * PAIR) * cdiv(L, run * BWD_RUNS) * batch;
        const int64_t cost = (ctas + 148 * 3 - 1) / (148 * 3) * (run + 4);
        if (cost < least) least = cost, best = run;
    }
    return (int)best;
}
static inline int64_t parts(int batch, int L, int D) {
    return (int64_t)batch * cdiv(L, bwd_run(batch, L, D) * BWD_RUNS);
}

template <typename T, int W, bool VEC>
static int backward_vec(const Args& a, cudaStream_t s) {
    constexpr int smem = bwd_smem<T, W, VEC>();
    static std::atomic<uint64_t> allowed{0};
    if (!allow_smem(bwd_kernel<T, W, VEC>, smem, allowed)) return MI_ERR_CUDA;
    const dim3 grid(cdiv(a.D, 32 * PAIR), cdiv(a.L, a.run * BWD_RUNS), a.batch);
    bwd_kernel<T, W, VEC><<<grid, 256, smem, s>>>(a);
    MI_CHECK_LAUNCH();
    return MI_OK;
}
template <typename T, int W>
static int backward(Args& a, cudaStream_t s) {
    a.run = bwd_run(a.batch, a.L, a.D);
    return a.vec ? backward_vec<T, W, true>(a, s) : backward_vec<T, W, false>(a, s);
}

static int check(int batch, int L, int D, int W, int dtype) {
    if (batch < 0 || L < 0 || D <= 0) return MI_ERR_INVALID;
    if (dtype != MI_DT_F32 && dtype != MI_DT_BF16 && dtype != MI_DT_F16) return MI_ERR_INVALID;
    if (W < 2 || W > MAXW || batch > 65535 || L > 65535 * 16 * BWD_RUNS) return MI_ERR_UNSUPPORTED;
    return MI_OK;
}

}  // namespace conv1d
}  // namespace mi

#define MI_CONV_TAPS(W, FN, T, ...)             \
    do {                                        \
        if ((W) == 2) return FN<T, 2>(__VA_ARGS__); \
        if ((W) == 3) return FN<T, 3>(__VA_ARGS__); \
        return FN<T, 4>(__VA_ARGS__);           \
    } while (0)

extern "C" int mi_causal_conv1d(const void* x, int64_t x_batch, int64_t x_row, const float* w, const float* bias,
                                const void* win, const int32_t* lengths, void* y, void* win_out, int batch, int L,
                                int D, int W, int silu, int dtype, void* stream) {
    using namespace mi::conv1d;
    const int rc = check(batch, L, D, W, dtype);
    if (rc != MI_OK) return rc;
    if (batch == 0 || (L == 0 && !win_out)) return MI_OK;
    if (!w || (L > 0 && (!x || !y))) return MI_ERR_INVALID;
    Args a = {};
    a.x = x, a.xb = x_batch, a.xl = x_row, a.w = w, a.bias = bias, a.win = win, a.lengths = lengths;
    a.y = y, a.win_out = win_out, a.batch = batch, a.L = L, a.D = D, a.silu = silu;
    a.vec = D % KF == 0 && x_batch % KF == 0 && x_row % KF == 0 && mi::aligned16(x) && mi::aligned16(y) &&
            mi::aligned16(win) && mi::aligned16(win_out) && mi::aligned16(w) && mi::aligned16(bias);
    MI_DISPATCH_DTYPE(dtype, T, MI_CONV_TAPS(W, forward, T, a, (cudaStream_t)stream));
    return MI_ERR_INVALID;
}

extern "C" int mi_causal_conv1d_step(const void* x, int64_t x_batch, const float* w, const float* bias, void* win,
                                     void* y, int batch, int D, int W, int silu, int dtype, void* stream) {
    using namespace mi::conv1d;
    const int rc = check(batch < 0 ? -1 : 0, 1, D, W, dtype);
    if (rc != MI_OK) return rc;
    if (batch == 0) return MI_OK;
    if (!x || !w || !win || !y) return MI_ERR_INVALID;
    Args a = {};
    a.x = x, a.xb = x_batch, a.w = w, a.bias = bias, a.win_out = win, a.y = y;
    a.batch = batch, a.L = 1, a.D = D, a.silu = silu;
    a.vec = D % KF == 0 && x_batch % KF == 0 && mi::aligned16(x) && mi::aligned16(y) && mi::aligned16(win) &&
            mi::aligned16(w) && mi::aligned16(bias);
    MI_DISPATCH_DTYPE(dtype, T, MI_CONV_TAPS(W, step, T, a, (cudaStream_t)stream));
    return MI_ERR_INVALID;
}

extern "C" int64_t mi_causal_conv1d_backward_workspace(int batch, int L, int D, int W) {
    if (batch <= 0 || L <= 0 || D <= 0 || W < 2 || W > mi::conv1d::MAXW) return 0;
    return (int64_t)sizeof(float) * mi::conv1d::parts(batch, L, D) * D * (W + 1);
}

extern "C" int mi_causal_conv1d_backward(const void* dy, int64_t dy_batch, int64_t dy_row, const void* dwin_out,
                                         const void* x, int64_t x_batch, int64_t x_row, const float* w,
                                         const float* bias, const void* win, const int32_t* lengths, void* dx,
                                         float* dw, float* dbias, void* dwin, void* workspace, int batch, int L, int D,
                                         int W, int silu, int dtype, void* stream) {
    using namespace mi::conv1d;
    const int rc = check(batch, L, D, W, dtype);
    if (rc != MI_OK) return rc;
    if (batch == 0 || L == 0) return MI_ERR_INVALID;  // nothing to walk: the caller's gradients are zeros and copies
    if (!dy || !x || !w || (!dx && !dw && !dbias && !dwin)) return MI_ERR_INVALID;
    if ((dw || dbias) && !workspace) return MI_ERR_INVALID;
    cudaStream_t s = (cudaStream_t)stream;
    Args a = {};
    a.x = x, a.xb = x_batch, a.xl = x_row, a.w = w, a.bias = bias, a.win = win, a.lengths = lengths;
    a.dy = dy, a.gb = dy_batch, a.gl = dy_row, a.dwin_out = dwin_out, a.dx = dx, a.dwin = dwin;
    a.part = dw || dbias ? static_cast<float*>(workspace) : nullptr;
    a.batch = batch, a.L = L, a.D = D, a.silu = silu;
    const int pack = dtype == MI_DT_F32 ? 4 : 8;
    a.vec = D % pack == 0 && x_batch % pack == 0 && x_row % pack == 0 && dy_batch % pack == 0 && dy_row % pack == 0 &&
            mi::aligned16(x) && mi::aligned16(dy) && mi::aligned16(win) && mi::aligned16(dwin_out) &&
            mi::aligned16(dx) && mi::aligned16(dwin) && mi::aligned16(w) && mi::aligned16(bias);
    int (*fn)(Args&, cudaStream_t) = nullptr;
    MI_DISPATCH_DTYPE(dtype, T, fn = W == 2 ? backward<T, 2> : W == 3 ? backward<T, 3> : backward<T, 4>);
    const int rc2 = fn(a, s);
    if (rc2 != MI_OK || !a.part) return rc2;
    const int64_t cols = (int64_t)D * (W + 1);
    sum_kernel<<<(unsigned)((cols + 31) / 32), 256, 0, s>>>(a.part, dw, dbias, (int)parts(batch, L, D), D, W);
    MI_CHECK_LAUNCH();
    return MI_OK;
}

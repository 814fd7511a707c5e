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

// Backward.  A CTA is 32 channel packs by 8 runs of one sequence.  A thread
// walks its run forward, 4 positions at a time: dc[t] needs x up to t, dx[t]
// needs dc up to t + W - 1, so it goes W - 1 positions past its run, and dx
// comes out W - 1 positions late.  Its own positions' terms of dw and dbias stay in registers;
// the CTA adds its 8 runs in shared memory, in order, and writes one partial
// row, which sum_kernel adds.
constexpr int BWD_RUNS = 8;  // of a.run positions: 16 or 32

template <typename T, int W, int K, bool VEC>
__global__ void __launch_bounds__(256, 2) bwd_kernel(const Args a) {
    using P = Pack<T, K>;
    constexpr int S = (W + 1) * K;
    __shared__ float sh[BWD_RUNS][32][S + 1];
    const int cx = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int c = (blockIdx.x * 32 + cx) * K, have = a.D - c;
    const int b = blockIdx.z;
    const int t0 = (blockIdx.y * BWD_RUNS + g) * a.run, t1 = t0 + a.run < a.L ? t0 + a.run : a.L;
    const int len = length_of(a.lengths, b, a.L);
    float dw[W][K], db[K];
#pragma unroll
    for (int i = 0; i < K; i++) {
        db[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < W; k++) dw[k][i] = 0.0f;
    }
    if (have > 0 && t0 < a.L) {
        const T* xb = static_cast<const T*>(a.x) + b * a.xb + c;
        const T* gb = static_cast<const T*>(a.dy) + b * a.gb + c;
        const T* gwin = static_cast<const T*>(a.dwin_out);
        const int last = len > 0 ? len - 1 : 0;
        P nx[4], ng[4];
        auto fetch = [&](int t) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int64_t r = t + j < last ? t + j : last;
                nx[j] = raw_row<VEC, K>(xb + r * a.xl, have);
                ng[j] = raw_row<VEC, K>(gb + r * a.gl, have);
            }
        };
        fetch(t0);
        float w[W][K], bias[K];
        float x[W + 3][K], dc[W + 3][K];  // inputs and dc from W - 1 positions before a group to its end
        rows_before<W, K, VEC, T>(a, b, t0, len, c, reinterpret_cast<float(&)[W - 1][K]>(x));
        load_w<W, K>(a, c, w, bias);
#pragma unroll
        for (int j = 0; j < W - 1; j++)
#pragma unroll
            for (int i = 0; i < K; i++) dc[j][i] = 0.0f;
        // the run that begins the sequence also makes the window's gradients, dx at t = -(W-1) .. -1
        const int first = t0 == 0 ? -(W - 1) : t0;
#pragma unroll 1
        for (int t = t0; t < t1 + W - 1; t += 4) {
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < K; i++) {
                    x[W - 1 + j][i] = t + j < len ? to_f(nx[j].v[i]) : 0.0f;
                    dc[W - 1 + j][i] = t + j < len ? to_f(ng[j].v[i]) : 0.0f;
                }
            fetch(t + 4);
            if (a.silu) {
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int i = 0; i < K; i++) {
                        float s = bias[i];
#pragma unroll
                        for (int k = 0; k < W; k++) s = __fmaf_rn(w[k][i], x[j + k][i], s);
                        const float sg = sigmoid(s);
                        const float f = __fmul_rn(sg, __fmaf_rn(s, __fsub_rn(1.0f, sg), 1.0f));
                        dc[W - 1 + j][i] = t + j < len ? __fmul_rn(dc[W - 1 + j][i], f) : 0.0f;
                    }
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (t + j < t1) {  // the run's own positions
#pragma unroll
                    for (int i = 0; i < K; i++) {
                        db[i] = __fadd_rn(db[i], dc[W - 1 + j][i]);
#pragma unroll
                        for (int k = 0; k < W; k++) dw[k][i] = __fmaf_rn(dc[W - 1 + j][i], x[j + k][i], dw[k][i]);
                    }
                }
            // dx of the positions W - 1 earlier
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int td = t + j - (W - 1);
                T* to = td >= 0 ? static_cast<T*>(a.dx) : static_cast<T*>(a.dwin);
                if (td < first || td >= t1 || !to) continue;
                float o[K];
#pragma unroll
                for (int i = 0; i < K; i++) {
                    float s = __fmul_rn(w[0][i], dc[j + W - 1][i]);
#pragma unroll
                    for (int k = 1; k < W; k++) s = __fmaf_rn(w[k][i], dc[j + W - 1 - k][i], s);
                    o[i] = s;
                }
                // this input's place in the window that leaves, if it has one
                const int kw = td - (len - (W - 1));
                if (gwin && kw >= 0 && kw < W - 1) {
                    const P p = raw_row<VEC, K>(gwin + ((int64_t)b * (W - 1) + kw) * a.D + c, have);
#pragma unroll
                    for (int i = 0; i < K; i++) o[i] = __fadd_rn(o[i], to_f(p.v[i]));
                }
                store_pack<K>(to + (td >= 0 ? (int64_t)b * a.L + td : (int64_t)b * (W - 1) + td + W - 1) * a.D + c, o, have,
                              VEC);
            }
#pragma unroll
            for (int j = 0; j < W - 1; j++)
#pragma unroll
                for (int i = 0; i < K; i++) x[j][i] = x[j + 4][i], dc[j][i] = dc[j + 4][i];
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < K; i++) {
#pragma unroll
        for (int k = 0; k < W; k++) sh[g][cx][i * (W + 1) + k] = dw[k][i];
        sh[g][cx][i * (W + 1) + W] = db[i];
    }
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

// Channels a thread.  Wider packs need fewer loads, but what a thread holds for
// each channel (4 taps, 7 inputs; backward 4 sums and 7 dc more) costs
// registers, and occupancy is worth more than the loads: 8 x 2048 x 1536 bf16
// took 41 us forward with 8 channels (209 registers) and 37 with 4.
constexpr int KF = 4, KB = 2;

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

// positions a thread: 32 where that still gives every SM 4 CTAs
static inline int bwd_run(int batch, int L, int D) {
    return (int64_t)cdiv(D, 32 * KB) * cdiv(L, 32 * BWD_RUNS) * batch >= 148 * 4 ? 32 : 16;
}
static inline int64_t parts(int batch, int L, int D) {
    return (int64_t)batch * cdiv(L, bwd_run(batch, L, D) * BWD_RUNS);
}

template <typename T, int W>
static int backward(Args& a, cudaStream_t s) {
    a.run = bwd_run(a.batch, a.L, a.D);
    const dim3 grid(cdiv(a.D, 32 * KB), cdiv(a.L, a.run * BWD_RUNS), a.batch);
    if (a.vec)
        bwd_kernel<T, W, KB, true><<<grid, 256, 0, s>>>(a);
    else
        bwd_kernel<T, W, KB, false><<<grid, 256, 0, s>>>(a);
    MI_CHECK_LAUNCH();
    return MI_OK;
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
    a.vec = D % KF == 0 && x_batch % KF == 0 && x_row % KF == 0 && dy_batch % KF == 0 && dy_row % KF == 0 &&
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

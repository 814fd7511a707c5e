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

constexpr int RUN = 16;   // positions a thread
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
#pragma unroll
    for (int i = 0; i < K; i++) {
        const bool in = c + i < a.D;
#pragma unroll
        for (int k = 0; k < W; k++) w[k][i] = in ? a.w[(int64_t)(c + i) * W + k] : 0.0f;
        bias[i] = in && a.bias ? a.bias[c + i] : 0.0f;
    }
}

template <typename T, int W, int K>
__global__ void __launch_bounds__(128) fwd_kernel(const Args a) {
    const int vecs = cdiv(a.D, K);
    const int runs = a.L > 0 ? cdiv(a.L, RUN) : 1;  // an empty sequence still passes its window on
    const int64_t item = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (item >= (int64_t)vecs * runs * a.batch) return;
    const int c = (int)(item % vecs) * K;
    const int run = (int)(item / vecs % runs), b = (int)(item / vecs / runs);
    const bool vec = a.vec != 0;
    const int len = length_of(a.lengths, b, a.L);
    const int t0 = run * RUN, t1 = t0 + RUN < a.L ? t0 + RUN : a.L;
    T* y = static_cast<T*>(a.y) + ((int64_t)b * a.L) * a.D + c;
    float w[W][K], bias[K];
    load_w<W, K>(a, c, w, bias);
    float row[W][K];  // the inputs of the last W positions, oldest first
#pragma unroll
    for (int k = 0; k < W - 1; k++) {
        const int t = t0 - (W - 1) + k;
        if (t < len) {
            const Pack<T, K> p = load_x<W, K, T>(a, b, t, c, vec);
#pragma unroll
            for (int i = 0; i < K; i++) row[k + 1][i] = to_f(p.v[i]);
        }
    }
#pragma unroll 1
    for (int t = t0; t < t1; t += 4) {
        Pack<T, K> p[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (t + j < t1 && t + j < len) p[j] = load_x<W, K, T>(a, b, t + j, c, vec);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (t + j >= t1) break;
            float o[K];
            if (t + j < len) {
#pragma unroll
                for (int i = 0; i < K; i++) {
#pragma unroll
                    for (int k = 0; k < W - 1; k++) row[k][i] = row[k + 1][i];
                    row[W - 1][i] = to_f(p[j].v[i]);
                    float s = bias[i];
#pragma unroll
                    for (int k = 0; k < W; k++) s = __fmaf_rn(w[k][i], row[k][i], s);
                    o[i] = a.silu ? __fmul_rn(s, sigmoid(s)) : s;
                }
            } else {
#pragma unroll
                for (int i = 0; i < K; i++) o[i] = 0.0f;
            }
            store_pack<K>(y + (int64_t)(t + j) * a.D, o, a.D - c, vec);
        }
    }
    // the window that leaves: inputs len - W + 1 .. len - 1, by the first run
    if (run == 0 && a.win_out) {
#pragma unroll
        for (int k = 0; k < W - 1; k++) {
            const Pack<T, K> p = load_x<W, K, T>(a, b, len - (W - 1) + k, c, vec);
            float o[K];
#pragma unroll
            for (int i = 0; i < K; i++) o[i] = to_f(p.v[i]);
            store_pack<K>(static_cast<T*>(a.win_out) + ((int64_t)b * (W - 1) + k) * a.D + c, o, a.D - c, vec);
        }
    }
}

// Backward.  A CTA is 32 channel packs by 8 runs of one sequence.  A thread
// walks its run forward: dc[t] needs x up to t, dx[t] needs dc up to
// t + W - 1, so it goes W - 1 positions past its run, and dx comes out W - 1
// positions late.  Its own positions' terms of dw and dbias stay in registers;
// the CTA adds its 8 runs in shared memory, in order, and writes one partial
// row, which sum_kernel adds.
constexpr int BWD_RUNS = 8;

template <typename T, int W, int K>
__global__ void __launch_bounds__(256) bwd_kernel(const Args a) {
    constexpr int S = (W + 1) * K;
    __shared__ float sh[BWD_RUNS][32][S + 1];
    const int cx = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int c = (blockIdx.x * 32 + cx) * K;
    const int b = blockIdx.z;
    const int t0 = (blockIdx.y * BWD_RUNS + g) * RUN, t1 = t0 + RUN < a.L ? t0 + RUN : a.L;
    const bool vec = a.vec != 0;
    const int len = length_of(a.lengths, b, a.L);
    float dw[W][K], db[K];
#pragma unroll
    for (int i = 0; i < K; i++) {
        db[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < W; k++) dw[k][i] = 0.0f;
    }
    if (c < a.D && t0 < a.L) {
        float w[W][K], bias[K];
        load_w<W, K>(a, c, w, bias);
        const T* dyp = static_cast<const T*>(a.dy) + b * a.gb + c;
        T* dxp = static_cast<T*>(a.dx) + (int64_t)b * a.L * a.D + c;
        const T* gwin = static_cast<const T*>(a.dwin_out);
        float row[W][K], dc[W][K];  // the last W inputs and the last W dc, oldest first
#pragma unroll
        for (int i = 0; i < K; i++)
#pragma unroll
            for (int k = 0; k < W; k++) row[k][i] = dc[k][i] = 0.0f;
        // the run that begins the sequence also makes the window's gradients,
        // dx at t = -(W-1) .. -1
        const int first = t0 == 0 ? -(W - 1) : t0;
#pragma unroll
        for (int k = 0; k < W - 1; k++) {
            const int t = t0 - (W - 1) + k;
            if (t < len) {
                const Pack<T, K> p = load_x<W, K, T>(a, b, t, c, vec);
#pragma unroll
                for (int i = 0; i < K; i++) row[k + 1][i] = to_f(p.v[i]);
            }
        }
#pragma unroll 1
        for (int tb = t0; tb < t1 + W - 1; tb += 4) {
            Pack<T, K> px[4], pg[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int t = tb + j;
                if (t < t1 + W - 1 && t < len) {
                    px[j] = load_x<W, K, T>(a, b, t, c, vec);
                    pg[j] = load_pack<K>(dyp + t * a.gl, a.D - c, vec);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int t = tb + j;
                if (t >= t1 + W - 1) break;
#pragma unroll
                for (int i = 0; i < K; i++)
#pragma unroll
                    for (int k = 0; k < W - 1; k++) dc[k][i] = dc[k + 1][i];
                if (t < len) {
#pragma unroll
                    for (int i = 0; i < K; i++) {
#pragma unroll
                        for (int k = 0; k < W - 1; k++) row[k][i] = row[k + 1][i];
                        row[W - 1][i] = to_f(px[j].v[i]);
                        float gr = to_f(pg[j].v[i]);
                        if (a.silu) {
                            float s = bias[i];
#pragma unroll
                            for (int k = 0; k < W; k++) s = __fmaf_rn(w[k][i], row[k][i], s);
                            const float sg = sigmoid(s);
                            gr = __fmul_rn(gr, __fmul_rn(sg, __fmaf_rn(s, __fsub_rn(1.0f, sg), 1.0f)));
                        }
                        dc[W - 1][i] = gr;
                        if (t < t1) {
                            db[i] = __fadd_rn(db[i], gr);
#pragma unroll
                            for (int k = 0; k < W; k++) dw[k][i] = __fmaf_rn(gr, row[k][i], dw[k][i]);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < K; i++) dc[W - 1][i] = 0.0f;
                }
                // dx at td = t - (W - 1), whose last reader is t; dc[j] is dc at td + j
                const int td = t - (W - 1);
                if (td >= first && td < t1 && (td < 0 ? a.dwin != nullptr : a.dx != nullptr)) {
                    float o[K];
#pragma unroll
                    for (int i = 0; i < K; i++) {
                        float s = 0.0f;
#pragma unroll
                        for (int k = 0; k < W; k++) s = __fmaf_rn(w[k][i], dc[W - 1 - k][i], s);
                        o[i] = s;
                    }
                    // this input's place in the window that leaves, if it has one
                    const int kw = td - (len - (W - 1));
                    if (gwin && kw >= 0 && kw < W - 1) {
                        const Pack<T, K> p = load_pack<K>(gwin + ((int64_t)b * (W - 1) + kw) * a.D + c, a.D - c, vec);
#pragma unroll
                        for (int i = 0; i < K; i++) o[i] = __fadd_rn(o[i], to_f(p.v[i]));
                    }
                    if (td < 0)
                        store_pack<K>(static_cast<T*>(a.dwin) + ((int64_t)b * (W - 1) + td + W - 1) * a.D + c, o,
                                      a.D - c, vec);
                    else
                        store_pack<K>(dxp + (int64_t)td * a.D, o, a.D - c, vec);
                }
            }
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

constexpr int KF = 4;  // channels a thread: 16 bytes of fp32, 8 of 16-bit types

template <typename T, int W>
static int forward(const Args& a, cudaStream_t s) {
    const int64_t items = (int64_t)cdiv(a.D, KF) * (a.L > 0 ? cdiv(a.L, RUN) : 1) * a.batch;
    fwd_kernel<T, W, KF><<<(unsigned)((items + 127) / 128), 128, 0, s>>>(a);
    MI_CHECK_LAUNCH();
    return MI_OK;
}

template <typename T, int W>
static int step(const Args& a, cudaStream_t s) {
    const int64_t items = (int64_t)cdiv(a.D, KF) * a.batch;
    MI_LAUNCH_DEPENDENT(step_kernel<T, W, KF>, (unsigned)((items + 127) / 128), 128, 0, s, a);
    return MI_OK;
}

template <typename T, int W>
static int backward(const Args& a, cudaStream_t s) {
    const dim3 grid(cdiv(a.D, 32 * KF), cdiv(cdiv(a.L, RUN), BWD_RUNS), a.batch);
    bwd_kernel<T, W, KF><<<grid, 256, 0, s>>>(a);
    MI_CHECK_LAUNCH();
    return MI_OK;
}

static int check(int batch, int L, int D, int W, int dtype) {
    if (batch < 0 || L < 0 || D <= 0) return MI_ERR_INVALID;
    if (dtype != MI_DT_F32 && dtype != MI_DT_BF16 && dtype != MI_DT_F16) return MI_ERR_INVALID;
    if (W < 2 || W > MAXW || batch > 65535 || L > 65535 * RUN * BWD_RUNS) return MI_ERR_UNSUPPORTED;
    return MI_OK;
}

static inline int64_t parts(int batch, int L) { return (int64_t)batch * cdiv(cdiv(L, RUN), BWD_RUNS); }

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
            mi::aligned16(win) && mi::aligned16(win_out);
    MI_DISPATCH_DTYPE(dtype, T, MI_CONV_TAPS(W, forward, T, a, (cudaStream_t)stream));
    return MI_ERR_INVALID;
}

extern "C" int mi_causal_conv1d_step(const void* x, int64_t x_batch, const float* w, const float* bias, void* win,
                                     void* y, int batch, int D, int W, int silu, int dtype, void* stream) {
    using namespace mi::conv1d;
    const int rc = check(batch, 1, D, W, dtype);
    if (rc != MI_OK) return rc;
    if (batch == 0) return MI_OK;
    if (!x || !w || !win || !y) return MI_ERR_INVALID;
    Args a = {};
    a.x = x, a.xb = x_batch, a.w = w, a.bias = bias, a.win_out = win, a.y = y;
    a.batch = batch, a.L = 1, a.D = D, a.silu = silu;
    a.vec = D % KF == 0 && x_batch % KF == 0 && mi::aligned16(x) && mi::aligned16(y) && mi::aligned16(win);
    MI_DISPATCH_DTYPE(dtype, T, MI_CONV_TAPS(W, step, T, a, (cudaStream_t)stream));
    return MI_ERR_INVALID;
}

extern "C" int64_t mi_causal_conv1d_backward_workspace(int batch, int L, int D, int W) {
    if (batch <= 0 || L <= 0 || D <= 0 || W < 2 || W > mi::conv1d::MAXW) return 0;
    return (int64_t)sizeof(float) * mi::conv1d::parts(batch, L) * D * (W + 1);
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
            mi::aligned16(dx) && mi::aligned16(dwin);
    int (*fn)(const Args&, cudaStream_t) = nullptr;
    MI_DISPATCH_DTYPE(dtype, T, fn = W == 2 ? backward<T, 2> : W == 3 ? backward<T, 3> : backward<T, 4>);
    const int rc2 = fn(a, s);
    if (rc2 != MI_OK || !a.part) return rc2;
    const int64_t cols = (int64_t)D * (W + 1);
    sum_kernel<<<(unsigned)((cols + 31) / 32), 256, 0, s>>>(a.part, dw, dbias, (int)parts(batch, L), D, W);
    MI_CHECK_LAUNCH();
    return MI_OK;
}

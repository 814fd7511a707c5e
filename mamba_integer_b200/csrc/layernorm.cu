// layernorm.cu -- layer norm with the residual's addition in front of it, and
// its backward pass.
//
//   s = x + r                     (kept in r's type; s = x without a residual)
//   mean = sum(s) / D;  var = sum((s - mean)^2) / D;  rstd = 1 / sqrt(var + eps)
//   xhat = (s - mean) rstd;  y = xhat w + b
// and, with g = w dy,
//   ds = rstd (g - mean(g) - xhat mean(g xhat)) + dsum
//   dw = sum over rows of dy xhat;  db = sum over rows of dy
//
// Every row is read once and held in registers between the reductions and the
// output, so the bound is HBM: x and r in, s and y out; backwards s, dy and dsum
// in, ds out.  The variance is that of the centred row: the difference of two
// means would lose what is left of a row far from 0.
//
// Layout: a row belongs to TPR threads of NV packs of 8 neighbouring elements.
// Rows within a warp reduce by shuffles alone, longer ones through shared memory
// behind a barrier of the row's own warps.  The next rows' packs come by
// asynchronous copies into slots of the thread's own.
#include "mi_elem.cuh"

namespace mi {
namespace ln {

constexpr int K = 8, MAX_BLOCK = 512, MAX_D = 16384;

struct Args {
    const void* x;
    const void* r;
    const float* w;
    const float* b;    // may be NULL
    void* y;
    void* sum;         // forward: s, in r's type (NULL without a residual); backward: s
    float2* stats;     // [T]: mean and rstd; forward out (may be NULL), backward in
    const void* dy;
    const void* dsum;  // may be NULL
    void* dx;          // may be NULL
    void* dr;          // in r's type, may be NULL
    float* part;       // [gridDim.x, 2, D]: sums of dw and db, or NULL
    int64_t ldx, ldr;  // row strides of x and of r (backward: of s) in elements
    int T, D, tpr;
    float eps;
};

__device__ __forceinline__ float2 dup(float v) { return make_float2(v, v); }

// Sums over the threads of a row, in a fixed order; N values at once.  `red`:
// 2 x MAX_BLOCK / 32 x N slots, whose halves are taken in turn, so that one
// barrier is enough.
template <typename V, int N>
struct Reduce {
    V (*red)[MAX_BLOCK / 32][N];
    int tpr, half;
    __device__ __forceinline__ static float add(float a, float b) { return __fadd_rn(a, b); }
    __device__ __forceinline__ static float2 add(float2 a, float2 b) { return __fadd2_rn(a, b); }
    __device__ __forceinline__ static float shift(float v, int m) { return __shfl_xor_sync(0xffffffffu, v, m); }
    __device__ __forceinline__ static float2 shift(float2 v, int m) {
        return make_float2(__shfl_xor_sync(0xffffffffu, v.x, m), __shfl_xor_sync(0xffffffffu, v.y, m));
    }
    __device__ __forceinline__ void operator()(V (&v)[N]) {
        if (tpr < 32) {
            for (int m = tpr >> 1; m; m >>= 1)
#pragma unroll
                for (int k = 0; k < N; k++) v[k] = add(v[k], shift(v[k], m));
            return;
        }
#pragma unroll
        for (int m = 16; m; m >>= 1)
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = add(v[k], shift(v[k], m));
        if (tpr > 32) {
            const int warps = tpr >> 5, group = threadIdx.x / tpr, first = group * warps;
            V(*at)[N] = red[half];
            if ((threadIdx.x & 31) == 0) {
#pragma unroll
                for (int k = 0; k < N; k++) at[threadIdx.x >> 5][k] = v[k];
            }
            asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(tpr) : "memory");
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = at[first][k];
            for (int i = 1; i < warps; i++)
#pragma unroll
                for (int k = 0; k < N; k++) v[k] = add(v[k], at[first + i][k]);
            half ^= 1;
        }
    }
};

// The columns of a thread.  VEC, where every row starts on 16 bytes and is whole
// packs: pack j is 8 neighbouring ones, copied into slots of the thread's own.
// Else element i of pack j lies (8 j + i) TPR behind the thread's first, so that a
// warp's accesses are one stretch; the row's threads copy the 16-byte blocks that
// hold the row into a window of the row's, which starts inside the first one.
// 16384 x 761 bf16 with a residual: forward 65 us and backward 58 with plain loads.
template <bool VEC>
struct Columns {
    int tpr, lane, D;
    __device__ __forceinline__ int at(int j, int i = 0) const { return VEC ? (j * tpr + lane) * K + i : (j * K + i) * tpr + lane; }
    __device__ __forceinline__ bool any(int j) const { return at(j) < D; }
    __device__ __forceinline__ bool has(int j, int i) const { return VEC ? any(j) : at(j, i) < D; }
    // pack j of a row, zeros where there is none (all of it without `some`)
    template <typename T>
    __device__ __forceinline__ Pack<T, K> read(const T* row, int j, bool some = true) const {
        Pack<T, K> v;
#pragma unroll
        for (int i = 0; i < K; i++) v.v[i] = from_f<T>(0.0f);
        if (VEC) {
            if (some && any(j)) v = *reinterpret_cast<const Pack<T, K>*>(row + at(j));
        } else {
#pragma unroll
            for (int i = 0; i < K; i++)
                if (some && has(j, i)) v.v[i] = row[at(j, i)];
        }
        return v;
    }
    template <typename T>
    __device__ __forceinline__ void write(T* row, int j, const Pack<T, K>& v) const {
        if (VEC) {
            if (any(j)) *reinterpret_cast<Pack<T, K>*>(row + at(j)) = v;
        } else {
#pragma unroll
            for (int i = 0; i < K; i++)
                if (has(j, i)) row[at(j, i)] = v.v[i];
        }
    }
    template <typename T>
    __device__ __forceinline__ void write(T* row, int j, const float (&f)[K]) const {
        Pack<T, K> v;
#pragma unroll
        for (int i = 0; i < K; i++) v.v[i] = from_f<T>(f[i]);
        write(row, j, v);
    }
};

// A whole pack into this thread's slot (`some`), or zeros.
template <typename T>
__device__ __forceinline__ void fetch_whole(Pack<T, K>& slot, const T* p, const void* any, bool some) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(Pack<T, K>) / 16; i++)
        cp_async<16>(reinterpret_cast<char*>(&slot) + 16 * i,
                     some ? reinterpret_cast<const char*>(p) + 16 * i : static_cast<const char*>(any), some ? 16 : 0);
}
template <typename T, int NV>
__host__ __device__ constexpr int window_bytes(int tpr) { return NV * tpr * (int)sizeof(Pack<T, K>) + 16; }
template <typename T>
__device__ __forceinline__ void fetch_window(char* to, const T* row, int D, int lane, int tpr) {
    const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15), all = off + D * (int)sizeof(T);
    const char* from = reinterpret_cast<const char*>(row) - off;
    for (int at = 16 * lane; at < all; at += 16 * tpr) cp_async<16>(to + at, from + at, all - at < 16 ? all - at : 16);
}
template <typename T>
__device__ __forceinline__ const T* in_window(const char* window, const T* row) {
    return reinterpret_cast<const T*>(window + (reinterpret_cast<uintptr_t>(row) & 15));
}
// All threads of a row have come here (their copies into its window are there).
__device__ __forceinline__ void row_sync(int tpr) {
    if (tpr > 32)
        asm volatile("bar.sync %0, %1;" ::"r"((int)threadIdx.x / tpr + 1), "r"(tpr) : "memory");
    else
        __syncwarp();
}
// Behind a reduction, before the row's window is filled again by all of its threads:
// every one has read it.  Rows of several warps have met at the reduction's barrier;
// the shuffles of those within a warp put no order on shared memory.
__device__ __forceinline__ void window_read() { __syncwarp(); }
template <typename T>
__device__ __forceinline__ float2 two(const Pack<T, K>& p, int i) {
    return make_float2(to_f(p.v[2 * i]), to_f(p.v[2 * i + 1]));
}

template <typename T, typename R, int NV>
constexpr int STAGES = NV * K * (sizeof(T) + sizeof(R)) <= 32 ? 2 : 1;

// BLOCK 256: rows within a warp (or 128 threads of few rows), two CTAs an SM.
template <typename T, typename R, int NV, bool VEC, int BLOCK>
__global__ void __launch_bounds__(BLOCK, BLOCK > 256 ? 1 : 2) fwd_kernel(const Args a) {
    constexpr int ST = STAGES<T, R, NV>;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float red[2][MAX_BLOCK / 32][1];
    const int tid = threadIdx.x, tpr = a.tpr, group = tid / tpr, rows = blockDim.x / tpr;
    const int lane = tid - group * tpr, block = blockDim.x;
    Pack<T, K>* xs = reinterpret_cast<Pack<T, K>*>(smem);                                          // [ST][NV][block]
    Pack<R, K>* rs = reinterpret_cast<Pack<R, K>*>(smem + sizeof(Pack<T, K>) * ST * NV * block);   // [ST][NV][block]
    const int wx = window_bytes<T, NV>(tpr), wr = window_bytes<R, NV>(tpr);  // not VEC: [ST][rows] of x's, then of r's
    auto x_window = [&](int k) { return reinterpret_cast<char*>(smem) + (k * rows + group) * wx; };
    auto r_window = [&](int k) { return reinterpret_cast<char*>(smem) + ST * rows * wx + (k * rows + group) * wr; };
    Reduce<float, 1> reduce = {red, tpr, 0};
    grid_dependency_sync();
    const Columns<VEC> cols = {tpr, lane, a.D};
    auto fetch = [&](int64_t t, int k) {
        if (!VEC && t < a.T) {
            fetch_window(x_window(k), static_cast<const T*>(a.x) + t * a.ldx, a.D, lane, tpr);
            if (a.r) fetch_window(r_window(k), static_cast<const R*>(a.r) + t * a.ldr, a.D, lane, tpr);
        }
#pragma unroll
        for (int j = 0; VEC && j < NV; j++) {
            const int c = cols.at(j);
            const bool some = t < a.T && cols.any(j);
            fetch_whole(xs[(k * NV + j) * block + tid], static_cast<const T*>(a.x) + t * a.ldx + c, a.x, some);
            if (a.r) fetch_whole(rs[(k * NV + j) * block + tid], static_cast<const R*>(a.r) + t * a.ldr + c, a.r, some);
        }
        cp_async_commit();
    };
    const int64_t step = (int64_t)gridDim.x * rows, first = (int64_t)blockIdx.x * rows + group;
#pragma unroll
    for (int i = 0; i < ST; i++) fetch(first + i * step, i);
    const float n = (float)a.D;
    int k = 0;
    // the threads of a row that does not exist still take part in the reductions
#pragma unroll 1
    for (int64_t t = first; t - group < a.T; t += step) {
        const bool live = t < a.T;
        float2 s[NV][K / 2];
        float2 acc = dup(0.0f);
        cp_async_wait<ST - 1>();
        if (!VEC) row_sync(tpr);
        const T* x_row = in_window(x_window(k), static_cast<const T*>(a.x) + t * a.ldx);
        const R* r_row = in_window(r_window(k), static_cast<const R*>(a.r) + t * a.ldr);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const Pack<T, K> px = VEC ? xs[(k * NV + j) * block + tid] : cols.read(x_row, j, live);
#pragma unroll
            for (int i = 0; i < K / 2; i++) s[j][i] = two(px, i);
            if (a.r) {  // the norm is of the sum as it is kept, so that a backward pass finds the same one
                Pack<R, K> pr = VEC ? rs[(k * NV + j) * block + tid] : cols.read(r_row, j, live);
#pragma unroll
                for (int i = 0; i < K / 2; i++) {
                    const float2 v = __fadd2_rn(s[j][i], two(pr, i));
                    pr.v[2 * i] = from_f<R>(v.x), pr.v[2 * i + 1] = from_f<R>(v.y);
                    s[j][i] = two(pr, i);
                }
                if (live) cols.write(static_cast<R*>(a.sum) + t * a.D, j, pr);
            }
#pragma unroll
            for (int i = 0; i < K / 2; i++) acc = __fadd2_rn(acc, s[j][i]);
        }
        if (VEC) fetch(t + ST * step, k);
        float sum[1] = {__fadd_rn(acc.x, acc.y)};
        reduce(sum);
        if (!VEC) {
            window_read();
            fetch(t + ST * step, k);
        }
        k = k + 1 == ST ? 0 : k + 1;
        const float mean = __fdiv_rn(sum[0], n);
        acc = dup(0.0f);
#pragma unroll
        for (int j = 0; j < NV; j++) {
#pragma unroll
            for (int i = 0; i < K / 2; i++) {
                s[j][i] = __fadd2_rn(s[j][i], dup(-mean));
                if (VEC) {
                    if (cols.any(j)) acc = __ffma2_rn(s[j][i], s[j][i], acc);
                } else {
                    if (cols.has(j, 2 * i)) acc.x = __fmaf_rn(s[j][i].x, s[j][i].x, acc.x);
                    if (cols.has(j, 2 * i + 1)) acc.y = __fmaf_rn(s[j][i].y, s[j][i].y, acc.y);
                }
            }
        }
        sum[0] = __fadd_rn(acc.x, acc.y);
        reduce(sum);
        const float rstd = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(sum[0], n), a.eps)));
        if (!live) continue;
        if (lane == 0 && a.stats) a.stats[t] = make_float2(mean, rstd);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if (!cols.any(j)) continue;
            const Pack<float, K> w = cols.read(a.w, j);
            Pack<float, K> b = {};
            if (a.b) b = cols.read(a.b, j);
            float o[K];
#pragma unroll
            for (int i = 0; i < K / 2; i++) {
                const float2 v = __ffma2_rn(__fmul2_rn(s[j][i], dup(rstd)), two(w, i), two(b, i));
                o[2 * i] = v.x, o[2 * i + 1] = v.y;
            }
            cols.write(static_cast<T*>(a.y) + t * a.D, j, o);
        }
    }
    cp_async_wait();
}

// Rows that a thread works on at once, and slots for them: two rows hide each
// other's reduction.  16384 x 768 bf16 with a residual 22.7 us without the sums'
// kernel; one row at a time, in two CTAs of 64 registers 31.3 (spills), in two of
// 288 threads 22.7, but with twice the partial rows for the sums.
template <typename T, typename R, int NV>
constexpr int AT_ONCE = NV * (sizeof(T) + sizeof(R)) <= 6 ? 2 : 1;
template <typename T, typename R, int NV>
constexpr int BSTAGES = NV * (sizeof(T) + 2 * sizeof(R)) <= 12 ? 2 : 1;
template <typename T, typename R, int NV>
struct BwdSlot {  // of a thread
    Pack<R, K> s[NV], d[NV];
    Pack<T, K> g[NV];
};

// What the rows of a CTA give to dw and db stays in its threads' registers; the
// row groups are added through shared memory at the end, and sums_kernel adds
// the CTAs' rows.  Rows are held as they were read and opened twice.
template <typename T, typename R, int NV, bool VEC>
__global__ void __launch_bounds__(MAX_BLOCK, 1) bwd_kernel(const Args a) {
    constexpr int ST = BSTAGES<T, R, NV>, AT = AT_ONCE<T, R, NV>;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float2 red[2][MAX_BLOCK / 32][AT];
    const int tid = threadIdx.x, tpr = a.tpr, group = tid / tpr, rows = blockDim.x / tpr;
    const int lane = tid - group * tpr, block = blockDim.x;
    // [ST][AT][NV][block] of s, of dsum and of dy; [ST][AT][block] of the statistics
    Pack<R, K>* ss = reinterpret_cast<Pack<R, K>*>(smem);
    Pack<R, K>* ds = ss + ST * AT * NV * block;
    Pack<T, K>* gs = reinterpret_cast<Pack<T, K>*>(ds + ST * AT * NV * block);
    float2* sts = reinterpret_cast<float2*>(gs + ST * AT * NV * block);
    // not VEC: windows [ST][AT][rows] of s, of dsum and of dy; then the statistics
    const int wr = window_bytes<R, NV>(tpr), wt = window_bytes<T, NV>(tpr);
    auto s_window = [&](int k, int q) { return reinterpret_cast<char*>(smem) + ((k * AT + q) * rows + group) * wr; };
    auto d_window = [&](int k, int q) { return s_window(k, q) + ST * AT * rows * wr; };
    auto g_window = [&](int k, int q) { return reinterpret_cast<char*>(smem) + 2 * ST * AT * rows * wr + ((k * AT + q) * rows + group) * wt; };
    if (!VEC) sts = reinterpret_cast<float2*>(smem + ST * AT * rows * (2 * wr + wt));
    Reduce<float2, AT> reduce = {red, tpr, 0};
    const Columns<VEC> cols = {tpr, lane, a.D};
    auto slot = [&](int k, int q, int j) { return ((k * AT + q) * NV + j) * block + tid; };
    const int64_t step = (int64_t)gridDim.x * rows, first = (int64_t)blockIdx.x * rows + group;
    auto fetch = [&](int64_t t0, int k) {
#pragma unroll
        for (int q = 0; q < AT; q++) {
            const int64_t t = t0 + q * step;
            const bool live = t < a.T;
            if (!VEC && live) {
                fetch_window(s_window(k, q), static_cast<const R*>(a.sum) + t * a.ldr, a.D, lane, tpr);
                fetch_window(g_window(k, q), static_cast<const T*>(a.dy) + t * a.D, a.D, lane, tpr);
                if (a.dsum) fetch_window(d_window(k, q), static_cast<const R*>(a.dsum) + t * a.D, a.D, lane, tpr);
            }
#pragma unroll
            for (int j = 0; VEC && j < NV; j++) {
                const int c = cols.at(j), at = slot(k, q, j);
                const bool some = live && cols.any(j);
                fetch_whole(ss[at], static_cast<const R*>(a.sum) + t * a.ldr + c, a.sum, some);
                fetch_whole(gs[at], static_cast<const T*>(a.dy) + t * a.D + c, a.dy, some);
                if (a.dsum) fetch_whole(ds[at], static_cast<const R*>(a.dsum) + t * a.D + c, a.dsum, some);
            }
            cp_async<8>(&sts[(k * AT + q) * block + tid], live ? a.stats + t : a.stats, live ? 8 : 0);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < ST; i++) fetch(first + i * AT * step, i);
    constexpr bool HOLD = NV == 1;  // w in registers
    Pack<float, K> w[NV];
    float2 dw[NV][K / 2], db[NV][K / 2];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        if (HOLD) w[j] = cols.read(a.w, j);
#pragma unroll
        for (int i = 0; i < K / 2; i++) dw[j][i] = db[j][i] = dup(0.0f);
    }
    const float share = __fdiv_rn(1.0f, (float)a.D);
    int k = 0;
#pragma unroll 1
    for (int64_t t0 = first; t0 - group < a.T; t0 += AT * step) {
        cp_async_wait<ST - 1>();
        if (!VEC) row_sync(tpr);
        float2 st[AT], sums[AT];
        Pack<R, K> ps[AT][NV], pd[AT][NV];
        Pack<T, K> pg[AT][NV];
#pragma unroll
        for (int q = 0; q < AT; q++) {
            const int64_t t = t0 + q * step;
            const bool live = t < a.T;
            // a row that does not exist is all zeros: it adds nothing
            st[q] = sts[(k * AT + q) * block + tid];
            sums[q] = dup(0.0f);
            float2 s1 = dup(0.0f), s2 = dup(0.0f);
#pragma unroll
            for (int j = 0; j < NV; j++) {
                if (VEC) {
                    const int at = slot(k, q, j);
                    ps[q][j] = ss[at], pg[q][j] = gs[at];
                    if (a.dsum) pd[q][j] = ds[at];
                } else {
                    ps[q][j] = cols.read(in_window(s_window(k, q), static_cast<const R*>(a.sum) + t * a.ldr), j, live);
                    pg[q][j] = cols.read(in_window(g_window(k, q), static_cast<const T*>(a.dy) + t * a.D), j, live);
                    if (a.dsum)
                        pd[q][j] = cols.read(in_window(d_window(k, q), static_cast<const R*>(a.dsum) + t * a.D), j, live);
                }
                if (!HOLD) w[j] = cols.read(a.w, j);
#pragma unroll
                for (int i = 0; i < K / 2; i++) {
                    const float2 xh = __fmul2_rn(__fadd2_rn(two(ps[q][j], i), dup(-st[q].x)), dup(st[q].y));
                    const float2 dy = two(pg[q][j], i), g = __fmul2_rn(two(w[j], i), dy);
                    dw[j][i] = __ffma2_rn(dy, xh, dw[j][i]);
                    db[j][i] = __fadd2_rn(db[j][i], dy);
                    s1 = __fadd2_rn(s1, g);
                    s2 = __ffma2_rn(g, xh, s2);
                }
            }
            sums[q] = make_float2(__fadd_rn(s1.x, s1.y), __fadd_rn(s2.x, s2.y));
        }
        if (VEC) fetch(t0 + ST * AT * step, k);
        reduce(sums);
        if (!VEC) {
            window_read();
            fetch(t0 + ST * AT * step, k);
        }
        k = k + 1 == ST ? 0 : k + 1;
        if (!a.dx && !a.dr) continue;
#pragma unroll
        for (int q = 0; q < AT; q++) {
            const int64_t t = t0 + q * step;
            if (t >= a.T) continue;
            const float m1 = __fmul_rn(sums[q].x, share), m2 = __fmul_rn(sums[q].y, share);
#pragma unroll
            for (int j = 0; j < NV; j++) {
                if (!cols.any(j)) continue;
                float o[K];
#pragma unroll
                for (int i = 0; i < K / 2; i++) {
                    const float2 xh = __fmul2_rn(__fadd2_rn(two(ps[q][j], i), dup(-st[q].x)), dup(st[q].y));
                    const float2 g = __fmul2_rn(two(w[j], i), two(pg[q][j], i));
                    float2 v = __fmul2_rn(dup(st[q].y), __ffma2_rn(xh, dup(-m2), __fadd2_rn(g, dup(-m1))));
                    if (a.dsum) v = __fadd2_rn(v, two(pd[q][j], i));
                    o[2 * i] = v.x, o[2 * i + 1] = v.y;
                }
                if (a.dx) cols.write(static_cast<T*>(a.dx) + t * a.D, j, o);
                if (a.dr) cols.write(static_cast<R*>(a.dr) + t * a.D, j, o);
            }
        }
    }
    cp_async_wait();
    if (!a.part) return;
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.D;
    float* sh = reinterpret_cast<float*>(smem);  // [rows][D], in the place of the slots
#pragma unroll
    for (int which = 0; which < 2; which++) {
        float* to = rows > 1 ? sh + group * a.D : part + which * a.D;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NV; j++) {
            if constexpr (VEC) {  // 16 bytes a store; with 4 the call took 60.0 us instead of 54.9 (4096 x 4096 bf16, fp32 residual)
                if (!cols.any(j)) continue;
#pragma unroll
                for (int i = 0; i < K; i += 4) {
                    const float2 u = which ? db[j][i / 2] : dw[j][i / 2], v = which ? db[j][i / 2 + 1] : dw[j][i / 2 + 1];
                    *reinterpret_cast<float4*>(to + cols.at(j) + i) = make_float4(u.x, u.y, v.x, v.y);
                }
            } else {
#pragma unroll
                for (int i = 0; i < K / 2; i++) {
                    const float2 v = which ? db[j][i] : dw[j][i];
                    if (cols.has(j, 2 * i)) to[cols.at(j, 2 * i)] = v.x;
                    if (cols.has(j, 2 * i + 1)) to[cols.at(j, 2 * i + 1)] = v.y;
                }
            }
        }
        if (rows == 1) continue;
        __syncthreads();
        for (int c = tid; c < a.D; c += block) {
            float v = sh[c];
            for (int i = 1; i < rows; i++) v = __fadd_rn(v, sh[i * a.D + c]);
            part[which * a.D + c] = v;
        }
    }
}

// out[c] = sum over p of part[p, c] for the columns of dw, then of db: 64 strands
// of rows, then the strands in order.  8 columns a CTA (a sector of each row),
// so that the rows are read by all SMs.
constexpr int SUM_COLS = 8, STRANDS = 64;
static __global__ void __launch_bounds__(SUM_COLS* STRANDS)
    sums_kernel(const float* __restrict__ part, float* __restrict__ dw, float* __restrict__ db, int P, int D) {
    __shared__ float sh[STRANDS][SUM_COLS + 1];
    const int l = threadIdx.x % SUM_COLS, c = blockIdx.x * SUM_COLS + l, g = threadIdx.x / SUM_COLS;
    grid_dependency_sync();
    float s = 0.0f;
    if (c < 2 * D) {
#pragma unroll 5
        for (int p = g; p < P; p += STRANDS) s = __fadd_rn(s, part[(int64_t)p * 2 * D + c]);
    }
    sh[g][l] = s;
    __syncthreads();
    if (g < 8) {
#pragma unroll
        for (int i = 1; i < STRANDS / 8; i++) s = __fadd_rn(s, sh[g + 8 * i][l]);
        sh[g][l] = s;
    }
    __syncthreads();
    if (g == 0 && c < 2 * D) {
#pragma unroll
        for (int i = 1; i < 8; i++) s = __fadd_rn(s, sh[i][l]);
        if (c < D) {
            if (dw) dw[c] = s;
        } else if (db) {
            db[c - D] = s;
        }
    }
}

struct Plan {
    int tpr, nv, block, grid;
};

static inline int within_warp(int packs) {  // threads of a row of few packs: a power of 2
    int tpr = 4;
    while (tpr < packs && tpr < 32) tpr *= 2;
    return tpr;
}

// Forward: a warp where 4 packs a thread hold the row, more threads where they do
// not, and for the few rows of a decode batch, which would leave most of the GPU
// without a warp.
static inline Plan forward_plan(int T, int D) {
    const int packs = cdiv(D, K);
    Plan p;
    if (packs <= 32)
        p.tpr = within_warp(packs);
    else if (packs > 4 * 128)
        p.tpr = 512;
    else
        p.tpr = packs > 4 * 32 || T <= 148 * 4 ? 128 : 32;
    p.nv = cdiv(packs, p.tpr);
    p.block = p.tpr > 256 ? p.tpr : 256;
    const int ctas = cdiv(T, p.block / p.tpr), most = p.block > 256 ? 148 : 148 * 2;
    p.grid = ctas < most ? ctas : most;
    return p;
}

// Backward: one pack a thread up to 512 of them, so that the sums of dw and db
// leave registers for the rows.
static inline Plan backward_plan(int T, int D) {
    const int packs = cdiv(D, K);
    Plan p;
    p.nv = packs <= MAX_BLOCK ? 1 : packs <= 2 * MAX_BLOCK ? 2 : 4;
    const int need = cdiv(packs, p.nv);
    p.tpr = need <= 32 ? within_warp(need) : cdiv(need, 32) * 32;
    int rows = MAX_BLOCK / p.tpr;
    if (rows > 15 && p.tpr > 32) rows = 15;
    const int share = cdiv(T, 148);  // few rows: a CTA each
    if (rows > share) rows = share;
    const int least = cdiv(32, p.tpr);  // whole warps
    rows = cdiv(rows, least) * least;
    p.block = rows * p.tpr;
    const int ctas = cdiv(T, rows);
    p.grid = ctas < 148 ? ctas : 148;
    return p;
}

template <typename T, typename R, int NV, bool VEC, int BLOCK>
static int forward(const Args& a, const Plan& p, cudaStream_t s) {
    constexpr size_t ST = STAGES<T, R, NV>, most = ST * BLOCK * NV * K * (sizeof(T) + sizeof(R)) + (VEC ? 0 : ST * 32 * (BLOCK / 4));
    const int rows = p.block / p.tpr;
    const size_t smem = VEC ? ST * p.block * NV * K * (sizeof(T) + sizeof(R))
                            : ST * rows * (window_bytes<T, NV>(p.tpr) + window_bytes<R, NV>(p.tpr));
    static std::atomic<uint64_t> allowed{0};
    if (!allow_smem(fwd_kernel<T, R, NV, VEC, BLOCK>, most, allowed)) return MI_ERR_CUDA;
    MI_LAUNCH_DEPENDENT(fwd_kernel<T, R, NV, VEC, BLOCK>, p.grid, p.block, smem, s, a);
    return MI_OK;
}

template <typename T, typename R, int NV>
static int forward(const Args& a, const Plan& p, bool vec, cudaStream_t s) {
    if (p.block <= 256) return vec ? forward<T, R, NV, true, 256>(a, p, s) : forward<T, R, NV, false, 256>(a, p, s);
    constexpr int MANY = NV > 1 ? NV : 2;  // such rows have more than 512 packs
    return vec ? forward<T, R, MANY, true, 512>(a, p, s) : forward<T, R, 4, false, 512>(a, p, s);
}

template <typename T, typename R, int NV, bool VEC>
static int backward(const Args& a, const Plan& p, cudaStream_t s) {
    constexpr size_t ROWS = BSTAGES<T, R, NV> * AT_ONCE<T, R, NV>, per = ROWS * (sizeof(BwdSlot<T, R, NV>) + sizeof(float2));
    constexpr size_t most = per * MAX_BLOCK + (VEC ? 0 : ROWS * 48 * (MAX_BLOCK / 4));
    constexpr size_t sums_most = sizeof(float) * K * NV * MAX_BLOCK;
    const int rows = p.block / p.tpr;
    size_t smem = VEC ? per * p.block
                      : ROWS * (rows * (2 * window_bytes<R, NV>(p.tpr) + window_bytes<T, NV>(p.tpr)) + p.block * sizeof(float2));
    const size_t sums = p.block > p.tpr ? sizeof(float) * (p.block / p.tpr) * a.D : 0;
    if (smem < sums) smem = sums;
    static std::atomic<uint64_t> allowed{0};
    if (!allow_smem(bwd_kernel<T, R, NV, VEC>, most > sums_most ? most : sums_most, allowed)) return MI_ERR_CUDA;
    bwd_kernel<T, R, NV, VEC><<<p.grid, p.block, smem, s>>>(a);
    MI_CHECK_LAUNCH();
    return MI_OK;
}

template <typename T, typename R, bool BWD>
static int by_width(const Args& a, const Plan& p, bool vec, cudaStream_t s) {
    if constexpr (BWD) {
        if (p.nv == 1) return vec ? backward<T, R, 1, true>(a, p, s) : backward<T, R, 1, false>(a, p, s);
        if (p.nv == 2) return vec ? backward<T, R, 2, true>(a, p, s) : backward<T, R, 2, false>(a, p, s);
        return vec ? backward<T, R, 4, true>(a, p, s) : backward<T, R, 4, false>(a, p, s);
    } else {
        if (p.nv == 1) return forward<T, R, 1>(a, p, vec, s);
        if (p.nv == 2) return forward<T, R, 2>(a, p, vec, s);
        if (p.nv == 3) return forward<T, R, 3>(a, p, vec, s);
        return forward<T, R, 4>(a, p, vec, s);
    }
}

template <bool BWD>
static int dispatch(Args& a, const Plan& p, bool vec, int dtype, int rdtype, cudaStream_t s) {
    a.tpr = p.tpr;
    MI_DISPATCH_DTYPE(dtype, T, {
        if (rdtype == dtype) return by_width<T, T, BWD>(a, p, vec, s);
        if (rdtype == MI_DT_F32) return by_width<T, float, BWD>(a, p, vec, s);
        return MI_ERR_INVALID;
    });
}

}  // namespace ln
}  // namespace mi

static int mi_ln_check(int T, int D) {
    if (T < 0 || D <= 0) return MI_ERR_INVALID;
    if (D > mi::ln::MAX_D) return MI_ERR_UNSUPPORTED;
    return MI_OK;
}

extern "C" int mi_layer_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, const float* weight,
                             const float* bias, void* y, void* sum, float* stats, int T, int D, float eps, int dtype,
                             int rdtype, void* stream) {
    if (!x || !weight || !y || (residual && !sum) || ldx < 0 || (residual && ldr < 0)) return MI_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(stats) & 7) return MI_ERR_INVALID;
    const int rc = mi_ln_check(T, D);
    if (rc != MI_OK) return rc;
    if (T == 0) return MI_OK;
    mi::ln::Args a = {};
    a.x = x, a.r = residual, a.w = weight, a.b = bias, a.y = y, a.sum = sum;
    a.stats = reinterpret_cast<float2*>(stats);
    a.ldx = ldx, a.ldr = ldr, a.T = T, a.D = D, a.eps = eps;
    bool vec = D % 8 == 0 && ldx % 8 == 0 && mi::aligned16(x) && mi::aligned16(weight) && mi::aligned16(y) &&
               (!bias || mi::aligned16(bias));
    if (residual) vec = vec && ldr % 8 == 0 && mi::aligned16(residual) && mi::aligned16(sum);
    return mi::ln::dispatch<false>(a, mi::ln::forward_plan(T, D), vec, dtype, residual ? rdtype : dtype, (cudaStream_t)stream);
}

extern "C" int64_t mi_layer_norm_backward_workspace(int T, int D) {
    if (T <= 0 || D <= 0 || D > mi::ln::MAX_D) return 0;
    return (int64_t)sizeof(float) * mi::ln::backward_plan(T, D).grid * 2 * D;
}

extern "C" int mi_layer_norm_backward(const void* dy, const void* dsum, const void* s, int64_t lds, const float* weight,
                                      const float* stats, void* dx, void* dresidual, float* dweight, float* dbias,
                                      void* workspace, int T, int D, int dtype, int rdtype, void* stream) {
    if (!dy || !s || !weight || !stats || (!dx && !dresidual && !dweight && !dbias)) return MI_ERR_INVALID;
    const bool sums = dweight || dbias;
    if ((sums && !workspace) || lds < 0 || (reinterpret_cast<uintptr_t>(stats) & 7)) return MI_ERR_INVALID;
    const int rc = mi_ln_check(T, D);
    if (rc != MI_OK) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (T == 0) {
        for (float* p : {dweight, dbias})
            if (p && cudaMemsetAsync(p, 0, sizeof(float) * D, st) != cudaSuccess) return MI_ERR_CUDA;
        return MI_OK;
    }
    mi::ln::Args a = {};
    a.dy = dy, a.dsum = dsum, a.sum = const_cast<void*>(s), a.ldr = lds, a.w = weight;
    a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats)), a.dx = dx, a.dr = dresidual;
    a.part = sums ? static_cast<float*>(workspace) : nullptr;
    a.T = T, a.D = D;
    const bool vec = D % 8 == 0 && lds % 8 == 0 && mi::aligned16(dy) && mi::aligned16(s) && mi::aligned16(weight) &&
                     (!dsum || mi::aligned16(dsum)) && (!sums || mi::aligned16(workspace)) &&
                     (!dx || mi::aligned16(dx)) && (!dresidual || mi::aligned16(dresidual));
    const mi::ln::Plan p = mi::ln::backward_plan(T, D);
    const int rc2 = mi::ln::dispatch<true>(a, p, vec, dtype, rdtype, st);
    if (rc2 != MI_OK || !sums) return rc2;
    MI_LAUNCH_DEPENDENT(mi::ln::sums_kernel, mi::cdiv(2 * D, mi::ln::SUM_COLS), mi::ln::SUM_COLS * mi::ln::STRANDS, 0, st, static_cast<const float*>(a.part), dweight,
                        dbias, p.grid, D);
    return MI_OK;
}

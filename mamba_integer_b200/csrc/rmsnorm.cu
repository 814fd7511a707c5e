// rmsnorm.cu -- RMS norm with the residual's addition in front of it, and an
// int8 output with row scales; its backward pass.
//
//   s = x + r                     (kept in r's type; s = x without a residual)
//   rstd = 1 / sqrt(mean(s^2) + eps)
//   y = s * rstd * w
//   int8: m = max(max|y|, 1e-8); q = rne(y * 127 / m); scale = m / 127, the
//         rows quantise_rows gives, ready for the ternary GEMMs
//   ds = rstd * (w dy - xhat * mean(w dy xhat)) + dsum,  xhat = s * rstd
//   dw = sum over rows of dy * xhat
//
// Every row is read once and held in registers between the reduction and the
// output, so the bound is HBM: x and r in, s and y out.  A row belongs to TPR
// threads (a warp up to 1024 columns of 16 bits); rows that need more than a
// warp reduce through shared memory.
#include <type_traits>

#include "mi_elem.cuh"

namespace mi {
namespace rms {

constexpr int THREADS = 256, CTAS = 148 * 2;  // two CTAs an SM at most

struct Args {
    const void* x;
    const void* r;
    const float* w;
    void* y;       // forward: y (NULL with xq)
    void* sum;     // s, in r's type (NULL without a residual)
    int8_t* xq;
    float* xscale;
    float* rstd;   // forward out (may be NULL), backward in
    const void* dy;
    const void* dsum;  // may be NULL
    void* dx;          // may be NULL
    void* dr;          // in r's type, may be NULL
    float* dw_part;    // [gridDim.x, D], may be NULL
    int64_t ldx, ldr;  // row strides of x and r in elements
    int T, D;
    float eps;
    int vec;           // every row starts on the packs' alignment
};

// Sum (or maximum) of one value over the TPR threads of a row, in a fixed order.
template <int TPR, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red) {
#pragma unroll
    for (int m = 16; m; m >>= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, v, m);
        v = MAX ? max_nan(v, o) : __fadd_rn(v, o);
    }
    if (TPR > 32) {
        constexpr int W = TPR / 32;
        const int warp = threadIdx.x >> 5, row = threadIdx.x / TPR;
        __syncthreads();  // the last round's reads of red are done
        if ((threadIdx.x & 31) == 0) red[warp] = v;
        __syncthreads();
        v = red[row * W];
#pragma unroll
        for (int i = 1; i < W; i++) v = MAX ? max_nan(v, red[row * W + i]) : __fadd_rn(v, red[row * W + i]);
    }
    return v;
}

// K elements from p on, `valid` of which exist.  VEC: all of them or none, and
// aligned, so that the load needs a predicate and no branch (behind a branch
// the warp would wait for it).
template <bool VEC, int K, typename T>
__device__ __forceinline__ Pack<T, K> row_pack(const T* p, int valid) {
    Pack<T, K> r;
    if (VEC) {
#pragma unroll
        for (int i = 0; i < K; i++) r.v[i] = from_f<T>(0.0f);
        if (valid > 0) r = *reinterpret_cast<const Pack<T, K>*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < K; i++) r.v[i] = i < valid ? p[i] : from_f<T>(0.0f);
    }
    return r;
}

template <typename T, typename R, int K, int NV, int TPR>
struct InSlots {  // by thread
    static constexpr int BLOCK = TPR > THREADS ? TPR : THREADS;
    Pack<T, K> x[NV][BLOCK];
    Pack<R, K> r[NV][BLOCK];
};

// Rows are dealt to at most CTAS CTAs; the next row's packs come into the
// thread's own slots while a row is worked on.  32768 x 768 bf16 to int8 with a
// residual 31 us (177 MB, 5.7 TB/s) against 40 with a warp for each row, whose
// loads and arithmetic take turns, and 39 with 3 CTAs an SM (80 registers
// instead of 102); 16384 x 768 to bf16 17 us (100 MB, 6.0 TB/s) against 21.
// T: element type of x and y; R: of the residual and s.  A thread holds NV
// packs of K elements, TPR * K apart.
template <typename T, typename R, int K, int NV, int TPR, bool VEC, bool QUANT>
__global__ void __launch_bounds__(TPR > THREADS ? TPR : THREADS, TPR > THREADS ? 1 : 2) fwd_kernel(const Args a) {
    __shared__ float red[32];
    extern __shared__ __align__(16) unsigned char smem[];
    InSlots<T, R, K, NV, TPR>& slots = *reinterpret_cast<InSlots<T, R, K, NV, TPR>*>(smem);
    constexpr int ROWS = (TPR > THREADS ? TPR : THREADS) / TPR;
    const int tid = threadIdx.x, lane = tid % TPR;
    grid_dependency_sync();
    auto fetch = [&](int64_t t) {
        const T* x = static_cast<const T*>(a.x) + t * a.ldx + lane * K;
        const R* r = static_cast<const R*>(a.r) + t * a.ldr + lane * K;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = j * TPR * K, valid = t < a.T ? a.D - c - lane * K : 0;
            fetch_pack<K>(slots.x[j][tid].v, x + c, a.x, valid, true);
            if (a.r) fetch_pack<K>(slots.r[j][tid].v, r + c, a.r, valid, true);
        }
        cp_async_commit();
    };
    if (VEC) fetch((int64_t)blockIdx.x * ROWS + tid / TPR);
#pragma unroll 1
    for (int64_t t0 = (int64_t)blockIdx.x * ROWS; t0 < a.T; t0 += (int64_t)gridDim.x * ROWS) {
        const int64_t t = t0 + tid / TPR;
        // the threads of a row that does not exist still take part in the barriers
        const bool live = t < a.T;
        float s[NV][K];
        float acc = 0.0f;
        Pack<T, K> px[NV];
        Pack<R, K> pr[NV];
        if constexpr (VEC) {
            cp_async_wait();
#pragma unroll
            for (int j = 0; j < NV; j++) {
                px[j] = slots.x[j][tid];
                if (a.r) pr[j] = slots.r[j][tid];
            }
            fetch(t + (int64_t)gridDim.x * ROWS);
        } else {
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int c = (j * TPR + lane) * K;
                const int valid = live ? a.D - c : 0;
                px[j] = row_pack<VEC, K>(static_cast<const T*>(a.x) + t * a.ldx + c, valid);
                if (a.r) pr[j] = row_pack<VEC, K>(static_cast<const R*>(a.r) + t * a.ldr + c, valid);
            }
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = (j * TPR + lane) * K;
            const int valid = live ? a.D - c : 0;
#pragma unroll
            for (int i = 0; i < K; i++) s[j][i] = to_f(px[j].v[i]);
            if (a.r) {  // the norm is of the sum as it is kept, so that a backward pass finds the same one
#pragma unroll
                for (int i = 0; i < K; i++) {
                    pr[j].v[i] = from_f<R>(__fadd_rn(s[j][i], to_f(pr[j].v[i])));
                    s[j][i] = to_f(pr[j].v[i]);
                }
                R* o = static_cast<R*>(a.sum) + t * a.D + c;
                if (VEC) {
                    if (valid > 0) *reinterpret_cast<Pack<R, K>*>(o) = pr[j];
                } else {
#pragma unroll
                    for (int i = 0; i < K; i++)
                        if (i < valid) o[i] = pr[j].v[i];
                }
            }
#pragma unroll
            for (int i = 0; i < K; i++) acc = __fmaf_rn(s[j][i], s[j][i], acc);
        }
        acc = row_reduce<TPR, false>(acc, red);
        const float rstd = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(acc, (float)a.D), a.eps)));
        if (live && lane == 0 && a.rstd) a.rstd[t] = rstd;
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = (j * TPR + lane) * K;
            const Pack<float, K> w = row_pack<VEC, K>(a.w + c, a.D - c);
#pragma unroll
            for (int i = 0; i < K; i++) {
                s[j][i] = __fmul_rn(__fmul_rn(s[j][i], rstd), w.v[i]);
                if (QUANT) amax = max_nan(amax, fabsf(s[j][i]));
            }
            if (!QUANT && live && c < a.D) store_pack<K>(static_cast<T*>(a.y) + t * a.D + c, s[j], a.D - c, VEC);
        }
        if (QUANT) {
            amax = row_reduce<TPR, true>(amax, red);
            float scale;
            const float inv = quant_inv_scale(amax, scale);
            const uint32_t some = amax < __int_as_float(0x7f800000) ? 0xffffffffu : 0u;
            if (live && lane == 0) a.xscale[t] = scale;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int c = (j * TPR + lane) * K;
                if (!live || c >= a.D) continue;
                int8_t* o = a.xq + t * a.D + c;
                static_assert(K == 8, "two words of 4");
                alignas(8) uint32_t word[2];
                // 1.5 2^23 + v holds v rounded to even in its low bits: |v| is at most 127 as it is rounded, or the
                // row has an infinity or a NaN, and then all of its q are 0 (infinity times 0, NaN) like quantise_rows'
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t b[4];
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        b[i] = __float_as_uint(__fadd_rn(__fmul_rn(s[j][4 * h + i], inv), 12582912.0f));
                    word[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410) & some;
                }
                const Pack<int8_t, K>& q = reinterpret_cast<const Pack<int8_t, K>&>(word);
                if (VEC) {
                    *reinterpret_cast<Pack<int8_t, K>*>(o) = q;
                } else {
#pragma unroll
                    for (int i = 0; i < K; i++)
                        if (i < a.D - c) o[i] = q.v[i];
                }
            }
        }
    }
    if (VEC) cp_async_wait();
}

// Rows are dealt to the CTAs in a fixed order; each thread keeps the sums of
// its columns' dy * xhat over its rows in registers, a CTA adds its row groups
// through shared memory and writes one row of partial sums, and
// column_sum_kernel adds those.  Those sums leave registers for two CTAs an SM
// and none for the next row, which asynchronous copies bring into the thread's
// own slots while a row is worked on.
// Registers that a thread of the backward pass holds for its packs; up to 92 of
// them it runs in two CTAs an SM, which leave it 128 in all.  Two packs of 8 fit
// those; three do not quite (without the bound they take about 195) and spill,
// bf16 180 bytes, fp16 96.  us with the sums' kernel (2.8), in two CTAs an SM
// and in one: 16384 x 512 bf16 20.5 and 23.0; x 768 bf16 32.7 and 28.8, fp16
// 26.7 and 28.8, with fp32 residuals 43.6 and 39.0, fp32 46.3 and 39.2; x 1024
// bf16 49.3 and 33.0.  So the bound is right but for three packs of bf16.
template <typename T, typename R, int K, int NV>
constexpr int held = (2 * K + (sizeof(T) + 2 * sizeof(R)) * K / 4) * NV;
template <typename T, typename R, int K, int NV, int TPR>
struct Slots {  // by thread
    static constexpr int BLOCK = TPR > THREADS ? TPR : THREADS;
    Pack<R, K> s[NV][BLOCK], d[NV][BLOCK];
    Pack<T, K> g[NV][BLOCK];
};
template <typename T, typename R, int K, int NV, int TPR, bool VEC>
__global__ void __launch_bounds__(TPR > THREADS ? TPR : THREADS, TPR <= THREADS && held<T, R, K, NV> <= 92 ? 2 : 1)
    bwd_kernel(const Args a) {
    __shared__ float red[32];
    extern __shared__ __align__(16) unsigned char smem[];
    Slots<T, R, K, NV, TPR>& slots = *reinterpret_cast<Slots<T, R, K, NV, TPR>*>(smem);
    constexpr int ROWS = (TPR > THREADS ? TPR : THREADS) / TPR;
    const int tid = threadIdx.x, lane = tid % TPR, row = tid / TPR;
    float dw[NV][K];
    Pack<float, K> w[NV];
    const R* ps_at = static_cast<const R*>(a.sum) + lane * K;
    const R* pd_at = static_cast<const R*>(a.dsum) + lane * K;
    const T* pg_at = static_cast<const T*>(a.dy) + lane * K;
    float next_rstd = 0.0f;
    auto fetch = [&](int64_t t) {
        const bool live = t < a.T;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = j * TPR * K, valid = live ? a.D - c - lane * K : 0;
            fetch_pack<K>(slots.s[j][tid].v, ps_at + t * a.ldr + c, a.sum, valid, true);
            fetch_pack<K>(slots.g[j][tid].v, pg_at + t * a.D + c, a.dy, valid, true);
        }
        cp_async_commit();
        next_rstd = live ? a.rstd[t] : 0.0f;
    };
    auto fetch_dsum = [&](int64_t t) {  // needed last, so it stays in its slots and its successor comes behind it
        if (a.dsum) {
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int c = j * TPR * K, valid = t < a.T ? a.D - c - lane * K : 0;
                fetch_pack<K>(slots.d[j][tid].v, pd_at + t * a.D + c, a.dsum, valid, true);
            }
        }
        cp_async_commit();
    };
    if (VEC) fetch((int64_t)blockIdx.x * ROWS + row), fetch_dsum((int64_t)blockIdx.x * ROWS + row);
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int c = (j * TPR + lane) * K;
        w[j] = row_pack<VEC, K>(a.w + c, a.D - c);
#pragma unroll
        for (int i = 0; i < K; i++) dw[j][i] = 0.0f;
    }
    for (int64_t t0 = (int64_t)blockIdx.x * ROWS; t0 < a.T; t0 += (int64_t)gridDim.x * ROWS) {
        const int64_t t = t0 + row;
        const bool live = t < a.T;
        Pack<R, K> ps[NV];
        Pack<T, K> pg[NV];
        Pack<R, K> pd[NV];
        float rstd;
        if constexpr (VEC) {
            cp_async_wait<1>();
#pragma unroll
            for (int j = 0; j < NV; j++) ps[j] = slots.s[j][tid], pg[j] = slots.g[j][tid];
            rstd = next_rstd;
            fetch(t + (int64_t)gridDim.x * ROWS);
        } else {
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int c = (j * TPR + lane) * K;
                const int valid = live ? a.D - c : 0;
                ps[j] = row_pack<VEC, K>(static_cast<const R*>(a.sum) + t * a.ldr + c, valid);
                pg[j] = row_pack<VEC, K>(static_cast<const T*>(a.dy) + t * a.D + c, valid);
                if (a.dsum) pd[j] = row_pack<VEC, K>(static_cast<const R*>(a.dsum) + t * a.D + c, valid);
            }
            rstd = live ? a.rstd[t] : 0.0f;
        }
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int i = 0; i < K; i++) {
                const float xh = __fmul_rn(to_f(ps[j].v[i]), rstd);
                const float g = to_f(pg[j].v[i]);
                dot = __fmaf_rn(__fmul_rn(w[j].v[i], g), xh, dot);
                dw[j][i] = __fmaf_rn(g, xh, dw[j][i]);
            }
        dot = row_reduce<TPR, false>(dot, red);
        const float mean = __fdiv_rn(dot, (float)a.D);
        if (VEC) cp_async_wait<1>();
        if (a.dx || a.dr) {
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int c = (j * TPR + lane) * K;
                if (!live || c >= a.D) continue;
                if (VEC && a.dsum) pd[j] = slots.d[j][tid];
                float o[K];
#pragma unroll
                for (int i = 0; i < K; i++) {
                    const float xh = __fmul_rn(to_f(ps[j].v[i]), rstd);
                    const float g = __fmul_rn(w[j].v[i], to_f(pg[j].v[i]));
                    o[i] = __fmul_rn(rstd, __fmaf_rn(-xh, mean, g));
                    if (a.dsum) o[i] = __fadd_rn(o[i], to_f(pd[j].v[i]));
                }
                if (a.dx) store_pack<K>(static_cast<T*>(a.dx) + t * a.D + c, o, a.D - c, VEC);
                if (a.dr) store_pack<K>(static_cast<R*>(a.dr) + t * a.D + c, o, a.D - c, VEC);
            }
        }
        if (VEC) fetch_dsum(t + (int64_t)gridDim.x * ROWS);
    }
    if (VEC) cp_async_wait();
    if (!a.dw_part) return;
    float* part = a.dw_part + (int64_t)blockIdx.x * a.D;
    float* sh = reinterpret_cast<float*>(smem);  // [ROWS][D], in the place of the slots
    if (ROWS > 1) __syncthreads();
    float* to = ROWS > 1 ? sh + row * a.D : part;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int i = 0; i < K; i++) {
            const int c = (j * TPR + lane) * K + i;
            if (c < a.D) to[c] = dw[j][i];
        }
    if (ROWS == 1) return;
    __syncthreads();
    for (int c = tid; c < a.D; c += Slots<T, R, K, NV, TPR>::BLOCK) {
        float v = sh[c];
#pragma unroll
        for (int g = 1; g < ROWS; g++) v = __fadd_rn(v, sh[g * a.D + c]);
        part[c] = v;
    }
}

constexpr int MAX_D = 16384;  // 512 threads of 4 packs

// Threads of a row: a warp where 4 packs of 8 a thread hold it, 128 or 512
// where they do not, and 128 too for the few rows of a decode batch, which
// would leave most of the GPU without a warp: 256 x 1024 2.7 us with 128 and
// 4.3 with 32; 32768 x 768 59 and 31.
static inline int threads_per_row(int T, int D, int K) {
    const int packs = cdiv(D, K);
    if (packs > 4 * 128) return 512;
    return packs > 4 * 32 || (packs > 32 && T <= 148 * 4) ? 128 : 32;
}

// the backward pass's CTAs: each keeps its sums of dw to the end
static inline int grid_of(int T, int D) {
    const int tpr = threads_per_row(T, D, 8);
    const int grid = cdiv(T, (tpr > THREADS ? tpr : THREADS) / tpr);
    return grid < CTAS ? grid : CTAS;
}

template <typename T, typename R, int K, int TPR, bool BWD, bool QUANT>
static int launch_nv(const Args& a, int grid, int block, cudaStream_t s) {
    const int nv = cdiv(cdiv(a.D, K), TPR);
#define MI_RMS_CASE(NV, VEC)                                                                     \
    do {                                                                                         \
        using S = std::conditional_t<BWD, Slots<T, R, K, NV, TPR>, InSlots<T, R, K, NV, TPR>>;   \
        constexpr int smem = sizeof(S);                                                          \
        static std::atomic<uint64_t> allowed{0};                                                 \
        if constexpr (BWD) {                                                                     \
            if (!allow_smem(bwd_kernel<T, R, K, NV, TPR, VEC>, smem, allowed)) return MI_ERR_CUDA; \
            bwd_kernel<T, R, K, NV, TPR, VEC><<<grid, block, smem, s>>>(a);                      \
        } else {                                                                                 \
            if (!allow_smem(fwd_kernel<T, R, K, NV, TPR, VEC, QUANT>, smem, allowed)) return MI_ERR_CUDA; \
            MI_LAUNCH_DEPENDENT(fwd_kernel<T, R, K, NV, TPR, VEC, QUANT>, grid, block, smem, s, a); \
        }                                                                                        \
    } while (0)
    if (!a.vec)
        MI_RMS_CASE(4, false);
    else if (nv <= 1)
        MI_RMS_CASE(1, true);
    else if (nv == 2)
        MI_RMS_CASE(2, true);
    else if (nv == 3)
        MI_RMS_CASE(3, true);
    else
        MI_RMS_CASE(4, true);
#undef MI_RMS_CASE
    MI_CHECK_LAUNCH();
    return MI_OK;
}

template <typename T, typename R, bool BWD, bool QUANT>
static int launch(const Args& a, int grid_cap, cudaStream_t s) {
    constexpr int K = 8;
    const int tpr = threads_per_row(a.T, a.D, K);
    const int block = tpr > THREADS ? tpr : THREADS;
    int grid = cdiv(a.T, block / tpr);
    if (grid > grid_cap) grid = grid_cap;
    switch (tpr) {
        case 32: return launch_nv<T, R, K, 32, BWD, QUANT>(a, grid, block, s);
        case 128: return launch_nv<T, R, K, 128, BWD, QUANT>(a, grid, block, s);
        default: return launch_nv<T, R, K, 512, BWD, QUANT>(a, grid, block, s);
    }
}

template <bool BWD, bool QUANT>
static int dispatch(const Args& a, int dtype, int rdtype, int grid_cap, cudaStream_t s) {
    MI_DISPATCH_DTYPE(dtype, T, {
        if (rdtype == dtype) return launch<T, T, BWD, QUANT>(a, grid_cap, s);
        if (rdtype == MI_DT_F32) return launch<T, float, BWD, QUANT>(a, grid_cap, s);
        return MI_ERR_INVALID;
    });
    return MI_ERR_INVALID;
}

}  // namespace rms
}  // namespace mi

static int mi_rms_check(int T, int D) {
    if (T < 0 || D <= 0) return MI_ERR_INVALID;
    if (D > mi::rms::MAX_D) return MI_ERR_UNSUPPORTED;
    return MI_OK;
}

static int mi_rms_forward(const void* x, int64_t ldx, const void* r, int64_t ldr, const float* w, void* y, void* sum,
                          int8_t* xq, float* xscale, float* rstd, int T, int D, float eps, int dtype, int rdtype,
                          void* stream) {
    if (!x || !w || (r && !sum)) return MI_ERR_INVALID;
    const int rc = mi_rms_check(T, D);
    if (rc != MI_OK) return rc;
    if (ldx < 0 || (r && ldr < 0)) return MI_ERR_INVALID;
    if (T == 0) return MI_OK;
    mi::rms::Args a = {};
    a.x = x, a.r = r, a.w = w, a.y = y, a.sum = sum, a.xq = xq, a.xscale = xscale, a.rstd = rstd;
    a.ldx = ldx, a.ldr = ldr, a.T = T, a.D = D, a.eps = eps;
    bool vec = D % 8 == 0 && ldx % 8 == 0 && mi::aligned16(x) && mi::aligned16(w);
    if (r) vec = vec && ldr % 8 == 0 && mi::aligned16(r) && mi::aligned16(sum);
    vec = vec && (xq ? (reinterpret_cast<uintptr_t>(xq) & 7) == 0 : mi::aligned16(y));
    a.vec = vec;
    if (xq) return mi::rms::dispatch<false, true>(a, dtype, r ? rdtype : dtype, mi::rms::CTAS, (cudaStream_t)stream);
    return mi::rms::dispatch<false, false>(a, dtype, r ? rdtype : dtype, mi::rms::CTAS, (cudaStream_t)stream);
}

extern "C" int mi_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, const float* weight, void* y,
                           void* sum, float* rstd, int T, int D, float eps, int dtype, int rdtype, void* stream) {
    if (!y) return MI_ERR_INVALID;
    return mi_rms_forward(x, ldx, residual, ldr, weight, y, sum, nullptr, nullptr, rstd, T, D, eps, dtype, rdtype,
                          stream);
}

extern "C" int mi_rms_norm_quant(const void* x, int64_t ldx, const void* residual, int64_t ldr, const float* weight,
                                 int8_t* xq, float* xscale, void* sum, int T, int D, float eps, int dtype, int rdtype,
                                 void* stream) {
    if (!xq || !xscale) return MI_ERR_INVALID;
    return mi_rms_forward(x, ldx, residual, ldr, weight, nullptr, sum, xq, xscale, nullptr, T, D, eps, dtype, rdtype,
                          stream);
}

extern "C" int64_t mi_rms_norm_backward_workspace(int T, int D) {
    if (T <= 0 || D <= 0 || D > mi::rms::MAX_D) return 0;
    return (int64_t)sizeof(float) * mi::rms::grid_of(T, D) * D;
}

extern "C" int mi_rms_norm_backward(const void* dy, const void* dsum, const void* s, int64_t lds, const float* weight,
                                    const float* rstd, void* dx, void* dresidual, float* dweight, void* workspace,
                                    int T, int D, int dtype, int rdtype, void* stream) {
    if (!dy || !s || !weight || !rstd || (!dx && !dresidual && !dweight)) return MI_ERR_INVALID;
    if (dweight && !workspace) return MI_ERR_INVALID;
    const int rc = mi_rms_check(T, D);
    if (rc != MI_OK) return rc;
    if (lds < 0) return MI_ERR_INVALID;
    cudaStream_t st = (cudaStream_t)stream;
    if (T == 0) {
        if (dweight && cudaMemsetAsync(dweight, 0, sizeof(float) * D, st) != cudaSuccess) return MI_ERR_CUDA;
        return MI_OK;
    }
    mi::rms::Args a = {};
    a.dy = dy, a.dsum = dsum, a.sum = const_cast<void*>(s), a.ldr = lds, a.w = weight;
    a.rstd = const_cast<float*>(rstd), a.dx = dx, a.dr = dresidual;
    a.dw_part = dweight ? static_cast<float*>(workspace) : nullptr;
    a.T = T, a.D = D;
    a.vec = D % 8 == 0 && lds % 8 == 0 && mi::aligned16(dy) && mi::aligned16(s) && mi::aligned16(weight) &&
            (!dsum || mi::aligned16(dsum)) && (!dx || mi::aligned16(dx)) && (!dresidual || mi::aligned16(dresidual));
    const int grid = mi::rms::grid_of(T, D);
    const int rc2 = mi::rms::dispatch<true, false>(a, dtype, rdtype, grid, st);
    if (rc2 != MI_OK || !dweight) return rc2;
    mi::column_sum_kernel<<<mi::cdiv(D, 32), 1024, 0, st>>>(a.dw_part, dweight, grid, D);
    MI_CHECK_LAUNCH();
    return MI_OK;
}

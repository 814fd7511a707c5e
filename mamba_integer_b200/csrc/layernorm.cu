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
// Layout: a row belongs to TPR threads of NV packs of 8 neighbouring elements,
// and a thread keeps its columns, so that w, b and the sums of dw and db stay in
// registers over the rows that its CTA is dealt.  Rows within a warp reduce by
// shuffles alone, longer ones through shared memory behind a barrier of the
// row's own warps.  The next rows' packs come by asynchronous copies into slots
// of the thread's own.
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

// Sums over the threads of a row, in a fixed order.  `red`: 2 x MAX_BLOCK / 32
// slots, of which rows take alternate halves, so that one barrier is enough.
template <typename V>
struct Reduce {
    V* red;
    int tpr, half;
    __device__ __forceinline__ static float add(float a, float b) { return __fadd_rn(a, b); }
    __device__ __forceinline__ static float2 add(float2 a, float2 b) { return __fadd2_rn(a, b); }
    __device__ __forceinline__ static float shift(float v, int m) { return __shfl_xor_sync(0xffffffffu, v, m); }
    __device__ __forceinline__ static float2 shift(float2 v, int m) {
        return make_float2(__shfl_xor_sync(0xffffffffu, v.x, m), __shfl_xor_sync(0xffffffffu, v.y, m));
    }
    __device__ __forceinline__ V operator()(V v) {
        if (tpr < 32) {
            for (int m = tpr >> 1; m; m >>= 1) v = add(v, shift(v, m));
            return v;
        }
#pragma unroll
        for (int m = 16; m; m >>= 1) v = add(v, shift(v, m));
        if (tpr > 32) {
            const int warps = tpr >> 5, group = threadIdx.x / tpr;
            V* at = red + half * (MAX_BLOCK / 32) + group * warps;
            if ((threadIdx.x & 31) == 0) at[(threadIdx.x >> 5) - group * warps] = v;
            asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(tpr) : "memory");
            v = at[0];
            for (int i = 1; i < warps; i++) v = add(v, at[i]);
            half ^= 1;
        }
        return v;
    }
};

template <typename T, typename R, int NV>
constexpr int STAGES = NV * K * (sizeof(T) + sizeof(R)) <= 96 ? 2 : 1;

// Elements of a pack that exist: where rows are whole packs (VEC), 0 or K.
template <bool VEC, typename T>
__device__ __forceinline__ Pack<T, K> pack_at(const T* p, int valid) {
    Pack<T, K> v;
#pragma unroll
    for (int i = 0; i < K; i++) v.v[i] = from_f<T>(0.0f);
    if (VEC) {
        if (valid > 0) v = *reinterpret_cast<const Pack<T, K>*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < K; i++)
            if (i < valid) v.v[i] = p[i];
    }
    return v;
}

template <typename T, typename R, int NV, bool VEC>
__global__ void __launch_bounds__(MAX_BLOCK, 1) fwd_kernel(const Args a) {
    constexpr int ST = STAGES<T, R, NV>;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float red[2 * MAX_BLOCK / 32];
    const int tid = threadIdx.x, tpr = a.tpr, group = tid / tpr, rows = blockDim.x / tpr;
    const int lane = tid - group * tpr, block = blockDim.x;
    Pack<T, K>* xs = reinterpret_cast<Pack<T, K>*>(smem);                                          // [ST][NV][block]
    Pack<R, K>* rs = reinterpret_cast<Pack<R, K>*>(smem + sizeof(Pack<T, K>) * ST * NV * block);   // [ST][NV][block]
    Reduce<float> reduce = {red, tpr, 0};
    grid_dependency_sync();
    auto column = [&](int j) { return (j * tpr + lane) * K; };
    auto fetch = [&](int64_t t, int k) {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = column(j), valid = t < a.T ? a.D - c : 0;
            fetch_pack<K>(xs[(k * NV + j) * block + tid].v, static_cast<const T*>(a.x) + t * a.ldx + c, a.x, valid, true);
            if (a.r)
                fetch_pack<K>(rs[(k * NV + j) * block + tid].v, static_cast<const R*>(a.r) + t * a.ldr + c, a.r, valid, true);
        }
        cp_async_commit();
    };
    const int64_t step = (int64_t)gridDim.x * rows, first = (int64_t)blockIdx.x * rows + group;
    if (VEC) {
#pragma unroll
        for (int i = 0; i < ST; i++) fetch(first + i * step, i);
    }
    Pack<float, K> w[NV], b[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        w[j] = pack_at<VEC>(a.w + column(j), a.D - column(j));
        if (a.b)
            b[j] = pack_at<VEC>(a.b + column(j), a.D - column(j));
        else
            b[j] = {};
    }
    const float n = (float)a.D;
    int k = 0;
    // the threads of a row that does not exist still take part in the reductions
    for (int64_t t = first; t - group < a.T; t += step) {
        const bool live = t < a.T;
        float s[NV][K];
        float acc = 0.0f;
        if (VEC) cp_async_wait<ST - 1>();
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = column(j), valid = live ? a.D - c : 0;
            const Pack<T, K> px = VEC ? xs[(k * NV + j) * block + tid]
                                      : pack_at<VEC>(static_cast<const T*>(a.x) + t * a.ldx + c, valid);
#pragma unroll
            for (int i = 0; i < K; i++) s[j][i] = to_f(px.v[i]);
            if (a.r) {  // the norm is of the sum as it is kept, so that a backward pass finds the same one
                Pack<R, K> pr = VEC ? rs[(k * NV + j) * block + tid]
                                    : pack_at<VEC>(static_cast<const R*>(a.r) + t * a.ldr + c, valid);
#pragma unroll
                for (int i = 0; i < K; i++) {
                    pr.v[i] = from_f<R>(__fadd_rn(s[j][i], to_f(pr.v[i])));
                    s[j][i] = to_f(pr.v[i]);
                }
                R* o = static_cast<R*>(a.sum) + t * a.D + c;
                if (VEC) {
                    if (valid > 0) *reinterpret_cast<Pack<R, K>*>(o) = pr;
                } else {
#pragma unroll
                    for (int i = 0; i < K; i++)
                        if (i < valid) o[i] = pr.v[i];
                }
            }
#pragma unroll
            for (int i = 0; i < K; i++) acc = __fadd_rn(acc, s[j][i]);
        }
        if (VEC) {
            fetch(t + ST * step, k);
            k = k + 1 == ST ? 0 : k + 1;
        }
        const float mean = __fdiv_rn(reduce(acc), n);
        acc = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int valid = a.D - column(j);
#pragma unroll
            for (int i = 0; i < K; i++) {
                s[j][i] = __fsub_rn(s[j][i], mean);
                if (i < valid) acc = __fmaf_rn(s[j][i], s[j][i], acc);
            }
        }
        const float rstd = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(reduce(acc), n), a.eps)));
        if (!live) continue;
        if (lane == 0 && a.stats) a.stats[t] = make_float2(mean, rstd);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = column(j);
#pragma unroll
            for (int i = 0; i < K; i++) s[j][i] = __fmaf_rn(__fmul_rn(s[j][i], rstd), w[j].v[i], b[j].v[i]);
            if (c < a.D) store_pack<K>(static_cast<T*>(a.y) + t * a.D + c, s[j], a.D - c, VEC);
        }
    }
    if (VEC) cp_async_wait();
}

template <typename T, typename R, int NV>
constexpr int BSTAGES = NV * K * (sizeof(T) + 2 * sizeof(R)) <= 96 ? 2 : 1;

// What the rows of a CTA give to dw and db stays in its threads' registers; the
// row groups are added through shared memory at the end, and
// column_sum_kernel adds the CTAs' rows.
template <typename T, typename R, int NV, bool VEC>
__global__ void __launch_bounds__(MAX_BLOCK, 1) bwd_kernel(const Args a) {
    constexpr int ST = BSTAGES<T, R, NV>;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float2 red[2 * MAX_BLOCK / 32];
    const int tid = threadIdx.x, tpr = a.tpr, group = tid / tpr, rows = blockDim.x / tpr;
    const int lane = tid - group * tpr, block = blockDim.x;
    Pack<R, K>* ss = reinterpret_cast<Pack<R, K>*>(smem);  // [ST][NV][block], then dsum's, dy's and the statistics
    Pack<R, K>* ds = ss + ST * NV * block;
    Pack<T, K>* gs = reinterpret_cast<Pack<T, K>*>(ds + ST * NV * block);
    float2* sts = reinterpret_cast<float2*>(gs + ST * NV * block);  // [ST][block]
    Reduce<float2> reduce = {red, tpr, 0};
    auto column = [&](int j) { return (j * tpr + lane) * K; };
    auto fetch = [&](int64_t t, int k) {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = column(j), at = (k * NV + j) * block + tid, valid = t < a.T ? a.D - c : 0;
            fetch_pack<K>(ss[at].v, static_cast<const R*>(a.sum) + t * a.ldr + c, a.sum, valid, true);
            fetch_pack<K>(gs[at].v, static_cast<const T*>(a.dy) + t * a.D + c, a.dy, valid, true);
            if (a.dsum) fetch_pack<K>(ds[at].v, static_cast<const R*>(a.dsum) + t * a.D + c, a.dsum, valid, true);
        }
        cp_async<8>(&sts[k * block + tid], t < a.T ? a.stats + t : a.stats, t < a.T ? 8 : 0);
        cp_async_commit();
    };
    const int64_t step = (int64_t)gridDim.x * rows, first = (int64_t)blockIdx.x * rows + group;
    if (VEC) {
#pragma unroll
        for (int i = 0; i < ST; i++) fetch(first + i * step, i);
    }
    Pack<float, K> w[NV];
    float dw[NV][K], db[NV][K];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        w[j] = pack_at<VEC>(a.w + column(j), a.D - column(j));
#pragma unroll
        for (int i = 0; i < K; i++) dw[j][i] = db[j][i] = 0.0f;
    }
    const float n = (float)a.D;
    int k = 0;
    for (int64_t t = first; t - group < a.T; t += step) {
        const bool live = t < a.T;
        if (VEC) cp_async_wait<ST - 1>();
        const float2 st = VEC ? sts[k * block + tid] : live ? a.stats[t] : make_float2(0.0f, 0.0f);
        float xh[NV][K], g[NV][K];
        Pack<R, K> pd[NV];
        float2 sums = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = column(j), at = (k * NV + j) * block + tid, valid = live ? a.D - c : 0;
            const Pack<R, K> ps = VEC ? ss[at] : pack_at<VEC>(static_cast<const R*>(a.sum) + t * a.ldr + c, valid);
            const Pack<T, K> pg = VEC ? gs[at] : pack_at<VEC>(static_cast<const T*>(a.dy) + t * a.D + c, valid);
            if (a.dsum) pd[j] = VEC ? ds[at] : pack_at<VEC>(static_cast<const R*>(a.dsum) + t * a.D + c, valid);
#pragma unroll
            for (int i = 0; i < K; i++) {
                xh[j][i] = __fmul_rn(__fsub_rn(to_f(ps.v[i]), st.x), st.y);
                const float dy = to_f(pg.v[i]);
                if (i < valid) dw[j][i] = __fmaf_rn(dy, xh[j][i], dw[j][i]);
                db[j][i] = __fadd_rn(db[j][i], dy);
                g[j][i] = __fmul_rn(w[j].v[i], dy);
                sums.x = __fadd_rn(sums.x, g[j][i]);
                if (i < valid) sums.y = __fmaf_rn(g[j][i], xh[j][i], sums.y);
            }
        }
        if (VEC) {
            fetch(t + ST * step, k);
            k = k + 1 == ST ? 0 : k + 1;
        }
        sums = reduce(sums);
        const float m1 = __fdiv_rn(sums.x, n), m2 = __fdiv_rn(sums.y, n);
        if (!live || (!a.dx && !a.dr)) continue;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = column(j);
            if (c >= a.D) continue;
#pragma unroll
            for (int i = 0; i < K; i++) {
                float o = __fmul_rn(st.y, __fmaf_rn(-xh[j][i], m2, __fsub_rn(g[j][i], m1)));
                if (a.dsum) o = __fadd_rn(o, to_f(pd[j].v[i]));
                g[j][i] = o;
            }
            if (a.dx) store_pack<K>(static_cast<T*>(a.dx) + t * a.D + c, g[j], a.D - c, VEC);
            if (a.dr) store_pack<K>(static_cast<R*>(a.dr) + t * a.D + c, g[j], a.D - c, VEC);
        }
    }
    if (VEC) cp_async_wait();
    if (!a.part) return;
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.D;
    float* sh = reinterpret_cast<float*>(smem);  // [rows][D], in the place of the slots
#pragma unroll
    for (int which = 0; which < 2; which++) {
        float* to = rows > 1 ? sh + group * a.D : part + which * a.D;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int i = 0; i < K; i++)
                if (column(j) + i < a.D) to[column(j) + i] = which ? db[j][i] : dw[j][i];
        if (rows == 1) continue;
        __syncthreads();
        for (int c = tid; c < a.D; c += block) {
            float v = sh[c];
            for (int i = 1; i < rows; i++) v = __fadd_rn(v, sh[i * a.D + c]);
            part[which * a.D + c] = v;
        }
    }
}

// out[c] = sum over p of part[p, c] for the columns of dw, then of db: 32 strands
// of rows, then the strands in order
static __global__ void __launch_bounds__(1024) sums_kernel(const float* __restrict__ part, float* __restrict__ dw,
                                                           float* __restrict__ db, int P, int D) {
    __shared__ float sh[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
    grid_dependency_sync();
    float s = 0.0f;
    if (c < 2 * D) {
#pragma unroll 10
        for (int p = g; p < P; p += 32) s = __fadd_rn(s, part[(int64_t)p * 2 * D + c]);
    }
    sh[g][threadIdx.x & 31] = s;
    __syncthreads();
    if (g == 0 && c < 2 * D) {
        float v = sh[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < 32; i++) v = __fadd_rn(v, sh[i][threadIdx.x]);
        if (c < D) {
            if (dw) dw[c] = v;
        } else if (db) {
            db[c - D] = v;
        }
    }
}

// Threads of a row: one pack each up to 512 of them, a power of 2 within a warp.
struct Plan {
    int tpr, nv, block, grid;
};
static inline Plan plan_of(int T, int D) {
    const int packs = cdiv(D, K);
    Plan p;
    p.nv = packs <= MAX_BLOCK ? 1 : packs <= 2 * MAX_BLOCK ? 2 : 4;
    const int need = cdiv(packs, p.nv);
    p.tpr = 4;
    while (p.tpr < need && p.tpr < 32) p.tpr *= 2;
    if (need > 32) p.tpr = cdiv(need, 32) * 32;
    int rows = MAX_BLOCK / p.tpr;
    if (rows > 15 && p.tpr > 32) rows = 15;
    // few rows: a CTA each
    const int share = cdiv(T, 148 * 2);
    if (rows > share) rows = share;
    const int least = cdiv(32, p.tpr);  // whole warps
    rows = cdiv(rows, least) * least;
    p.block = rows * p.tpr;
    const int ctas = cdiv(T, rows);
    p.grid = ctas < 148 * 2 ? ctas : 148 * 2;
    return p;
}

template <typename T, typename R, int NV, bool VEC, bool BWD>
static int launch(const Args& a, const Plan& p, cudaStream_t s) {
    size_t smem;
    static std::atomic<uint64_t> allowed{0};
    if constexpr (BWD) {
        constexpr size_t most = 227 * 1024 - sizeof(float2) * 2 * MAX_BLOCK / 32 - 1024;
        smem = (size_t)BSTAGES<T, R, NV> * p.block * (NV * K * (sizeof(T) + 2 * sizeof(R)) + 8);
        const size_t sums = p.block > p.tpr ? sizeof(float) * (p.block / p.tpr) * a.D : 0;
        if (smem < sums) smem = sums;
        if (!allow_smem(bwd_kernel<T, R, NV, VEC>, most, allowed)) return MI_ERR_CUDA;
        bwd_kernel<T, R, NV, VEC><<<p.grid, p.block, smem, s>>>(a);
        MI_CHECK_LAUNCH();
    } else {
        constexpr size_t most = 227 * 1024 - sizeof(float) * 2 * MAX_BLOCK / 32 - 1024;
        smem = VEC ? (size_t)STAGES<T, R, NV> * p.block * NV * K * (sizeof(T) + sizeof(R)) : 0;
        if (!allow_smem(fwd_kernel<T, R, NV, VEC>, most, allowed)) return MI_ERR_CUDA;
        MI_LAUNCH_DEPENDENT(fwd_kernel<T, R, NV, VEC>, p.grid, p.block, smem, s, a);
    }
    return MI_OK;
}

template <typename T, typename R, bool BWD>
static int by_width(const Args& a, const Plan& p, bool vec, cudaStream_t s) {
    if (p.nv == 1) return vec ? launch<T, R, 1, true, BWD>(a, p, s) : launch<T, R, 1, false, BWD>(a, p, s);
    if (p.nv == 2) return vec ? launch<T, R, 2, true, BWD>(a, p, s) : launch<T, R, 2, false, BWD>(a, p, s);
    return vec ? launch<T, R, 4, true, BWD>(a, p, s) : launch<T, R, 4, false, BWD>(a, p, s);
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
    return mi::ln::dispatch<false>(a, mi::ln::plan_of(T, D), vec, dtype, residual ? rdtype : dtype, (cudaStream_t)stream);
}

extern "C" int64_t mi_layer_norm_backward_workspace(int T, int D) {
    if (T <= 0 || D <= 0 || D > mi::ln::MAX_D) return 0;
    return (int64_t)sizeof(float) * mi::ln::plan_of(T, D).grid * 2 * D;
}

extern "C" int mi_layer_norm_backward(const void* dy, const void* dsum, const void* s, int64_t lds, const float* weight,
                                      const float* stats, void* dx, void* dresidual, float* dweight, float* dbias,
                                      void* workspace, int T, int D, int dtype, int rdtype, void* stream) {
    if (!dy || !s || !weight || !stats || (!dx && !dresidual && !dweight && !dbias)) return MI_ERR_INVALID;
    const bool sums = dweight || dbias;
    if ((sums && !workspace) || lds < 0) return MI_ERR_INVALID;
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
                     (reinterpret_cast<uintptr_t>(stats) & 7) == 0 && (!dsum || mi::aligned16(dsum)) &&
                     (!dx || mi::aligned16(dx)) && (!dresidual || mi::aligned16(dresidual));
    const mi::ln::Plan p = mi::ln::plan_of(T, D);
    const int rc2 = mi::ln::dispatch<true>(a, p, vec, dtype, rdtype, st);
    if (rc2 != MI_OK || !sums) return rc2;
    MI_LAUNCH_DEPENDENT(mi::ln::sums_kernel, mi::cdiv(2 * D, 32), 1024, 0, st, static_cast<const float*>(a.part), dweight,
                        dbias, p.grid, D);
    return MI_OK;
}

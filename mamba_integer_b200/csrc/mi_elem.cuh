// mi_elem.cuh -- element types of the float operators (fp32, bf16, fp16) and
// the loads and stores that move 8 neighbouring elements of them.
//
// All arithmetic on these is fp32; a result is rounded to its type once, when
// it is stored.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "mi_common.cuh"

namespace mi {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// K neighbouring elements as they lie in memory.
template <typename T, int K>
struct alignas((K * sizeof(T)) < 16 ? (K * sizeof(T)) : 16) Pack {
    T v[K];
};

// K elements at p, of which the first `valid` exist (the others read as zero).
// `vec`: p is aligned to the pack (16 bytes at most), so a whole pack is read
// with wide loads.
template <int K, typename T>
__device__ __forceinline__ Pack<T, K> load_pack(const T* __restrict__ p, int valid, bool vec) {
    if (vec && valid >= K) return *reinterpret_cast<const Pack<T, K>*>(p);
    Pack<T, K> r;
#pragma unroll
    for (int i = 0; i < K; i++) r.v[i] = i < valid ? p[i] : from_f<T>(0.0f);
    return r;
}

template <int K, typename T>
__device__ __forceinline__ void store_pack(T* __restrict__ p, const float (&f)[K], int valid, bool vec) {
    Pack<T, K> r;
#pragma unroll
    for (int i = 0; i < K; i++) r.v[i] = from_f<T>(f[i]);
    if (vec && valid >= K) {
        *reinterpret_cast<Pack<T, K>*>(p) = r;
    } else {
#pragma unroll
        for (int i = 0; i < K; i++)
            if (i < valid) p[i] = r.v[i];
    }
}

// Asynchronous copies into shared memory: `src` of BYTES bytes exist, the rest are zeros.
template <int BYTES>
__device__ __forceinline__ void cp_async(void* to, const void* from, int src) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(to);
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(from), "r"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(s), "l"(from), "n"(BYTES), "r"(src)
                     : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int PENDING = 0>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(PENDING) : "memory");
}

// Starts the copy of K elements at p, of which `valid` exist, into this
// thread's own slot; the others become zeros.  `vec`: p is aligned to the pack
// (16 bytes at most); elements one by one otherwise.  `any` is an address that
// can be named where nothing is read.
template <int K, typename T>
__device__ __forceinline__ void fetch_pack(T* slot, const T* p, const void* any, int valid, bool vec) {
    constexpr int BYTES = K * sizeof(T) < 16 ? K * sizeof(T) : 16, N = K * sizeof(T) / BYTES;
    if (vec) {
        const int have = valid <= 0 ? 0 : (valid < K ? valid : K) * (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int src = have - i * BYTES < 0 ? 0 : (have - i * BYTES < BYTES ? have - i * BYTES : BYTES);
            cp_async<BYTES>(reinterpret_cast<char*>(slot) + i * BYTES,
                            src ? reinterpret_cast<const char*>(p) + i * BYTES : reinterpret_cast<const char*>(any), src);
        }
    } else {
#pragma unroll
        for (int i = 0; i < K; i++) slot[i] = i < valid ? p[i] : from_f<T>(0.0f);
    }
}

// Lets `kernel` have its shared memory, once for each device (by bit).  `regs`:
// the registers a thread that its launch must bring along (what setmaxnreg
// deals out has to be there, or the workers would wait for it without end).
template <typename K>
static bool allow_smem(K* kernel, size_t bytes, std::atomic<uint64_t>& done, int regs = 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return true;
    if (regs) {
        cudaFuncAttributes f;
        if (cudaFuncGetAttributes(&f, kernel) != cudaSuccess || f.numRegs < regs) return false;
    }
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return false;
    done.fetch_or(bit, std::memory_order_relaxed);
    return true;
}

// 2^x to 2 ulp; results below the normal range are zero.
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// 1 / (1 + e^-x): e^-x overflows to inf and the reciprocal of that is 0.
__device__ __forceinline__ float sigmoid(float x) {
    return rcp_fast(__fadd_rn(1.0f, exp2_fast(__fmul_rn(x, -LOG2E))));
}

// softplus(x) = max(x, 0) + log(1 + e), e = e^-|x| in (0, 1].  With
// s = e / (2 + e) in (0, 1/3], log(1 + e) = 2 artanh(s)
// = 2 s (1 + s^2/3 + s^4/5 + ...), which keeps its relative precision where
// the result is small (step sizes of 1e-3 and less) and log(1 + e) would lose
// it to the rounding of 1 + e.  Cut after s^12/13: the rest is below
// 2^-25 of the sum at s = 1/3.
__device__ __forceinline__ float softplus(float x) {
    const float e = exp2_fast(__fmul_rn(fabsf(x), -LOG2E));
    const float s = __fmul_rn(e, rcp_fast(__fadd_rn(2.0f, e)));
    const float q = __fmul_rn(s, s);
    float p = 1.0f / 13.0f;
    p = __fmaf_rn(p, q, 1.0f / 11.0f);
    p = __fmaf_rn(p, q, 1.0f / 9.0f);
    p = __fmaf_rn(p, q, 1.0f / 7.0f);
    p = __fmaf_rn(p, q, 1.0f / 5.0f);
    p = __fmaf_rn(p, q, 1.0f / 3.0f);
    p = __fmaf_rn(p, q, 1.0f);
    const float l = __fmul_rn(__fadd_rn(s, s), p);
    // a NaN stays one (fmaxf alone would drop it; l carries it)
    return __fadd_rn(fmaxf(x, 0.0f), l);
}

// out[c] = sum over p of part[p, c]: 32 strands of rows, then the strands in order
static __global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ part, float* __restrict__ out,
                                                                 int P, int D) {
    __shared__ float sh[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
    float s = 0.0f;
    if (c < D) {
#pragma unroll 8
        for (int p = g; p < P; p += 32) s = __fadd_rn(s, part[(int64_t)p * D + c]);
    }
    sh[g][threadIdx.x & 31] = s;
    __syncthreads();
    if (g == 0 && c < D) {
        float v = sh[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < 32; i++) v = __fadd_rn(v, sh[i][threadIdx.x]);
        out[c] = v;
    }
}

__host__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace mi

// Calls fn.template operator()<T>() for the element type of code `dtype`.
#define MI_DISPATCH_DTYPE(dtype, T, ...)                   \
    do {                                                   \
        if ((dtype) == MI_DT_F32) {                        \
            using T = float;                               \
            __VA_ARGS__;                                   \
        } else if ((dtype) == MI_DT_BF16) {                \
            using T = __nv_bfloat16;                       \
            __VA_ARGS__;                                   \
        } else if ((dtype) == MI_DT_F16) {                 \
            using T = __half;                              \
            __VA_ARGS__;                                   \
        } else {                                           \
            return MI_ERR_INVALID;                         \
        }                                                  \
    } while (0)

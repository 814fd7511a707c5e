// mi_folds.cuh -- what stretches of positions do to a recurrence's state, and how the
// warps of a CTA and the CTAs of a cluster tell one another.
#pragma once

#include <cooperative_groups.h>

#include "mi_elem.cuh"

namespace mi {
namespace rec {

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int MAX_CLUSTER = 16;

__device__ __forceinline__ float2 dup(float v) { return make_float2(v, v); }

// what a stretch of positions does to the state of two channels: s -> p s + q
struct Fold {
    float2 p, q;
};
__device__ __forceinline__ float2 fold(float2 s, const Fold& f) { return __ffma2_rn(f.p, s, f.q); }
__device__ __forceinline__ float2 some(float2 p) {
    return make_float2(max_nan(p.x, 1.17549435e-38f), max_nan(p.y, 1.17549435e-38f));
}
__device__ __forceinline__ Fold join(const Fold& a, const Fold& b) {  // a, then b
    return {some(__fmul2_rn(a.p, b.p)), __ffma2_rn(b.p, a.q, b.q)};
}

// The folds of a round, in order: `mine` is this warp's, `s` the state that the
// round starts from.  Returns the state that this warp starts from; s becomes
// the state after the round.  Rounds alternate between two sets of slots: whoever
// writes to one has seen the other's round end, which all read the first before.
//
// A CTA that has waited in vain (about 2 s) goes on without: it sets the device's
// error word, sends and awaits no more, and its states are NaN from there on.  Then
// the others wait in vain once too, and all of them come to the kernel's last barrier.
struct Exchange {
    Fold warp[2][WARPS][32];
    uint64_t arrived[2];
    int lost;  // a wait ran out
    int pad[3];
};
constexpr size_t CTA_FOLDS = sizeof(Fold) * 2 * 32;  // bytes for each CTA of a cluster, [2][cluster][32]

__device__ __forceinline__ float2 exchange(Exchange& ex, Fold* folds, int round, int cs, int rank, Fold mine,
                                           float2& s, long long limit = WAIT_CYCLES) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, k = round & 1;
    mine.p = some(mine.p);
    ex.warp[k][warp][lane] = mine;
    __syncthreads();
    float2 from = s;
    if (cs == 1) {
#pragma unroll
        for (int i = 0; i < WARPS; i++) {
            if (i == warp) from = s;
            s = fold(s, ex.warp[k][i][lane]);
        }
        return from;
    }
    // the same for all threads: a wait of the last round was over before the barrier
    if (*static_cast<volatile int*>(&ex.lost)) return s = dup(__int_as_float(0x7fffffff));
    if (threadIdx.x == 0) mbar_expect_tx(smem_u32(&ex.arrived[k]), cs * 32 * sizeof(Fold));
    if (warp < cs) {  // warp i tells CTA i (and i + 8)
        Fold all = ex.warp[k][0][lane];
#pragma unroll
        for (int i = 1; i < WARPS; i++) all = join(all, ex.warp[k][i][lane]);
        for (int i = warp; i < cs; i += WARPS) {
            uint32_t to, bar;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(&folds[(k * cs + rank) * 32 + lane])), "r"(i));
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_u32(&ex.arrived[k])), "r"(i));
            asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to),
                         "f"(all.p.x), "f"(all.p.y), "f"(all.q.x), "f"(all.q.y), "r"(bar)
                         : "memory");
        }
    }
    if (!mbar_wait(smem_u32(&ex.arrived[k]), (round >> 1) & 1, &ex.lost, limit)) return s = dup(__int_as_float(0x7fffffff));
    for (int i = 0; i < cs; i++) {
        if (i == rank) from = s;
        s = fold(s, folds[(k * cs + i) * 32 + lane]);
    }
    for (int i = 0; i < warp; i++) from = fold(from, ex.warp[k][i][lane]);
    return from;
}

__device__ __forceinline__ void begin(Exchange& ex, int cs) {
    if (threadIdx.x < 2) mbar_init(smem_u32(&ex.arrived[threadIdx.x]), 1);
    if (threadIdx.x == 0) ex.lost = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (cs > 1)
        cooperative_groups::this_cluster().sync();
    else
        __syncthreads();
}

}  // namespace rec
}  // namespace mi

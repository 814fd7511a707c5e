"""The exchange of folds between the CTAs of a cluster (csrc/mi_folds.cuh), by itself: the states of every round, and what a
CTA does when another one sends nothing more (a wait of 0.1 s that runs out, at most once a CTA)."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = r"""
#include "mi_common.cuh"
#include "mi_folds.cuh"
using namespace mi;
using namespace mi::rec;

// CTA r of the cluster takes part in the first rounds[r] rounds; out [cs, most, 2, 256]: s and the warps' starts
__global__ void __launch_bounds__(THREADS) run(const int* rounds, int most, int cs, long long limit, float* out, long long* spent) {
    extern __shared__ __align__(16) unsigned char smem[];
    Exchange& ex = *reinterpret_cast<Exchange*>(smem);
    Fold* folds = reinterpret_cast<Fold*>(smem + sizeof(Exchange));
    const int rank = blockIdx.x, warp = threadIdx.x >> 5;
    begin(ex, cs);
    float2 s = dup(1.0f);
    const long long t0 = clock64();
    for (int r = 0; r < rounds[rank]; r++) {
        const Fold mine = {dup(0.5f), dup((float)(warp + 8 * rank + r))};
        const float2 from = exchange(ex, folds, r, cs, rank, mine, s, limit);
        float* o = out + ((rank * most + r) * 2) * THREADS + threadIdx.x;
        o[0] = s.x, o[THREADS] = from.y;
    }
    if (threadIdx.x == 0) spent[rank] = clock64() - t0;
    if (cs > 1) cooperative_groups::this_cluster().sync();
}

extern "C" int run_folds(const int* rounds, int most, int cs, long long limit, float* out, long long* spent, int* error) {
    const size_t smem = sizeof(Exchange) + cs * CTA_FOLDS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cs);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cs;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const int zero = 0;
    cudaMemcpyToSymbol(g_dev_error, &zero, sizeof(int));
    if (cudaLaunchKernelEx(&cfg, run, rounds, most, cs, limit, out, spent) != cudaSuccess) return 1;
    if (cudaDeviceSynchronize() != cudaSuccess) return 2;
    return cudaMemcpyFromSymbol(error, g_dev_error, sizeof(int)) == cudaSuccess ? 0 : 3;
}
"""
LIMIT = 200_000_000  # cycles


@pytest.fixture(scope="module")
def lib(cuda_dev, tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    from mamba_integer_b200.build import CSRC, NVCC_FLAGS
    at = tmp_path_factory.mktemp("folds")
    (at / "folds.cu").write_text(SOURCE)
    subprocess.run([nvcc, *NVCC_FLAGS, "-I" + CSRC, "-o", str(at / "folds.so"), str(at / "folds.cu")], check=True)
    return ctypes.CDLL(str(at / "folds.so"))


def run(lib, dev, rounds):
    cs, most = len(rounds), max(rounds)
    n = torch.tensor(rounds, dtype=torch.int32, device=dev)
    out = torch.full((cs, most, 2, 256), -1.0, device=dev)
    spent = torch.zeros(cs, dtype=torch.int64, device=dev)
    error = ctypes.c_int(-1)
    torch.cuda.synchronize()
    rc = lib.run_folds(ctypes.c_void_p(n.data_ptr()), most, cs, ctypes.c_longlong(LIMIT), ctypes.c_void_p(out.data_ptr()),
                       ctypes.c_void_p(spent.data_ptr()), ctypes.byref(error))
    assert rc == 0
    return out.cpu().numpy(), spent.tolist(), error.value


def want(cs, rounds):
    s, states, starts = np.float32(1), [], []
    for r in range(rounds):
        row = []
        for i in range(8 * cs):
            row.append(s)
            s = np.float32(np.float32(0.5) * s + np.float32(i + r))
        states.append(s), starts.append(row)
    return states, starts


def check_rounds(out, cs, rank, rounds):
    states, starts = want(cs, rounds)
    for r in range(rounds):
        assert np.allclose(out[rank, r, 0], states[r], rtol=1e-5), (rank, r)
        assert np.allclose(out[rank, r, 1].reshape(8, 32), np.array(starts[r][8 * rank:8 * rank + 8])[:, None], rtol=1e-5)


@pytest.mark.parametrize("cs", [2, 4, 8])
def test_every_round_comes(lib, cuda_dev, cs):
    out, spent, error = run(lib, cuda_dev, [11] * cs)
    for rank in range(cs):
        check_rounds(out, cs, rank, 11)
    assert error == 0 and max(spent) < LIMIT


@pytest.mark.parametrize("rounds,silent", [([40, 3], 1), ([0, 40], 0), ([40, 40, 2, 40], 2), ([40] * 7 + [5], 7)])
def test_a_cta_that_sends_no_more(lib, cuda_dev, rounds, silent):
    from mamba_integer_b200 import _lib
    cs, last = len(rounds), rounds[silent]
    out, spent, error = run(lib, cuda_dev, rounds)
    assert error == _lib.MI_DEV_TIMEOUT
    for rank in range(cs):
        check_rounds(out, cs, rank, last)  # what came before is right
        if rank != silent:
            assert np.isnan(out[rank, last:]).all()  # and nothing after it is taken for a state
    # each CTA waits in vain once, not once a round
    assert max(spent) < 2 * LIMIT

"""Multi-rank host logic on CPU (gloo, world size 2 and 3): batch partition,
ordered gather of last-position logits, and a missing rank surfacing as an
error rather than a hang."""
import os
import socket
import sys

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _free_port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _worker(rank, world, port, global_batch, V, q):
    sys.path.insert(0, ROOT)
    from mamba_integer_b200 import distributed as mdist

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    mdist.init_from_env("gloo", timeout_s=30)
    lo, hi = mdist.shard_range(global_batch, world, rank)
    # each rank's "logits": row i of the global batch holds value i in every column
    local = torch.arange(lo, hi, dtype=torch.float32).unsqueeze(1).repeat(1, V)
    full = mdist.gather_last_logits(local, global_batch)
    # the reusable gather bench.py times: twice with the same buffers, fed a strided view
    # (the last position of [b, L, V] logits) as the prefill engine's output is
    g = mdist.LastLogitsGather(global_batch, V)
    seq = torch.zeros(hi - lo, 3, V)
    for step in range(2):
        seq[:, -1, :] = local + 1000 * step
        got = g(seq[:, -1, :])
        assert got.shape == (global_batch, V)
        assert got[:, 0].tolist() == [float(i + 1000 * step) for i in range(global_batch)]
    ids = mdist.gather_ids(torch.arange(lo, hi, dtype=torch.int64).unsqueeze(1).repeat(1, 2), global_batch)
    assert ids[:, 1].tolist() == list(range(global_batch))
    q.put((rank, (lo, hi), full[:, 0].tolist()))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("world,global_batch", [(2, 64), (3, 64), (2, 5)])
def test_partition_and_ordered_gather(world, global_batch):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, global_batch, 4, q)) for r in range(world)]
    for p in procs:
        p.start()
    res = [q.get(timeout=120) for _ in procs]
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    ranges = sorted(r[1] for r in res)
    assert ranges[0][0] == 0 and ranges[-1][1] == global_batch
    assert all(a[1] == b[0] for a, b in zip(ranges, ranges[1:]))
    for _, _, col in res:
        assert col == [float(i) for i in range(global_batch)]


def _lonely(port, q):
    sys.path.insert(0, ROOT)
    from mamba_integer_b200 import distributed as mdist

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK="0", WORLD_SIZE="2")
    try:
        mdist.init_from_env("gloo", timeout_s=3)
        q.put("joined")
    except Exception as e:  # rendezvous times out: the peer never joined
        q.put(type(e).__name__)


def test_missing_rank_is_an_error_not_a_hang():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    p = ctx.Process(target=_lonely, args=(_free_port(), q))
    p.start()
    msg = q.get(timeout=120)
    p.join(timeout=30)
    if p.is_alive():
        p.kill()
    assert msg != "joined"


def test_shard_counts():
    from mamba_integer_b200.distributed import shard_counts, shard_range

    assert shard_counts(64, 8) == [8] * 8
    assert shard_counts(5, 2) == [3, 2]
    assert shard_range(64, 4, 3) == (48, 64)
    with pytest.raises(ValueError):
        shard_counts(4, 0)


def toy_engine():
    """DecodeEngine.generate over logits of a toy rule, the choice by the 64-bit formula."""
    from types import SimpleNamespace

    import recurrent_ref as ref
    from mamba_integer_b200 import decode, kernels

    kernels.argmax_rows = lambda x, V=None, out=None: torch.argmax(x, -1) if out is None else out.copy_(torch.argmax(x, -1))

    class Toy(decode.DecodeEngine):
        def __init__(self):
            self.pre = SimpleNamespace(dev=torch.device("cpu"))

        def start(self, prompt_ids):
            self.ws = SimpleNamespace(next_ids=torch.zeros(prompt_ids.shape[0], dtype=torch.int64))
            return self.step(prompt_ids.sum(1))

        def step(self, ids):
            return torch.cos(torch.arange(60.0)[None] * (1 + ids[:, None].float() % 7))

        @staticmethod
        def sample(logits, u, temperature, top_k, top_p, min_p, out=None):
            got = [ref.sample(row, float(v), temperature, top_k, top_p, min_p)[0] for row, v in zip(logits, u)]
            return out.copy_(torch.tensor(got))
    return Toy()


def _sampling_worker(rank, world, port, prompts, n_new, kw, q):
    for path in (ROOT, os.path.join(ROOT, "tests")):
        sys.path.insert(0, path)
    from mamba_integer_b200 import distributed as mdist
    from mamba_integer_b200.decode import Sampling

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    mdist.init_from_env("gloo", timeout_s=30)
    torch.manual_seed(21)  # as a program that seeds every rank alike
    ids, total = torch.tensor(prompts), len(prompts)
    lo, hi = mdist.shard_range(total, world, rank)
    mine = toy_engine().generate(ids[lo:hi], n_new, sampling=Sampling(**kw), first=lo, total=total)
    q.put((rank, mdist.gather_ids(mine, total).tolist()))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("kw", [dict(temperature=1.0, seed=3), dict(temperature=0.8, top_k=20, top_p=0.9)])
def test_sampled_streams_do_not_depend_on_the_number_of_ranks(kw):
    from mamba_integer_b200 import kernels
    from mamba_integer_b200.decode import Sampling

    prompts, n_new = [[5, 9, 2]] * 7, 9
    keep = kernels.argmax_rows
    try:
        eng = toy_engine()
        torch.manual_seed(21)
        want = eng.generate(torch.tensor(prompts), n_new, sampling=Sampling(**kw)).tolist()
        assert len({tuple(t) for t in want}) == 7  # equal prompts, numbers of their own
        for first, total in ((1, None), (5, 7), (-1, 9), (0, 2)):
            with pytest.raises(ValueError):
                eng.generate(torch.tensor(prompts)[:3], n_new, sampling=Sampling(**kw), first=first, total=total)
    finally:
        kernels.argmax_rows = keep
    ctx = mp.get_context("spawn")
    for world in (2, 3):
        q, port = ctx.Queue(), _free_port()
        procs = [ctx.Process(target=_sampling_worker, args=(r, world, port, prompts, n_new, kw, q)) for r in range(world)]
        for p in procs:
            p.start()
        res = [q.get(timeout=120) for _ in procs]
        for p in procs:
            p.join(timeout=60)
            assert p.exitcode == 0
        assert all(ids == want for _, ids in res), world

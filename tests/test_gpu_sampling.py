"""Generation that samples: the engine's and the server's tokens are those that the 64-bit formula (tests/recurrent_ref.py)
chooses from the oracle's logits of the whole sequence, whatever shares the slots."""
import numpy as np
import pytest
import torch

import cases
import recurrent_ref as ref

pytestmark = pytest.mark.gpu


def _f32(v):
    return float(torch.tensor(v, dtype=torch.float32))


def _alone(p, cfg, prompt, n_new, s, eos=None):
    from oracle import model as om
    seq, out = np.asarray(prompt, np.int64)[None, :], []
    u = None if s is None else s.numbers(n_new).tolist()
    for i in range(n_new):
        row = torch.from_numpy(om.forward(p, cfg, seq)[0, -1].copy())
        if s is None:
            tok = int(torch.argmax(row))
        else:
            tok, _, near = ref.sample(row, u[i], _f32(s.temperature), s.top_k, _f32(s.top_p), _f32(s.min_p))
            assert near > 2.0 ** -30  # no choice of this run lies on a border
        out.append(tok)
        if tok == eos:
            break
        seq = np.concatenate([seq, [[tok]]], axis=1)
    return out


@pytest.fixture(scope="module")
def model(cuda_dev):
    from mamba_integer_b200.mamba_integer_model import MambaIntegerModel
    from oracle import model as om
    cfg, sd, _ = cases.model_inputs("c1")
    m = MambaIntegerModel(cfg)
    m.load_state_dict(sd)
    return m.to(cuda_dev).eval(), om.prepare(sd), cfg


@pytest.mark.parametrize("use_graph", [True, False])
def test_server_samples(model, use_graph):
    from mamba_integer_b200.decode import DecodeEngine, Sampling
    from mamba_integer_b200.serve import DecodeServer
    m, p, cfg = model
    g = torch.Generator().manual_seed(11)
    settings = [Sampling(0.8, seed=1), None, Sampling(1.2, 40, 0.9, 0.02, seed=2), Sampling(0.0, seed=3),
                Sampling(0.5, top_p=0.7, seed=4), None, Sampling(2.0, min_p=0.1, seed=5)]
    lens, news = [5, 9, 5, 12, 3, 7, 5], [4, 6, 3, 5, 1, 2, 4]
    prompts = [torch.randint(0, cfg["vocab_size"], (n,), generator=g).tolist() for n in lens]
    srv = DecodeServer(m, slots=3, engine=DecodeEngine(m, use_graph=use_graph))
    rids = [srv.submit(pr, k, s) for pr, k, s in zip(prompts[:5], news, settings)]
    srv.step(), srv.step()
    rids += [srv.submit(pr, k, s) for pr, k, s in zip(prompts[5:], news[5:], settings[5:])]
    out = srv.run()
    for rid, pr, k, s in zip(rids, prompts, news, settings):
        assert out[rid] == _alone(p, cfg, pr, k, s if s is not None and s.temperature > 0 else None), rid


def test_generate_samples(model, cuda_dev):
    from mamba_integer_b200.decode import DecodeEngine, Sampling
    m, p, cfg = model
    ids = torch.randint(0, cfg["vocab_size"], (3, 8), generator=torch.Generator().manual_seed(4))
    eng, s = DecodeEngine(m), Sampling(0.9, 50, 0.95, seed=7)
    got = eng.generate(ids.to(cuda_dev), 6, sampling=s)
    assert torch.equal(got, eng.generate(ids.to(cuda_dev), 6, sampling=s))
    u = s.numbers(6, 3)
    for b in range(3):
        one = Sampling(0.9, 50, 0.95)
        object.__setattr__(one, "numbers", lambda n, b=b: u[:, b])
        assert got[b].tolist() == _alone(p, cfg, ids[b].tolist(), 6, one)
    greedy = eng.generate(ids.to(cuda_dev), 6)
    assert torch.equal(greedy, eng.generate(ids.to(cuda_dev), 6, sampling=Sampling(0.0)))
    assert eng.generate(ids.to(cuda_dev), 0, sampling=s).shape == (3, 0)

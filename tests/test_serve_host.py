"""DecodeServer's slot management on the CPU, with a stand-in engine whose
"model" is a toy rule: the first token of a prompt is sum(prompt) % V and
every next token is (previous + 1) % V.  Checks admission (equal-length
grouping, queueing beyond the slots), per-slot inputs, retirement and EOS."""
import pytest
import torch

from mamba_integer_b200.serve import DecodeServer

V = 50


class FakeEngine:
    def __init__(self):
        self.prefill_calls = []

    def reserve(self, batch):
        self.ws = type("WS", (), {})()
        self.ws.ids = torch.zeros(batch, dtype=torch.int64)
        self._next = torch.zeros(batch, dtype=torch.int64)

    def prefill_slots(self, slots, prompt_ids):
        self.prefill_calls.append((list(slots), prompt_ids.shape[1]))
        logits = torch.zeros(prompt_ids.shape[0], V)
        logits[torch.arange(prompt_ids.shape[0]), prompt_ids.sum(1) % V] = 1.0
        return logits

    @staticmethod
    def argmax(logits):
        return torch.argmax(logits, dim=-1)

    def step(self, ids):
        self.ws.ids.copy_(ids)
        self._next = (self.ws.ids + 1) % V

    def next_ids(self):
        return self._next


def expected(prompt, n, eos=None):
    out, tok = [], sum(prompt) % V
    for _ in range(n):
        out.append(tok)
        if tok == eos:
            break
        tok = (tok + 1) % V
    return out


def test_slots_queueing_and_per_request_tokens():
    eng = FakeEngine()
    srv = DecodeServer(None, slots=2, engine=eng)
    reqs = [([1, 2, 3], 4), ([4, 5, 6], 2), ([7, 8], 5), ([9, 9, 9], 1), ([1], 3)]
    rids = [srv.submit(p, n) for p, n in reqs]
    out = srv.run()
    for rid, (p, n) in zip(rids, reqs):
        assert out[rid] == expected(p, n), rid
    # the first admission took both equal-length prompts together
    assert eng.prefill_calls[0] == ([0, 1], 3)
    assert all(r is None for r in srv.active) and not srv.queue


def test_eos_and_late_arrivals():
    eng = FakeEngine()
    srv = DecodeServer(None, slots=3, eos_id=12, engine=eng)
    a = srv.submit([10], 8)        # 10, 11, 12 -> stops at eos
    srv.step()
    b = srv.submit([3, 3], 3)      # arrives while a is running
    out = srv.run()
    assert out[a] == [10, 11, 12]
    assert out[b] == expected([3, 3], 3, eos=12)


class SamplingEngine(FakeEngine):
    """Logits of a toy rule, and the choice by the 64-bit formula."""

    @staticmethod
    def logits_of(prev):
        base = torch.arange(V).float()[None]
        return 3 * torch.cos(base * (1 + prev[:, None].float() % 7)) + (base == (prev[:, None] + 1) % V)

    def prefill_slots(self, slots, prompt_ids):
        self.prefill_calls.append((list(slots), prompt_ids.shape[1]))
        return self.logits_of(prompt_ids.sum(1) % V)

    def step(self, ids):
        self.ws.ids.copy_(ids)
        self.ws.logits = self.logits_of(self.ws.ids)
        self._next = torch.argmax(self.ws.logits, dim=-1)

    @staticmethod
    def sample(logits, u, temperature, top_k, top_p, min_p, out=None):
        import recurrent_ref as ref
        got = torch.tensor([ref.sample(*row)[0] for row in zip(logits, *(t.tolist() for t in (u, temperature, top_k, top_p, min_p)))])
        return got if out is None else out.copy_(got)


def sampled_alone(prompt, n, s, eos=None):
    import recurrent_ref as ref
    f32 = lambda v: float(torch.tensor(v))  # noqa: E731
    prev, out = torch.tensor([sum(prompt) % V]), []
    u = [0.0] * n if s is None else s.numbers(n).tolist()
    for i in range(n):
        row = SamplingEngine.logits_of(prev)[0]
        tok = (int(torch.argmax(row)) if s is None else
               ref.sample(row, u[i], f32(s.temperature), s.top_k, f32(s.top_p), f32(s.min_p))[0])
        out.append(tok)
        if tok == eos:
            break
        prev = torch.tensor([tok])
    return out


def test_sampled_requests_have_their_own_numbers():
    from mamba_integer_b200.decode import Sampling
    reqs = [([1, 2, 3], 6, Sampling(0.9, seed=1)), ([4, 5, 6], 3, None), ([7, 8], 5, Sampling(1.2, 8, 0.9, 0.01, seed=2)),
            ([9, 9, 9], 1, Sampling(0.7, top_p=0.5, seed=3)), ([1], 4, Sampling(0.0, seed=9)), ([2], 7, Sampling(0.9, seed=1)),
            ([3, 3], 6, None)]
    for slots in (1, 2, 4):
        srv = DecodeServer(None, slots=slots, engine=SamplingEngine())
        rids = [srv.submit(p, n, s) for p, n, s in reqs[:4]]
        srv.step(), srv.step()
        rids += [srv.submit(p, n, s) for p, n, s in reqs[4:]]
        out = srv.run()
        for rid, (p, n, s) in zip(rids, reqs):
            assert out[rid] == sampled_alone(p, n, None if s is not None and s.temperature == 0 else s), (slots, rid)


def test_sampling_settings_are_checked():
    import pytest
    from mamba_integer_b200.decode import Sampling
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1),
                dict(top_k=1.5), dict(top_k=2 ** 31), dict(top_p=1.1), dict(top_p=float("nan")), dict(min_p=-0.5)):
        with pytest.raises(ValueError):
            Sampling(**bad)
    a, b = Sampling(seed=4).numbers(5), Sampling(seed=4).numbers(5)
    assert torch.equal(a, b) and not torch.equal(a, Sampling(seed=5).numbers(5))


def test_sampling_whole_top_k_of_any_number_type():
    """A whole number given as a float is kept as an int, which is what the kernel's call takes."""
    import pytest
    from mamba_integer_b200.decode import Sampling
    for k in (5, 5.0):
        s = Sampling(top_k=k)
        assert s.top_k == 5 and type(s.top_k) is int
    with pytest.raises(ValueError):
        Sampling(top_k=5.5)


def test_a_sampled_request_with_a_large_cap_holds_few_numbers():
    """Its numbers are those of Sampling.numbers, the default generator's too, but not all at once."""
    import tracemalloc

    from mamba_integer_b200.decode import Sampling
    eng, cap = SamplingEngine(), 3_000_000
    srv = DecodeServer(None, slots=2, eos_id=12, engine=eng)
    for kw in (dict(seed=6), dict()):
        torch.manual_seed(8)
        want = Sampling(1.0, **kw).numbers(cap)
        after = torch.rand(3)
        torch.manual_seed(8)
        tracemalloc.start()
        rid = srv.submit([4, 5], cap, Sampling(1.0, **kw))
        peak = tracemalloc.get_traced_memory()[1]
        tracemalloc.stop()
        assert peak < 1 << 20
        if not kw:
            assert torch.equal(after, torch.rand(3))
        r = srv.queue[-1]
        spots = [0, 1, 4095, 4096, 10000, 10000, 10001, 2_500_000, cap - 1]
        assert [r.numbers[i] for i in spots] == want[spots].tolist()
        with pytest.raises(IndexError):
            r.numbers[cap]
        srv.queue.remove(r)
    # served to its end token
    s = Sampling(1.0, seed=6)
    rid = srv.submit([4, 5], 20000, s)
    want = sampled_alone([4, 5], 20000, s, eos=12)
    assert srv.run()[rid] == want and want[-1] == 12 and len(want) < 20000
    for n in (1, 2, 4095, 4096, 4097, 9000):
        got = s.one_by_one(n)
        assert [got[i] for i in range(n)] == s.numbers(n).tolist()


def test_sampling_refuses_top_k_that_is_no_number_by_the_same_error():
    from mamba_integer_b200.decode import Sampling
    for k in (float("inf"), float("nan"), -float("inf"), 2.0 ** 31, -0.5):
        with pytest.raises(ValueError, match="top_k"):
            Sampling(top_k=k)
    assert Sampling(top_k=2 ** 31 - 1).top_k == 2 ** 31 - 1

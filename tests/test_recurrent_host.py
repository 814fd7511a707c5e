"""The float recurrent layer's operators without a GPU: the refusals of the Python functions and of the C entry points, and
the 64-bit formulas that the GPU tests compare with against differences."""
import pytest
import torch

import recurrent_ref as ref
from mamba_integer_b200 import _lib, kernels, selective


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float64)


@pytest.mark.parametrize("change,error", [
    (dict(x=_t(2, 5, 8, dtype=torch.float64)), TypeError),
    (dict(x=_t(2, 8)), ValueError),
    (dict(x=_t(2, 5, 0), gate=_t(2, 5, 0)), ValueError),
    (dict(gate=_t(2, 5, 7)), ValueError),
    (dict(gate=_t(2, 5, 8, dtype=torch.bfloat16)), TypeError),
    (dict(x=_t(2, 8, 5).transpose(1, 2)), ValueError),
    (dict(gate=_t(2, 8, 5).transpose(1, 2)), ValueError),
    (dict(z=_t(2, 4, 8)), ValueError),
    (dict(z=_t(2, 5, 8, dtype=torch.float16)), TypeError),
    (dict(gate_bias=_t(7)), ValueError),
    (dict(gate_bias=_t(8, dtype=torch.bfloat16)), TypeError),
    (dict(h0=_t(2, 7)), ValueError),
    (dict(h0=_t(2, 8, dtype=torch.float64)), TypeError),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(), ValueError),  # CPU tensors
])
def test_recurrence_refuses(change, error):
    with pytest.raises(error):
        selective.gated_recurrence(**{**dict(x=_t(2, 5, 8), gate=_t(2, 5, 8)), **change})


@pytest.mark.parametrize("change,error", [
    (dict(h=_t(2, 7)), ValueError),
    (dict(h=_t(2, 8, dtype=torch.bfloat16)), TypeError),
    (dict(h=_t(8, 2).t()), ValueError),
    (dict(h=_t(17)[1:].view(2, 8)), ValueError),  # off the 16-byte boundary
    (dict(x=_t(2, 1, 8)), ValueError),
    (dict(gate=_t(3, 8)), ValueError),
    (dict(z=_t(2, 8, dtype=torch.float16)), TypeError),
    (dict(gate_bias=_t(8).requires_grad_(True)), RuntimeError),
    (dict(), ValueError),
])
def test_recurrence_step_refuses(change, error):
    with pytest.raises(error):
        selective.gated_recurrence_step(**{**dict(h=_t(2, 8), x=_t(2, 8), gate=_t(2, 8)), **change})


@pytest.mark.parametrize("change,error", [
    (dict(x=_t(4, 8, dtype=torch.float64)), TypeError),
    (dict(weight=_t(7)), ValueError),
    (dict(weight=_t(8, dtype=torch.bfloat16)), TypeError),
    (dict(bias=_t(9)), ValueError),
    (dict(bias=_t(8, dtype=torch.float16)), TypeError),
    (dict(residual=_t(4, 7)), ValueError),
    (dict(residual=_t(4, 8, dtype=torch.bfloat16)), TypeError),
    (dict(x=_t(1, selective.MAX_NORM_WIDTH + 1), weight=_t(selective.MAX_NORM_WIDTH + 1)), ValueError),
    (dict(x=torch.zeros(())), ValueError),
    (dict(), ValueError),
])
def test_layer_norm_refuses(change, error):
    with pytest.raises(error):
        selective.layer_norm(**{**dict(x=_t(4, 8), weight=_t(8)), **change})


@pytest.mark.parametrize("change,error", [
    (dict(logits=_t(4, 9, dtype=torch.float64)), TypeError),
    (dict(logits=_t(4)), ValueError),
    (dict(logits=_t(4, 0)), ValueError),
    (dict(logits=_t(9, 4).t()), ValueError),
    (dict(logits=_t(4, 1).expand(4, 262145)), ValueError),
    (dict(logits=_t(4, 9).requires_grad_(True)), RuntimeError),
    (dict(u=_t(5)), ValueError),
    (dict(u=_t(4, 1)), ValueError),
    (dict(u=_t(4, dtype=torch.float64)), TypeError),
    (dict(temperature=-0.1), ValueError),
    (dict(temperature=float("nan")), ValueError),
    (dict(temperature=_t(5)), ValueError),
    (dict(temperature=_t(4, dtype=torch.bfloat16)), TypeError),
    (dict(temperature="hot"), TypeError),
    (dict(top_k=-1), ValueError),
    (dict(top_k=2.5), TypeError),
    (dict(top_k=torch.zeros(4, dtype=torch.int64)), TypeError),
    (dict(top_p=1.1), ValueError),
    (dict(top_p=-0.1), ValueError),
    (dict(top_p=float("nan")), ValueError),
    (dict(top_p=_t(1)), ValueError),
    (dict(min_p=1.5), ValueError),
    (dict(min_p=torch.zeros(4, dtype=torch.int32)), TypeError),
    (dict(out=torch.zeros(4, dtype=torch.int32)), TypeError),
    (dict(out=torch.zeros(5, dtype=torch.int64)), ValueError),
    (dict(out=torch.zeros(8, dtype=torch.int64)[::2]), ValueError),
    (dict(), ValueError),  # CPU tensors
])
def test_sample_refuses(change, error):
    with pytest.raises(error):
        kernels.sample_rows(**{**dict(logits=_t(4, 9), u=_t(4)), **change})


def test_sample_refuses_to_lose_derivatives():
    """Of a setting or the numbers as of the logits: prob would come without them."""
    from torch.autograd import forward_ad

    args = lambda: dict(logits=_t(4, 9), u=_t(4), temperature=torch.ones(4), top_p=torch.ones(4), min_p=_t(4))  # noqa: E731
    for name in args():
        with pytest.raises(RuntimeError, match="no backward pass"):
            kernels.sample_rows(**{**args(), name: args()[name].requires_grad_(True)})
        with torch.no_grad(), pytest.raises(ValueError, match="must be a CUDA tensor"):
            kernels.sample_rows(**{**args(), name: args()[name].requires_grad_(True)})
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            kernels.sample_rows(**{**args(), name: forward_ad.make_dual(args()[name], torch.ones_like(args()[name]))})


def test_sizes_past_the_counters_are_refused():
    """Expanded views: no such memory is there."""
    for shape, what in (((1, (1 << 30) + 1, 1), "too long"), ((65536, 1, 1), "at most 65535"),
                        ((65536, 0, 1), "at most 65535"), ((1, 1, (1 << 24) + 1), "channels")):
        x = _t(1).as_strided(shape, (0, 0, 0))
        with pytest.raises(ValueError, match=what):
            selective.gated_recurrence(x, x)
    with pytest.raises(ValueError, match="at most 65535 streams"):
        selective.gated_recurrence_step(_t(65536, 1), _t(65536, 1), _t(65536, 1))


def test_entry_points_refuse_on_the_host():
    """Before any CUDA call; the pointers are not touched."""
    lib = _lib.load()
    p, s, none = 256, (256, 512, 64), (None, 0, 0)

    def fwd(x=s, f=s, z=none, y=p, batch=2, L=8, D=64, dtype=0):
        return lib.mi_gated_recurrence(*x, *f, *z, None, None, None, y, p, None, None, batch, L, D, 1, dtype, None)
    assert fwd(x=none) == -1 and fwd(f=none) == -1 and fwd(y=None) == -1
    assert fwd(L=0) == -1 and fwd(L=-1) == -1 and fwd(D=0) == -1 and fwd(batch=-1) == -1
    assert fwd(dtype=3) == -1 and fwd(dtype=-1) == -1 and fwd(z=(256, -1, 64)) == -1
    assert fwd(batch=65536) == -2
    assert fwd(batch=0) == 0
    bwd = lambda dy=s, ck=p, dx=p, df=p, dz=p, dbias=p, ws=p, z=s: lib.mi_gated_recurrence_backward(  # noqa: E731
        *dy, None, *s, *s, *z, None, None, ck, dx, df, dz, dbias, None, ws, 2, 8, 64, 1, 0, None)
    assert bwd(dy=none) == -1 and bwd(ck=None) == -1 and bwd(dx=None) == -1 and bwd(df=None) == -1 and bwd(dz=None) == -1
    assert bwd(ws=None) == -1
    step = lambda h=p, y=p, dtype=0, D=64: lib.mi_gated_recurrence_step(p, 64, p, 64, None, 0, None, h, y, 2, D, 1, dtype,  # noqa: E731
                                                                       None)
    assert step(h=None) == -1 and step(y=None) == -1 and step(dtype=7) == -1 and step(D=0) == -1
    norm = lambda x=p, y=p, r=None, s_=None, D=64, rdtype=0, dtype=0, w=p: lib.mi_layer_norm(  # noqa: E731
        x, 64, r, 64, w, None, y, s_, None, 4, D, 1e-5, dtype, rdtype, None)
    assert norm(x=None) == -1 and norm(y=None) == -1 and norm(w=None) == -1 and norm(r=p) == -1
    assert norm(D=16385) == -2 and norm(D=0) == -1 and norm(dtype=3) == -1 and norm(r=p, s_=p, rdtype=1) == -1
    back = lambda dx=p, dw=None, db=None, ws=None, stats=p: lib.mi_layer_norm_backward(  # noqa: E731
        p, None, p, 64, p, stats, dx, None, dw, db, ws, 4, 64, 0, 0, None)
    assert back(dx=None) == -1 and back(dw=p) == -1 and back(db=p) == -1 and back(stats=None) == -1
    pick = lambda x=p, u=p, token=p, rows=4, V=64, ld=64, dtype=0: lib.mi_sample_rows(  # noqa: E731
        x, ld, u, None, None, None, None, 1.0, 0, 1.0, 0.0, token, None, rows, V, dtype, None)
    assert pick(x=None) == -1 and pick(u=None) == -1 and pick(token=None) == -1 and pick(rows=-1) == -1 and pick(V=0) == -1
    assert pick(ld=-1) == -1 and pick(dtype=3) == -1 and pick(V=262145) == -2 and pick(rows=0) == 0
    assert lib.mi_gated_recurrence_checkpoints(2, 17, 5) == 2 * 3 * 5
    assert lib.mi_gated_recurrence_workspace(1, 64, 64, 1, 1) == 4 * 64
    assert lib.mi_gated_recurrence_workspace(1, 64, 64, 0, 1) == 0
    assert lib.mi_gated_recurrence_workspace(1, 65536, 64, 0, 1) > 0 and fwd(batch=1, L=65536) == -1  # it wants the workspace


def test_entry_points_refuse_buffers_off_their_pairs():
    """What the kernels store two floats at a time: the states kept for the backward pass, the norm's mean and rstd."""
    lib = _lib.load()
    p, s = 256, (256, 512, 64)
    for off in (4, 12, 1):
        assert lib.mi_gated_recurrence(*s, *s, None, 0, 0, None, None, None, p, p, p + off, None, 2, 8, 64, 1, 0, None) == -1
        assert lib.mi_layer_norm(p, 64, None, 0, p, None, p, None, p + off, 4, 64, 1e-5, 0, 0, None) == -1
        assert lib.mi_layer_norm_backward(p, None, p, 64, p, p + off, p, None, None, None, None, 4, 64, 0, 0, None) == -1
    # on the boundary the call goes on (nothing to do)
    assert lib.mi_gated_recurrence(*s, *s, None, 0, 0, None, None, None, p, p, p + 8, None, 0, 8, 64, 1, 0, None) == 0
    assert lib.mi_layer_norm(p, 64, None, 0, p, None, p, None, p + 8, 0, 64, 1e-5, 0, 0, None) == 0


@pytest.mark.parametrize("size,forward16,forward32,backward", [
    # chunks (> 0 bytes of folds) where they were measured to be faster than clusters, None where the two are alike
    ((1, 4096, 128), False, False, False), ((1, 4096, 256), False, False, False), ((1, 4096, 1024), True, True, True),
    ((1, 6144, 256), False, None, True), ((1, 8192, 256), None, True, True), ((1, 16384, 256), True, True, True),
    ((2, 4096, 1024), False, False, False), ((4, 8192, 512), False, False, False), ((1, 32768, 512), True, True, True),
    ((1, 2048, 1536), False, False, False), ((8, 2048, 1536), False, False, False), ((1, 100, 64), False, False, False),
    ((1, 4096, 2176), True, True, True), ((1, 4096, 2112), False, False, False),
])
def test_chunks_are_taken_where_they_are_faster(size, forward16, forward32, backward):
    lib = _lib.load()
    b, n, d = size
    for dtype, want in ((0, forward32), (1, forward16), (2, forward16)):
        assert want is None or (lib.mi_gated_recurrence_workspace(b, n, d, 0, dtype) > 0) == want, dtype
    # backward: the folds of chunks, and a row of sums for each CTA of a block of channels
    rows = lib.mi_gated_recurrence_workspace(b, n, d, 1, 1) / (4 * b * d)
    assert (rows == int(rows) and rows % 3 == 0) if backward else rows in (1, 2, 4, 8, 16)


def slopes(value, leaves, got, prefix="d"):
    """Central differences of 1e-6 in 64 bits: 1e-12 of curvature and 1e-10 of rounding next to values of order 10."""
    g = torch.Generator().manual_seed(77)
    for name, t in leaves.items():
        v = _rand(g, *t.shape)
        up, down = (value({**leaves, name: t + s * 1e-6 * v}) for s in (1, -1))
        slope = float(up - down) / 2e-6
        have = float((got[prefix + name][0] * v).sum())
        assert abs(have - slope) < 1e-7 * max(1, abs(slope)) + 1e-7, (name, have, slope)


@pytest.mark.parametrize("convex", [True, False])
def test_recurrence_formula_against_differences(convex):
    g = torch.Generator().manual_seed(0)
    b, n, d = 3, 7, 4
    leaves = dict(x=_rand(g, b, n, d), f=_rand(g, b, n, d), z=_rand(g, b, n, d), bias=_rand(g, d), h0=_rand(g, b, d))
    rest = dict(convex=convex, lengths=torch.tensor([7, 4, 0], dtype=torch.int32))
    dy, dh = _rand(g, b, n, d), _rand(g, b, d)

    def value(vals):
        out = ref.recurrence({**vals, **rest})
        return (out["y"][0] * dy).sum() + (out["h"][0] * dh).sum()
    slopes(value, leaves, ref.recurrence({**leaves, **rest, "dy": dy, "dh": dh}))
    # the formula itself, written out for one channel
    one = {k: (t[:1, :, :1] if t.dim() == 3 else t[..., :1] if t.dim() == 1 else t[:1, :1]) for k, t in leaves.items()}
    out, h = ref.recurrence({**one, "convex": convex}), float(one["h0"])
    for t in range(n):
        a = float(torch.sigmoid(one["f"][0, t, 0] + one["bias"][0]))
        h = a * h + (1 - a if convex else 1) * float(one["x"][0, t, 0])
        z = float(one["z"][0, t, 0])
        assert abs(float(out["y"][0][0, t, 0]) - h * z / (1 + 2.718281828459045 ** -z)) < 1e-12


def test_norm_formula_against_differences():
    g = torch.Generator().manual_seed(2)
    leaves = dict(s=_rand(g, 5, 9), w=_rand(g, 9), bias=_rand(g, 9))
    dy, dsum = _rand(g, 5, 9), _rand(g, 5, 9)

    def value(v):
        return (ref.norm(v["s"], v["w"], v["bias"], 1e-5)["y"][0] * dy).sum() + (v["s"] * dsum).sum()
    slopes(value, leaves, ref.norm(leaves["s"], leaves["w"], leaves["bias"], 1e-5, dy, dsum))
    y = ref.norm(leaves["s"], leaves["w"], leaves["bias"], 1e-5)["y"][0]
    assert torch.allclose(y, torch.nn.functional.layer_norm(leaves["s"], (9,), leaves["w"], leaves["bias"], 1e-5), rtol=1e-12)


def test_forward_mode_is_refused():
    """A tangent would be lost; any argument may carry it, a view of a dual tensor too."""
    from torch.autograd import forward_ad

    x = lambda: _t(2, 5, 8)  # noqa: E731
    calls = [
        (selective.gated_recurrence, dict(x=x(), gate=x(), z=x(), gate_bias=_t(8), h0=_t(2, 8))),
        (selective.gated_recurrence_step, dict(h=_t(2, 8), x=_t(2, 8), gate=_t(2, 8), z=_t(2, 8), gate_bias=_t(8))),
        (selective.layer_norm, dict(x=_t(4, 8), weight=_t(8), bias=_t(8), residual=_t(4, 8))),
    ]
    for fn, args in calls:
        for name, t in args.items():
            with forward_ad.dual_level():
                wide = forward_ad.make_dual(torch.zeros(2, *t.shape), torch.ones(2, *t.shape))
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                        fn(**{**args, name: wide[0]})
        with pytest.raises(ValueError, match="must be a CUDA tensor"):  # and without one the call goes on
            fn(**args)


def test_the_choice_by_hand():
    x = torch.log(torch.tensor([1.0, 4.0, 2.0, 4.0, 1.0, 8.0], dtype=torch.float64))  # shares of 20; order 5 1 3 2 0 4
    pick = lambda u, t=1.0, k=0, p=1.0, m=0.0: ref.sample(x, u, t, k, p, m)[:2]  # noqa: E731
    assert pick(0.0) == (0, pytest.approx(1 / 20)) and pick(0.049)[0] == 0 and pick(0.051)[0] == 1 and pick(0.99)[0] == 5
    assert pick(0.6, t=0.0) == (5, 1.0)
    assert pick(0.3, k=2) == (1, pytest.approx(1 / 3)) and pick(0.34, k=2)[0] == 5  # the lower index of the equal ones
    assert pick(0.1, p=0.39) == (5, 1.0) and pick(0.1, p=0.41)[0] == 1  # 8 of 20 before the second
    assert pick(0.0, m=0.4)[0] == 1 and pick(0.0, m=0.2)[0] == 1 and pick(0.0, m=0.12)[0] == 0
    assert pick(0.3, t=2.0, k=2)[1] == pytest.approx(2 ** 0.5 / (1 + 2 ** 0.5) / 2 ** 0.5)
    inf = float("inf")
    assert ref.sample(torch.tensor([-inf, -inf]), 0.5, 1.0, 0, 1.0, 0.0)[:2] == (0, 1.0)
    assert ref.sample(torch.tensor([1.0, float("nan"), inf]), 0.5, 1.0, 0, 1.0, 0.0)[:2] == (1, 1.0)

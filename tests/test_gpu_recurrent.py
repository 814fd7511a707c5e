"""The float recurrent layer's operators against their 64-bit formulas (tests/recurrent_ref.py, where the tolerances are
derived)."""
import numpy as np
import pytest
import torch

import recurrent_ref as ref
from mamba_integer_b200 import _lib

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def sel(cuda_dev):
    from mamba_integer_b200 import selective
    return selective


def rec_inputs(dev, dtype, b, n, d, seed=0, z=True, bias=True, h0=False, convex=True, lengths=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    a = dict(x=r(b, n, d).to(dtype), f=(r(b, n, d) + (0 if bias else 2)).to(dtype), z=r(b, n, d).to(dtype) if z else None,
             bias=2 + 2 * r(d) if bias else None, h0=r(b, d) if h0 else None, convex=convex)
    a["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return {k: t.to(dev) if isinstance(t, torch.Tensor) else t for k, t in a.items()}


def call_rec(sel, a, **over):
    a = {**a, **over}
    return sel.gated_recurrence(a["x"], a["f"], z=a["z"], gate_bias=a["bias"], convex=a["convex"], h0=a["h0"],
                                lengths=a["lengths"], return_state=True)


def check_rec(y, h, a):
    want = ref.recurrence(a)
    ref.check(y, want["y"], "y")
    ref.check(h, want["h"], "h")


REC_SIZES = [
    # batch, L, channels: blocks of 64 channels, stretches of 8 and 16 positions, tiles of 64 and 128, clusters of 1 to 8
    (1, 1, 1), (2, 1, 64), (1, 2, 33), (3, 7, 31), (2, 8, 64), (2, 9, 65), (1, 15, 100), (2, 16, 128), (1, 17, 8),
    (2, 63, 72), (1, 64, 2), (1, 65, 130), (3, 128, 40), (2, 129, 64), (1, 255, 16), (1, 257, 66), (1, 513, 24),
    (1, 1100, 72), (40, 70, 520), (2, 2050, 12),
]


@pytest.mark.parametrize("size", REC_SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_recurrence_prompt(sel, cuda_dev, size, dtype):
    a = rec_inputs(cuda_dev, dtype, *size, h0=size[1] % 2 == 1)
    check_rec(*call_rec(sel, a), a)


def rec_grads(sel, a, dy, dh, need=None):
    names = [k for k in ("x", "f", "z", "bias", "h0") if a[k] is not None and (need is None or k in need)]
    leaves = {k: a[k].detach().clone().requires_grad_(True) for k in names}
    y, h = call_rec(sel, a, **leaves)
    outs = [(o, g) for o, g in ((y, dy), (h, dh)) if g is not None]
    got = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)
    return y, h, dict(zip(names, got))


def check_rec_grads(got, a, dy, dh):
    want = ref.recurrence(dict(a, dy=dy, dh=dh))
    for name, t in got.items():
        assert t.dtype == a[name].dtype
        ref.check(t, want["d" + name], "d" + name)


@pytest.mark.parametrize("size", REC_SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_recurrence_gradients(sel, cuda_dev, size, dtype):
    b, n, d = size
    a = rec_inputs(cuda_dev, dtype, *size, h0=True)
    g = torch.Generator().manual_seed(5)
    dy, dh = torch.randn(b, n, d, generator=g).to(cuda_dev, dtype), torch.randn(b, d, generator=g).to(cuda_dev)
    y, h, got = rec_grads(sel, a, dy, dh)
    check_rec(y, h, a)
    check_rec_grads(got, a, dy, dh)


@pytest.mark.parametrize("convex", [True, False])
@pytest.mark.parametrize("z,bias,h0", [(False, False, False), (True, False, True), (False, True, True)])
@pytest.mark.parametrize("n", [40, 300])
def test_recurrence_options(sel, cuda_dev, n, convex, z, bias, h0):
    a = rec_inputs(cuda_dev, F32, 2, n, 48, z=z, bias=bias, h0=h0, convex=convex)
    dy = torch.randn(2, n, 48, device=cuda_dev)
    y, h, got = rec_grads(sel, a, dy, None)
    check_rec(y, h, a)
    check_rec_grads(got, a, dy, None)
    dh = torch.randn(2, 48, device=cuda_dev)
    _, _, got = rec_grads(sel, a, None, dh, need=("x", "f"))
    check_rec_grads(got, a, None, dh)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("d", [66, 72])
def test_recurrence_long_sequences(sel, cuda_dev, dtype, d):
    """Few channels and many positions, which are shared out in chunks; lengths that end at a chunk's border, inside one, in
    front of all."""
    n, lens = 4500, [4500, 1024, 1027, 0, 3333]
    a = rec_inputs(cuda_dev, dtype, 5, n, d, h0=True, lengths=lens)
    a["bias"] += 3  # memories long enough to reach through chunks
    dy, dh = torch.randn(5, n, d, device=cuda_dev).to(dtype), torch.randn(5, d, device=cuda_dev)
    y, h, got = rec_grads(sel, a, dy, dh)
    check_rec(y, h, a)
    check_rec_grads(got, a, dy, dh)
    with torch.no_grad():
        again = call_rec(sel, a)
    assert torch.equal(again[0], y) and torch.equal(again[1], h)


@pytest.mark.parametrize("n", [37, 260])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_recurrence_lengths(sel, cuda_dev, n, dtype):
    # 0, 1, inside and at a stretch's border, past the end (clamped), negative (clamped)
    lens = [0, 1, 8, 16, 20, n, n + 5, -3]
    a = rec_inputs(cuda_dev, dtype, len(lens), n, 40, h0=True, lengths=lens)
    clamped = dict(a, lengths=torch.tensor([min(max(v, 0), n) for v in lens], dtype=torch.int32))
    dy, dh = torch.randn(len(lens), n, 40, device=cuda_dev).to(dtype), torch.randn(len(lens), 40, device=cuda_dev)
    for i, v in enumerate(clamped["lengths"].tolist()):  # what lies behind a length is not used
        for name in ("x", "f", "z"):
            a[name][i, v:] = float("nan") if i % 2 else float("inf")
        dy[i, v:] = float("nan")
    y, h, got = rec_grads(sel, a, dy, dh)
    check_rec(y, h, clamped)
    check_rec_grads(got, clamped, dy, dh)
    for i, v in enumerate(clamped["lengths"].tolist()):
        assert not y[i, v:].any() and not got["x"][i, v:].any() and not got["f"][i, v:].any() and not got["z"][i, v:].any()
    assert torch.equal(h[0], a["h0"][0]) and torch.equal(got["h0"][0], dh[0])


def test_recurrence_strides_slices_and_broadcasts(sel, cuda_dev):
    b, n, d = 3, 70, 48
    a = rec_inputs(cuda_dev, BF16, b, n, d)
    want = call_rec(sel, a)
    for pad in (8, 3):  # columns of wider rows, aligned and not; every other row
        wide = torch.randn(b, 2 * n, 3 * d + pad, device=cuda_dev).to(BF16)
        cut = {}
        for i, key in enumerate(("x", "f", "z")):
            cut[key] = wide[:, ::2, pad + i * d:pad + (i + 1) * d]
            cut[key].copy_(a[key])
        got = call_rec(sel, a, **cut)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = {key: a[key][:1] for key in ("x", "f", "z")}
    spread = call_rec(sel, a, **{key: t.expand(b, -1, -1) for key, t in one.items()})
    copied = call_rec(sel, a, **{key: t.repeat(b, 1, 1) for key, t in one.items()})
    assert torch.equal(spread[0], copied[0]) and torch.equal(spread[1], copied[1])
    flat = torch.empty(d + 1, device=cuda_dev)
    flat[1:].copy_(a["bias"])
    assert torch.equal(call_rec(sel, a, bias=flat[1:])[0], want[0])
    # gradients of a sequence that several share
    dy = torch.randn(b, n, d, device=cuda_dev).to(BF16)
    x = one["x"].detach().clone().requires_grad_(True)
    y, _ = call_rec(sel, a, x=x.expand(b, -1, -1))
    got, = torch.autograd.grad(y, x, dy)
    xs = one["x"].repeat(b, 1, 1).requires_grad_(True)
    y, _ = call_rec(sel, a, x=xs)
    each, = torch.autograd.grad(y, xs, dy.transpose(1, 2).contiguous().transpose(1, 2))  # a gradient with another layout
    assert torch.equal(got, each.sum(0, keepdim=True))


def test_recurrence_offsets_past_32_bits(sel, cuda_dev):
    n, d = 20, 32
    a = rec_inputs(cuda_dev, BF16, 2, n, d)
    want = call_rec(sel, a)
    big = torch.empty(2 ** 31 + 64 * n, dtype=BF16, device=cuda_dev)
    for i, key in enumerate(("x", "f", "z")):
        far = big[i * 8 * d:].as_strided((2, n, d), (2 ** 31 + 3 * d - 2 ** 10, d, 1))
        far.copy_(a[key])
        got = call_rec(sel, a, **{key: far})
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_recurrence_extreme_gates(sel, cuda_dev, dtype):
    """Gates that keep the state, that drop it at once, and NaN and infinities of inputs and states."""
    n = 300
    a = rec_inputs(cuda_dev, dtype, 1, n, 64, h0=True, bias=False, z=False)
    a["f"][0, ::3], a["f"][0, 1::7] = 60.0, -60.0
    dy, dh = torch.randn_like(a["x"]), torch.randn(1, 64, device=cuda_dev)
    y, h, got = rec_grads(sel, a, dy, dh)
    check_rec(y, h, a)
    check_rec_grads(got, a, dy, dh)
    a["f"][0, ::3], a["f"][0, 1::7] = float("inf"), float("-inf")  # a convention: 2^-126 is as good as 0
    y2, h2 = call_rec(sel, a)
    assert torch.isfinite(y2).all() and torch.isfinite(h2).all()
    a = rec_inputs(cuda_dev, dtype, 1, n, 64, h0=True)
    a["x"][0, 150, :32] = float("inf")
    a["h0"][0, 40] = float("-inf")
    a["x"][0, 200, 50] = float("nan")
    y, h = call_rec(sel, a, z=None)
    assert (y[0, 150:, :32] == float("inf")).all() and torch.isfinite(y[0, :150, :32]).all()
    assert (y[0, :, 40] == float("-inf")).all() and h[0, 40] == float("-inf")
    assert torch.isfinite(y[0, :200, 50]).all() and y[0, 200:, 50].isnan().all() and h[0, 50].isnan()
    rest = [i for i in range(32, 64) if i not in (40, 50)]
    assert torch.isfinite(y[..., rest]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("size", [(1, 1), (3, 33), (4, 512), (2, 130), (256, 64), (5, 1021)])
@pytest.mark.parametrize("convex,z,bias", [(True, True, True), (False, False, False), (True, False, True), (False, True, False)])
def test_recurrence_step(sel, cuda_dev, dtype, size, convex, z, bias):
    b, d = size
    a = rec_inputs(cuda_dev, dtype, b, 3, d, z=z, bias=bias, h0=True, convex=convex)
    h = a["h0"].clone()
    ys = []
    for t in range(3):
        with torch.no_grad():
            ys.append(sel.gated_recurrence_step(h, a["x"][:, t], a["f"][:, t], z=None if a["z"] is None else a["z"][:, t],
                                                gate_bias=a["bias"], convex=convex))
    check_rec(torch.stack(ys, 1), h, a)


# Output gates over the types' whole range.  sigmoid reaches 0 within 110 of 0, where z sigmoid(z) and its slope are 0 too.
GATES = [-85.0, -87.5, -89.0, -95.0, -110.0, -1e4, -1e30, -1e34, -1e37, "lowest", 60.0, 86.0, 88.0, 100.0, 1e3]


def gate_rows(dtype, dev, b, n, d):
    """A z of each of GATES at every channel, between ordinary ones."""
    z = torch.randn(b, n, d, generator=torch.Generator().manual_seed(9))
    low = torch.finfo(dtype).min
    for i, v in enumerate(GATES):
        z[:, 1 + 2 * i] = low if v == "lowest" else max(v, low)
    return z.to(dtype).to(dev)


def check_gated(got, want, error, name):
    """`error`: absolute, before the result's own rounding (half a step, or half the smallest subnormal)."""
    dtype = got.dtype
    tol = error + torch.finfo(dtype).eps / 2 * (want.abs() + error) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2
    off = (got.detach().cpu().double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (name, bad.nonzero()[:6].tolist(), got.cpu()[bad][:6], want[bad][:6])


def check_output_gate(a, y, dz=None, dy=None):
    """y and dz from the states' own errors (the formula without a gate) and the gate's.

    sigmoid(z) and sigmoid(-z) are off by 10 units and 3 |z| more of the smaller one (tests/recurrent_ref.py).  One below
    e^-87 (fp32) or 2^-126 (16 bits) counts as 0; with the roundings of z and of the power, up to 1.0001 times that."""
    z = ref.d64(a["z"])
    plain, mags = dict(a, z=None), dict(a, z=None, x=a["x"].abs(), h0=None if a["h0"] is None else a["h0"].abs())
    want = ref.recurrence(plain)
    h, e_h = want["y"]
    m_h = ref.recurrence(mags)["y"][0]
    s, n = torch.sigmoid(z), torch.sigmoid(-z)
    r_s, r_n = (torch.where(q > 0.5, 10.0, 9 + 3 * z.abs()) for q in (s, n))
    U, least = 2.0 ** -24, 1.0001 * (np.exp(-87.0) if y.dtype == F32 else 2.0 ** -126)
    lost = lambda q: torch.where(q < least, q, 0.0)  # noqa: E731
    gate, slope, m_slope = z * s, s + z * s * n, s + z.abs() * s * n
    e_gate = U * (r_s + 2) * gate.abs() + z.abs() * lost(s)
    e_slope = U * ((r_s + 2) * s + (r_s + r_n + 4) * z.abs() * s * n) + lost(s) * (1 + z.abs() * n) + lost(n) * z.abs() * s
    check_gated(y, h * gate, U * e_h * gate.abs() + m_h * e_gate + 2.0 ** -149, "y")
    if dz is not None:
        g = ref.d64(dy).abs()
        error = g * (U * e_h * m_slope + m_h * (e_slope + 2 * U * m_slope)) + 2.0 ** -149 * (1 + g)
        check_gated(dz, ref.d64(dy) * h * slope, error, "dz")


@pytest.mark.parametrize("d", [40, 41])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_recurrence_output_gate_over_its_whole_range(sel, cuda_dev, dtype, d):
    n = 37
    a = rec_inputs(cuda_dev, dtype, 2, n, d, h0=True)
    a["z"] = gate_rows(dtype, cuda_dev, 2, n, d)
    dy, dh = torch.randn(2, n, d, device=cuda_dev).to(dtype), torch.randn(2, d, device=cuda_dev)
    y, h, got = rec_grads(sel, a, dy, dh)
    check_output_gate(a, y, got["z"], dy)
    check_rec_grads({k: t for k, t in got.items() if k != "z"}, a, dy, dh)  # a gate of 0 passes nothing on
    with torch.no_grad():
        assert torch.equal(call_rec(sel, a)[0], y)
    for v in (float("-inf"), float("nan")):  # 0 times an infinity, as in the formula
        a["z"][:, 5] = v
        assert call_rec(sel, a)[0][:, 5].isnan().all() and not call_rec(sel, a)[0][:, 6].isnan().any()


@pytest.mark.parametrize("d", [40, 41])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_recurrence_step_output_gate_over_its_whole_range(sel, cuda_dev, dtype, d):
    n = 37
    a = rec_inputs(cuda_dev, dtype, 2, n, d, h0=True)
    a["z"] = gate_rows(dtype, cuda_dev, 2, n, d)
    h, ys = a["h0"].clone(), []
    for t in range(n):
        with torch.no_grad():
            ys.append(sel.gated_recurrence_step(h, a["x"][:, t], a["f"][:, t], z=a["z"][:, t], gate_bias=a["bias"]))
    check_output_gate(a, torch.stack(ys, 1))


@pytest.mark.parametrize("n,d", [(37, 40), (37, 41), (8300, 24)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_recurrence_inputs_of_weight_zero(sel, cuda_dev, dtype, n, d):
    """Where the gate keeps the whole state, an input counts for nothing, the type's lowest value included."""
    a = rec_inputs(cuda_dev, dtype, 1, n, d, h0=True, bias=False)
    most = torch.finfo(dtype).max
    for i, (f, x) in enumerate([(200.0, -most), (1e4, most), (most, -most), (most, -1e4), (200.0, -min(most, 1e30)), (1e30, most)]):
        a["f"][0, 2 + 5 * i], a["x"][0, 2 + 5 * i] = min(f, most), x
    dy, dh = torch.randn(1, n, d, device=cuda_dev).to(dtype), torch.randn(1, d, device=cuda_dev)
    y, h, got = rec_grads(sel, a, dy, dh)
    check_rec(y, h, a)
    check_rec_grads(got, a, dy, dh)
    assert not got["x"][0, 2:30:5].any() and not got["f"][0, 2:30:5].any()
    s, ys = a["h0"].clone(), []
    for t in range(min(n, 37)):
        with torch.no_grad():
            ys.append(sel.gated_recurrence_step(s, a["x"][:, t], a["f"][:, t], z=a["z"][:, t]))
    check_rec(torch.stack(ys, 1), s, {k: v[:, :37] if k in ("x", "f", "z") else v for k, v in a.items()})
    a["f"][0, 2:30:5] = float("inf")
    assert torch.equal(call_rec(sel, a)[0], y)


# Sequences of 8229 positions of few channels go in chunks (of 384), both ways and in every type; with rows off 16 bytes those
# of 16421.
CHUNK_LENGTHS = [30000, 5376, 5377, 2687, 0, 5000]  # all; at a border of each, behind it, in front of it; none; inside


@pytest.mark.parametrize("d", [72, 33])
@pytest.mark.parametrize("z,bias,convex", [(True, True, True), (False, True, True), (True, False, False), (False, False, False)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_recurrence_in_chunks(sel, cuda_dev, dtype, z, bias, convex, d):
    b, n = len(CHUNK_LENGTHS), 8229 if d == 72 else 16421
    a = rec_inputs(cuda_dev, dtype, b, n, d, z=z, bias=bias, h0=True, convex=convex, lengths=[min(v, n) for v in CHUNK_LENGTHS])
    if bias:
        a["bias"] += 3  # memories that reach through chunks
    if z:
        a["z"][0, 100::1000] = torch.finfo(dtype).min  # closed output gates
    dy, dh = torch.randn(b, n, d, device=cuda_dev).to(dtype), torch.randn(b, d, device=cuda_dev)
    lib = _lib.load()
    for backward in (0, 1):  # (a row of sums a cluster's CTA, or three a chunk)
        assert lib.mi_gated_recurrence_workspace(b, n, d, backward, {F32: 0, BF16: 1, F16: 2}[dtype]) > 4 * b * d * 16 * backward
    y, h, got = rec_grads(sel, a, dy, dh)
    check_rec(y, h, a)
    check_rec_grads(got, a, dy, dh)
    if z:
        assert not y[0, 100::1000].any() and not got["z"][0, 100::1000].any()
    with torch.no_grad():
        again = call_rec(sel, a)
    assert torch.equal(again[0], y) and torch.equal(again[1], h)


@pytest.mark.parametrize("n", [8192, 20000])
def test_recurrence_one_long_sequence(sel, cuda_dev, n):
    a = rec_inputs(cuda_dev, BF16, 1, n, 24, z=False)
    a["bias"] += 4
    dy = torch.randn(1, n, 24, device=cuda_dev).to(BF16)
    y, h, got = rec_grads(sel, a, dy, None)
    check_rec(y, h, a)
    check_rec_grads(got, a, dy, None)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_recurrence_extreme_values_in_chunks(sel, cuda_dev, dtype):
    """Gates that keep and that drop the state, and infinite and NaN inputs, states and gradients, through chunks that they
    do not lie in."""
    n, d = 8300, 64
    a = rec_inputs(cuda_dev, dtype, 1, n, d, h0=True, bias=False, z=False)
    a["f"][0, ::3], a["f"][0, 1::7] = 60.0, -60.0
    dy, dh = torch.randn(1, n, d, device=cuda_dev).to(dtype), torch.randn(1, d, device=cuda_dev)
    y, h, got = rec_grads(sel, a, dy, dh)
    check_rec(y, h, a)
    check_rec_grads(got, a, dy, dh)
    inf, nan = float("inf"), float("nan")
    a["x"][0, 3000, :32] = inf
    a["h0"][0, 40] = -inf
    a["x"][0, 6000, 50] = nan
    dy[0, 7000, 33], dh[0, 34] = nan, inf
    y, h, got = rec_grads(sel, a, dy, dh)
    assert (y[0, 3000:, :32] == inf).all() and torch.isfinite(y[0, :3000, :32]).all() and (h[0, :32] == inf).all()
    assert (y[0, :, 40] == -inf).all() and h[0, 40] == -inf
    assert torch.isfinite(y[0, :6000, 50]).all() and y[0, 6000:, 50].isnan().all() and h[0, 50].isnan()
    rest = [i for i in range(32, 64) if i not in (40, 50)]
    assert torch.isfinite(y[..., rest]).all() and torch.isfinite(h[..., rest]).all()
    dx = got["x"]
    assert dx[0, :7001, 33].isnan().all() and torch.isfinite(dx[0, 7001:, 33]).all() and got["h0"][0, 33].isnan()
    # 1 - a is e^-60 at the least, so an infinite gradient reaches every input
    assert (dx[0, :, 34] == inf).all() and got["h0"][0, 34] == inf
    rest = [i for i in range(64) if i not in (33, 34)]
    assert torch.isfinite(dx[..., rest]).all() and torch.isfinite(got["h0"][..., rest]).all()


def test_recurrence_same_bits_and_streams(sel, cuda_dev):
    """The same inputs give the same bits, on another stream and captured in a graph that is replayed."""
    a = rec_inputs(cuda_dev, BF16, 2, 700, 192, h0=True)
    dy, dh = torch.randn(2, 700, 192, device=cuda_dev).to(BF16), torch.randn(2, 192, device=cuda_dev)
    y, h, got = rec_grads(sel, a, dy, dh)
    y, h, got = y.detach(), h.detach(), {k: t.clone() for k, t in got.items()}
    for _ in range(3):
        y2, h2, got2 = rec_grads(sel, a, dy, dh)
        assert torch.equal(y, y2) and torch.equal(h, h2) and all(torch.equal(got[k], got2[k]) for k in got)
    del y2, h2, got2
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    leaves = {k: a[k].detach().clone().requires_grad_(True) for k in got}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        call_rec(sel, a, **leaves)
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            y3, h3 = call_rec(sel, a, **leaves)
            got3 = torch.autograd.grad([y3, h3], list(leaves.values()), [dy, dh])
    for _ in range(2):
        y3.detach().zero_(), h3.detach().zero_(), [t.zero_() for t in got3]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, y3) and torch.equal(h, h3)
        assert all(torch.equal(got[k], t) for k, t in zip(leaves, got3))


def test_recurrence_empty_calls(sel, cuda_dev):
    for b, n in ((0, 5), (2, 0)):
        a = rec_inputs(cuda_dev, F32, b, n, 8, h0=True)
        leaves = {k: a[k].detach().clone().requires_grad_(True) for k in ("x", "f", "z", "bias", "h0")}
        y, h = call_rec(sel, a, **leaves)
        assert y.shape == (b, n, 8) and torch.equal(h, a["h0"])
        got = torch.autograd.grad([y.sum() + h.sum()], list(leaves.values()))
        assert not got[3].any() and (got[4] == 1).all()
    none = torch.zeros(0, 8, device=cuda_dev)
    assert sel.gated_recurrence_step(none, none, none).shape == (0, 8)


def test_recurrence_second_order_is_refused(sel, cuda_dev):
    a = rec_inputs(cuda_dev, F32, 1, 9, 8)
    x = a["x"].requires_grad_(True)
    y, _ = call_rec(sel, a)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="first order"):
        torch.autograd.grad(g.sum(), x)


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
EPS = 1e-5
NORM_SIZES = [
    # rows, width: rows within a warp (4 to 32 threads), of several warps, of 1, 2 and 4 packs a thread, odd widths
    (1, 1), (5, 8), (3, 31), (70, 32), (9, 72), (33, 129), (2, 256), (700, 264), (17, 509), (4, 512), (37, 768), (300, 1024),
    (6, 1032), (3, 2000), (5, 4096), (3, 4100), (2, 5000), (2, 8192), (3, 8200), (1, 9001), (2, 16384), (1, 16380),
]


def norm_inputs(dev, dtype, t, d, rdtype=None, bias=True, seed=0, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    a = dict(x=(r(t, d) + offset).to(dtype), w=1 + 0.5 * r(d), b=r(d) if bias else None,
             r=None if rdtype is None else (2 * r(t, d)).to(rdtype), dy=r(t, d).to(dtype))
    a["dsum"] = None if rdtype is None else r(t, d).to(rdtype)
    return {k: None if v is None else v.to(dev) for k, v in a.items()}


def check_norm(sel, a):
    names = [k for k in ("x", "w", "b", "r") if a[k] is not None]
    leaves = {k: a[k].detach().clone().requires_grad_(True) for k in names}
    y, s = sel.layer_norm(leaves["x"], leaves["w"], leaves.get("b"), eps=EPS, residual=leaves.get("r"))
    outs = [(y, a["dy"])] + ([] if s is None else [(s, a["dsum"])])
    got = dict(zip(names, torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs])))
    kept = a["x"] if s is None else (a["x"].float() + a["r"].float()).to(a["r"].dtype)
    if s is not None:
        assert torch.equal(s, kept)
    want = ref.norm(kept, a["w"], a["b"], EPS, a["dy"], a["dsum"])
    ref.check(y, want["y"], "y")
    ref.check(got["x"], want["ds"], "dx")
    ref.check(got["w"], want["dw"], "dw")
    if a["b"] is not None:
        ref.check(got["b"], want["dbias"], "db")
    if a["r"] is not None:
        ref.check(got["r"], want["ds"], "dr")
    with torch.no_grad():
        again, s2 = sel.layer_norm(a["x"], a["w"], a["b"], eps=EPS, residual=a["r"])
    assert torch.equal(again, y) and (s is None or torch.equal(s, s2))


@pytest.mark.parametrize("size", NORM_SIZES)
@pytest.mark.parametrize("dtype,rdtype", [(F32, None), (F32, F32), (BF16, None), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
def test_layer_norm(sel, cuda_dev, size, dtype, rdtype):
    check_norm(sel, norm_inputs(cuda_dev, dtype, *size, rdtype=rdtype, bias=size[0] % 3 != 0))


@pytest.mark.parametrize("t,d", [(5000, 64), (2500, 768), (1301, 509), (700, 4096)])
def test_layer_norm_many_rows(sel, cuda_dev, t, d):
    check_norm(sel, norm_inputs(cuda_dev, BF16, t, d, rdtype=BF16))


@pytest.mark.parametrize("d", [3, 31, 33, 65, 129, 255])
@pytest.mark.parametrize("dtype,rdtype", [(F32, F32), (BF16, BF16), (F16, F32)])
def test_layer_norm_many_narrow_odd_rows(sel, cuda_dev, dtype, rdtype, d):
    """Rows of 4 to 32 threads whose windows are filled many times over by other lanes, the sum's gradient among them; the
    same bits in every run."""
    t = 20011
    a = norm_inputs(cuda_dev, dtype, t, d, rdtype=rdtype)
    check_norm(sel, a)
    leaves = {k: a[k].detach().clone().requires_grad_(True) for k in ("x", "w", "b", "r")}
    runs = []
    for _ in range(5):
        y, s = sel.layer_norm(leaves["x"], leaves["w"], leaves["b"], eps=EPS, residual=leaves["r"])
        runs.append([y.detach(), s.detach(), *torch.autograd.grad([y, s], list(leaves.values()), [a["dy"], a["dsum"]])])
    assert all(torch.equal(p, q) for run in runs[1:] for p, q in zip(runs[0], run))


def test_layer_norm_rows_far_from_zero(sel, cuda_dev):
    """A mean a thousand times the spread, rows that are constant, and rows of zeros."""
    a = norm_inputs(cuda_dev, F32, 40, 700, offset=1000.0)
    a["x"][3], a["x"][4] = 7.25, 0.0
    check_norm(sel, a)
    y, _ = sel.layer_norm(a["x"], a["w"], a["b"], eps=EPS)
    assert torch.allclose(y[4], a["b"])
    a["x"][5, 9], a["x"][6, 2] = float("nan"), float("inf")
    y, _ = sel.layer_norm(a["x"], a["w"], a["b"], eps=EPS)
    assert y[5].isnan().all() and y[6].isnan().all() and torch.isfinite(y[[0, 1, 2, 3, 4, 7]]).all()


def test_layer_norm_shapes_strides_and_parts(sel, cuda_dev):
    a = norm_inputs(cuda_dev, BF16, 24, 96, rdtype=F32)
    want = sel.layer_norm(a["x"], a["w"], a["b"], residual=a["r"])
    got = sel.layer_norm(a["x"].view(2, 3, 4, 96), a["w"], a["b"], residual=a["r"].view(2, 3, 4, 96))
    assert got[0].shape == (2, 3, 4, 96) and torch.equal(got[0].view(24, 96), want[0]) and torch.equal(got[1].view(24, 96), want[1])
    for pad in (8, 3):
        wide = torch.empty(24, 96 + 2 * pad, dtype=BF16, device=cuda_dev)
        x = wide[:, pad:pad + 96]
        x.copy_(a["x"])
        got = sel.layer_norm(x, a["w"], a["b"], residual=a["r"])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    flat = torch.empty(97, device=cuda_dev)
    flat[1:].copy_(a["w"])
    assert torch.equal(sel.layer_norm(a["x"], flat[1:], a["b"], residual=a["r"])[0], want[0])
    row = a["x"][:1].detach().clone().requires_grad_(True)  # a row that many share
    y, _ = sel.layer_norm(row.expand(24, -1), a["w"], a["b"])
    g, = torch.autograd.grad(y, row, a["dy"])
    each = a["x"][:1].repeat(24, 1).requires_grad_(True)
    y, _ = sel.layer_norm(each, a["w"], a["b"])
    assert torch.equal(g, torch.autograd.grad(y, each, a["dy"])[0].sum(0, keepdim=True))
    # gradients of some of the arguments, and of the sum alone
    full = {}
    for names in (("x", "w", "b", "r"), ("x",), ("w",), ("b",), ("r",)):
        leaves = {k: a[k].detach().clone().requires_grad_(k in names) for k in ("x", "w", "b", "r")}
        y, s = sel.layer_norm(leaves["x"], leaves["w"], leaves["b"], residual=leaves["r"])
        outs, givens = ([y, s], [a["dy"], a["dsum"]]) if set(names) & {"x", "r"} else ([y], [a["dy"]])
        got = dict(zip(names, torch.autograd.grad(outs, [leaves[k] for k in names], givens)))
        full = full or got
        assert all(torch.equal(full[k], got[k]) for k in names)
    x, r = a["x"].detach().requires_grad_(True), a["r"].detach().requires_grad_(True)
    _, s = sel.layer_norm(x, a["w"], a["b"], residual=r)
    gx, gr = torch.autograd.grad(s, [x, r], a["dsum"])
    assert torch.equal(gx, a["dsum"].to(BF16)) and torch.equal(gr, a["dsum"])


def test_layer_norm_empty_and_refused(sel, cuda_dev):
    w = torch.ones(8, device=cuda_dev, requires_grad=True)
    b = torch.ones(8, device=cuda_dev, requires_grad=True)
    y, s = sel.layer_norm(torch.zeros(0, 8, device=cuda_dev), w, b)
    assert y.shape == (0, 8) and s is None
    gw, gb = torch.autograd.grad(y.sum(), [w, b])
    assert not gw.any() and not gb.any()
    x = torch.randn(3, 8, device=cuda_dev, requires_grad=True)
    y, _ = sel.layer_norm(x, w, b)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="first order"):
        torch.autograd.grad(g.sum(), x)


def test_layer_norm_captured(sel, cuda_dev):
    a = norm_inputs(cuda_dev, BF16, 333, 768, rdtype=BF16)
    leaves = {k: a[k].detach().clone().requires_grad_(True) for k in ("x", "w", "b", "r")}

    def step():
        y, s = sel.layer_norm(leaves["x"], leaves["w"], leaves["b"], residual=leaves["r"])
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], list(leaves.values()), [a["dy"], a["dsum"]])]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        want = [t.clone() for t in step()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            got = step()
    for _ in range(2):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got))


# ---------------------------------------------------------------------------
# the choice of a token
# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def kernels(cuda_dev):
    from mamba_integer_b200 import kernels
    return kernels


# masses are whole numbers of 2^-44 from powers right to 2^-37: sums of up to 2^17 of them are off by less than 2^-30 of
# the total, and a border that lies nearer than that to the number asked for may be taken from either side
NEAR = 2.0 ** -30


def check_sample(kernels, dev, logits, u, t, k, p, m):
    """Settings: numbers, or lists of one a row."""
    rows = logits.shape[0]
    each = lambda v: v if isinstance(v, list) else [v] * rows  # noqa: E731
    send = lambda v, d: torch.tensor(v, dtype=d, device=dev) if isinstance(v, list) else v  # noqa: E731
    token, prob = kernels.sample_rows(logits.to(dev), torch.tensor(u, device=dev), send(t, F32), send(k, torch.int32),
                                      send(p, F32), send(m, F32), return_prob=True)
    f32 = lambda v: torch.tensor(v, dtype=F32).double().tolist()  # noqa: E731
    token, prob = token.tolist(), prob.tolist()
    unsure = 0
    for i, row in enumerate(zip(f32(u), f32(each(t)), each(k), f32(each(p)), f32(each(m)))):
        want, share, near = ref.sample(logits[i], *row)
        if near < NEAR:
            unsure += 1
            continue
        assert token[i] == want, (i, row, token[i], want, near)
        # its own rounding, and the total's 2^-30
        assert abs(prob[i] - share) <= share * (2.0 ** -24 + NEAR), (i, row, prob[i], share)
    assert unsure <= max(1, rows // 50)


def sample_logits(rows, v, seed=0, spread=2.5, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, v, generator=g)
    return torch.where(torch.rand(rows, v, generator=g) < 30 / v, 4 + 8 * torch.rand(rows, v, generator=g), x).to(dtype)


def uniform(rows, seed=1):
    return torch.rand(rows, generator=torch.Generator().manual_seed(seed)).tolist()


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.1), (0.9, 40, 0.8, 0.05),
            (0.0, 5, 0.5, 0.5), (1.5, 1, 1.0, 0.0), (1.0, 700, 0.97, 0.0), (0.2, 0, 0.5, 0.01), (50.0, 0, 0.7, 0.0)]


@pytest.mark.parametrize("setting", SETTINGS)
@pytest.mark.parametrize("rows,v", [(1, 1), (3, 2), (5, 64), (7, 1000), (4, 4096), (9, 32768), (2, 50021), (1, 131072)])
def test_sample(kernels, cuda_dev, rows, v, setting):
    check_sample(kernels, cuda_dev, sample_logits(rows, v, seed=v), uniform(rows, v), *setting)


# More than 131072 tokens take clusters whatever the number of rows.
@pytest.mark.parametrize("setting", SETTINGS)
@pytest.mark.parametrize("rows,v", [(2, 131073), (3, 200003), (2, 262144)])
def test_sample_large_vocabularies(kernels, cuda_dev, rows, v, setting):
    check_sample(kernels, cuda_dev, sample_logits(rows, v, seed=v), uniform(rows, v), *setting)


@pytest.mark.parametrize("v", [131073, 262144])
def test_sample_many_rows_of_large_vocabularies(kernels, cuda_dev, v):
    rows = 160
    g = torch.Generator().manual_seed(v)
    r = lambda: torch.rand(rows, generator=g)  # noqa: E731
    t = torch.where(r() < 0.1, 0.0, 0.3 + 1.5 * r()).tolist()
    k = torch.where(r() < 0.5, 0, (r() * 2000).int() + 1).int().tolist()
    p = torch.where(r() < 0.4, 1.0, r()).tolist()
    m = torch.where(r() < 0.5, 0.0, 0.3 * r()).tolist()
    logits = sample_logits(rows, v, seed=v, dtype=BF16)
    logits[3] = 0.0  # ties all over
    logits[4, : v - 5] = -float("inf")
    check_sample(kernels, cuda_dev, logits, uniform(rows, v), t, k, p, m)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("v", [300, 4100, 32768, 40000])
def test_sample_rows_with_settings_of_their_own(kernels, cuda_dev, v, dtype):
    rows = 160
    g = torch.Generator().manual_seed(v)
    r = lambda: torch.rand(rows, generator=g)  # noqa: E731
    t = torch.where(r() < 0.2, 0.0, 0.3 + 1.5 * r()).tolist()
    k = torch.where(r() < 0.4, 0, (r() * 2000).int() + 1).int().tolist()
    p = torch.where(r() < 0.4, 1.0, r()).tolist()
    m = torch.where(r() < 0.5, 0.0, 0.3 * r()).tolist()
    check_sample(kernels, cuda_dev, sample_logits(rows, v, seed=v, dtype=dtype), uniform(rows, v), t, k, p, m)


@pytest.mark.parametrize("v", [600, 5000, 32768, 100003])
@pytest.mark.parametrize("spread", [0.01, 0.3, 1.0, 8.0])
def test_sample_nuclei_of_flat_and_steep_rows(kernels, cuda_dev, v, spread):
    """Top-p (and large k) that keep a few tokens, some thousands, and nearly all."""
    logits = torch.cat([spread * torch.randn(4, v, generator=torch.Generator().manual_seed(v)), sample_logits(4, v)])
    p = [0.05, 0.5, 0.9, 0.999, 0.3, 0.8, 0.99, 0.9999]
    check_sample(kernels, cuda_dev, logits, uniform(8, v), 1.0, 0, p, 0.0)
    check_sample(kernels, cuda_dev, logits, uniform(8, v + 1), 0.6, 0, p, [0.0, 0.01, 0.2, 0.0, 1e-4, 0.5, 0.0, 1e-6])
    check_sample(kernels, cuda_dev, logits, uniform(8, v + 2), 2.0, v // 3, p[::-1], 0.0)
    check_sample(kernels, cuda_dev, logits.repeat(40, 1), uniform(320, v + 3), 1.0, 0, p * 40, 0.0)


@pytest.mark.parametrize("v", [999, 32768, 70000])
def test_sample_equal_logits(kernels, cuda_dev, v):
    """Ties go to the lower index: rows of one value, of few values, and of values that differ in their last bits."""
    flat = torch.zeros(1, v)
    steps = torch.randint(0, 3, (1, v), generator=torch.Generator().manual_seed(3)).float()
    close = 1000 + 2 ** -13 * torch.randint(0, 40, (1, v), generator=torch.Generator().manual_seed(4)).float()
    zeros = torch.where(torch.arange(v)[None] % 2 == 0, -0.0, 0.0)
    logits = torch.cat([flat, steps, close, zeros, torch.full((1, v), -3e38)])
    for setting in ((1.0, 0, 1.0, 0.0), (1.0, 500, 1.0, 0.0), (1.0, 0, 0.37, 0.0), (0.5, 600, 0.9, 0.3), (0.0, 0, 1.0, 0.0),
                    (1e-3, 0, 0.5, 0.0), (1e30, 300, 0.5, 0.0)):
        check_sample(kernels, cuda_dev, logits, uniform(5, v), *setting)


@pytest.mark.parametrize("v", [77, 32768])
def test_sample_masks(kernels, cuda_dev, v):
    """Banned tokens of -inf and of the type's lowest value, rows with one token left, rows with none, NaN and +inf."""
    inf = float("inf")
    base = sample_logits(8, v, seed=5)
    base[0, v // 2:] = -inf
    base[1, : v - 3] = torch.finfo(F32).min
    base[2] = -inf
    base[2, 40] = -7.0
    base[3] = -inf
    base[4, 50], base[4, 60] = inf, inf
    base[5, 70], base[5, 30], base[5, 20] = float("nan"), float("nan"), inf
    base[6] = torch.finfo(F32).min
    base[7] = torch.where(torch.arange(v) % 2 == 0, 3.4e38, -3.4e38)
    for setting in SETTINGS + [(1.0, v - 1, 0.999, 0.0), (1.0, 60, 1.0, 1.0), (1.0, 3, 0.0, 0.0)]:
        check_sample(kernels, cuda_dev, base, uniform(8, v), *setting)


def test_sample_numbers_at_the_ends(kernels, cuda_dev):
    """u of 0, just below 1, 1, beyond and NaN; settings beyond their range, by row."""
    nan = float("nan")
    v = 5000
    logits = sample_logits(1, v).repeat(9, 1)
    u = [0.0, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, nan, 0.5, 0.5, 0.5]
    check_sample(kernels, cuda_dev, logits, u, 1.0, 0, 1.0, 0.0)
    check_sample(kernels, cuda_dev, logits, u, 1.0, 20, 0.9, 0.0)
    check_sample(kernels, cuda_dev, logits, [0.7] * 9, [1.0, -1.0, nan, float("inf"), 1e-38, 1e-45, 3e38, 1.0, 1.0],
                 [-5, 3, 3, 0, 0, 0, 0, 2 ** 31 - 1, v + 1], [1.0, 0.5, 0.5, 1.0, 1.0, 0.5, 0.5, nan, 2.0],
                 [nan, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, -1.0, 5.0])


def test_sample_frequencies(kernels, cuda_dev):
    """Many numbers over one row give every token its share: within 6 standard deviations."""
    v, n = 200, 40000
    row = sample_logits(1, v, seed=9)
    u = (torch.arange(n, device=cuda_dev) + 0.5) / n
    token = kernels.sample_rows(row.to(cuda_dev).expand(n, -1), u, temperature=0.8, top_p=0.9)
    got = torch.bincount(token, minlength=v).cpu().double() / n
    w = torch.softmax(row[0].double() / 0.8, 0)
    s, order = torch.sort(w, descending=True, stable=True)
    s = torch.where(torch.cumsum(s, 0) - s < torch.tensor(0.9).double(), s, 0)
    want = torch.zeros(v, dtype=torch.float64).scatter_(0, order, s / s.sum())
    assert (got - want).abs().max() <= 2.0 / n  # evenly spread numbers: two borders, half a number each


def test_sample_strides_out_and_argmax(kernels, cuda_dev):
    x = sample_logits(40, 3001).to(cuda_dev)
    u = torch.rand(40, device=cuda_dev)
    want = kernels.sample_rows(x, u, top_k=30)
    wide = torch.zeros(40, 4000, device=cuda_dev)
    for pad in (4, 3):
        cut = wide[:, pad:pad + 3001]
        cut.copy_(x)
        assert torch.equal(kernels.sample_rows(cut, u, top_k=30), want)
    out = torch.full((40,), -1, dtype=torch.int64, device=cuda_dev)
    assert kernels.sample_rows(x, u, top_k=30, out=out) is not None and torch.equal(out, want)
    assert torch.equal(kernels.sample_rows(x, u, temperature=0.0), kernels.argmax_rows(x))
    assert torch.equal(kernels.sample_rows(x, u, top_k=1), kernels.argmax_rows(x))
    assert kernels.sample_rows(x[:0], u[:0]).shape == (0,)
    back = torch.flip(u, (0,)).flip(0)[::1]
    assert torch.equal(kernels.sample_rows(x, torch.stack([u, back], 1)[:, 0], top_k=30), want)


def test_sample_captured_and_on_streams(kernels, cuda_dev):
    x = sample_logits(6, 32768).to(cuda_dev)
    u, k = torch.rand(6, device=cuda_dev), torch.tensor([0, 5, 50, 500, 5000, 1], dtype=torch.int32, device=cuda_dev)
    want = [t.clone() for t in kernels.sample_rows(x, u, 0.9, k, 0.95, 0.01, return_prob=True)]
    for _ in range(20):
        assert all(torch.equal(p, q) for p, q in zip(want, kernels.sample_rows(x, u, 0.9, k, 0.95, 0.01, return_prob=True)))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            got = kernels.sample_rows(x, u, 0.9, k, 0.95, 0.01, return_prob=True)
    for _ in range(2):
        got[0].zero_(), got[1].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_sample_offsets_past_32_bits(kernels, cuda_dev):
    v, rows = 70000, 3
    x = sample_logits(rows, v, dtype=BF16).to(cuda_dev)
    u = torch.rand(rows, device=cuda_dev)
    big = torch.empty(2 * 2 ** 31 + 2 ** 20, dtype=BF16, device=cuda_dev)
    far = big.as_strided((rows, v), (2 ** 31 - 8, 1))
    far.copy_(x)
    assert torch.equal(kernels.sample_rows(far, u, 0.9, 40, 0.9), kernels.sample_rows(x, u, 0.9, 40, 0.9))


# ---------------------------------------------------------------------------
# the three together: a small recurrent language model, trained, prompted and stepped
# ---------------------------------------------------------------------------
class Net:
    """Two layers of norm, gates and recurrence, a norm and a head; `ops`: the framework's calls, or the formulas."""

    def __init__(self, dev, dtype, d=64, v=500, seed=0):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g).to(dev, dtype)  # noqa: E731
        self.p = {"emb": r(v, d), "head": r(v, d) / d ** 0.5, "fw": 1 + 0.1 * r(d), "fb": 0.1 * r(d)}
        for i in range(2):
            self.p.update({f"w{i}": 1 + 0.1 * r(d), f"b{i}": 0.1 * r(d), f"in{i}": r(3 * d, d) / d ** 0.5,
                           f"out{i}": r(d, d) / d ** 0.5, f"bias{i}": 2 + r(d)})
        self.d = d

    def forward(self, ops, ids, states=None, lengths=None):
        """ids [batch, L] (or [batch] with states, one token each): logits, and the states behind the prompt."""
        p, d = self.p, self.d
        x, kept = p["emb"][ids], []
        delta = torch.zeros_like(x)
        for i in range(2):
            n, x = ops.norm(delta, p[f"w{i}"], p[f"b{i}"], x)
            rows = n @ p[f"in{i}"].t()
            y, h = ops.rec(rows[..., :d], rows[..., d:2 * d], rows[..., 2 * d:], p[f"bias{i}"],
                           None if states is None else states[i], lengths)
            kept.append(h)
            delta = y @ p[f"out{i}"].t()
        n, _ = ops.norm(delta, p["fw"], p["fb"], x)
        return n @ p["head"].t(), kept


class Ours:
    def __init__(self, sel, step=False):
        self.sel, self.step = sel, step

    def norm(self, x, w, b, r):
        return self.sel.layer_norm(x, w, b, residual=r)

    def rec(self, x, f, z, bias, h, lengths):
        if self.step:
            return self.sel.gated_recurrence_step(h, x, f, z=z, gate_bias=bias), h
        return self.sel.gated_recurrence(x, f, z=z, gate_bias=bias, h0=h, lengths=lengths, return_state=True)


class Formula:
    @staticmethod
    def norm(x, w, b, r):
        s = x + r
        c = s - s.mean(-1, keepdim=True)
        return c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * w + b, s

    @staticmethod
    def rec(x, f, z, bias, h, lengths):
        a, out = torch.sigmoid(f + bias), []
        h = torch.zeros_like(x[:, 0]) if h is None else h
        for t in range(x.shape[1]):
            new = a[:, t] * h + (1 - a[:, t]) * x[:, t]
            h = new if lengths is None else torch.where((t < lengths)[:, None], new, h)
            out.append(new if lengths is None else torch.where((t < lengths)[:, None], new, 0.0))
        return torch.stack(out, 1) * z * torch.sigmoid(z), h


def test_a_training_step_of_all(sel, cuda_dev):
    net, ref64 = Net(cuda_dev, F32), Net(cuda_dev, torch.float64)
    ids = torch.randint(0, 500, (3, 33), generator=torch.Generator().manual_seed(1)).to(cuda_dev)
    lengths = torch.tensor([33, 20, 7], dtype=torch.int32, device=cuda_dev)
    grads = []
    for n, ops in ((net, Ours(sel)), (ref64, Formula())):
        for k in n.p:
            n.p[k] = n.p[k].double().to(n.p[k].dtype).requires_grad_(True)
        logits, _ = n.forward(ops, ids[:, :-1], lengths=lengths - 1)
        lp = torch.log_softmax(logits, -1).gather(2, ids[:, 1:, None])[..., 0]
        live = torch.arange(32, device=cuda_dev)[None] < (lengths - 1)[:, None]
        loss = -(lp * live).sum() / live.sum()
        grads.append(torch.autograd.grad(loss, list(n.p.values())))
    for name, a, b in zip(net.p, *grads):
        # fp32 through two layers and products of 64 terms: each value's error is some hundred roundings of its terms,
        # which the norm of the whole gradient bounds (2^-24 * 1000 = 6e-5); a wrong term would be of order 1
        assert (a.double() - b).norm() <= 1e-3 * b.norm(), name


def test_prompt_steps_and_choices_of_all(sel, kernels, cuda_dev):
    """Tokens chosen step by step from the carried states are those chosen from the whole sequence in 64 bits."""
    net, ref64 = Net(cuda_dev, F32), Net(cuda_dev, torch.float64)
    for k in net.p:
        ref64.p[k] = net.p[k].double()
    prompt = torch.randint(0, 500, (4, 21), generator=torch.Generator().manual_seed(2)).to(cuda_dev)
    u = torch.rand(12, 4, generator=torch.Generator().manual_seed(3)).to(cuda_dev)
    t, k, p = 0.8, 40, 0.95
    with torch.no_grad():
        logits, states = net.forward(Ours(sel), prompt)
        logits, seq = logits[:, -1].contiguous(), prompt
        for i in range(12):
            want64 = ref64.forward(Formula(), seq)[0][:, -1]
            # a hundred roundings per layer on logits of order 1 to 10
            assert (logits.double() - want64).abs().max() < 1e-3
            tok = kernels.sample_rows(logits, u[i], t, k, p)
            for b in range(4):
                want, _, near = ref.sample(logits[b], float(u[i, b]), 0.8, k, 0.95, 0.0)
                assert near < 1e-6 or int(tok[b]) == want  # 0.8 and 0.95 as fp32 numbers move a border by 1e-7
            seq = torch.cat([seq, tok[:, None]], 1)
            logits, states = net.forward(Ours(sel, step=True), tok, states)


def test_integration_example(sel, kernels, cuda_dev):
    """The recurrent layer's calls of INTEGRATION.md as they are written there."""
    import os
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")) as f:
        code = f.read().split("## 1b.")[1].split("```python\n")[2].split("```")[0]
    b, n, d, width = 3, 10, 64, 32
    r = lambda *s: torch.randn(*s, device=cuda_dev)  # noqa: E731
    v = dict(torch=torch, selective=sel, kernels=kernels, d=d, x=r(b, n, width), residual=r(b, n, width), ln_w=r(width),
             ln_b=r(width), w_in=r(3 * d, width), gate_b=r(d) + 2, rows1=r(b, 3 * d), logits=r(b, 500), u=torch.rand(b, device=cuda_dev),
             lengths=torch.tensor([10, 4, 0], dtype=torch.int32, device=cuda_dev))
    exec(code, v)
    for i, e in enumerate((10, 4, 0)):  # the tokens go on from each sequence's own length
        rows = torch.cat([v["rows"][i:i + 1, :e], v["rows1"][i:i + 1, None]], 1)
        want = ref.recurrence(dict(x=rows[..., :d], f=rows[..., d:2 * d], z=rows[..., 2 * d:], bias=v["gate_b"]))
        ref.check(v["s1"][i], tuple(t[0, -1] for t in want["y"]), "s1")
    assert v["tok"].tolist() == [ref.sample(v["logits"][i], float(v["u"][i]), float(torch.tensor(0.8)), 50, 1.0, 0.0)[0] for i in range(b)]

"""The float Mamba operators against their 64-bit formulas (tests/selective_ref.py).

Tolerances.  A result is a sum of terms; each term meets a number of fp32 roundings (2^-24 of the term each) on its way.
Scan: a state passes at most L positions.  A position costs it at most 8: the decay a = 2^x, x = dt A log2(e), is off by
x times the 8 roundings behind x (softplus 5, two products, the constant) plus 4 for ex2 itself, and a (4 + 8 |x|) =
e^-v (4 + 8 v / ln 2 ln 2) <= 4 + 8 / e < 7; the multiply-add is one more.  Around it the inputs, gates and sums over
states and channels cost less than 64, so 8 L + 64 for y and h.  A gradient meets the recurrence twice, and its sums
over batch and positions add at most batch * L roundings: 16 L + 128 + batch * L.
Convolution: 4 taps, bias, SiLU's sigmoid and products: 32; its parameters' sums batch * L more.
Norm: a row's squares are added at most 32 in a thread, then over at most 16 warps and 5 + 15 steps: 64, and 16 around.
"""
import pytest
import torch

import selective_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def sel(cuda_dev):
    from mamba_integer_b200 import selective
    return selective


def scan_inputs(dev, dtype, b, n, d, k, seed=0, D=True, z=True, bias=True, softplus=True, h0=False, lengths=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    a = dict(u=r(b, n, d).to(dtype), A=-(0.2 * r(d, k)).exp() * torch.arange(1, k + 1), B=r(b, n, k).to(dtype),
             C=r(b, n, k).to(dtype), D=r(d) if D else None, z=r(b, n, d).to(dtype) if z else None,
             h0=r(b, d, k) if h0 else None, softplus=softplus)
    if softplus:
        a["delta"] = (r(b, n, d) - (0 if bias else 3)).to(dtype)
        a["bias"] = r(d) - 4 if bias else None
    else:
        a["delta"] = (0.05 * r(b, n, d).exp()).to(dtype)
        a["bias"] = None if not bias else 0.01 * r(d).exp()
    a["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return {key: t.to(dev) if isinstance(t, torch.Tensor) else t for key, t in a.items()}


def call_scan(sel, a, **over):
    a = {**a, **over}
    return sel.selective_scan(a["u"], a["delta"], a["A"], a["B"], a["C"], D=a["D"], z=a["z"], delta_bias=a["bias"],
                              delta_softplus=a["softplus"], h0=a["h0"], lengths=a["lengths"], return_state=True)


def check_scan(y, h, a):
    want, mag = ref.scan(a), ref.scan(a, mag=True)
    units = 8 * a["u"].shape[1] + 64
    ref.check(y, want["y"], mag["y"], units, "y")
    ref.check(h, want["h"], mag["h"], units, "h")


SCAN_SIZES = [
    # batch, L, channels, states: tiles of 16 and 32 positions, blocks of 32 and 64 channels, lanes of 4 states
    (1, 1, 1, 1), (2, 1, 64, 16), (1, 2, 33, 3), (3, 15, 31, 8), (2, 16, 32, 16), (2, 17, 65, 17), (1, 31, 100, 5),
    (2, 33, 64, 24), (1, 64, 40, 32), (2, 65, 24, 33), (1, 40, 17, 64), (2, 127, 8, 16), (1, 128, 96, 16),
    (2, 200, 72, 16), (1, 333, 40, 64), (1, 161, 130, 8),
]


@pytest.mark.parametrize("size", SCAN_SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scan_prompt(sel, cuda_dev, size, dtype):
    a = scan_inputs(cuda_dev, dtype, *size, h0=size[1] % 2 == 1)
    check_scan(*call_scan(sel, a), a)


@pytest.mark.parametrize("D,z,bias,softplus,h0", [(False, False, False, False, False), (True, False, False, True, True),
                                                  (False, True, True, False, True), (False, False, True, True, False)])
def test_scan_options(sel, cuda_dev, D, z, bias, softplus, h0):
    a = scan_inputs(cuda_dev, F32, 2, 37, 48, 16, D=D, z=z, bias=bias, softplus=softplus, h0=h0)
    check_scan(*call_scan(sel, a), a)


@pytest.mark.parametrize("n", [37, 260])
def test_scan_lengths(sel, cuda_dev, n):
    # 0, 1, inside and at a tile's border, past the end (clamped), negative (clamped)
    lens = [0, 1, 16, 20, n, n + 5, -3]
    a = scan_inputs(cuda_dev, BF16, len(lens), n, 40, 16, h0=True, lengths=lens)
    clamped = dict(a, lengths=torch.tensor([min(max(v, 0), n) for v in lens], dtype=torch.int32))
    for name in ("u", "delta", "B", "C", "z"):
        for i, v in enumerate(clamped["lengths"].tolist()):
            a[name][i, v:] = float("nan")  # what lies behind a length is not used
    y, h = call_scan(sel, a)
    check_scan(y, h, clamped)
    for i, v in enumerate(clamped["lengths"].tolist()):
        assert not y[i, v:].any()
    assert torch.equal(h[0], a["h0"][0])


def test_scan_strides_slices_and_broadcasts(sel, cuda_dev):
    b, n, d, k = 3, 70, 48, 16
    a = scan_inputs(cuda_dev, BF16, b, n, d, k)
    want = call_scan(sel, a)
    # columns of wider rows, aligned and not; every other row; sequences expanded from one
    for pad in (8, 3):
        wide = torch.randn(b, 2 * n, 2 * d + pad, device=cuda_dev).to(BF16)
        z = wide[:, ::2, pad:pad + d]
        z.copy_(a["z"])
        rows = torch.randn(b, n, pad + 2 * k, device=cuda_dev).to(BF16)
        B, C = rows[..., pad:pad + k], rows[..., pad + k:]
        B.copy_(a["B"]), C.copy_(a["C"])
        got = call_scan(sel, a, z=z, B=B, C=C)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = {key: a[key][:1] for key in ("u", "delta", "B", "C", "z")}
    spread = call_scan(sel, a, **{key: t.expand(b, -1, -1) for key, t in one.items()})
    copied = call_scan(sel, a, **{key: t.repeat(b, 1, 1) for key, t in one.items()})
    assert torch.equal(spread[0], copied[0]) and torch.equal(spread[1], copied[1])
    # parameters off the 16-byte boundary, and transposed
    flat = torch.empty(d * k + 1, device=cuda_dev)
    A = flat[1:].view(d, k)
    A.copy_(a["A"])
    got = call_scan(sel, a, A=A)
    assert torch.equal(got[0], want[0])
    got = call_scan(sel, a, A=a["A"].t().contiguous().t())
    assert torch.equal(got[0], want[0])


def test_scan_offsets_past_32_bits(sel, cuda_dev):
    n, d, k = 20, 32, 16
    a = scan_inputs(cuda_dev, BF16, 2, n, d, k)
    want = call_scan(sel, a)
    big = torch.empty(2 ** 31 + 64 * n, dtype=BF16, device=cuda_dev)
    far = {}
    for i, key in enumerate(("u", "delta", "z")):
        far[key] = big[i * 8 * d:].as_strided((2, n, d), (2 ** 31 + 3 * d - 2 ** 10, d, 1))
        far[key].copy_(a[key])
        got = call_scan(sel, a, **{key: far[key]})
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_scan_extreme_steps(sel, cuda_dev):
    """A step that forgets the state at once, one that keeps it exactly, softplus far on both sides."""
    a = scan_inputs(cuda_dev, F32, 1, 40, 32, 16, h0=True, bias=False)
    a["delta"][0, ::3] = 60.0
    a["delta"][0, 1::3] = -80.0
    check_scan(*call_scan(sel, a), a)
    a["delta"][0, 5] = float("nan")
    y, h = call_scan(sel, a)
    assert not y[0, :5].isnan().any() and y[0, 5:].isnan().all() and h.isnan().all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [21, 300])
def test_scan_infinite_decays(sel, cuda_dev, n, dtype):
    """States that are forgotten at once: the formula with a large A, also behind a length and in the backward pass."""
    a = scan_inputs(cuda_dev, dtype, 3, n, 40, 16, h0=True, lengths=[n, n - 9, 2])
    large = dict(a, A=a["A"].clone())
    a["A"][:, 3::5], large["A"][:, 3::5] = float("-inf"), -1e12
    a["A"][::7], large["A"][::7] = float("-inf"), -1e12
    check_scan(*call_scan(sel, a), large)
    dy, dh = torch.randn_like(a["u"]), torch.randn(3, 40, 16, device=cuda_dev)
    _, _, got = scan_grads(sel, a, dy, dh)
    # what only such a decay passes on: fp32 decays end at 2^-126 = 1.2e-38, so dh0 = a g and dA = sum a g h dt are at
    # most that many times values of order 10 (and 300 positions of 3 sequences for dA), where the formula has 0
    for name, gone in (("A", a["A"].isinf()), ("h0", a["A"].isinf().expand(3, -1, -1))):
        assert (got[name][gone].abs() < 1e-30).all()
        got[name] = got[name].masked_fill(gone, 0.0)
    check_scan_grads(got, large, dy, dh)
    h = a["h0"].clone()
    y = sel.selective_scan_step(h, a["u"][:, 0], a["delta"][:, 0], a["A"], a["B"][:, 0], a["C"][:, 0], D=a["D"],
                                z=a["z"][:, 0], delta_bias=a["bias"], delta_softplus=True)
    first = {key: large[key][:, :1] for key in ("u", "delta", "B", "C", "z")}
    check_scan(y[:, None], h, dict(large, **first, lengths=None))


def scan_grads(sel, a, dy, dh):
    names = [k for k in ("u", "delta", "A", "B", "C", "D", "z", "bias", "h0") if a[k] is not None]
    leaves = {k: a[k].detach().clone().requires_grad_(True) for k in names}
    y, h = call_scan(sel, a, **leaves)
    outs = [(o, g) for o, g in ((y, dy), (h, dh)) if g is not None]
    got = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)
    return y, h, dict(zip(names, got))


def check_scan_grads(got, a, dy, dh):
    args = dict(a, dy=dy, dh=dh)
    want, mag = ref.scan(args), ref.scan(args, mag=True)
    b, n, _ = a["u"].shape
    for name, t in got.items():
        assert t.dtype == a[name].dtype
        ref.check(t, want["d" + name], mag["d" + name], 16 * n + 128 + b * n, "d" + name)


@pytest.mark.parametrize("size", SCAN_SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scan_gradients(sel, cuda_dev, size, dtype):
    b, n, d, k = size
    a = scan_inputs(cuda_dev, dtype, *size, h0=True)
    g = torch.Generator().manual_seed(5)
    dy = torch.randn(b, n, d, generator=g).to(cuda_dev, dtype)
    dh = torch.randn(b, d, k, generator=g).to(cuda_dev)
    y, h, got = scan_grads(sel, a, dy, dh)
    check_scan(y, h, a)
    check_scan_grads(got, a, dy, dh)


@pytest.mark.parametrize("D,z,bias,softplus", [(False, False, False, False), (True, False, False, True),
                                               (False, True, True, False)])
@pytest.mark.parametrize("only", ["y", "h"])
def test_scan_gradients_of_options(sel, cuda_dev, D, z, bias, softplus, only):
    a = scan_inputs(cuda_dev, F32, 2, 37, 72, 16, D=D, z=z, bias=bias, softplus=softplus)
    dy = torch.randn(2, 37, 72, device=cuda_dev) if only == "y" else None
    dh = torch.randn(2, 72, 16, device=cuda_dev) if only == "h" else None
    _, _, got = scan_grads(sel, a, dy, dh)
    check_scan_grads(got, a, dy, dh)


@pytest.mark.parametrize("n", [37, 260])
def test_scan_gradients_with_lengths(sel, cuda_dev, n):
    lens = [0, 1, 16, 20, n]
    a = scan_inputs(cuda_dev, BF16, len(lens), n, 40, 16, h0=True, lengths=lens)
    dy = torch.randn(len(lens), n, 40, device=cuda_dev).to(BF16)
    dh = torch.randn(len(lens), 40, 16, device=cuda_dev)
    dirty = dict(a)
    for name in ("u", "delta", "B", "C", "z"):
        dirty[name] = a[name].clone()
        for i, v in enumerate(lens):
            dirty[name][i, v:] = float("inf")
    dirty_dy = dy.clone()
    for i, v in enumerate(lens):
        dirty_dy[i, v:] = float("nan")
    _, _, got = scan_grads(sel, dirty, dirty_dy, dh)
    check_scan_grads(got, a, dy, dh)
    for name in ("u", "delta", "B", "C", "z"):
        for i, v in enumerate(lens):
            assert not got[name][i, v:].any()


def test_scan_gradients_follow_differences(sel, cuda_dev):
    """<gradient, v> against a central difference of the operator itself along v."""
    a = scan_inputs(cuda_dev, F32, 2, 24, 32, 16, h0=True)
    dy = torch.randn(2, 24, 32, device=cuda_dev)
    _, _, got = scan_grads(sel, a, dy, torch.zeros(2, 32, 16, device=cuda_dev))
    g = torch.Generator(device=cuda_dev).manual_seed(3)
    # a step of 2^-7 of each value: the curvature gives ~(2^-7)^2 of the slope's terms, rounding 2^-24 * 2^7 of y's
    for name in got:
        v = torch.randn(a[name].shape, generator=g, device=cuda_dev) * a[name].abs()
        up, down = (call_scan(sel, a, **{name: a[name] + s * 2 ** -7 * v})[0].double() for s in (1, -1))
        terms = (up - down) * 2 ** 6 * dy
        assert abs(float((got[name].double() * v).sum() - terms.sum())) <= 2e-2 * float(terms.norm()) + 1e-3, name


def test_scan_gradients_of_shared_inputs(sel, cuda_dev):
    """One leaf for every sequence (expanded), and the same leaf as two inputs: their gradients add up."""
    a = scan_inputs(cuda_dev, F32, 3, 20, 32, 16)
    B = a["B"][:1].clone().requires_grad_(True)
    y, _ = call_scan(sel, a, B=B.expand(3, -1, -1), C=B.expand(3, -1, -1))
    (got,) = torch.autograd.grad(y.sum(), B)  # the gradient of a sum is expanded too
    full = dict(a, B=B.detach().expand(3, -1, -1), C=B.detach().expand(3, -1, -1), dy=torch.ones_like(y))
    want, mag = ref.scan(full), ref.scan(full, mag=True)
    ref.check(got, (want["dB"] + want["dC"]).sum(0, keepdim=True), (mag["dB"] + mag["dC"]).sum(0, keepdim=True),
              16 * 20 + 128 + 60, "shared")


def test_gradients_are_of_first_order(sel, cuda_dev):
    x = torch.randn(4, 8, device=cuda_dev, requires_grad=True)
    w = torch.ones(8, device=cuda_dev, requires_grad=True)
    y, _ = sel.rms_norm(x, w)
    dy = torch.ones_like(y, requires_grad=True)
    (g,) = torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="first order"):
        g.sum().backward()
    c = sel.causal_conv1d(x.unsqueeze(0), torch.ones(8, 4, device=cuda_dev), silu=True)
    torch.autograd.grad(c.sum(), x, create_graph=True)  # one order is there, whatever the mode


def test_scan_repeats_its_bits(sel, cuda_dev):
    a = scan_inputs(cuda_dev, BF16, 2, 300, 96, 16, h0=True)
    dy = torch.randn(2, 300, 96, device=cuda_dev).to(BF16)
    dh = torch.randn(2, 96, 16, device=cuda_dev)
    one, two = (scan_grads(sel, a, dy, dh) for _ in range(2))
    assert torch.equal(one[0], two[0]) and all(torch.equal(one[2][k], two[2][k]) for k in one[2])
    y, h = call_scan(sel, a)  # the form without a backward pass gives the training form's bits
    assert torch.equal(y, one[0]) and torch.equal(h, one[1])


@pytest.mark.parametrize("size", [(1, 1, 1), (3, 33, 5), (5, 64, 16), (2, 100, 24), (4, 32, 64), (70, 17, 33)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scan_step(sel, cuda_dev, size, dtype):
    b, d, k = size
    a = scan_inputs(cuda_dev, dtype, b, 3, d, k, h0=True)
    h = a["h0"].clone()
    rows = torch.empty(b, 3, 2 * d + 1, dtype=dtype, device=cuda_dev)
    z = rows[..., 1:d + 1]
    z.copy_(a["z"])
    ys = [sel.selective_scan_step(h, a["u"][:, t], a["delta"][:, t], a["A"], a["B"][:, t], a["C"][:, t], D=a["D"],
                                  z=z[:, t], delta_bias=a["bias"], delta_softplus=True) for t in range(3)]
    check_scan(torch.stack(ys, 1), h, a)


def test_steps_in_place_are_seen_by_autograd(sel, cuda_dev):
    """A state that a graph has saved and a step then overwrites is an error in that graph's backward pass."""
    h = torch.randn(1, 8, 4, device=cuda_dev)
    w = torch.ones(1, 8, 4, device=cuda_dev, requires_grad=True)
    out = (h * w).sum()  # saves h
    z = lambda *s: torch.randn(*s, device=cuda_dev)  # noqa: E731
    with torch.no_grad():
        sel.selective_scan_step(h, z(1, 8), z(1, 8), -z(8, 4).exp(), z(1, 4), z(1, 4))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


def test_empty_calls(sel, cuda_dev):
    z = lambda *s, dtype=F32: torch.randn(*s, device=cuda_dev).to(dtype)  # noqa: E731
    for b, n in ((0, 5), (2, 0)):
        h0 = z(b, 8, 4).requires_grad_(True)
        y, h = sel.selective_scan(z(b, n, 8), z(b, n, 8), z(8, 4), z(b, n, 4), z(b, n, 4), h0=h0, return_state=True)
        assert y.shape == (b, n, 8) and torch.equal(h, h0)
        (g,) = torch.autograd.grad(h.sum(), h0)
        assert torch.equal(g, torch.ones_like(h0))
        win = z(b, 3, 8)
        y, out = sel.causal_conv1d(z(b, n, 8), z(8, 4), win=win, return_window=True)
        assert y.shape == (b, n, 8) and torch.equal(out, win)
        # all that could have changed the result gets a gradient of zeros
        leaves = [t.requires_grad_(True) for t in (z(b, n, 8), z(b, n, 8), z(8, 4), z(b, n, 4), z(b, n, 4), z(8), z(8))]
        y = sel.selective_scan(*leaves[:5], D=leaves[5], delta_bias=leaves[6])
        assert not any(t.any() for t in torch.autograd.grad(y.sum(), leaves))
        leaves = [t.requires_grad_(True) for t in (z(b, n, 8, dtype=BF16), z(8, 4), z(8))]
        assert not any(t.any() for t in torch.autograd.grad(sel.causal_conv1d(*leaves).sum(), leaves))
    leaves = [t.requires_grad_(True) for t in (z(0, 8, dtype=BF16), z(8), z(0, 8))]
    y, s = sel.rms_norm(leaves[0], leaves[1], residual=leaves[2])
    assert s.dtype == F32 and not any(t.any() for t in torch.autograd.grad(y.sum() + s.sum(), leaves))
    assert sel.selective_scan_step(z(0, 8, 4), z(0, 8), z(0, 8), z(8, 4), z(0, 4), z(0, 4)).shape == (0, 8)
    assert sel.causal_conv1d_step(z(0, 8), z(8, 4), z(0, 3, 8)).shape == (0, 8)
    y, s = sel.rms_norm(z(0, 8), z(8), residual=z(0, 8))
    assert y.shape == s.shape == (0, 8)
    q, scale, s = sel.rms_norm_quant(z(2, 0, 8), z(8))
    assert q.shape == (2, 0, 8) and scale.shape == (2, 0) and s is None


# ---------------------------------------------------------------------------
# convolution
# ---------------------------------------------------------------------------
def conv_inputs(dev, dtype, b, n, d, k, bias=True, silu=True, win=False, lengths=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    a = dict(x=r(b, n, d).to(dtype), w=r(d, k), bias=r(d) if bias else None, silu=silu,
             win=r(b, k - 1, d).to(dtype) if win else None,
             lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32))
    return {key: t.to(dev) if isinstance(t, torch.Tensor) else t for key, t in a.items()}


def call_conv(sel, a, **over):
    a = {**a, **over}
    return sel.causal_conv1d(a["x"], a["w"], bias=a["bias"], silu=a["silu"], win=a["win"], lengths=a["lengths"],
                             return_window=True)


CONV_SIZES = [(1, 1, 1, 4), (2, 2, 5, 4), (3, 3, 64, 4), (1, 16, 8, 2), (2, 17, 33, 3), (2, 19, 128, 4), (1, 130, 36, 4),
              (2, 257, 20, 3), (1, 128, 260, 2)]


@pytest.mark.parametrize("size", CONV_SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("bias,silu,win", [(True, True, True), (False, False, False), (True, False, True)])
def test_conv(sel, cuda_dev, size, dtype, bias, silu, win):
    b, n, d, k = size
    a = conv_inputs(cuda_dev, dtype, *size, bias=bias, silu=silu, win=win)
    g = torch.Generator().manual_seed(9)
    dy = torch.randn(b, n, d, generator=g).to(cuda_dev, dtype)
    dwin = torch.randn(b, k - 1, d, generator=g).to(cuda_dev, dtype) if win else None
    y, out = call_conv(sel, a)
    args = dict(a, dy=dy, dwin=dwin)
    want, mag = ref.conv(args), ref.conv(args, mag=True)
    ref.check(y, want["y"], mag["y"], 32, "y")
    assert torch.equal(out.cpu().double(), want["win"])
    names = [m for m in ("x", "w", "bias", "win") if a[m] is not None]
    leaves = {m: a[m].clone().requires_grad_(True) for m in names}
    y2, out2 = call_conv(sel, a, **leaves)
    assert torch.equal(y2, y)
    got = torch.autograd.grad([y2, out2] if win else [y2], list(leaves.values()), [dy, dwin] if win else [dy])
    for m, t in zip(names, got):
        ref.check(t, want["d" + m], mag["d" + m], 64 + (b * n if m in ("w", "bias") else 0), "d" + m)


@pytest.mark.parametrize("size", [(222, 509, 8, 4), (444, 510, 8, 3), (2, 300, 72, 4)])
def test_conv_gradients_of_long_runs(sel, cuda_dev, size):
    """Runs of 32 and of 64 positions, lengths that end in them, lanes beyond the last channel."""
    b, n, d, k = size
    lens = [(37 * i) % (n + 1) for i in range(b)]
    a = conv_inputs(cuda_dev, BF16, *size, win=True, lengths=lens)
    clean = {key: t.clone() if isinstance(t, torch.Tensor) else t for key, t in a.items()}
    dy = torch.randn(b, n, d, device=cuda_dev).to(BF16)
    dwin = torch.randn(b, k - 1, d, device=cuda_dev).to(BF16)
    for i, v in enumerate(lens):
        a["x"][i, v:] = dy[i, v:] = float("nan")
        clean["x"][i, v:] = 0
    args = dict(clean, dy=dy.nan_to_num(0.0), dwin=dwin)
    want, mag = ref.conv(args), ref.conv(args, mag=True)
    leaves = {m: a[m].clone().requires_grad_(True) for m in ("x", "w", "bias", "win")}
    y, out = call_conv(sel, a, **leaves)
    ref.check(y, want["y"], mag["y"], 32, "y")
    got = torch.autograd.grad([y, out], list(leaves.values()), [dy, dwin])
    for m, t in zip(leaves, got):
        ref.check(t, want["d" + m], mag["d" + m], 64 + (b * n if m in ("w", "bias") else 0), "d" + m)
    assert not any(got[0][i, v:].any() for i, v in enumerate(lens))


@pytest.mark.parametrize("n", [5, 40, 150])
def test_conv_lengths(sel, cuda_dev, n):
    lens = [0, 1, 2, n - 1, n, n + 7, -1]
    a = conv_inputs(cuda_dev, BF16, len(lens), n, 24, 4, win=True, lengths=lens)
    clamped = [min(max(v, 0), n) for v in lens]
    dy = torch.randn(len(lens), n, 24, device=cuda_dev).to(BF16)
    dwin = torch.randn(len(lens), 3, 24, device=cuda_dev).to(BF16)
    clean = dict(a, lengths=torch.tensor(clamped, dtype=torch.int32), dy=dy.clone(), dwin=dwin)
    want, mag = ref.conv(clean), ref.conv(clean, mag=True)
    a["x"] = a["x"].clone()
    for i, v in enumerate(clamped):
        a["x"][i, v:] = float("nan")
        dy[i, v:] = float("nan")
    leaves = {m: a[m].clone().requires_grad_(True) for m in ("x", "w", "bias", "win")}
    y, out = call_conv(sel, a, **leaves)
    got = torch.autograd.grad([y, out], list(leaves.values()), [dy, dwin])
    ref.check(y, want["y"], mag["y"], 32, "y")
    assert torch.equal(out.cpu().double(), want["win"])
    for m, t in zip(leaves, got):
        ref.check(t, want["d" + m], mag["d" + m], 64 + (len(lens) * n if m in ("w", "bias") else 0), "d" + m)


def test_conv_strides_and_weight_forms(sel, cuda_dev):
    a = conv_inputs(cuda_dev, BF16, 2, 50, 40, 4)
    want, win = call_conv(sel, a)
    for pad in (8, 1):
        wide = torch.zeros(2, 100, 80 + pad, dtype=BF16, device=cuda_dev)
        x = wide[:, ::2, pad:pad + 40]
        x.copy_(a["x"])
        got = call_conv(sel, a, x=x)
        assert torch.equal(got[0], want) and torch.equal(got[1], win)
    got = call_conv(sel, a, w=a["w"].unsqueeze(1))
    assert torch.equal(got[0], want)
    big = torch.empty(2 ** 31 + 4096, dtype=BF16, device=cuda_dev)
    far = big.as_strided((2, 50, 40), (2 ** 31 - 1024, 40, 1))
    far.copy_(a["x"])
    got = call_conv(sel, a, x=far)
    assert torch.equal(got[0], want)
    x = a["x"][:1].clone().requires_grad_(True)  # one sequence for both, and an expanded gradient
    (g,) = torch.autograd.grad(call_conv(sel, a, x=x.expand(2, -1, -1))[0].sum(), x)
    one = dict(a, x=x.detach(), dy=torch.ones(1, 50, 40, device=cuda_dev))
    r, m = ref.conv(one), ref.conv(one, mag=True)
    # two rounded halves and their rounded sum
    assert ((g.cpu().double() - 2 * r["dx"]).abs() <= 2 ** -8 * 4 * r["dx"].abs() + 2 ** -24 * 200 * m["dx"]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d,k,silu", [(1, 2, True), (33, 3, False), (64, 4, True), (1030, 4, True)])
def test_conv_step(sel, cuda_dev, dtype, d, k, silu):
    a = conv_inputs(cuda_dev, dtype, 3, 5, d, k, silu=silu, win=True)
    win = a["win"].clone()
    ys = [sel.causal_conv1d_step(a["x"][:, t], a["w"], win, bias=a["bias"], silu=silu) for t in range(5)]
    y, out = call_conv(sel, a)
    assert torch.equal(torch.stack(ys, 1), y) and torch.equal(win, out)


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------
NORM_SIZES = [(1, 1), (3, 7), (2, 32), (5, 100), (9, 256), (4, 768), (3, 1000), (2, 1025), (1, 2048), (2, 4096), (3, 8191),
              (1, 16384), (700, 264), (2500, 40), (1250, 1032), (900, 4104)]  # the last: several rows a warp, or block


@pytest.mark.parametrize("size", NORM_SIZES)
@pytest.mark.parametrize("dtype,rdtype", [(F32, None), (F32, F32), (BF16, None), (BF16, BF16), (BF16, F32), (F16, F16),
                                          (F16, F32)])
def test_norm(sel, cuda_dev, size, dtype, rdtype):
    T, d = size
    g = torch.Generator().manual_seed(T + d)
    r = lambda *s: torch.randn(*s, generator=g).to(cuda_dev)  # noqa: E731
    x, w = r(T, d).to(dtype).requires_grad_(True), (1 + 0.3 * r(d)).requires_grad_(True)
    res = None if rdtype is None else (2 * r(T, d)).to(rdtype).requires_grad_(True)
    dy, ds = r(T, d).to(dtype), None if rdtype is None else r(T, d).to(rdtype)
    y, s = sel.rms_norm(x, w, eps=1e-5, residual=res)
    kept = x.detach() if res is None else (x.detach().float() + res.detach().float()).to(rdtype)
    assert s is None if res is None else torch.equal(s, kept)
    want = ref.norm(kept, w, 1e-5, dy, ds)
    ref.check(y, want["y"], want["y"].abs(), 80, "y")
    outs = ([y], [dy]) if res is None else ([y, s], [dy, ds])
    got = torch.autograd.grad(outs[0], [x, w] + ([] if res is None else [res]), outs[1])
    assert all(t.dtype == o.dtype for t, o in zip(got, [x, w, res]))
    ref.check(got[0], want["ds"], want["ds_mag"], 200, "dx")
    ref.check(got[1], want["dw"], want["dw_mag"], 100 + T, "dw")
    if res is not None:
        ref.check(got[2], want["ds"], want["ds_mag"], 200, "dresidual")
    with torch.no_grad():
        y2, s2 = sel.rms_norm(x, w, eps=1e-5, residual=res)
        assert torch.equal(y, y2)
        # the int8 form: the scale is max|y| / 127, a value half a step off at most
        q, scale, s3 = sel.rms_norm_quant(x, w, eps=1e-5, residual=res)
    assert s3 is None if res is None else torch.equal(s3, kept)
    most = want["y"].abs().amax(1)
    assert ((scale.cpu().double() - most.clamp(min=1e-8) / 127).abs() <= 82 * 2 ** -24 * most / 127 + 1e-12).all()
    off = (q.cpu().double() * scale.cpu().double()[:, None] - want["y"]).abs()
    assert (off <= scale.cpu().double()[:, None] * (0.5 + 127 * 90 * 2 ** -24)).all()
    assert int(q.abs().max()) <= 127


def test_norm_strides_zeros_and_infinities(sel, cuda_dev):
    wide = torch.randn(6, 2, 300, device=cuda_dev).to(BF16)
    w = torch.randn(96, device=cuda_dev)
    for x in (wide[:, 0, :96], wide[:, 1, 3:99], wide[:1, 0, :96].expand(4, -1), wide[..., 8:104]):
        y, _ = sel.rms_norm(x, w)
        y2, _ = sel.rms_norm(x.contiguous(), w)
        assert y.shape == x.shape and torch.equal(y, y2)
    lead = torch.randn(96, device=cuda_dev)
    y, s = sel.rms_norm(lead, w, residual=lead)
    assert y.shape == (96,) and torch.equal(s, 2 * lead)
    x = torch.zeros(3, 96, device=cuda_dev)
    x[1] = 1e30  # its square is infinite: the norm is 0, as the formula says in 32 bits
    x[2, 5] = float("nan")
    y, _ = sel.rms_norm(x, w)
    assert not y[0].any() and not y[1].any() and y[2].isnan().all()
    q, scale, _ = sel.rms_norm_quant(x[:2], w)
    assert not q.any() and torch.equal(scale.cpu(), torch.full((2,), 1e-8) / 127)  # a true division
    x2 = wide[:, 0, :96].float().requires_grad_(True)  # a strided row, an expanded gradient, one gradient of two
    _, s = sel.rms_norm(x2, w, residual=x2)
    (g,) = torch.autograd.grad(s.sum(), x2)
    assert torch.equal(g, torch.full_like(x2, 2))


def test_norm_quant_gives_the_rows_of_quantize_rows(sel, cuda_dev):
    """Bit for bit from the fp32 norm, rows with infinities and NaN (no value of theirs is kept) too."""
    from mamba_integer_b200 import kernels
    x, w = 3 * torch.randn(3000, 200, device=cuda_dev), torch.randn(200, device=cuda_dev)
    x[5, 7], x[6, 199] = float("nan"), float("inf")
    x[7] = 0
    y, _ = sel.rms_norm(x, w)
    one = torch.ones(200, device=cuda_dev)
    q, scale, _ = sel.rms_norm_quant(x, w)
    want, wscale = kernels.quantize_rows(y[:8])
    assert torch.equal(q[:8], want[:, :200]) and torch.equal(scale[:8].isnan(), wscale.isnan())
    fine = ~wscale.isnan()
    assert torch.equal(scale[:8][fine], wscale[fine])
    want, wscale = kernels.quantize_rows(y[10:])
    assert torch.equal(q[10:], want[:, :200]) and torch.equal(scale[10:], wscale)
    # infinite values of the norm itself: an infinite weight
    one[4] = float("inf")
    y, _ = sel.rms_norm(x[10:], one)
    q, scale, _ = sel.rms_norm_quant(x[10:], one)
    want, wscale = kernels.quantize_rows(y)
    assert torch.equal(q, want[:, :200]) and torch.equal(scale, wscale)


def test_norm_quant_feeds_the_ternary_product(sel, cuda_dev):
    from mamba_integer_b200 import kernels, synth
    from mamba_integer_b200.rational_bitnet import BitLinear
    g = torch.Generator().manual_seed(0)
    lin = BitLinear(256, 128)
    lin.weight.data.copy_(synth.ternary_weight(128, 256, g))
    lin = lin.to(cuda_dev)
    x, r = (torch.randn(37, 256, generator=g).to(cuda_dev) for _ in range(2))
    w = torch.ones(256, device=cuda_dev)
    q, scale, s = sel.rms_norm_quant(x, w, residual=r)
    tw = lin.device_weights(cuda_dev)
    got = kernels.bitlinear_packed(q, tw.w2, scale, tw.scale)
    with torch.no_grad():
        y, _ = sel.rms_norm(x, w, residual=r)
        assert torch.equal(got, lin(y))  # quantising the fp32 rows apart gives the same int8 rows


# ---------------------------------------------------------------------------
# together, on other streams, in graphs
# ---------------------------------------------------------------------------
class FloatLayer(torch.nn.Module):
    """norm, input projection, convolution, scan, output projection: a float Mamba layer as a user writes it."""

    def __init__(self, d=48, k=16, R=6, taps=4, seed=0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        p = lambda *s, scale=1.0: torch.nn.Parameter(torch.randn(*s, generator=g) * scale)  # noqa: E731
        di = 2 * d
        self.di, self.k, self.R = di, k, R
        self.norm_w = torch.nn.Parameter(torch.ones(d))
        self.w_in, self.w_x = p(2 * di, d, scale=d ** -0.5), p(R + 2 * k, di, scale=di ** -0.5)
        self.w_dt, self.w_out = p(di, R, scale=R ** -0.5), p(d, di, scale=di ** -0.5)
        self.conv_w, self.conv_b = p(di, taps, scale=0.5), p(di, scale=0.1)
        self.A = torch.nn.Parameter(-torch.arange(1, k + 1).float().repeat(di, 1))
        self.D, self.dt_bias = torch.nn.Parameter(torch.ones(di)), torch.nn.Parameter(torch.full((di,), -3.0))

    def forward(self, sel, x, residual, win=None, h0=None):
        F = torch.nn.functional
        y, residual = sel.rms_norm(x, self.norm_w, residual=residual)
        xz = F.linear(y, self.w_in)
        c, win = sel.causal_conv1d(xz[..., :self.di], self.conv_w, bias=self.conv_b, silu=True, win=win,
                                   return_window=True)
        xp = F.linear(c, self.w_x)
        delta = F.linear(xp[..., :self.R], self.w_dt)
        s, h = sel.selective_scan(c, delta, self.A, xp[..., self.R:self.R + self.k], xp[..., self.R + self.k:], D=self.D,
                                  z=xz[..., self.di:], delta_bias=self.dt_bias, delta_softplus=True, h0=h0,
                                  return_state=True)
        return F.linear(s, self.w_out), residual, win, h

    def step(self, sel, x, residual, win, h):
        F = torch.nn.functional
        y, residual = sel.rms_norm(x, self.norm_w, residual=residual)
        xz = F.linear(y, self.w_in)
        c = sel.causal_conv1d_step(xz[:, :self.di], self.conv_w, win, bias=self.conv_b, silu=True)
        xp = F.linear(c, self.w_x)
        delta = F.linear(xp[:, :self.R], self.w_dt)
        s = sel.selective_scan_step(h, c, delta, self.A, xp[:, self.R:self.R + self.k], xp[:, self.R + self.k:], D=self.D,
                                    z=xz[:, self.di:], delta_bias=self.dt_bias, delta_softplus=True)
        return F.linear(s, self.w_out), residual

    def plain(self, x, residual):
        """the same in torch, for 64 bits"""
        F = torch.nn.functional
        residual = residual + x
        y = residual / torch.sqrt((residual ** 2).mean(-1, keepdim=True) + 1e-6) * self.norm_w
        xz = F.linear(y, self.w_in)
        n, taps = x.shape[1], self.conv_w.shape[1]
        rows = F.pad(xz[..., :self.di], (0, 0, taps - 1, 0))
        c = F.silu(sum(rows[:, i:i + n] * self.conv_w[:, i] for i in range(taps)) + self.conv_b)
        xp = F.linear(c, self.w_x)
        dt = F.softplus(F.linear(xp[..., :self.R], self.w_dt) + self.dt_bias)
        B, C = xp[..., self.R:self.R + self.k], xp[..., self.R + self.k:]
        h, out = torch.zeros(x.shape[0], self.di, self.k, dtype=x.dtype, device=x.device), []
        for t in range(n):
            h = torch.exp(dt[:, t, :, None] * self.A) * h + (dt[:, t] * c[:, t])[..., None] * B[:, t, None]
            out.append((h * C[:, t, None]).sum(-1) + self.D * c[:, t])
        return F.linear(torch.stack(out, 1) * F.silu(xz[..., self.di:]), self.w_out), residual


@pytest.fixture
def exact_products(cuda_dev):
    kept = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = kept


def test_layer_forward_and_gradients(sel, cuda_dev, exact_products):
    layer = FloatLayer().to(cuda_dev)
    x, r = (torch.randn(2, 45, 48, device=cuda_dev).requires_grad_(True) for _ in range(2))
    y, res, _, _ = layer(sel, x, r)
    g, gr = torch.randn_like(y), torch.randn_like(res)
    leaves = [x, r, *layer.parameters()]
    got = torch.autograd.grad([y, res], leaves, [g, gr])
    exact = FloatLayer().double().to(cuda_dev)
    xd, rd = (t.detach().double().requires_grad_(True) for t in (x, r))
    yd, resd = exact.plain(xd, rd)
    want = torch.autograd.grad([yd, resd], [xd, rd, *exact.parameters()], [g.double(), gr.double()])
    # five products and three operators in a row, each within 1e-6 of what enters it in the 2-norm, gains of order 10
    for a, b in [(y.detach(), yd.detach()), (res.detach(), resd.detach()), *zip(got, want)]:
        assert float((a.double() - b).norm()) <= 1e-4 * float(b.norm())


def test_layer_prompt_then_tokens(sel, cuda_dev, exact_products):
    layer = FloatLayer().to(cuda_dev)
    x, r = (torch.randn(3, 24, 48, device=cuda_dev) for _ in range(2))
    with torch.no_grad():
        whole, res, win_w, h_w = layer(sel, x, r)
        y, _, win, h = layer(sel, x[:, :17], r[:, :17])
        parts = [y]
        y, _, win, h = layer(sel, x[:, 17:20], r[:, 17:20], win=win, h0=h)
        parts.append(y)
        for t in range(20, 24):
            y, _ = layer.step(sel, x[:, t], r[:, t], win, h)
            parts.append(y.unsqueeze(1))
    got = torch.cat(parts, 1)
    # the products of other shapes round differently: 1e-6 of the rows' norm through three operators
    assert float((got - whole).norm()) <= 2e-5 * float(whole.norm())
    assert float((h - h_w).norm()) <= 2e-5 * float(h_w.norm())
    assert float((win - win_w).norm()) <= 2e-5 * float(win_w.norm())


def test_other_stream(sel, cuda_dev):
    a = scan_inputs(cuda_dev, BF16, 2, 300, 64, 16)
    dy = torch.randn(2, 300, 64, device=cuda_dev).to(BF16)
    want = scan_grads(sel, a, dy, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = scan_grads(sel, a, dy, None)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and all(torch.equal(got[2][k], want[2][k]) for k in want[2])


def _capture(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fn()
    return g, out


def test_graphs_of_prompts_and_training_steps(sel, cuda_dev):
    """Two graphs of different sizes, replayed in turn on new values: each keeps its own workspaces."""
    made = []
    for seed, size in ((0, (1, 320, 64, 16)), (1, (2, 150, 40, 24))):
        a = scan_inputs(cuda_dev, F32, *size, seed=seed, h0=True)
        dy = torch.randn(*a["u"].shape, device=cuda_dev)
        leaves = {k: a[k].requires_grad_(True) for k in ("u", "A", "B", "h0")}

        def train(a=a, dy=dy, leaves=leaves):
            y, h = call_scan(sel, a)
            grads = torch.autograd.grad(y, list(leaves.values()), dy)
            return y.detach(), grads  # no autograd graph outlives the call
        made.append((a, dy, train, *_capture(train)))
    for round_ in range(2):
        for a, dy, train, graph, out in made:
            with torch.no_grad():
                a["u"].copy_(torch.randn_like(a["u"]))
                a["h0"].mul_(0.5)
        for a, dy, train, graph, out in made:
            graph.replay()
        torch.cuda.synchronize()
        for a, dy, train, graph, out in made:
            y, grads = train()
            assert torch.equal(y, out[0]) and all(torch.equal(p, q) for p, q in zip(grads, out[1]))


def test_capture_beside_an_eager_graph_is_refused(sel, cuda_dev):
    """The leaves' gradients would be added on the default stream, which a capture cannot join."""
    x, w = torch.randn(1, 9, 8, device=cuda_dev), torch.randn(8, device=cuda_dev, requires_grad=True)
    taps = torch.randn(8, 4, device=cuda_dev, requires_grad=True)
    A = torch.randn(8, 4, device=cuda_dev, requires_grad=True)
    calls = {"norm": lambda: sel.rms_norm(x, w)[0], "conv": lambda: sel.causal_conv1d(x, taps * 2),
             "scan": lambda: sel.selective_scan(x, x, A, x[..., :4], x[..., :4])}
    for call in calls.values():
        call()
        alive = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = x * 2  # a graph is not empty
            with pytest.raises(RuntimeError, match="autograd graph made on the default stream is alive"):
                call()
            with torch.no_grad():
                y = call()
        graph.replay()
        assert torch.equal(y, alive) and torch.equal(kept, x * 2)


def test_many_streams(sel, cuda_dev):
    """Steps have no limit of 65535 streams."""
    b = 65537
    a = scan_inputs(cuda_dev, F32, 1, 1, 3, 4, h0=True)
    step = {k: a[k][:, 0].expand(b, -1).contiguous() for k in ("u", "delta", "B", "C")}
    h = a["h0"].expand(b, -1, -1).contiguous()
    y = sel.selective_scan_step(h, step["u"], step["delta"], a["A"], step["B"], step["C"])
    assert torch.equal(y, y[:1].expand(b, -1)) and torch.equal(h, h[:1].expand(b, -1, -1))
    assert not torch.equal(h[:1], a["h0"])
    win = torch.zeros(b, 3, 3, device=cuda_dev)
    taps = torch.ones(3, 4, device=cuda_dev)
    assert torch.equal(sel.causal_conv1d_step(step["u"], taps, win), step["u"])
    assert torch.equal(win[:, 2], step["u"]) and not win[:, :2].any()


def test_graph_of_decode_steps(sel, cuda_dev):
    a = scan_inputs(cuda_dev, BF16, 5, 6, 64, 16, h0=True)
    c = conv_inputs(cuda_dev, BF16, 5, 6, 64, 4, win=True)
    w = torch.randn(64, device=cuda_dev)
    x, h, win = a["u"][:, 0].clone(), a["h0"].clone(), c["win"].clone()

    def token():
        q, scale, _ = sel.rms_norm_quant(x, w, residual=x)
        y = sel.causal_conv1d_step(x, c["w"], win, bias=c["bias"], silu=True)
        return q, scale, y, sel.selective_scan_step(h, y, a["delta"][:, 0], a["A"], a["B"][:, 0], a["C"][:, 0], D=a["D"],
                                                    delta_bias=a["bias"], delta_softplus=True)
    graph, out = _capture(token)
    h.copy_(a["h0"]), win.copy_(c["win"])
    got = []
    for t in range(6):
        x.copy_(a["u"][:, t])
        graph.replay()
        got.append([o.clone() for o in out])
    h2, win2 = h.clone(), win.clone()
    h.copy_(a["h0"]), win.copy_(c["win"])
    for t in range(6):
        x.copy_(a["u"][:, t])
        assert all(torch.equal(p, q) for p, q in zip(token(), got[t]))
    assert torch.equal(h, h2) and torch.equal(win, win2)


# ---------------------------------------------------------------------------
# second order, values that are not finite, the variants that only large calls take
# ---------------------------------------------------------------------------
def test_gradients_of_gradients_are_refused(sel, cuda_dev):
    """Under create_graph every gradient refuses a second pass, whatever the incoming one; without it none has a graph."""
    z = lambda *s: torch.randn(*s, device=cuda_dev).requires_grad_(True)  # noqa: E731
    x, w, A, B = z(2, 9, 8), z(8), z(8, 4), z(2, 9, 4)
    calls = {"norm": (lambda: sel.rms_norm(x, w)[0], [x, w]),
             "residual": (lambda: sel.rms_norm(x, w, residual=x * 2)[0], [x, w]),
             "conv": (lambda: sel.causal_conv1d(x, A, bias=w, silu=True), [x, A, w]),
             "scan": (lambda: sel.selective_scan(x, x, A, B, B, D=w, z=x, delta_softplus=True), [x, A, B, w])}
    for name, (call, leaves) in calls.items():
        got = torch.autograd.grad(call().sum(), leaves, create_graph=True)
        for g in got:
            assert g.requires_grad, name
            with pytest.raises(RuntimeError, match="first order"):
                g.sum().backward(retain_graph=True)
        y = call()
        plain = torch.autograd.grad(y, leaves, torch.ones_like(y).requires_grad_(True))
        assert not any(g.requires_grad for g in plain), name
        assert all(torch.equal(g, p) for g, p in zip(got, plain)), name
    # beside another way to the leaf too: the term is not left out
    y, _ = sel.rms_norm(x, w)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="first order"):
        torch.autograd.grad(y.sum() + (g * g).sum(), x)
    # the sum alone is linear: its gradient may be differentiated
    _, s = sel.rms_norm(x, w, residual=x * 2)
    (g,) = torch.autograd.grad((s * s).sum(), x, create_graph=True)
    (gg,) = torch.autograd.grad(g.sum(), x)
    assert torch.equal(gg, torch.full_like(x, 18))


def same_infinities(got, want, name):
    """Where the formula has no finite value the result is the same; elsewhere it is finite."""
    got, odd = got.detach().cpu().double(), want.isinf()
    assert torch.equal(got.isnan(), want.isnan()), (name, int(got.isnan().sum()), int(want.isnan().sum()))
    assert torch.equal(got[odd], want[odd]) and got[want.isfinite()].isfinite().all(), name


def infinite_inputs(dev, dtype, n, k):
    """Inputs whose formula has infinities and, in y, no NaN; no single decay leaves the range of fp32."""
    a = scan_inputs(dev, dtype, 3, n, 40, k, h0=True)
    for name in ("B", "C", "D"):
        a[name] = a[name].abs() + 0.125
    a["A"] *= 2 / k
    a["u"][0, 7, 3] = float("inf")
    a["delta"][1, 9, 5], a["u"][1, 9, 5] = float("inf"), 1.0
    return a


INFINITE = [(k, n, dtype) for k in (1, 5, 16, 20, 24, 33) for n in (20,) for dtype in (F32, BF16)]


@pytest.mark.parametrize("k,n,dtype", INFINITE)
def test_scan_infinite_inputs(sel, cuda_dev, k, n, dtype):
    """States that only fill a lane up are reached by an infinite input or step size, and stay 0."""
    a = infinite_inputs(cuda_dev, dtype, n, k)
    want = ref.scan(a)
    assert not want["y"].isnan().any() and want["y"][0, 7:, 3].isinf().all() and want["y"][1, 9:, 5].isinf().all()
    y, h = call_scan(sel, a)
    same_infinities(y, want["y"], "y")
    same_infinities(h, want["h"], "h")
    h, ys = a["h0"].clone(), []
    for t in range(11):  # one token at a time
        ys.append(sel.selective_scan_step(h, a["u"][:, t], a["delta"][:, t], a["A"], a["B"][:, t], a["C"][:, t], D=a["D"],
                                          z=a["z"][:, t], delta_bias=a["bias"], delta_softplus=True))
    same_infinities(torch.stack(ys, 1), want["y"][:, :11], "steps")


@pytest.mark.parametrize("k,n,dtype", INFINITE)
def test_scan_infinite_gradients(sel, cuda_dev, k, n, dtype):
    a = infinite_inputs(cuda_dev, dtype, n, k)
    a["u"][0, 7, 3], a["delta"][1, 9, 5] = 1.0, 0.5
    g = torch.Generator().manual_seed(1)
    dy, dh = torch.randn(3, n, 40, generator=g).to(cuda_dev, dtype), torch.randn(3, 40, k, generator=g).to(cuda_dev)
    dy[0, 12, 4] = float("inf")
    _, _, got = scan_grads(sel, a, dy, dh)
    want = ref.scan(dict(a, dy=dy, dh=dh))
    for name, t in got.items():
        same_infinities(t, want["d" + name], "d" + name)


@pytest.mark.parametrize("k", [1, 5, 16])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [20, 300])
def test_scan_nan_steps_reach_the_gradients(sel, cuda_dev, n, dtype, k):
    """A step size that is NaN makes the same gradients NaN as in the formula, those of earlier positions among them."""
    a = scan_inputs(cuda_dev, dtype, 2, n, 40, k, h0=True)
    a["delta"][0, 9, 5] = float("nan")
    dy, dh = torch.randn(2, n, 40, device=cuda_dev).to(dtype), torch.randn(2, 40, k, device=cuda_dev)
    y, h, got = scan_grads(sel, a, dy, dh)
    want = ref.scan(dict(a, dy=dy, dh=dh))
    assert want["dh0"][0, 5].isnan().all() and not want["dD"].isnan().any()
    for name, t in dict(got, y=y, h=h).items():
        same_infinities(t, want[name if name in ("y", "h") else "d" + name], name)



@pytest.mark.parametrize("lengths", [None, [20, 13, 17]])
@pytest.mark.parametrize("k,n,dtype", INFINITE)
def test_scan_gradients_of_infinite_states(sel, cuda_dev, k, n, dtype, lengths):
    """Positions behind the end, whose step size is 0, add nothing to dA, also where the state is infinite."""
    a = infinite_inputs(cuda_dev, dtype, n, k)
    a["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda_dev)
    g = torch.Generator().manual_seed(1)
    # gradients of one sign: the formula's dA is an infinity for the infinite input, and NaN for the infinite step
    dy, dh = torch.rand(3, n, 40, generator=g).to(cuda_dev, dtype), torch.rand(3, 40, k, generator=g).to(cuda_dev)
    a["z"] = a["z"].abs()
    _, _, got = scan_grads(sel, a, dy, dh)
    want = ref.scan(dict(a, dy=dy, dh=dh))
    assert want["dA"][3].isinf().all()
    for name, t in got.items():
        same_infinities(t, want["d" + name], "d" + name)


@pytest.mark.parametrize("k,dtype", [(k, dtype) for k in (1, 16, 20) for dtype in (F32, BF16)])
def test_scan_infinities_over_chunks(sel, cuda_dev, k, dtype):
    """An infinite state, and an infinite gradient, stay infinite over chunks whose decay as a whole is 0 in fp32."""
    n = 300
    a = infinite_inputs(cuda_dev, dtype, n, k)
    a["A"] *= 4
    a["delta"] += 2
    want = ref.scan(a)
    y, h = call_scan(sel, a)
    same_infinities(y, want["y"], "y")
    same_infinities(h, want["h"], "h")
    a["u"][0, 7, 3], a["delta"][1, 9, 5] = 1.0, 0.5
    g = torch.Generator().manual_seed(1)
    dy, dh = torch.randn(3, n, 40, generator=g).to(cuda_dev, dtype), torch.randn(3, 40, k, generator=g).to(cuda_dev)
    dy[0, 290, 4] = float("inf")
    _, _, got = scan_grads(sel, a, dy, dh)
    want = ref.scan(dict(a, dy=dy, dh=dh))
    same_infinities(got["u"], want["du"], "du")
    same_infinities(got["h0"], want["dh0"], "dh0")


def test_scan_growth_over_chunks(sel, cuda_dev):
    """Growing states: a chunk's growth leaves the range of fp32, the states do not, being 0 there."""
    n = 2048
    a = scan_inputs(cuda_dev, F32, 1, n, 8, 16, softplus=False, bias=False, z=False)
    a["A"] = a["A"].abs().clamp(0.5, 1.0)
    a["delta"].fill_(2.0)
    a["u"][:, :n - 20] = 0
    dy = torch.randn(1, n, 8, device=cuda_dev)
    dy[:, 20:] = 0
    y, h, got = scan_grads(sel, a, dy, None)
    args = dict(a, dy=dy)
    want, mag = ref.scan(args), ref.scan(args, mag=True)
    # a factor e^2 = 2^2.9 has 4 + 8 * 2.9 roundings, the step one more; 20 positions and what lies around them; twice for gradients
    ref.check(y, want["y"], mag["y"], 28 * 20 + 64, "y")
    ref.check(h, want["h"], mag["h"], 28 * 20 + 64, "h")
    for name, t in got.items():
        ref.check(t, want["d" + name], mag["d" + name], 2 * (28 * 20 + 64) + n, "d" + name)


@pytest.mark.parametrize("softplus,sign", [(False, 1), (False, -1), (True, 1)])
def test_scan_growth_to_the_end_of_fp32(sel, cuda_dev, softplus, sign):
    """Factors between 2^126 and 2^128, and one beyond, which ends in an infinity or next to it."""
    a = scan_inputs(cuda_dev, F32, 1, 1, 8, 16, softplus=softplus, bias=False, z=False, h0=True)
    a["A"] = sign * torch.ones(8, 16, device=cuda_dev)
    a["delta"].fill_(sign * 88.0)
    a["C"] *= 2.0 ** -10
    a["h0"] = a["h0"].clamp(-1, 1)
    dh = torch.randn(1, 8, 16, device=cuda_dev).clamp(-1, 1)
    y, h, got = scan_grads(sel, a, None, dh)
    args = dict(a, dh=dh)
    want, mag = ref.scan(args), ref.scan(args, mag=True)
    # the factor: x = 127, 4 + 8 * 127 roundings; 64 around it
    ref.check(h, want["h"], mag["h"], 1100, "h")
    ref.check(y, want["y"], mag["y"], 1100, "y")
    ref.check(got["h0"], want["dh0"], mag["dh0"], 1100, "dh0")
    a["delta"][:] = sign * 200.0
    a["h0"] = a["h0"].sign() * 2
    h = call_scan(sel, a)[1]
    assert torch.equal(h, a["h0"] * float("inf"))
    if not softplus:  # the other way, what is left is the input's part
        a["delta"][:] = sign * -200.0
        h = call_scan(sel, a)[1]
        want, mag = ref.scan(a), ref.scan(a, mag=True)
        ref.check(h, want["h"], mag["h"], 64, "h")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("d", [24, 21])
@pytest.mark.parametrize("n", [33, 160])
def test_conv_infinite_weights_behind_lengths(sel, cuda_dev, n, d, silu, dtype):
    """What lies behind a length has gradients of 0 and adds nothing to others, also where a weight is infinite or NaN."""
    lens = [0, 1, 7, 30, n]
    a = conv_inputs(cuda_dev, dtype, 5, n, d, 4, silu=silu, win=True, lengths=lens)
    a["w"][3, 1], a["w"][5, 0], a["w"][5, 3] = float("inf"), float("nan"), float("-inf")
    leaves = {m: a[m].clone().requires_grad_(True) for m in ("x", "w", "bias", "win")}
    y, out = call_conv(sel, a, **leaves)
    for given in ((y,), (out,), (y, out)):
        grads = [torch.randn_like(t) for t in given]
        dx, dwin = torch.autograd.grad(given, [leaves["x"], leaves["win"]], grads, retain_graph=True)
        for i, v in enumerate(lens):
            assert not y[i, v:].any() and not dx[i, v:].any()
        assert torch.equal(dwin[0], torch.zeros_like(dwin[0]) if given[-1] is y else grads[-1][0])  # the empty sequence's


@pytest.mark.parametrize("size", [(600, 33, 40, 16), (300, 20, 72, 13), (592, 49, 64, 9)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scan_two_channels_a_lane(sel, cuda_dev, size, dtype):
    """From 592 CTAs of 64 channels on, a lane of a scan of 9 to 16 states carries two channels."""
    b, n, d, k = size
    assert b * -(-d // 64) >= 592
    lens = [(7 * i) % (n + 1) for i in range(b)]
    a = scan_inputs(cuda_dev, dtype, *size, h0=True, lengths=lens)
    g = torch.Generator().manual_seed(5)
    dy, dh = torch.randn(b, n, d, generator=g).to(cuda_dev, dtype), torch.randn(b, d, k, generator=g).to(cuda_dev)
    y, h, got = scan_grads(sel, a, dy, dh)
    check_scan(y, h, a)
    check_scan_grads(got, a, dy, dh)
    y2, h2 = call_scan(sel, a)
    assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.parametrize("b,k,lanes", [(8193, 8, 2), (4099, 16, 4), (2051, 24, 8), (2050, 32, 8), (1027, 64, 16),
                                       (1029, 44, 16)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scan_step_of_many_streams(sel, cuda_dev, b, k, lanes, dtype):
    """From 606208 lanes on a thread takes 4 streams, the last ones fewer."""
    assert b * 37 * lanes >= 606208 and b % 4
    a = scan_inputs(cuda_dev, dtype, b, 1, 37, k, h0=True)
    h = a["h0"].clone()
    y = sel.selective_scan_step(h, a["u"][:, 0], a["delta"][:, 0], a["A"], a["B"][:, 0], a["C"][:, 0], D=a["D"],
                                z=a["z"][:, 0], delta_bias=a["bias"], delta_softplus=True)
    check_scan(y[:, None], h, a)


@pytest.mark.parametrize("b,d,run", [(57000, 4, 64), (28500, 5, 64), (40000, 4, 32), (20000, 5, 32), (24000, 4, 16),
                                     (12000, 5, 16)])
@pytest.mark.parametrize("dtype,k", [(F32, 4), (BF16, 4), (F16, 3), (BF16, 2)])
def test_conv_forward_runs(sel, cuda_dev, b, d, run, dtype, k):
    """The longest runs that leave 113664 threads, each with a run of one position behind the full ones."""
    n = 65
    threads = lambda r: b * -(-d // 4) * -(-n // r)  # noqa: E731
    assert threads(run) >= 113664 and (run == 64 or threads(2 * run) < 113664)
    lens = [(11 * i) % (n + 1) for i in range(b)]
    a = conv_inputs(cuda_dev, dtype, b, n, d, k, win=True, lengths=lens)
    y, out = call_conv(sel, a)
    want, mag = ref.conv(a), ref.conv(a, mag=True)
    ref.check(y, want["y"], mag["y"], 32, "y")
    assert torch.equal(out.cpu().double(), want["win"])


def test_integration_example(sel, cuda_dev):
    """The calls of INTEGRATION.md as they are written there."""
    import os
    from mamba_integer_b200.rational_bitnet import BitLinear
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")) as f:
        code = f.read().split("## 1b.")[1].split("```python\n")[1].split("```")[0]
    b, n, d, k, width = 3, 10, 64, 16, 32
    r = lambda *s: torch.randn(*s, device=cuda_dev)  # noqa: E731
    linear = BitLinear(width, 48).to(cuda_dev)
    v = dict(torch=torch, d=d, x=r(b, n, width), residual=r(b, n, width), norm_w=torch.ones(width, device=cuda_dev),
             xz=r(b, n, 2 * d), conv_w=r(d, 4), conv_b=r(d), delta=r(b, n, d), A=-r(d, k).exp(), B=r(b, n, k), C=r(b, n, k),
             D=r(d), dt_bias=r(d) - 4, lengths=torch.tensor([10, 4, 0], dtype=torch.int32, device=cuda_dev), xz1=r(b, 2 * d),
             delta1=r(b, d), B1=r(b, k), C1=r(b, k), linear=linear)
    exec(code, v)
    # the tokens go on from each sequence's own length
    for i, e in enumerate((10, 4, 0)):
        one = lambda t, t1: torch.cat([t[i:i + 1, :e], t1[i:i + 1, None]], 1)  # noqa: E731
        xz = one(v["xz"], v["xz1"])
        c = sel.causal_conv1d(xz[..., :d], v["conv_w"], bias=v["conv_b"], silu=True)
        assert torch.equal(c[0, -1], v["c1"][i])
        whole = dict(u=c, delta=one(v["delta"], v["delta1"]), A=v["A"], B=one(v["B"], v["B1"]), C=one(v["C"], v["C1"]),
                     D=v["D"], z=xz[..., d:], bias=v["dt_bias"], softplus=True)
        want, mag = ref.scan(whole), ref.scan(whole, mag=True)
        ref.check(v["s1"][i], want["y"][0, -1], mag["y"][0, -1], 8 * (e + 1) + 64, "s1")
    with torch.no_grad():
        y, total = sel.rms_norm(v["x"], v["norm_w"], residual=v["residual"])
        assert torch.equal(v["out"], linear(y).flatten(0, -2)) and torch.equal(v["total"], total)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("d", [24, 21])
@pytest.mark.parametrize("n,lens", [(33, [33, 32, 9]), (162, [162, 160, 131]), (30, None)])
def test_conv_gradients_of_infinities_at_the_end(sel, cuda_dev, n, lens, d, silu, dtype):
    """Infinite inputs in a sequence's last positions, and infinite weights: the formula's gradients, in which there are
    no positions behind them."""
    a = conv_inputs(cuda_dev, dtype, 3, n, d, 4, silu=silu, win=True, lengths=lens)
    ends = [n] * 3 if lens is None else lens
    for i, e in enumerate(ends):
        for back in (1, 2, 3):
            a["x"][i, e - back, back] = float("inf")
    a["w"][7, 0], a["w"][8, 1], a["w"][9, 2] = (float("inf"),) * 3
    a["w"][10, 0] = float("nan")
    dy = torch.randn(3, n, d, generator=torch.Generator().manual_seed(9)).to(cuda_dev, dtype)
    dwin = torch.randn(3, 3, d, generator=torch.Generator().manual_seed(8)).to(cuda_dev, dtype)
    leaves = {m: a[m].clone().requires_grad_(True) for m in ("x", "w", "bias", "win")}
    y, out = call_conv(sel, a, **leaves)
    for given in (dy, None), (dy, dwin):
        outs = [y] if given[1] is None else [y, out]
        got = torch.autograd.grad(outs, list(leaves.values()), [g for g in given if g is not None], retain_graph=True)
        got = dict(zip(leaves, got), y=y)
        parts = []  # each sequence by itself, as long as it is
        for i, e in enumerate(ends):
            one = {m: None if t is None else t[i:i + 1] for m, t in (("win", a["win"]), ("dwin", given[1]))}
            parts.append(ref.conv(dict(a, x=a["x"][i:i + 1, :e], dy=given[0][i:i + 1, :e], lengths=None, **one)))
            for m in ("x", "y"):
                same_infinities(got[m][i:i + 1, :e], parts[-1]["dx" if m == "x" else "y"], m)
                assert not got[m][i, e:].any()
            same_infinities(got["win"][i:i + 1], parts[-1]["dwin"], "dwin")
        for m in ("w", "bias"):
            same_infinities(got[m], sum(p["d" + m] for p in parts), "d" + m)


@pytest.mark.parametrize("k,d", [(1, 40), (5, 33), (8, 70), (16, 40), (16, 65), (16, 64), (20, 33), (32, 31), (64, 33), (50, 1)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [20, 300])
def test_scan_infinite_B_and_C(sel, cuda_dev, n, dtype, k, d):
    """dB and dC are sums over the channels that there are, and no others of a block of channels."""
    a = scan_inputs(cuda_dev, dtype, 2, n, d, k, h0=True)
    for name in ("u", "B", "C", "D", "h0", "z"):
        a[name] = a[name].abs() + 0.125
    a["A"] *= 2 / k
    a["B"][0, 7, k - 1] = a["C"][1, 12, 0] = float("inf")
    g = torch.Generator().manual_seed(1)
    dy, dh = torch.rand(2, n, d, generator=g).to(cuda_dev, dtype), torch.rand(2, d, k, generator=g).to(cuda_dev)
    dy += 0.125
    y, h, got = scan_grads(sel, a, dy, dh)
    want = ref.scan(dict(a, dy=dy, dh=dh))
    assert want["dC"][0, 7:, k - 1].isinf().all() and want["dB"][1, :13, 0].isinf().all()
    assert want["dB"][0].isfinite().all() and want["dC"][1].isfinite().all()
    for name, t in dict(got, y=y, h=h).items():
        same_infinities(t, want[name if name in ("y", "h") else "d" + name], name)

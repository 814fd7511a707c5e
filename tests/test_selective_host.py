"""The float Mamba operators without a GPU: the refusals of the Python functions and of the C entry points, and the
64-bit formulas that the GPU tests compare with against autograd and against differences."""
import pytest
import torch

import selective_ref as ref
from mamba_integer_b200 import _lib, selective


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def scan_args(batch=2, n=5, d=8, k=4, dtype=torch.float32):
    return dict(u=_t(batch, n, d, dtype=dtype), delta=_t(batch, n, d, dtype=dtype), A=_t(d, k),
                B=_t(batch, n, k, dtype=dtype), C=_t(batch, n, k, dtype=dtype))


@pytest.mark.parametrize("change,error", [
    (dict(u=_t(2, 5, 8, dtype=torch.float64)), TypeError),
    (dict(delta=_t(2, 5, 7)), ValueError),
    (dict(delta=_t(2, 5, 8, dtype=torch.bfloat16)), TypeError),
    (dict(A=_t(7, 4)), ValueError),
    (dict(A=_t(8, 65)), ValueError),
    (dict(A=_t(8, 0)), ValueError),
    (dict(A=_t(8, 4, dtype=torch.bfloat16)), TypeError),
    (dict(B=_t(2, 5, 5)), ValueError),
    (dict(C=_t(2, 4, 4)), ValueError),
    (dict(u=_t(2, 8, 5).transpose(1, 2)), ValueError),
    (dict(D=_t(7)), ValueError),
    (dict(z=_t(2, 5, 8, dtype=torch.float16)), TypeError),
    (dict(delta_bias=_t(8, dtype=torch.float64)), TypeError),
    (dict(h0=_t(2, 8, 5)), ValueError),
    (dict(h0=_t(2, 8, 4, dtype=torch.bfloat16)), TypeError),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(u=_t(2, 8)), ValueError),
    (dict(), ValueError),  # CPU tensors
])
def test_scan_refuses(change, error):
    with pytest.raises(error):
        selective.selective_scan(**{**scan_args(), **change})


@pytest.mark.parametrize("change,error", [
    (dict(h=_t(2, 8, 5)), ValueError),
    (dict(h=_t(2, 8, 4, dtype=torch.bfloat16)), TypeError),
    (dict(h=_t(2, 4, 8).transpose(1, 2)), ValueError),
    (dict(u=_t(2, 1, 8)), ValueError),
    (dict(B=_t(3, 4)), ValueError),
    (dict(h=_t(2, 8, 4).requires_grad_(True)), RuntimeError),
    (dict(), ValueError),
])
def test_scan_step_refuses(change, error):
    args = dict(h=_t(2, 8, 4), u=_t(2, 8), delta=_t(2, 8), A=_t(8, 4), B=_t(2, 4), C=_t(2, 4))
    with pytest.raises(error):
        selective.selective_scan_step(**{**args, **change})


@pytest.mark.parametrize("change,error", [
    (dict(x=_t(2, 5, 8, dtype=torch.int32)), TypeError),
    (dict(x=_t(2, 8)), ValueError),
    (dict(weight=_t(8, 5)), ValueError),
    (dict(weight=_t(8, 1)), ValueError),
    (dict(weight=_t(7, 4)), ValueError),
    (dict(weight=_t(8, 2, 4)), ValueError),
    (dict(weight=_t(8, 4, dtype=torch.float16)), TypeError),
    (dict(bias=_t(4)), ValueError),
    (dict(win=_t(2, 4, 8)), ValueError),
    (dict(win=_t(2, 3, 8, dtype=torch.bfloat16)), TypeError),
    (dict(lengths=torch.zeros(2)), ValueError),
    (dict(), ValueError),
])
def test_conv_refuses(change, error):
    with pytest.raises(error):
        selective.causal_conv1d(**{**dict(x=_t(2, 5, 8), weight=_t(8, 4)), **change})


def test_conv_step_refuses():
    with pytest.raises(ValueError):
        selective.causal_conv1d_step(_t(2, 8), _t(8, 4), _t(2, 2, 8))
    with pytest.raises(TypeError):
        selective.causal_conv1d_step(_t(2, 8), _t(8, 4), _t(2, 3, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        selective.causal_conv1d_step(_t(2, 8), _t(8, 4), _t(2, 8, 3).transpose(1, 2))
    with pytest.raises(RuntimeError):
        selective.causal_conv1d_step(_t(2, 8), _t(8, 4).requires_grad_(True), _t(2, 3, 8))
    with pytest.raises(ValueError):
        selective.causal_conv1d_step(_t(2, 8), _t(8, 4), _t(2, 3, 8))


@pytest.mark.parametrize("change,error", [
    (dict(x=_t(4, 8, dtype=torch.float64)), TypeError),
    (dict(weight=_t(7)), ValueError),
    (dict(weight=_t(8, dtype=torch.bfloat16)), TypeError),
    (dict(residual=_t(4, 7)), ValueError),
    (dict(residual=_t(4, 8, dtype=torch.bfloat16)), TypeError),
    (dict(x=_t(1, selective.MAX_NORM_WIDTH + 1), weight=_t(selective.MAX_NORM_WIDTH + 1)), ValueError),
    (dict(), ValueError),
])
def test_norm_refuses(change, error):
    for fn in (selective.rms_norm, selective.rms_norm_quant):
        with pytest.raises(error):
            fn(**{**dict(x=_t(4, 8), weight=_t(8)), **change})


def test_sizes_past_32_bits_are_refused():
    """Expanded views: no such memory is there."""
    n = (1 << 30) + 1
    one = _t(1, 1, 1)
    with pytest.raises(ValueError, match="too long"):
        selective.selective_scan(one.expand(1, n, 1), one.expand(1, n, 1), _t(1, 1), one.expand(1, n, 1),
                                 one.expand(1, n, 1))
    with pytest.raises(ValueError, match="too long"):
        selective.causal_conv1d(one.expand(1, n, 1), _t(1, 4))


def test_too_many_sequences_are_refused():
    one = _t(1, 1, 1)
    for b, n in ((65536, 1), (65536, 0)):
        rows = one.expand(b, 1, 1)[:, :n]
        with pytest.raises(ValueError, match="at most 65535 sequences"):
            selective.selective_scan(rows, rows, _t(1, 1), rows, rows)
    for b, n in ((65536, 1), (1, 65535 * 128 + 1)):
        with pytest.raises(ValueError, match="at most 65535 sequences of 8388480"):
            selective.causal_conv1d(one.expand(b, n, 1), _t(1, 4))


def test_entry_points_refuse_on_the_host():
    """Before any CUDA call; the pointers are not touched."""
    lib = _lib.load()
    p, s = 256, (256, 512, 64)
    none = (None, 0, 0)

    def fwd(u=s, A=p, L=8, N=16, dtype=0, D=64, ck=None, ws=None):
        return lib.mi_selective_scan(*u, *s, A, *s, *s, None, *none, None, None, None, p, p, ck, ws, 2, L, D, N, 1,
                                     dtype, None)
    assert fwd(u=none) == -1
    assert fwd(A=p + 4) == -1      # rows of states are read 16 bytes at a time
    assert fwd(ck=p + 4) == -1
    assert fwd(L=0) == -1
    assert fwd(L=-1) == -1
    assert fwd(dtype=3) == -1
    assert fwd(N=65) == -2
    assert fwd(N=0) == -1
    assert fwd(L=4096) == -1       # few channels, a long sequence: it wants a workspace
    assert lib.mi_selective_scan_workspace(2, 4096, 64, 16, 0) > 0
    assert lib.mi_selective_scan_workspace(2, 8, 64, 16, 0) == 0
    assert lib.mi_selective_scan_checkpoints(2, 17, 64, 5) == 2 * 2 * 64 * 8
    bwd = lambda ck=p, dz=p, ws=p, z=s: lib.mi_selective_scan_backward(  # noqa: E731
        *s, None, *s, *s, p, *s, *s, None, *z, None, None, ck, p, p, None, None, None, None, dz, None, None, ws, 2, 8,
        64, 16, 1, 0, None)
    assert bwd(ck=None) == -1 and bwd(dz=None) == -1 and bwd(ws=None) == -1
    assert lib.mi_selective_scan_step(p, 64, p, 64, p, p, 16, p, 16, None, None, 0, None, p + 8, p, 2, 64, 16, 1, 0,
                                      None) == -1
    conv = lambda W=4, dtype=0, x=s, y=p: lib.mi_causal_conv1d(*x, p, None, None, None, y, None, 2, 8, 64, W, 1,  # noqa: E731
                                                              dtype, None)
    assert conv(W=5) == -2 and conv(W=1) == -2 and conv(dtype=-1) == -1 and conv(x=none) == -1 and conv(y=None) == -1
    assert lib.mi_causal_conv1d_backward(*s, None, *s, p, None, None, None, None, p, None, None, None, 2, 8, 64, 4, 1, 0,
                                         None) == -1
    assert lib.mi_causal_conv1d_step(p, 64, p, None, None, p, 2, 64, 4, 1, 0, None) == -1
    assert lib.mi_rms_norm(p, 64, None, 0, p, None, None, None, 4, 64, 1e-6, 0, 0, None) == -1
    assert lib.mi_rms_norm(p, 64, p, 64, p, p, None, None, 4, 64, 1e-6, 0, 0, None) == -1   # the sum has no place
    assert lib.mi_rms_norm(p, 16385, None, 0, p, p, None, None, 4, 16385, 1e-6, 0, 0, None) == -2
    assert lib.mi_rms_norm(p, 64, p, 64, p, p, p, None, 4, 64, 1e-6, 0, 1, None) == -1      # fp32 rows, bf16 residual
    assert lib.mi_rms_norm_quant(p, 64, None, 0, p, p, None, None, 4, 64, 1e-6, 0, 0, None) == -1
    assert lib.mi_rms_norm_backward(p, None, p, 64, p, p, p, None, p, None, 4, 64, 0, 0, None) == -1


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float64)


def test_scan_formula_against_autograd_and_differences():
    g = torch.Generator().manual_seed(0)
    b, n, d, k = 2, 7, 3, 4
    leaves = dict(u=_rand(g, b, n, d), delta=_rand(g, b, n, d), A=-_rand(g, d, k).exp(), B=_rand(g, b, n, k),
                  C=_rand(g, b, n, k), D=_rand(g, d), z=_rand(g, b, n, d), bias=_rand(g, d), h0=_rand(g, b, d, k))
    rest = dict(softplus=True, lengths=torch.tensor([7, 4], dtype=torch.int32), dy=_rand(g, b, n, d),
                dh=_rand(g, b, d, k))
    got = ref.scan({**leaves, **rest})

    def value(vals):
        out = ref.scan({**vals, "softplus": True, "lengths": rest["lengths"]})
        return (out["y"] * rest["dy"]).sum() + (out["h"] * rest["dh"]).sum()
    for name, t in leaves.items():
        v = _rand(g, *t.shape)
        up, down = ({**leaves, name: t + s * 1e-6 * v} for s in (1, -1))
        slope = float(value(up) - value(down)) / 2e-6
        # central differences of 1e-6 in 64 bits: 1e-12 of curvature and 1e-10 of rounding, relative to terms of order 10
        assert abs(float((got["d" + name] * v).sum()) - slope) < 1e-7 * max(1, abs(slope)) + 1e-7, name


def test_conv_formula_against_differences():
    g = torch.Generator().manual_seed(1)
    b, n, d, k = 3, 6, 4, 4
    leaves = dict(x=_rand(g, b, n, d), w=_rand(g, d, k), bias=_rand(g, d), win=_rand(g, b, k - 1, d))
    rest = dict(silu=True, lengths=torch.tensor([6, 2, 0], dtype=torch.int32))
    dy, dwin = _rand(g, b, n, d), _rand(g, b, k - 1, d)
    got = ref.conv({**leaves, **rest, "dy": dy, "dwin": dwin})

    def value(vals):
        out = ref.conv({**vals, **rest})
        return (out["y"] * dy).sum() + (out["win"] * dwin).sum()
    for name, t in leaves.items():
        v = _rand(g, *t.shape)
        slope = float(value({**leaves, name: t + 1e-6 * v}) - value({**leaves, name: t - 1e-6 * v})) / 2e-6
        assert abs(float((got["d" + name] * v).sum()) - slope) < 1e-7 * max(1, abs(slope)) + 1e-7, name


def test_norm_formula_against_autograd():
    g = torch.Generator().manual_seed(2)
    s, w, dy = _rand(g, 5, 9).requires_grad_(True), _rand(g, 9).requires_grad_(True), _rand(g, 5, 9)
    y = s / torch.sqrt((s * s).mean(1, keepdim=True) + 1e-6) * w
    ds, dw = torch.autograd.grad(y, [s, w], dy)
    got = ref.norm(s, w, 1e-6, dy)
    assert torch.allclose(got["ds"], ds, rtol=1e-12, atol=1e-12) and torch.allclose(got["dw"], dw, rtol=1e-12)


def test_forward_mode_is_refused():
    """A tangent would be lost; any argument may carry it, a view of a dual tensor too."""
    from torch.autograd import forward_ad

    step = dict(h=_t(2, 8, 4), u=_t(2, 8), delta=_t(2, 8), A=_t(8, 4), B=_t(2, 4), C=_t(2, 4), D=_t(8), z=_t(2, 8),
                delta_bias=_t(8))
    calls = [
        (selective.selective_scan, dict(scan_args(), D=_t(8), z=_t(2, 5, 8), delta_bias=_t(8), h0=_t(2, 8, 4))),
        (selective.selective_scan_step, step),
        (selective.causal_conv1d, dict(x=_t(2, 5, 8), weight=_t(8, 4), bias=_t(8), win=_t(2, 3, 8))),
        (selective.causal_conv1d_step, dict(x=_t(2, 8), weight=_t(8, 4), win=_t(2, 3, 8), bias=_t(8))),
        (selective.rms_norm, dict(x=_t(4, 8), weight=_t(8), residual=_t(4, 8))),
        (selective.rms_norm_quant, dict(x=_t(4, 8), weight=_t(8), residual=_t(4, 8))),
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


def test_the_native_calls_are_built_again_for_another_torch(tmp_path, monkeypatch):
    from mamba_integer_b200 import build

    monkeypatch.setattr(build, "TORCH_SO", str(tmp_path / "x.so"))
    monkeypatch.setattr(build, "TORCH_STAMP", str(tmp_path / "x.so.stamp"))
    assert build.torch_needs_build()
    (tmp_path / "x.so").write_bytes(b"")
    assert build.torch_needs_build()  # of unknown origin
    (tmp_path / "x.so.stamp").write_text(build.torch_stamp())
    assert not build.torch_needs_build()
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build.torch_needs_build()


def test_the_most_states():
    most = selective.MAX_STATES
    with pytest.raises(ValueError, match="CUDA tensor"):
        selective.selective_scan(**scan_args(k=most))
    with pytest.raises(ValueError, match=f"1 to {most} states"):
        selective.selective_scan(**scan_args(k=most + 1))


def test_the_error_of_the_decays_polynomial():
    """2^r on [-1/2, 1/2] by the kernels' coefficients: 2^-26.1, as the source says; the fp32 backward pass has them doubled."""
    import os
    import re

    import numpy as np
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "mamba_integer_b200", "csrc", "selective.cu")) as f:
        source = f.read()
    found = []
    for head in ("exp2_poly(float A, float2 dt) {", "exp2_poly(float2 x) {"):
        body = source.split(head)[1].split("return")[0]
        body = body[body.index("float2 p ="):]
        found.append([float(np.float32(v)) for v in re.findall(r"dup\((?:2 \* )?([0-9.e-]+)f\)", body)])
    assert len(found[0]) == 7 and found[0][:6] == found[1][:6] and found[0][6] == 1 and found[1][6] == 2
    r = np.linspace(-0.5, 0.5, 200001)
    p = np.zeros_like(r)
    for c in found[0]:
        p = p * r + c
    worst = np.abs(p / np.exp2(r) - 1).max()
    assert 2 ** -26.2 < worst < 2 ** -26.1

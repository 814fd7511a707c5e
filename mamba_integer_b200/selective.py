"""The operators of a float Mamba layer (exponential decays, SiLU, RMS norm),
beside the dyadic ones in ``kernels``: for training (each has its backward
pass), for prompts, and for single tokens.

    y, h = selective_scan(u, delta, A, B, C, D=.., z=.., return_state=True)
    y    = selective_scan_step(h, u, delta, A, B, C, D=.., z=..)      # h in place
    y, w = causal_conv1d(x, weight, bias=.., silu=True, return_window=True)
    y    = causal_conv1d_step(x, weight, w, bias=.., silu=True)       # w in place
    y, s = rms_norm(x, weight, residual=r)                            # s = x + r
    q, scale, s = rms_norm_quant(x, weight, residual=r)               # int8 rows for the ternary GEMMs

Activations are fp32, bf16 or fp16, one type for all of a call's; parameters
(A, D, delta_bias, the convolution's weight and bias, the norm's weight), scan
states and scales are fp32.  Arithmetic is fp32 throughout; a result is rounded
to its type once.  Operands need a unit last stride and may be column slices
(``xz[..., d:]``) or expanded over the batch.  The prompt and training forms
take ``lengths`` (int32 [batch], right-padded sequences): what lies at and
behind a sequence's length is not used, outputs and gradients there are 0, and
the state or window returned is the one at the length.

Every call launches on the current stream of its tensors' device, allocates its
outputs and workspaces with torch, and gives the same bits for the same inputs.
CUDA tensors only; gradients are of first order.  To capture a training step in
a CUDA graph, drop any earlier result that still holds an autograd graph over
the same leaves first (torch ties a leaf's gradient to the stream of the graph
that is alive).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.MI_DT_F32, torch.bfloat16: _lib.MI_DT_BF16, torch.float16: _lib.MI_DT_F16}
MAX_STATES = 64
MAX_NORM_WIDTH = 16384


# ---------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------
def _activation(t: torch.Tensor, name: str) -> None:
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")


def _on_gpu(t: torch.Tensor, name: str) -> None:
    """Checked last: the other refusals do not need a GPU."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")


def _like(t: torch.Tensor, first: torch.Tensor, shape, name: str) -> None:
    """An activation of a call whose first one is `first`."""
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype != first.dtype:
        raise TypeError(f"{name} must be {first.dtype} like the call's other activations, got {t.dtype}")
    if t.device != first.device:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on {first.device}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have a unit last stride")


def _plain(t: Optional[torch.Tensor], first: torch.Tensor, shape, name: str, dtype=torch.float32):
    """A contiguous operand of a fixed type (parameters, states), or None."""
    if t is None:
        return None
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != first.device:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on {first.device}")
    return _aligned(t)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and on a 16-byte boundary (a copy where it is not)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _in_place(t: torch.Tensor, first: torch.Tensor, shape, name: str, dtype) -> None:
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != first.device:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on {first.device}")
    if not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError(f"{name} is advanced in place: it must be contiguous and start on a 16-byte boundary")


def _no_grad_needed(*ts) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise RuntimeError("the single-token forms have no backward pass: call them under torch.no_grad()")


def _wanted(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _seq(t: Optional[torch.Tensor]):
    """pointer, batch stride, row stride of a [batch, L, *] operand"""
    return (None, 0, 0) if t is None else (t.data_ptr(), t.stride(0), t.stride(1))


def _row(t: Optional[torch.Tensor]):
    return (None, 0) if t is None else (t.data_ptr(), t.stride(0))


def _call(name: str, dev: torch.device, *args) -> None:
    """The entry point `name` on `dev`'s current stream."""
    fn = getattr(_lib.load(), name)
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    _lib.check(rc, name)


def _workspace(nbytes: int, dev) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _unit(t: torch.Tensor) -> torch.Tensor:
    """An incoming gradient as the kernels read it."""
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


# ---------------------------------------------------------------------------
# selective scan
# ---------------------------------------------------------------------------
def _scan_forward(u, delta, A, B, C, D, z, delta_bias, softplus, h0, lengths, keep: bool):
    batch, L, d = u.shape
    N = A.shape[1]
    lib = _lib.load()
    y = torch.empty(batch, L, d, dtype=u.dtype, device=u.device)
    h = torch.empty(batch, d, N, dtype=torch.float32, device=u.device)
    ckpt = None
    if keep:
        ckpt = torch.empty(lib.mi_selective_scan_checkpoints(batch, L, d, N), dtype=torch.float32, device=u.device)
    ws = _workspace(lib.mi_selective_scan_workspace(batch, L, d, N, 0), u.device)
    _call("mi_selective_scan", u.device, *_seq(u), *_seq(delta), A.data_ptr(), *_seq(B), *_seq(C), _p(D), *_seq(z),
          _p(delta_bias), _p(h0), _p(lengths), y.data_ptr(), h.data_ptr(), _p(ckpt), _p(ws), batch, L, d, N,
          int(softplus), _DTYPES[u.dtype])
    return y, h, ckpt


class SelectiveScanFunction(torch.autograd.Function):
    """selective_scan on checked arguments; saves the inputs and the states at every 16th position."""

    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, delta_bias, h0, lengths, softplus):
        y, h, ckpt = _scan_forward(u, delta, A, B, C, D, z, delta_bias, softplus, h0, lengths, True)
        ctx.save_for_backward(u, delta, A, B, C, D, z, delta_bias, lengths, ckpt)
        ctx.softplus = softplus
        ctx.has_h0 = h0 is not None
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        u, delta, A, B, C, D, z, delta_bias, lengths, ckpt = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 11
        batch, L, d = u.shape
        N = A.shape[1]
        dev = u.device
        need = ctx.needs_input_grad
        dy = torch.zeros_like(u, memory_format=torch.contiguous_format) if dy is None else _unit(dy)
        dh = None if dh is None else _aligned(dh)
        like = lambda t, want=True: torch.empty(t.shape, dtype=t.dtype, device=dev) if want and t is not None else None  # noqa: E731
        du, ddelta, dz = like(u), like(delta), like(z)
        dA, dB, dC = like(A, need[2]), like(B, need[3]), like(C, need[4])
        dD, dbias = like(D, need[5]), like(delta_bias, need[7])
        dh0 = torch.empty(batch, d, N, dtype=torch.float32, device=dev) if ctx.has_h0 and need[8] else None
        ws = _workspace(_lib.load().mi_selective_scan_workspace(batch, L, d, N, 1), dev)
        _call("mi_selective_scan_backward", dev, *_seq(dy), _p(dh), *_seq(u), *_seq(delta), A.data_ptr(), *_seq(B),
              *_seq(C), _p(D), *_seq(z), _p(delta_bias), _p(lengths), ckpt.data_ptr(), du.data_ptr(),
              ddelta.data_ptr(), _p(dA), _p(dB), _p(dC), _p(dD), _p(dz), _p(dbias), _p(dh0), _p(ws), batch, L, d, N,
              int(ctx.softplus), _DTYPES[u.dtype])
        return du, ddelta, dA, dB, dC, dD, dz, dbias, dh0, None, None


def _scan_arguments(lead, u, delta, A, B, C, D, z, delta_bias):
    _activation(u, "u")
    d = u.shape[-1]
    if A.dim() != 2 or A.shape[0] != d:
        raise ValueError(f"A must be [{d}, states], got {list(A.shape)}")
    N = A.shape[1]
    if d == 0 or not 1 <= N <= MAX_STATES:
        raise ValueError(f"selective scans have 1 to {MAX_STATES} states and at least one channel: A is {list(A.shape)}")
    _like(u, u, (*lead, d), "u")
    _like(delta, u, u.shape, "delta")
    _like(B, u, (*lead, N), "B")
    _like(C, u, (*lead, N), "C")
    if z is not None:
        _like(z, u, u.shape, "z")
    return _plain(A, u, (d, N), "A"), _plain(D, u, (d,), "D"), _plain(delta_bias, u, (d,), "delta_bias")


def _lengths(lengths, u, batch):
    if lengths is None:
        return None
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (batch,) or lengths.device != u.device:
        raise ValueError(f"lengths must be int32 [{batch}] on {u.device}")
    return lengths.contiguous()


def selective_scan(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                   delta_bias: Optional[torch.Tensor] = None, delta_softplus: bool = False,
                   h0: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                   return_state: bool = False):
    """Selective scan over [batch, L, channels]:

        dt = delta + delta_bias, softplus of it with delta_softplus
        h[t] = exp(dt A) h[t-1] + dt B[t] u[t],  h[-1] = h0 (zeros without one)
        y[t] = (sum over the states of C[t] h[t] + D u[t]) * z sigmoid(z)

    u, delta, z [batch, L, channels]; B, C [batch, L, states]; A [channels,
    states]; D, delta_bias [channels]; h0 [batch, channels, states].  Returns
    y, or (y, final state) with ``return_state``.  1 to 64 states."""
    if u.dim() != 3:
        raise ValueError(f"u must be [batch, L, channels], got {list(u.shape)}")
    batch, L, d = u.shape
    A, D, delta_bias = _scan_arguments((batch, L), u, delta, A, B, C, D, z, delta_bias)
    N = A.shape[1]
    h0 = _plain(h0, u, (batch, d, N), "h0")
    lengths = _lengths(lengths, u, batch)
    _on_gpu(u, "u")
    if batch == 0 or L == 0:  # nothing to scan
        y = u * 1
        h = torch.zeros(batch, d, N, dtype=torch.float32, device=u.device) if h0 is None else h0 * 1
    elif _wanted(u, delta, A, B, C, D, z, delta_bias, h0):
        y, h = SelectiveScanFunction.apply(u, delta, A, B, C, D, z, delta_bias, h0, lengths, bool(delta_softplus))
    else:
        y, h, _ = _scan_forward(u, delta, A, B, C, D, z, delta_bias, delta_softplus, h0, lengths, False)
    return (y, h) if return_state else y


def selective_scan_step(h: torch.Tensor, u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                        C: torch.Tensor, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        delta_bias: Optional[torch.Tensor] = None, delta_softplus: bool = False) -> torch.Tensor:
    """One position of selective_scan for every stream: u, delta, z [batch,
    channels], B, C [batch, states]; h [batch, channels, states] is advanced in
    place.  Returns y [batch, channels].  No backward pass."""
    if u.dim() != 2:
        raise ValueError(f"u must be [batch, channels], got {list(u.shape)}")
    batch, d = u.shape
    _no_grad_needed(h, u, delta, A, B, C, D, z, delta_bias)
    A, D, delta_bias = _scan_arguments((batch,), u, delta, A, B, C, D, z, delta_bias)
    N = A.shape[1]
    _in_place(h, u, (batch, d, N), "h", torch.float32)
    _on_gpu(u, "u")
    y = torch.empty(batch, d, dtype=u.dtype, device=u.device)
    _call("mi_selective_scan_step", u.device, *_row(u), *_row(delta), A.data_ptr(), *_row(B), *_row(C), _p(D),
          *_row(z), _p(delta_bias), h.data_ptr(), y.data_ptr(), batch, d, N, int(delta_softplus), _DTYPES[u.dtype])
    return y


# ---------------------------------------------------------------------------
# causal convolution
# ---------------------------------------------------------------------------
def _conv_forward(x, w, bias, win, lengths, silu):
    batch, L, d = x.shape
    W = w.shape[1]
    y = torch.empty(batch, L, d, dtype=x.dtype, device=x.device)
    out = torch.empty(batch, W - 1, d, dtype=x.dtype, device=x.device)
    _call("mi_causal_conv1d", x.device, *_seq(x), w.data_ptr(), _p(bias), _p(win), _p(lengths), y.data_ptr(),
          out.data_ptr(), batch, L, d, W, int(silu), _DTYPES[x.dtype])
    return y, out


class CausalConv1dFunction(torch.autograd.Function):
    """causal_conv1d on checked arguments."""

    @staticmethod
    def forward(ctx, x, w, bias, win, lengths, silu):
        y, out = _conv_forward(x, w, bias, win, lengths, silu)
        ctx.save_for_backward(x, w, bias, win, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dout):
        x, w, bias, win, lengths = ctx.saved_tensors
        if dy is None and dout is None:
            return (None,) * 6
        batch, L, d = x.shape
        W = w.shape[1]
        dev = x.device
        need = ctx.needs_input_grad
        dy = torch.zeros_like(x, memory_format=torch.contiguous_format) if dy is None else _unit(dy)
        dout = None if dout is None else _aligned(dout)
        like = lambda t, want: torch.empty(t.shape, dtype=t.dtype, device=dev) if want and t is not None else None  # noqa: E731
        dx, dw, dbias, dwin = like(x, need[0]), like(w, need[1]), like(bias, need[2]), like(win, need[3])
        ws = None
        if dw is not None or dbias is not None:
            ws = _workspace(_lib.load().mi_causal_conv1d_backward_workspace(batch, L, d, W), dev)
        _call("mi_causal_conv1d_backward", dev, *_seq(dy), _p(dout), *_seq(x), w.data_ptr(), _p(bias), _p(win),
              _p(lengths), _p(dx), _p(dw), _p(dbias), _p(dwin), _p(ws), batch, L, d, W, int(ctx.silu),
              _DTYPES[x.dtype])
        return dx, dw, dbias, dwin, None, None


def _conv_arguments(lead, x, weight, bias):
    _activation(x, "x")
    d = x.shape[-1]
    if weight.dim() == 3 and weight.shape[1] == 1:  # nn.Conv1d's [channels, 1, taps]
        weight = weight.squeeze(1)
    if weight.dim() != 2 or weight.shape[0] != d or d == 0 or not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"weight must be [{d}, taps] or [{d}, 1, taps] with 2 to 4 taps, got {list(weight.shape)}")
    _like(x, x, (*lead, d), "x")
    return _plain(weight, x, weight.shape, "weight"), _plain(bias, x, (d,), "bias")


def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, silu: bool = False,
                  win: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                  return_window: bool = False):
    """Causal depthwise convolution over [batch, L, channels]:

        c[t] = bias + sum_k weight[:, k] x[t - taps + 1 + k];  y = c sigmoid(c) with silu, else c

    weight [channels, taps] (or nn.Conv1d's [channels, 1, taps]), 2 to 4 taps;
    win [batch, taps - 1, channels] of x's type holds the inputs before
    position 0 (zeros without one).  Returns y, or (y, window) with
    ``return_window``: the last taps - 1 inputs, as causal_conv1d_step takes it."""
    if x.dim() != 3:
        raise ValueError(f"x must be [batch, L, channels], got {list(x.shape)}")
    batch, L, d = x.shape
    weight, bias = _conv_arguments((batch, L), x, weight, bias)
    W = weight.shape[1]
    win = _plain(win, x, (batch, W - 1, d), "win", x.dtype)
    lengths = _lengths(lengths, x, batch)
    _on_gpu(x, "x")
    if batch == 0 or L == 0:
        y = x * 1
        out = torch.zeros(batch, W - 1, d, dtype=x.dtype, device=x.device) if win is None else win * 1
    elif _wanted(x, weight, bias, win):
        y, out = CausalConv1dFunction.apply(x, weight, bias, win, lengths, bool(silu))
    else:
        y, out = _conv_forward(x, weight, bias, win, lengths, silu)
    return (y, out) if return_window else y


def causal_conv1d_step(x: torch.Tensor, weight: torch.Tensor, win: torch.Tensor,
                       bias: Optional[torch.Tensor] = None, silu: bool = False) -> torch.Tensor:
    """One position of causal_conv1d for every stream: x [batch, channels];
    win [batch, taps - 1, channels] is advanced in place.  Returns y [batch,
    channels].  No backward pass."""
    if x.dim() != 2:
        raise ValueError(f"x must be [batch, channels], got {list(x.shape)}")
    batch, d = x.shape
    _no_grad_needed(x, weight, win, bias)
    weight, bias = _conv_arguments((batch,), x, weight, bias)
    W = weight.shape[1]
    _in_place(win, x, (batch, W - 1, d), "win", x.dtype)
    _on_gpu(x, "x")
    y = torch.empty(batch, d, dtype=x.dtype, device=x.device)
    _call("mi_causal_conv1d_step", x.device, *_row(x), weight.data_ptr(), _p(bias), win.data_ptr(), y.data_ptr(),
          batch, d, W, int(silu), _DTYPES[x.dtype])
    return y


# ---------------------------------------------------------------------------
# RMS norm
# ---------------------------------------------------------------------------
def _rms_forward(x, weight, eps, residual, keep: bool):
    T, d = x.shape
    y = torch.empty(T, d, dtype=x.dtype, device=x.device)
    total = None if residual is None else torch.empty(T, d, dtype=residual.dtype, device=x.device)
    rstd = torch.empty(T, dtype=torch.float32, device=x.device) if keep else None
    code = _DTYPES[x.dtype]
    _call("mi_rms_norm", x.device, *_row(x), *_row(residual), weight.data_ptr(), y.data_ptr(), _p(total), _p(rstd), T,
          d, eps, code, code if residual is None else _DTYPES[residual.dtype])
    return y, total, rstd


class RMSNormFunction(torch.autograd.Function):
    """rms_norm on checked arguments ([rows, width]); saves the sum and each row's 1 / rms."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, total, rstd = _rms_forward(x, weight, eps, residual, True)
        ctx.save_for_backward(x if total is None else total, weight, rstd)
        ctx.x_dtype = x.dtype
        ctx.has_residual = residual is not None
        ctx.set_materialize_grads(False)
        return y if total is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dtotal=None):
        s, weight, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dy is None:
            if dtotal is None:
                return None, None, None, None
            return dtotal.to(ctx.x_dtype), None, dtotal, None
        T, d = s.shape
        dev = s.device
        dy = _aligned(dy)
        dtotal = None if dtotal is None else _aligned(dtotal)
        same = s.dtype == ctx.x_dtype
        want_r = ctx.has_residual and need[2]
        dx = torch.empty(T, d, dtype=ctx.x_dtype, device=dev) if need[0] or (same and want_r) else None
        dr = torch.empty(T, d, dtype=s.dtype, device=dev) if want_r and not same else None
        dw = torch.empty(d, dtype=torch.float32, device=dev) if need[1] else None
        ws = _workspace(_lib.load().mi_rms_norm_backward_workspace(T, d), dev) if need[1] else None
        _call("mi_rms_norm_backward", dev, dy.data_ptr(), _p(dtotal), s.data_ptr(), s.stride(0), weight.data_ptr(),
              rstd.data_ptr(), _p(dx), _p(dr), _p(dw), _p(ws), T, d, _DTYPES[ctx.x_dtype], _DTYPES[s.dtype])
        return dx if need[0] else None, dw, (dx if same else dr) if want_r else None, None


def _rms_arguments(x, weight, residual):
    _activation(x, "x")
    d = x.shape[-1] if x.dim() else 0
    if not 1 <= d <= MAX_NORM_WIDTH:
        raise ValueError(f"rows of 1 to {MAX_NORM_WIDTH} columns, got x {list(x.shape)}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must be {list(x.shape)}, got {list(residual.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"residual must be {x.dtype} or float32, got {residual.dtype}")
        if residual.device != x.device:
            raise ValueError(f"residual is on {residual.device}, x on {x.device}")
    weight = _plain(weight, x, (d,), "weight")
    _on_gpu(x, "x")
    rows = lambda t: _unit(t if t.dim() == 2 else t.reshape(-1, d))  # noqa: E731
    return rows(x), weight, None if residual is None else rows(residual)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None
             ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RMS norm over the last dimension, with the residual's addition:

        s = x + residual (s = x without one), in the residual's type
        y = s / sqrt(mean(s^2) + eps) * weight

    x and residual [..., width]; residual is of x's type or fp32; the norm is of
    s as it is kept.  Returns (y, s), s None without a residual."""
    x2, weight, r2 = _rms_arguments(x, weight, residual)
    if x2.shape[0] == 0:
        return x * 1, None if residual is None else residual * 1
    if _wanted(x2, weight, r2):
        out = RMSNormFunction.apply(x2, weight, r2, float(eps))
        y, total = (out, None) if residual is None else out
    else:
        y, total, _ = _rms_forward(x2, weight, float(eps), r2, False)
    return y.view(x.shape), None if total is None else total.view(x.shape)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None
                   ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """rms_norm with its rows quantised to int8 as kernels.quantize_rows does:
    returns (q int8 [..., width], scale fp32 [...], s), y = q * scale; q and
    scale feed ternary_matmul.  No backward pass."""
    _no_grad_needed(x, weight, residual)
    x2, weight, r2 = _rms_arguments(x, weight, residual)
    T, d = x2.shape
    q = torch.empty(T, d, dtype=torch.int8, device=x.device)
    scale = torch.empty(T, dtype=torch.float32, device=x.device)
    total = None if r2 is None else torch.empty(T, d, dtype=r2.dtype, device=x.device)
    code = _DTYPES[x.dtype]
    if T:
        _call("mi_rms_norm_quant", x.device, *_row(x2), *_row(r2), weight.data_ptr(), q.data_ptr(), scale.data_ptr(),
              _p(total), T, d, float(eps), code, code if r2 is None else _DTYPES[r2.dtype])
    return q.view(x.shape), scale.view(x.shape[:-1]), None if total is None else total.view(x.shape)

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
Wrong shapes and placements raise ValueError, wrong types TypeError.  The calls
are native (csrc/torch_ops.cpp, over the C ABI of include/mi_b200.h).
CUDA tensors only; gradients are of first order and by backward passes (dual
tensors of forward-mode differentiation raise NotImplementedError); a prompt or
training call has at most 65535 sequences.  To capture a training step in a CUDA graph, drop any
earlier result that still holds an autograd graph over the same leaves first
(torch ties a leaf's gradient to the stream of the graph that is alive; the
calls refuse such a capture where that is the default stream).
"""
from __future__ import annotations

import ctypes
import importlib.util
import os
from typing import Optional, Tuple

import torch

from . import _lib

MAX_STATES = 64
MAX_NORM_WIDTH = 16384

SO_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_mi_torch.so")
_ops = None


def _load():
    """The native calls, bound to the library's entry points."""
    global _ops
    if _ops is None:
        if not os.path.exists(SO_PATH):
            raise ImportError(f"{SO_PATH} is missing: build it with `python -m mamba_integer_b200.build`")
        spec = importlib.util.spec_from_file_location("_mi_torch", SO_PATH)
        ops = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(ops)
        bind(ops)
        _ops = ops
    return _ops


def bind(ops=None) -> None:
    """(Re)binds the native calls to the entry points of the loaded library."""
    lib = _lib.load()
    (ops or _load()).bind({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _lib.SIGNATURES
                           if hasattr(lib, name)})


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
    y, or (y, final state) with ``return_state``.  1 to 64 states.  An infinite
    A counts as a very large one (0 times it is 0)."""
    y, h = (_ops or _load()).selective_scan(u, delta, A, B, C, D, z, delta_bias, delta_softplus, h0, lengths)
    return (y, h) if return_state else y


def selective_scan_step(h: torch.Tensor, u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                        C: torch.Tensor, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        delta_bias: Optional[torch.Tensor] = None, delta_softplus: bool = False) -> torch.Tensor:
    """One position of selective_scan for every stream: u, delta, z [batch,
    channels], B, C [batch, states]; h [batch, channels, states] is advanced in
    place.  Returns y [batch, channels].  No backward pass."""
    return (_ops or _load()).selective_scan_step(h, u, delta, A, B, C, D, z, delta_bias, delta_softplus)


def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, silu: bool = False,
                  win: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                  return_window: bool = False):
    """Causal depthwise convolution over [batch, L, channels]:

        c[t] = bias + sum_k weight[:, k] x[t - taps + 1 + k];  y = c sigmoid(c) with silu, else c

    weight [channels, taps] (or nn.Conv1d's [channels, 1, taps]), 2 to 4 taps;
    win [batch, taps - 1, channels] of x's type holds the inputs before
    position 0 (zeros without one).  Returns y, or (y, window) with
    ``return_window``: the last taps - 1 inputs, as causal_conv1d_step takes it.
    Sequences of up to 8388480 positions."""
    y, out = (_ops or _load()).causal_conv1d(x, weight, bias, silu, win, lengths)
    return (y, out) if return_window else y


def causal_conv1d_step(x: torch.Tensor, weight: torch.Tensor, win: torch.Tensor,
                       bias: Optional[torch.Tensor] = None, silu: bool = False) -> torch.Tensor:
    """One position of causal_conv1d for every stream: x [batch, channels];
    win [batch, taps - 1, channels] is advanced in place.  Returns y [batch,
    channels].  No backward pass."""
    return (_ops or _load()).causal_conv1d_step(x, weight, win, bias, silu)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None
             ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RMS norm over the last dimension, with the residual's addition:

        s = x + residual (s = x without one), in the residual's type
        y = s / sqrt(mean(s^2) + eps) * weight

    x and residual [..., width]; residual is of x's type or fp32; the norm is of
    s as it is kept.  Returns (y, s), s None without a residual."""
    return (_ops or _load()).rms_norm(x, weight, eps, residual)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None
                   ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """rms_norm with its rows quantised to int8 as kernels.quantize_rows does:
    returns (q int8 [..., width], scale fp32 [...], s), y = q * scale; q and
    scale feed ternary_matmul.  No backward pass."""
    return (_ops or _load()).rms_norm_quant(x, weight, eps, residual)

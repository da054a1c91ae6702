"""Rotary positions, alone and with the per-head RMSNorm of queries and keys in the same pass.

Upstream's rotary embedding (model/forgetting_transformer/rotary.py, kernel 22-153; the layer's ``use_rope``) rotates by a
kernel of its own, from tables of cosines and sines; here the kernel forms the angles of the positions that it meets, product and reduction in
64 bits, so that there is no table and no longest position, and each value is rounded once.
"""
from __future__ import annotations

import math
from typing import Literal, Optional, Tuple, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["rotary_frequencies", "rotary_embedding", "qk_norm_rotary", "RotaryEmbedding"]

_host = None
Positions = Optional[Union[int, torch.Tensor]]


def _load_host():
    global _host
    _host = _lib.host()
    return _host


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: Literal["none", "linear", "ntk", "yarn"] = "none",
                       factor: float = 1.0, original_length: Optional[int] = None, beta_fast: float = 32.0,
                       beta_slow: float = 1.0, device=None) -> Tuple[torch.Tensor, float]:
    """(inv_freq, scale) for ``rotary_embedding``: ``base ** (-2 i / dim)``, i < dim / 2, in fp32, and 1.0; for contexts
    ``factor`` times as long as a model was trained on:

    - "linear": all frequencies divided by ``factor``;
    - "ntk": the base raised to ``base * factor ** (dim / (dim - 2))``, which leaves the fastest frequency as it is and
      divides the slowest by ``factor``;
    - "yarn" (arXiv 2309.00071, section 3.2): frequencies that turn less than ``beta_slow`` times over ``original_length``
      tokens divided by ``factor``, those that turn more than ``beta_fast`` times as they are, between them a mixture linear in
      the number of turns; scale = 0.1 ln(factor) + 1."""
    if dim < 2 or dim % 2:
        raise ValueError(f"the rotated part must have an even number of channels, but got {dim}")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"Unsupported scaling: {scaling}")
    if not factor > 0 or not base > 0:
        raise ValueError("base and factor must be positive")
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling needs more than one frequency")
        base = base * factor ** (dim / (dim - 2))
    freq = torch.pow(float(base), -torch.arange(0, dim, 2, dtype=torch.float64, device="cpu") / dim)
    scale = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if original_length is None or original_length < 1 or not beta_fast > beta_slow:
            raise ValueError("yarn scaling needs original_length >= 1 and beta_fast > beta_slow")
        turns = original_length * freq / (2 * math.pi)
        kept = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0, 1)
        freq = freq * kept + freq / factor * (1 - kept)
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return freq.to(torch.float32).to(torch.get_default_device() if device is None else device), scale


class _Rotate(torch.autograd.Function):
    """The calls that the native node leaves to Python (tracing, tensor subclasses, tangents, which this refuses)."""

    @staticmethod
    def forward(ctx, x, inv_freq, positions, head_first, interleaved, scale):
        ctx.rest = (head_first, interleaved, scale)
        ctx.first = None if isinstance(positions, torch.Tensor) else positions
        ctx.save_for_backward(inv_freq, positions if ctx.first is None else None)
        return _lib.host().rotary_apply(x, inv_freq, positions, head_first, interleaved, scale, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        inv_freq, positions = ctx.saved_tensors
        at = positions if ctx.first is None else ctx.first
        return (_lib.host().rotary_apply(dy, inv_freq, at, *ctx.rest, True), None, None, None, None, None)


class _NormRotate(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, inv_freq, positions, eps, head_first, interleaved, scale):
        ctx.rest = (eps, head_first, interleaved, scale)
        ctx.first = None if isinstance(positions, torch.Tensor) else positions
        ctx.save_for_backward(q, k, q_weight, k_weight, inv_freq, positions if ctx.first is None else None)
        return _lib.host().qk_norm_rotary_forward(q, k, q_weight, k_weight, inv_freq, positions, *ctx.rest)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        *tensors, positions = ctx.saved_tensors
        at = positions if ctx.first is None else ctx.first
        return (*_lib.host().qk_norm_rotary_backward(*tensors, at, *ctx.rest, dq, dk), None, None, None, None, None, None)


def _no_frequency_gradient(what: str, inv_freq: torch.Tensor) -> None:
    """(The native nodes look for themselves; inside an autograd function's forward gradients are off.)"""
    if torch.is_grad_enabled() and inv_freq.requires_grad:
        raise _lib.FoxError(f"{what} has no gradient for inv_freq: detach it, or call it under torch.no_grad()")


def rotary_embedding(x: torch.Tensor, inv_freq: torch.Tensor, positions: Positions = None, *, head_first: bool = False,
                     interleaved: bool = False, scale: float = 1.0) -> torch.Tensor:
    """``x`` with the first ``2 * inv_freq.numel()`` channels of every head turned by ``position * inv_freq`` and multiplied
    by ``scale``; the other channels as they are.

    - x (B, T, H, D) or (T, H, D), with ``head_first`` the H and T axes swapped, fp16 / bf16, D in {16, 32, 64, 128},
      any strides;
    - inv_freq fp32, up to D / 2 elements (``rotary_frequencies``);
    - positions: (T,) or (B, T) int32 / int64 on the device, an int (the first token's), or None: 0, 1, 2, ...;
    - pairs: channels i and i + half, with ``interleaved`` channels 2 i and 2 i + 1.

    Differentiable w.r.t. x, any number of times."""
    pos = 0 if positions is None else positions
    out = (_host or _load_host()).rotary(x, inv_freq, pos, head_first, interleaved, scale)
    if out is None:
        _no_frequency_gradient("rotary_embedding", inv_freq)
        out = _Rotate.apply(x, inv_freq, pos, head_first, interleaved, scale)
    return out


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, inv_freq: torch.Tensor,
                   positions: Positions = None, *, eps: float = 1e-5, head_first: bool = False, interleaved: bool = False,
                   scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``rotary_embedding`` of the per-head RMSNorms of q and k (``GroupNorm``) in one kernel, without rounding between the two.

    q (B, T, H, D) and k (B, T, Hk, D), or (T, H, D), as for ``rotary_embedding``; q_weight (H * D,) or (D,) for all heads
    alike, k_weight likewise, fp16 / bf16 / fp32.  Returns (q, k); differentiable, once, w.r.t. q, k and both weights."""
    pos = 0 if positions is None else positions
    out = (_host or _load_host()).qk_norm_rotary(q, k, q_weight, k_weight, inv_freq, pos, eps, head_first, interleaved, scale)
    if out is None:
        _no_frequency_gradient("qk_norm_rotary", inv_freq)
        out = _NormRotate.apply(q, k, q_weight, k_weight, inv_freq, pos, eps, head_first, interleaved, scale)
    return out


class RotaryEmbedding(nn.Module):
    """Rotary positions of a layer: ``rotary_frequencies``' arguments, kept with the layout of the pairs.  ``forward`` rotates
    q and k; ``norm`` norms them first.  The frequencies stay in fp32 whatever type the module is moved to; they come from the
    arguments, so that a module built on the meta device has them too, and what is pickled holds no device's copy.  They are copied
    to a device at the first call there, which may not be one that is captured in a CUDA graph."""

    def __init__(self, dim: int, base: float = 10000.0, interleaved: bool = False, **scaling):
        super().__init__()
        self.dim, self.base, self.interleaved = dim, float(base), interleaved
        with torch.inference_mode(False):
            self._freq, self.scale = rotary_frequencies(dim, base, device="cpu", **scaling)
        self._on_device = {}

    def __getstate__(self):
        return {**self.__dict__, "_on_device": {}}

    def inv_freq(self, device) -> torch.Tensor:
        got = self._on_device.get(device)
        if got is None:
            if torch.device(device).type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise _lib.FoxError("the frequencies come to a device at the first call there, which cannot be captured in a graph: "
                                    "call the module, or its inv_freq(device), once before")
            with torch.inference_mode(False):   # (the copy serves training too)
                got = self._freq.to(device)
            if type(got) is torch.Tensor:       # (a tracer's stand-in is not kept)
                self._on_device[device] = got
        return got

    def extra_repr(self) -> str:
        return f"{self.dim}, base={self.base}, interleaved={self.interleaved}, scale={self.scale}"

    def forward(self, q: torch.Tensor, k: torch.Tensor, positions: Positions = None, *, head_first: bool = False):
        f = self.inv_freq(q.device)
        return tuple(rotary_embedding(x, f, positions, head_first=head_first, interleaved=self.interleaved, scale=self.scale)
                     for x in (q, k))

    def norm(self, q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
             positions: Positions = None, *, eps: float = 1e-5, head_first: bool = False):
        return qk_norm_rotary(q, k, q_weight, k_weight, self.inv_freq(q.device), positions, eps=eps, head_first=head_first,
                              interleaved=self.interleaved, scale=self.scale)

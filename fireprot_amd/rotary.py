"""Rotary positions on gfx950: queries and keys turned in one launch.

``apply_rotary(q, k, positions, frequencies)`` turns the first ``rotary_dim``
channels of every head in pairs by the angle ``position * inv_freq[i]`` and
copies the rest (``fpx_rotary``): the half layout pairs channels ``i`` and
``i + rotary_dim / 2``, the interleaved one ``2i`` and ``2i + 1``.  FP32,
BF16 and FP16 rows in any strides with unit channel stride, out of place or in
place; arithmetic in FP32 with one rounding at the end, the angles in FP64, so
positions far into a long context keep their digits.

The map is orthogonal up to its factor: its gradient is the same kernel with
the angles negated, ``rotary_backward``.
Stands in for the reference's rotary kernel of its protein language models
(kernels/amd/fireprot_esmc_rope.hip).
"""
from __future__ import annotations

import dataclasses
import math
from typing import Any

import torch

from . import _native

MAX_HEAD_DIM = 512
LAYOUTS = {"half": 0, "interleaved": 1}
DTYPES = {torch.float32: _native.FPX_F32, torch.bfloat16: _native.FPX_BF16,
          torch.float16: _native.FPX_F16}
POSITION_DTYPES = {torch.int32: 0, torch.int64: 1}


@dataclasses.dataclass(frozen=True, eq=False)
class RotaryFrequencies:
    """``inv_freq``: contiguous float64 ``[rotary_dim / 2]``, radians a position
    of each pair; ``scale``: factor of the rotated channels."""

    inv_freq: torch.Tensor
    scale: float = 1.0

    def __post_init__(self) -> None:
        f = self.inv_freq
        if f.dtype != torch.float64 or f.dim() != 1 or f.numel() < 1 or not f.is_contiguous():
            raise ValueError("inv_freq must be a contiguous float64 vector, not empty")
        if f.requires_grad:
            raise ValueError("inv_freq gets no gradient: detach it")

    @property
    def rotary_dim(self) -> int:
        return 2 * self.inv_freq.shape[0]

    def to(self, device: Any) -> "RotaryFrequencies":
        return RotaryFrequencies(self.inv_freq.to(device), self.scale)


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str | None = None,
                       factor: float = 1.0, original_length: int | None = None,
                       slow: float = 1.0, fast: float = 32.0, scale: float | None = None,
                       device: Any = None) -> RotaryFrequencies:
    """``f_i = base ** (-2i / rotary_dim)``, scaled for contexts ``factor``
    times the trained one:

    * ``"linear"``: ``f_i / factor``, positions interpolated;
    * ``"ntk"``: ``base * factor ** (r / (r - 2))`` in place of ``base``, which
      interpolates the slowest pair and leaves the fastest;
    * ``"by_parts"``: pairs that turn more than ``fast`` times over
      ``original_length`` keep ``f_i``, those that turn less than ``slow``
      times get ``f_i / factor``, a linear blend between; the outputs' factor
      is ``0.1 ln(factor) + 1`` unless ``scale`` is given.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    if scaling not in (None, "linear", "ntk", "by_parts"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if not base > 0.0 or not factor >= 1.0:
        raise ValueError("base must be positive and factor at least 1")
    if scaling is None and factor != 1.0:
        raise ValueError("factor needs a scaling")
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    inv_freq = torch.pow(torch.tensor(float(base), dtype=torch.float64), -2.0 * i / rotary_dim)
    default_scale = 1.0
    if scaling == "linear":
        inv_freq = inv_freq / factor
    elif scaling == "by_parts":
        if original_length is None or not original_length > 0 or not fast > slow:
            raise ValueError("by_parts needs original_length > 0 and fast > slow")
        turns = original_length * inv_freq / (2.0 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        inv_freq = inv_freq / factor * (1.0 - keep) + inv_freq * keep
        default_scale = 0.1 * math.log(factor) + 1.0
    return RotaryFrequencies(inv_freq.to(device) if device is not None else inv_freq,
                             default_scale if scale is None else float(scale))


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """``t`` as [batch, tokens, heads, head_dim] with unit channel stride."""
    if t.dim() == 3:
        t = t.unsqueeze(0)
    elif t.dim() != 4:
        raise ValueError(f"{name} must be [batch, tokens, heads, head_dim] or "
                         f"[tokens, heads, head_dim], got {tuple(t.shape)}")
    return t if t.stride(3) == 1 else t.contiguous()


def _output(given: torch.Tensor | None, like: torch.Tensor, rows: torch.Tensor, name: str):
    """(the four-axis output, what the caller gets) for an input and its rows."""
    if given is None:
        out = torch.empty_like(rows, memory_format=torch.contiguous_format)
        return out, out if like.dim() == 4 else out[0]
    if (given.shape != like.shape or given.dtype != like.dtype or given.device != like.device
            or given.stride(-1) != 1 or _native.repeats(given)):
        raise ValueError(f"{name} must have its input's shape, type and device, unit channel "
                         "stride and no repeated elements")
    return given if given.dim() == 4 else given.unsqueeze(0), given


def _launch(q, k, positions, frequencies, layout, inverse, q_out, k_out):
    """Checks, then one fpx_rotary call into q_out and k_out (new where None)."""
    lib = _native.library()
    mode = LAYOUTS.get(layout)
    if mode is None:
        raise ValueError(f"layout must be one of {sorted(LAYOUTS)}")
    kind, device = DTYPES.get(q.dtype), q.get_device()
    if kind is None or device < 0:
        raise ValueError("q must be a float32, bfloat16 or float16 tensor on a HIP device")
    x = q if q.dim() == 4 and q.stride(3) == 1 else _rows(q, "q")
    batch, tokens, q_heads, head_dim = x.shape
    inv_freq = frequencies.inv_freq
    rotary_dim = 2 * inv_freq.shape[0]
    if rotary_dim > head_dim or head_dim > MAX_HEAD_DIM:
        raise ValueError(f"needs rotary_dim ({rotary_dim}) <= head_dim ({head_dim}) "
                         f"<= {MAX_HEAD_DIM}")
    wide = positions.dim() == 2
    place = POSITION_DTYPES.get(positions.dtype)
    if (place is None or positions.get_device() != device or inv_freq.get_device() != device
            or positions.shape != ((batch, tokens) if wide else (tokens,))):
        raise ValueError("positions must be int32 or int64 [batch, tokens] or [tokens], and they "
                         "and inv_freq on q's device")
    a, q_ret = _output(q_out, q, x, "q_out")
    if k is None:
        k_heads, k_ret = 0, None
        k_args = k_out_args = (None, 0, 0, 0)
    else:
        if (k.dtype != q.dtype or k.get_device() != device or k.dim() != q.dim()
                or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != head_dim):
            raise ValueError("k must have q's type, device, batch, tokens and head_dim")
        y = k if k.dim() == 4 and k.stride(3) == 1 else _rows(k, "k")
        k_heads = y.shape[2]
        b, k_ret = _output(k_out, k, y, "k_out")
        if a.data_ptr() == b.data_ptr() and a.numel() and b.numel():
            raise ValueError("q_out and k_out must not share memory")
        k_args = (y.data_ptr(), *y.stride()[:3])
        k_out_args = (b.data_ptr(), *b.stride()[:3])
    if q_heads == 0 and k_heads == 0:
        return q_ret, k_ret
    code = _native.launch(
        device, lib.fpx_rotary, kind, mode, x.data_ptr(), *x.stride()[:3],
        a.data_ptr(), *a.stride()[:3], q_heads, *k_args, *k_out_args, k_heads,
        positions.data_ptr(), place, positions.stride(0) if wide else 0, positions.stride(-1),
        inv_freq.data_ptr(), frequencies.scale, inverse, batch, tokens, head_dim, rotary_dim)
    if code:
        _native.check(code, "fpx_rotary")
    return q_ret, k_ret


def _apply(q, k, positions, frequencies, layout, inverse, q_out, k_out):
    if _native.differentiated(q, k, q_out, k_out):
        raise ValueError("no autograd graph is recorded: call without gradients "
                         "(torch.no_grad, detach); rotary_backward gives the gradients")
    outs = _launch(q, k, positions, frequencies, layout, inverse, q_out, k_out)
    return outs[0] if k is None else outs


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                 frequencies: RotaryFrequencies, *, layout: str = "half",
                 q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """``(q', k')``, or ``q'`` alone where ``k`` is None.

    ``q`` ``[batch, tokens, q_heads, head_dim]`` and ``k`` ``[batch, tokens,
    k_heads, head_dim]`` (or both without the batch axis) in any non-negative
    strides: views of a fused projection, head-first tensors transposed, a
    channel slice of wider heads.  ``positions`` ``[batch, tokens]`` or
    ``[tokens]``, int32 or int64.  ``q_out=q, k_out=k`` works in place; an output
    that shares an element with anything else is refused, views of one buffer that
    only interleave are not.

    As every operator here it records no autograd graph (tensors that require
    a gradient are refused under grad mode, those with a forward-mode tangent
    always): a training step calls
    ``rotary_backward`` from its own ``torch.autograd.Function``, or directly.
    """
    return _apply(q, k, positions, frequencies, layout, False, q_out, k_out)


def rotary_backward(grad_q: torch.Tensor, grad_k: torch.Tensor | None, positions: torch.Tensor,
                    frequencies: RotaryFrequencies, *, layout: str = "half",
                    q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """Gradients of ``apply_rotary``'s inputs from those of its outputs: the
    same arguments, the angles negated."""
    return _apply(grad_q, grad_k, positions, frequencies, layout, True, q_out, k_out)

"""Rotary positions in their general form: half and interleaved layouts, part of
the head, tables scaled for long contexts, forward and backward.

CUDA tensors go to the kernel (csrc/kernels/rotary.cu), CPU tensors to the
reference math in :mod:`turbol_b200.ops.reference`.  ``ops.rope`` is the older
in-place kernel of the decoder's default (bf16, half layout, whole head).
"""
from __future__ import annotations

import functools
import math
from typing import Optional

import torch

from .._native import core as _core
from . import reference as ref


def rotary_inv_freq(rot_dim: int, theta: float = 1e4, scaling: Optional[dict] = None):
    """(inverse frequencies fp64 [rot_dim / 2], factor on cos and sin).

    ``scaling`` stretches them for contexts beyond the trained length:

    * ``{"type": "linear", "factor": f}``: every frequency / f;
    * ``{"type": "ntk", "factor": f}``: theta * f^(R / (R - 2)), so that the
      lowest frequency is divided by f and the highest kept;
    * ``{"type": "llama3", "factor": f, "low_freq_factor": a, "high_freq_factor": b,
      "original_max_pos": n}``: kept above b turns over n positions, / f below a,
      mixed linearly (in turns) between;
    * ``{"type": "yarn", "factor": f, "original_max_pos": n, "beta_fast": 32,
      "beta_slow": 1, "attention_factor": m}``: kept above beta_fast turns, / f
      below beta_slow, mixed linearly (in the dimension's index) between; cos
      and sin times m (default 0.1 ln f + 1)."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rotary: an even rotary dimension of at least 2, not {rot_dim}")
    if not theta > 0:
        raise ValueError(f"rotary: theta is positive, not {theta}")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    inv = theta ** (-i / rot_dim)
    if not scaling:
        return inv, 1.0
    kind, f = scaling.get("type"), float(scaling.get("factor", 1.0))
    if not f >= 1.0:
        raise ValueError(f"rotary: a scaling factor of at least 1, not {f}")
    if kind == "linear":
        return inv / f, 1.0
    if kind == "ntk":
        if rot_dim < 4:
            raise ValueError("rotary: NTK scaling needs a rotary dimension of at least 4")
        return (theta * f ** (rot_dim / (rot_dim - 2))) ** (-i / rot_dim), 1.0
    if kind in ("llama3", "yarn"):
        n = scaling.get("original_max_pos")
        if not n:
            raise ValueError(f"rotary: {kind} scaling needs original_max_pos")
    if kind == "llama3":
        lo, hi = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
        if not (hi > lo and n > 0):
            raise ValueError("rotary: llama3 scaling needs high_freq_factor above low_freq_factor and a positive "
                             "original_max_pos")
        keep = ((n * inv / (2 * math.pi) - lo) / (hi - lo)).clamp(0, 1)
        return inv * (keep + (1 - keep) / f), 1.0
    if kind == "yarn":
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
        if not (fast >= slow > 0 and theta > 1 and n > 0):
            raise ValueError("rotary: yarn scaling needs beta_slow above 0 and not above beta_fast, theta above 1 and a "
                             "positive original_max_pos")

        def index_of(turns):  # the (fractional) pair index that makes this many turns over n positions
            return rot_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo = max(math.floor(index_of(fast)), 0)
        hi = min(math.ceil(index_of(slow)), rot_dim - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        m = scaling.get("attention_factor")
        return inv * (1 - ramp) + inv / f * ramp, float(0.1 * math.log(f) + 1.0 if m is None else m)
    raise ValueError(f"rotary: unknown scaling type {kind!r}")


def rotary_table(rot_dim: int, max_pos: int, theta: float = 1e4, scaling: Optional[dict] = None,
                 device="cuda") -> torch.Tensor:
    """fp32 [max_pos, rot_dim / 2, 2] of (cos, sin); the angles are formed in 64
    bits, so far positions keep their phase."""
    if max_pos < 1:
        raise ValueError("rotary_table: at least one position")
    inv, m = rotary_inv_freq(rot_dim, theta, scaling)
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv[None, :]
    return (torch.stack([torch.cos(ang), torch.sin(ang)], -1) * m).to(device=device, dtype=torch.float32).contiguous()


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    c = _core()
    return getattr(c.ops if hasattr(c, "ops") else c.host_ops, name)


def _call(name: str, *args):
    """A kernel entry point: checks, launches and returns its result; None for CPU tensors."""
    return _entry(name)(*args)


def _apply(x, pos, table, interleaved, transpose, out, error):
    y = _call("rotary", x, pos, table, out, interleaved, transpose, error)
    if y is None:
        y = ref.rotary(x, pos, table, interleaved, transpose, torch.empty_like(x) if out is None else out, error)
    return y if out is None else out


class _Rotary(torch.autograd.Function):
    """The differentiable form for CPU tensors."""

    @staticmethod
    def forward(ctx, x, pos, table, interleaved, transpose, error):
        ctx.save_for_backward(pos, table)
        ctx.how = (interleaved, transpose, error)
        return _apply(x, pos, table, interleaved, transpose, None, error)

    @staticmethod
    def backward(ctx, dy):
        pos, table = ctx.saved_tensors
        interleaved, transpose, error = ctx.how
        if dy.dim() == 3 and dy.stride(2) != 1:  # a broadcast gradient
            dy = dy.contiguous()
        # the transpose of a rotation (times the table's factor) is linear too
        return _Rotary.apply(dy, pos, table, interleaved, not transpose, error), None, None, None, None, None


def rotary(x: torch.Tensor, pos: torch.Tensor, table: torch.Tensor, interleaved: bool = False,
           transpose: bool = False, out: Optional[torch.Tensor] = None,
           error: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates the first R = 2 * table.shape[1] dimensions of x [T, H, D] (bf16,
    fp16 or fp32; any row and head strides) by the rows of ``table``
    (:func:`rotary_table`) that the int32 positions ``pos`` [T] name, in fp32
    with one rounding; the other dimensions are copied.

    interleaved: pairs (2i, 2i + 1) instead of (i, i + R / 2).  transpose: the
    backward's rotation (by the negative angles).  Differentiable in x, backward or
    in forward mode (not both at once), unless ``out`` is given (x itself for
    in-place use, or a tensor that does not overlap it); a table that requires a
    gradient is refused.  A row with a negative position is padding and copied
    unrotated; one at or beyond the table's end becomes NaN and sets ``error``
    (an int32 device tensor, optional) to 1."""
    if out is None:
        if x.requires_grad and torch.is_grad_enabled():
            if x.is_cuda:
                return _core().ops.rotary_grad(x, pos, table, interleaved, transpose, error)
            if table.requires_grad:
                raise ValueError("rotary: the table has no gradient (call it under torch.no_grad)")
            return _Rotary.apply(x, pos, table, interleaved, transpose, error)
    elif torch.is_grad_enabled() and (x.requires_grad or out.requires_grad):
        raise ValueError("rotary: out= has no gradient")
    return _apply(x, pos, table, interleaved, transpose, out, error)

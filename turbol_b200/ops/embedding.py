"""The embedding lookup with a scale, and its gradient as sums over sorted tokens.

``ops.embed_fwd`` / ``ops.embed_bwd`` are the older kernels (bf16 rows, no scale; a
gradient by atomics, whose last bits differ from run to run).  Here the gradient of a
row is summed in fp32 in the order of its tokens (long runs of one token in pieces of a
fixed length), so the same inputs give the same bits.  The decoder's gradient is this one.

CUDA tensors go to the kernels (csrc/kernels/embedding.cu), CPU tensors to the reference
math in :mod:`turbol_b200.ops.reference`.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import reference as ref
from .rotary import _call


class _Embedding(torch.autograd.Function):
    """The differentiable form for CPU tensors."""

    @staticmethod
    def forward(ctx, weight, ids, scale, error):
        ctx.save_for_backward(ids)
        ctx.how = (scale, weight.shape)
        return ref.embedding(ids, weight, scale, None, error)

    @staticmethod
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        scale, shape = ctx.how
        return _EmbeddingGrad.apply(dy, ids, scale, shape), None, None, None


class _EmbeddingGrad(torch.autograd.Function):
    """The gradient as a function of dy."""

    @staticmethod
    def forward(ctx, dy, ids, scale, shape):
        ctx.save_for_backward(ids)
        ctx.scale = scale
        return ref.embedding_grad(ids, dy, torch.empty(shape, dtype=dy.dtype), scale, False)

    @staticmethod
    def backward(ctx, g):
        return _Embedding.apply(g, ctx.saved_tensors[0], ctx.scale, None), None, None, None


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, out: Optional[torch.Tensor] = None,
              error: Optional[torch.Tensor] = None, first_row: bool = False) -> torch.Tensor:
    """scale * weight[ids] [*ids.shape, H] for ids of any shape (int32 or int64, contiguous) and
    rows ``weight`` [V, H] (bf16, fp16 or fp32; any row stride), rounded once.

    A negative id is padding: a row of zeros, without a gradient.  An id past the last
    row gives NaN, no gradient, and sets ``error`` (an int32 device tensor, optional) to 1.
    ``first_row``: ids outside the table, negative ones too, read row 0 instead and set ``error``,
    as ``ops.embed_fwd`` does (not with a gradient).
    Differentiable in ``weight`` (a dense gradient of its type), unless ``out`` is given."""
    if out is None and not first_row and weight.requires_grad and torch.is_grad_enabled():
        if weight.is_cuda:
            return _call("embedding_autograd", ids, weight, scale, error)
        _call("embedding", ids, weight, scale, None, error)  # the checks
        return _Embedding.apply(weight, ids, scale, error)
    y = _call("embedding", ids, weight, scale, out, error, first_row)
    if y is None:
        y = ref.embedding(ids, weight, scale, out, error, first_row)
    return y if out is None else out


def embedding_grad(ids: torch.Tensor, dy: torch.Tensor, grad: torch.Tensor, scale: float = 1.0,
                   accumulate: bool = True, error: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Adds scale * sum of the rows dy[t] with ids[t] == v to row v of ``grad`` [V, H] (bf16,
    fp16 or fp32; any row stride) and returns it, for training loops without autograd; dy
    [*ids.shape, H] (bf16, fp16 or fp32).  The sum is formed in fp32, in token order, and
    added with one rounding.  accumulate=False: grad is overwritten, rows that no id names
    with zeros.  Negative ids are padding; ids past the last row are left out and set
    ``error``.  (fp32 rows: values below 2^-126 may be added as zero.)"""
    if not _call("embedding_grad", ids, dy, grad, scale, accumulate, error):
        ref.embedding_grad(ids, dy, grad, scale, accumulate, error)
    return grad

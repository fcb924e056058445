"""Distillation from a teacher's top logits: the teacher's list of each row, and
the student's loss on it with the gradient.

The list of a row are ids a_k and log-probabilities l_k (:func:`topk_logprobs`,
or any other source); t_k = exp(l_k), S the set of the ids.  With p =
softmax(z / T) of the student's row and, where ``rest`` is on, everything outside
the list as one more class of mass t_R = 1 - sum t_k (teacher) and p_R (student):

* ``kind="forward"``: KL(t || p) = sum_k t_k (l_k - log p_{a_k}) + t_R (log t_R - log p_R);
  without ``rest`` the t_k are divided by their sum and the last term is gone.
* ``kind="reverse"`` (with ``rest``): KL(p || t) = sum_k p_{a_k} (log p_{a_k} - l_k) +
  p_R (log p_R - log t_R), t_R at least 2^-20 (what fp32 log-probabilities can tell from none).

A row counts weight * KL, plus target_weight * -log p[target] where a target is
given (a label, or a sampled token with minus its policy gradient).

Entries with a negative id or l_k = -inf are padding.  An id that occurs more than
once counts with the sum of its t_k.  Ids and targets past the vocabulary are left out
and set ``error`` (an int32 device tensor, optional) to 1; a negative target is none.
Rows whose weights are 0 are not read: loss 0, gradient 0, whatever the logits hold.
In a row with weight, NaN, +inf or no logit above -inf give NaN.  A student without
any mass outside the list (all its logits there -inf) leaves out the p_R term.
Log-probabilities are held in fp32: a logit whose distance to the row's largest, over
T, passes 3.4e38 (a mask of bf16's or fp32's lowest value with T < 1) counts as -inf.

CUDA tensors go to the kernels (csrc/kernels/topk_logprobs.cu,
csrc/kernels/distill.cu), CPU tensors to the reference math in
:mod:`turbol_b200.ops.reference`.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import reference as ref
from .rotary import _call


class TopLogprobs(NamedTuple):
    logprobs: torch.Tensor
    ids: torch.Tensor
    lse: torch.Tensor


def topk_logprobs(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogprobs:
    """The k (up to 256) largest logits of each row of ``logits`` [R, V] (bf16, fp16 or
    fp32; any row stride, V up to 2^20), largest first, equal ones by the lowest id:
    (log_softmax(logits / temperature) there fp32 [R, k], ids int32 [R, k],
    log-sum-exps of logits / temperature fp32 [R]).  NaN ranks as -inf and makes the
    row's numbers NaN; a row without a logit above -inf gives -inf.  Not
    differentiable (refused outside torch.no_grad)."""
    y = _call("topk_logprobs", logits, k, temperature)
    if y is None:
        y = ref.topk_logprobs(logits, k, temperature)
    return TopLogprobs(*y)


def distill_loss_grad(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor,
                      weight: Optional[torch.Tensor] = None, kind: str = "forward", rest: bool = True,
                      temperature: float = 1.0, target: Optional[torch.Tensor] = None,
                      target_weight: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                      error: Optional[torch.Tensor] = None,
                      kl: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss fp32 [R], its gradient: d loss[r] / d logits[r] in logits' type) of the rows
    ``logits`` [R, V] (bf16, fp16 or fp32; any row stride), for training loops without
    autograd.  ids int32 [R, K], logprobs fp32 [R, K] (K up to 256); weight,
    target_weight fp32 [R] (None: ones), target int32 [R].  ``out`` receives the
    gradient (logits itself for in-place use), ``kl`` (fp32 [R]) the rows' KL without weight
    or target (0 where weight is 0)."""
    y = _call("distill_loss_grad", logits, ids, logprobs, weight, kind, rest, temperature, target, target_weight, out,
              error, kl)
    if y is None:
        y = ref.distill(logits, ids, logprobs, weight, kind, rest, temperature, target, target_weight, error, out_kl=kl)
        y = (y[0], y[1] if out is None else out.copy_(y[1]))
    return (y[0], y[1] if out is None else out)


class _Distill(torch.autograd.Function):
    """The differentiable form for CPU tensors."""

    @staticmethod
    def forward(ctx, logits, *args):
        loss, d = ref.distill(logits, *args, dtype=torch.float64)
        ctx.save_for_backward(d)
        ctx.type = logits.dtype
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        return ((ctx.saved_tensors[0] * dloss.double()[:, None]).to(ctx.type),) + (None,) * 9


def distill_loss(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor,
                 weight: Optional[torch.Tensor] = None, kind: str = "forward", rest: bool = True,
                 temperature: float = 1.0, target: Optional[torch.Tensor] = None,
                 target_weight: Optional[torch.Tensor] = None, error: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The loss fp32 [R] of :func:`distill_loss_grad`, differentiable once in ``logits``
    (lists and weights that require a gradient are refused)."""
    args = (ids, logprobs, weight, kind, rest, temperature, target, target_weight, error)
    grad = logits.requires_grad and torch.is_grad_enabled()
    y = _call("distill_loss_autograd" if grad and logits.is_cuda else "distill_loss", logits, *args)
    if y is None:
        y = _Distill.apply(logits, *args) if grad else ref.distill(logits, *args)[0]
    return y

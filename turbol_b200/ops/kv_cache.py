"""The 8-bit paged KV cache of the rollout: rows quantised as they are written
(with rotary positions of q and k in the same launch where wanted), read back,
and the attention of one new token per sequence over them.

A cache is four tensors (:func:`quant_kv_cache`): codes ``kc`` / ``vc``
float8_e4m3fn [num_blocks, Hk, block_size, D] and scales ``ks`` / ``vs`` fp32
[num_blocks, Hk, block_size]; a value is code * scale, with the scale chosen per
token and KV head, so that the largest of the row's D values maps to code 448.
The slot of position p of sequence s is (block_table[s, p // block_size],
p % block_size).  Against bf16 pages this is 0.52 of the bytes at D = 128.

CUDA tensors go to the kernels (csrc/kernels/kv_quant.cu,
csrc/kernels/decode_attn_quant.cu), CPU tensors to the reference math in
:mod:`turbol_b200.ops.reference`.  ``error`` is an optional int32 device tensor
that a kernel sets to 1 when it meets an index out of range.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import reference as ref
from .rotary import _call


class QuantKV(NamedTuple):
    kc: torch.Tensor
    vc: torch.Tensor
    ks: torch.Tensor
    vs: torch.Tensor


def quant_kv_cache(num_blocks: int, n_kv_heads: int, block_size: int, head_dim: int, device="cuda") -> QuantKV:
    """An empty cache (codes and scales zero)."""
    if head_dim not in (64, 128, 256):
        raise ValueError(f"quant_kv_cache: head dimension 64, 128 or 256, not {head_dim}")
    if num_blocks < 1 or n_kv_heads < 1 or block_size < 1:
        raise ValueError("quant_kv_cache: at least one block, KV head and slot")
    shape = (num_blocks, n_kv_heads, block_size)
    codes = [torch.zeros(*shape, head_dim, device=device, dtype=torch.uint8).view(torch.float8_e4m3fn)
             for _ in range(2)]
    return QuantKV(*codes, *(torch.zeros(shape, device=device) for _ in range(2)))


def kv_quant_write(k: torch.Tensor, v: torch.Tensor, seq_of_token: torch.Tensor, pos: torch.Tensor,
                   block_table: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor,
                   q: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None, interleaved: bool = False,
                   q_out: Optional[torch.Tensor] = None, error: Optional[torch.Tensor] = None):
    """Quantises the rows k, v [T, Hk, D] (bf16, fp16 or fp32; any row and head
    strides) into the slots that (seq_of_token, pos) (int32 [T]) name.

    With ``table`` (:func:`~turbol_b200.ops.rotary.rotary_table`, a multiple of 8
    rotated dimensions) k is rotated by its position first, unrounded, and left
    as it was; with ``q`` [T, Hq, D] too, q is rotated into ``q_out`` (new if not
    given; q itself for in-place use), which is returned.

    A token with a negative position or sequence is padding: nothing is written
    and its q row is copied.  A sequence, position or block out of range writes
    nothing and sets ``error``; a position beyond the table also makes the q row
    NaN.  No two tokens of a call may name the same slot.  Not differentiable:
    tensors that require a gradient are refused outside torch.no_grad, tangents of
    forward mode always."""
    y = _call("kv_quant_write", k, v, seq_of_token, pos, block_table, kc, vc, ks, vs, q, q_out, table, interleaved, error)
    if not kc.is_cuda:
        y = torch.empty_like(q) if q is not None and q_out is None else q_out
        ref.kv_quant_write(k, v, seq_of_token, pos, block_table, kc, vc, ks, vs, q, table, interleaved, y, error)
    return y if q_out is None else q_out


def kv_quant_read(kc: torch.Tensor, vc: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor, seq_of_token: torch.Tensor,
                  pos: torch.Tensor, block_table: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                  out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, error: Optional[torch.Tensor] = None):
    """(k, v) [T, Hk, D] of the tokens that (seq_of_token, pos) (int32 [T]) name:
    code * scale, rounded once to ``dtype`` (bf16, fp16, fp32).  ``out``: the
    pair to write into (its type counts); rows of padding tokens (a negative
    position or sequence) are left as they were there, and zero in new tensors.
    Indexes out of range count as padding and set ``error``."""
    if out is None:
        shape = (pos.shape[0], kc.shape[1], kc.shape[3])
        out = (torch.zeros(shape, dtype=dtype, device=kc.device), torch.zeros(shape, dtype=dtype, device=kc.device))
    if not _call("kv_quant_read", kc, vc, ks, vs, seq_of_token, pos, block_table, out[0], out[1], error):
        ref.kv_quant_read(kc, vc, ks, vs, seq_of_token, pos, block_table, out, error)
    return out


def decode_attention_quant(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor,
                           block_table: torch.Tensor, ctx_len: torch.Tensor, scale: Optional[float] = None,
                           out: Optional[torch.Tensor] = None, error: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one token per sequence, q [B, Hq, D] (bf16 or fp16), over the
    first ctx_len[b] (int32) tokens of row b of ``block_table``: [B, Hq, D], q's
    type, without a backward pass (as :func:`kv_quant_write`).  Query head h reads
    KV head h // (Hq / Hk).  scale: default 1 / sqrt(D).  An empty context gives
    zeros, one whose scores are all -inf gives NaN.  Tokens behind the table or in
    blocks out of range are left out and set ``error``.  Weights are rounded to
    fp16 (sums stay in fp32).  The result does not depend on what the pages hold
    behind a context; it can depend, within rounding, on the other sequences of the
    batch (where contexts are split)."""
    y = _call("decode_attention_quant", q, kc, vc, ks, vs, block_table, ctx_len, out, scale, error)
    if y is None:
        y = ref.decode_attention_quant(q, kc, vc, ks, vs, block_table, ctx_len,
                                       1.0 / math.sqrt(q.shape[-1]) if scale is None else scale,
                                       torch.empty_like(q) if out is None else out, error)
    return y if out is None else out

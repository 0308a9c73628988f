"""Attention that trains: ragged batches with grouped heads, windows, first tokens that stay visible, and a learned bias by
distance, with its backward pass.

A layer of a model over users' histories, in training and when it recomputes its keys:

    q, k = rope(q, k, positions)                              # QKNormRope, where there is one
    bias = rel()                                              # RelativeBias: [heads, distances]
    out = jagged_attention(q, k, v, cu_seqlens, window=1024, sinks=4, bias=bias, bias_start=rel.start)

and serving the same model over a cache of its keys and values, with the same three:

    out = cache.attend(q, cu_seqlens, page_table, seq_lens, window=1024, sinks=4, bias=bias, bias_start=rel.start)

:func:`jagged_attention` and :func:`bucket_bias` are functions of tensors; no call waits for the device, and each may be captured
into a HIP graph.  No counterpart in the reference: its attention (primus_dlrm/models/onetrans.py:85-169) is dense and takes
positions from an embedding.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn

from . import ops
from .kv_cache import _fp32, _heads, _no_tangent, _traced

__all__ = ["jagged_attention", "bucket_bias", "relative_buckets", "RelativeBias"]


class _JaggedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, cu_seqlens_k, bias, scale, causal, window, sinks, bias_start, return_lse, err_flag):
        keep = 2 if ctx.needs_input_grad[5] else 1
        out, lse, stats, rest = ops.jagged_attention_raw(q, k, v, cu_seqlens, cu_seqlens_k, bias, scale, causal, window, sinks,
                                                         bias_start, return_lse, keep, err_flag)
        ctx.save_for_backward(q, k, v, cu_seqlens, cu_seqlens_k, bias, out, stats, rest)
        ctx.args = scale, causal, window, sinks, bias_start
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out, grad_lse):
        q, k, v, cu_seqlens, cu_seqlens_k, bias, out, stats, rest = ctx.saved_tensors
        if grad_out is None:
            grad_out = torch.zeros_like(out)
        grads = ops.jagged_attention_backward_raw(q, k, v, cu_seqlens, cu_seqlens_k, bias, out, stats, rest, grad_out,
                                                  grad_lse, *ctx.args)
        gq, gk, gv, gb = (g if ctx.needs_input_grad[i] else None for g, i in zip(grads, (0, 1, 2, 5)))
        return gq, gk, gv, None, None, gb, None, None, None, None, None, None, None


def jagged_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     cu_seqlens_k: Optional[torch.Tensor] = None, *, scale: Optional[float] = None, causal: bool = True,
                     window: int = 0, sinks: int = 0, bias: Optional[torch.Tensor] = None, bias_start: int = 0,
                     return_lse: bool = False, err_flag: Optional[torch.Tensor] = None):
    """Attention of q [T, Hq, D] to k and v [S, Hk, D] (bf16 or fp16, D 64 or 128) of the same sequences; query head h reads key
    head ``h // (Hq / Hk)``.  Differentiable in q, k, v, the bias and (through the returned ``lse``) all of them.

    Sequence b's queries are rows ``cu_seqlens[b] : cu_seqlens[b + 1]``, its keys and values rows ``cu_seqlens_k[b] :
    cu_seqlens_k[b + 1]`` (default: the same; both int32 on the device).  The queries are its last tokens: query i of n_q
    stands at position ``p = n_k - n_q + i`` and sees the keys j with ``j <= p`` (``causal``) and, where ``window`` > 0, those with
    ``j > p - window`` or ``j < sinks``.  Scores are ``scale * q . k`` (default D^-1/2) plus ``bias[h, p - j - bias_start]``, the
    column held within [0, distances): bias [Hq, distances], fp32 or q's dtype (:func:`bucket_bias`), smaller distances than the
    first column's take that, larger ones the last's.

    Returns out [T, Hq, D], and with ``return_lse`` the fp32 logarithm of each row's sum of exponentials [T, Hq].  Rows that see no
    key (or only scores of -inf) and rows that no sequence covers are zeros, with lse -inf, and have and give no gradient.
    ``err_flag`` (int32, never cleared) is set where spans decrease or leave the batch; outputs then hold nothing of use.

    Where the bias wants a gradient, weights meet the values in two parts: outputs are nearer to exact ones than without, and not
    the same bits.  A recomputation that has to give the same bits runs with the same tensors requiring gradients.

    Before a backward pass is captured into a HIP graph, let go of eager outputs of the same leaves: torch accumulates their
    gradients on the stream that those were made on, which a capture does not survive."""
    _no_tangent("jagged_attention", q, k, v, bias)
    cu_k = cu_seqlens if cu_seqlens_k is None else cu_seqlens_k
    if bias is not None:
        if bias.dtype not in (torch.float32, q.dtype):
            raise TypeError(f"bias must be float32 or {q.dtype}, got {bias.dtype}")
        bias = _fp32(bias)
    shape, q, k, v = q.shape, _heads(q), _heads(k), _heads(v)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, bias))
    if _traced(q, direct=err_flag is not None):
        if err_flag is not None:
            raise ValueError("err_flag is not available in a compiled or traced graph")
        keep = 0 if not grad else 2 if bias is not None and bias.requires_grad else 1
        out, lse, _, _ = torch.ops.pdm.jagged_attention(q, k, v, cu_seqlens, cu_k, bias, scale, causal, window, sinks,
                                                        bias_start, keep)
    elif grad:
        out, lse = _JaggedAttention.apply(q, k, v, cu_seqlens, cu_k, bias, scale, causal, window, sinks, bias_start, return_lse,
                                          err_flag)
    else:
        out, lse, _, _ = ops.jagged_attention_raw(q, k, v, cu_seqlens, cu_k, bias, scale, causal, window, sinks, bias_start,
                                                  return_lse, 0, err_flag)
    if len(shape) != 3:
        out, lse = out.view(shape), lse.view(shape[:-1]) if return_lse else None
    return (out, lse) if return_lse else out


class _BucketBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, buckets):
        ctx.save_for_backward(buckets)
        ctx.num, ctx.dtype = table.shape[0], table.dtype
        return ops.bucket_bias_raw(table, buckets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        return ops.bucket_bias_backward_raw(grad_out, ctx.saved_tensors[0], ctx.num, ctx.dtype), None


def bucket_bias(table: torch.Tensor, buckets: torch.Tensor) -> torch.Tensor:
    """A table [num_buckets, heads] (fp32, fp16 or bf16) spread over distances: fp32 [heads, distances] with
    ``out[h, c] = table[buckets[c], h]`` (0 where the bucket is none of the table's).  buckets: int32 [distances], any map.
    Differentiable in the table; the gradient is summed in one fixed order and rounded once, to the table's dtype."""
    _no_tangent("bucket_bias", table)
    if _traced(table):
        return torch.ops.pdm.bucket_bias(table, buckets)
    if torch.is_grad_enabled() and table.requires_grad:
        return _BucketBias.apply(table, buckets)
    return ops.bucket_bias_raw(table, buckets)


def relative_buckets(num_buckets: int, max_distance: int, both_sides: bool = False, device=None) -> torch.Tensor:
    """Buckets of the distances 0 .. max_distance (``both_sides``: -max_distance .. max_distance), int32: the nearer half of them
    for one distance each, the others in logarithmic steps up to ``max_distance``.  With ``both_sides`` keys behind a query (positive
    distances and 0) have the first ``ceil(num_buckets / 2)`` buckets, keys ahead of it the others."""
    if num_buckets < (2 if both_sides else 1) or max_distance < 0:
        raise ValueError("relative_buckets needs a bucket for each side, and max_distance >= 0")

    def side(n, d):
        near = n // 2 if max_distance >= n else n
        if d < near or near == n:
            return min(d, n - 1)
        steps = math.log(d / near) / math.log((max_distance + 1) / near) if near else d / (max_distance + 1)
        return min(near + int((n - near) * steps), n - 1)

    n = (num_buckets + 1) // 2 if both_sides else num_buckets
    out = [side(n, d) for d in range(max_distance + 1)]
    if both_sides:
        out = [n + side(num_buckets - n, d - 1) for d in range(max_distance, 0, -1)] + out
    return torch.tensor(out, dtype=torch.int32, device=device)


class RelativeBias(nn.Module):
    """The learned bias of a layer's heads by distance: ``table`` [num_buckets, n_heads], spread by :func:`relative_buckets`.

    ``forward()`` gives the bias [n_heads, distances] that :func:`jagged_attention` and :func:`kv_attention` take together with
    ``start``, the distance of its first column (0, or -max_distance with ``both_sides``, for attention that is not causal).  A
    serving program spreads it once."""

    def __init__(self, n_heads: int, num_buckets: int = 32, max_distance: int = 128, both_sides: bool = False, device=None):
        super().__init__()
        self.num_buckets, self.max_distance, self.both_sides = num_buckets, max_distance, both_sides
        self.start = -max_distance if both_sides else 0
        self.table = nn.Parameter(torch.zeros(num_buckets, n_heads, device=device))
        self.register_buffer("buckets", relative_buckets(num_buckets, max_distance, both_sides, device), persistent=False)

    def _apply(self, fn, *args, **kwargs):
        empty = self.buckets.is_meta
        super()._apply(fn, *args, **kwargs)
        if empty and not self.buckets.is_meta:
            self.buckets = relative_buckets(self.num_buckets, self.max_distance, self.both_sides, self.buckets.device)
        return self

    def forward(self) -> torch.Tensor:
        return bucket_bias(self.table, self.buckets)

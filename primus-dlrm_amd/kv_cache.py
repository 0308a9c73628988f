"""Cached attention: query / key norms with rotation, an 8-bit paged key-value cache, and attention over it.

For models that keep a user's history between requests: the keys and values of the tokens a model has seen stay in the
pages of a :class:`PagedKVCache`, a request computes those of its new tokens alone (new events, the NS-tokens of a
candidate) and attends from them over everything the cache holds.  One step of a layer is

    q, _ = rope(q, None, positions)                           # QKNormRope: norm of each head, rotation
    cache.append(k, v, cu_seqlens, page_table, seq_lens, rope=rope)
    out = cache.attend(q, cu_seqlens, page_table, seq_lens)

and a model is trained with ``q, k = rope(q, k, positions)``, which has a backward pass.  :func:`qk_norm_rope`,
:func:`kv_append` and :func:`kv_attention` are the same as functions of tensors.  No call waits for the device: lengths,
page tables and positions are read there, and every call may be captured into a HIP graph and replayed with other
lengths in the same tensors.  No counterpart in the reference (its attention, primus_dlrm/models/onetrans.py:85-169,
recomputes all keys and values and takes its positions from an embedding).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import ops
from .onetrans import RMSNorm

__all__ = ["rotary_tables", "qk_norm_rope", "kv_append", "kv_attention", "QKNormRope", "PagedKVCache"]


def rotary_tables(max_positions: int, rotary_dim: int, theta: float = 10000.0, device=None
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin of ``position * theta^(-2 i / rotary_dim)``, fp32 [max_positions, rotary_dim / 2] each.  The angles are
    computed in 64 bits: in 32 a position of 100,000 would be off by 0.004 radians."""
    freq = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _heads(t: torch.Tensor) -> torch.Tensor:
    """[..., heads, D] -> [tokens, heads, D], a view wherever the strides allow one."""
    dims = t.dim()
    if dims != 3:
        if dims < 3:
            raise ValueError(f"expected [..., heads, head_dim], got {tuple(t.shape)}")
        t = t.flatten(0, -3)
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _traced(t: torch.Tensor, direct: bool = False) -> bool:
    """True where a call has to be seen by the dispatcher: in compiled and traced graphs, for tensors without memory (fake, meta)
    or with a dispatch of their own, and under a dispatch mode.  ``direct``: the call has an argument that the registered
    operator has not; a mode that records no graph then does without it."""
    if torch.compiler.is_compiling() or isinstance(t, torch.fx.Proxy):
        return True
    if t.is_meta or type(t).__torch_dispatch__ is not torch.Tensor.__torch_dispatch__ or torch._C._is_tracing():
        return True
    return torch._C._len_torch_dispatch_stack() > 0 and not (direct and get_proxy_mode() is None)


def _no_tangent(name: str, *tensors: Optional[torch.Tensor]) -> None:
    if forward_ad._current_level < 0 or torch.compiler.is_compiling():
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no forward-mode derivative: give it the primals of its inputs")


def _fp32(w: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return w if w is None or (w.dtype == torch.float32 and w.is_contiguous()) else w.float().contiguous()


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved, err_flag):
        q_out, k_out = ops.qk_norm_rope_raw(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved, err_flag)
        ctx.save_for_backward(q, k, positions, cos, sin, q_weight, k_weight)
        ctx.eps, ctx.interleaved = eps, interleaved
        return q_out, k_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_q_out, grad_k_out):
        q, k, positions, cos, sin, q_weight, k_weight = ctx.saved_tensors
        grads = ops.qk_norm_rope_backward_raw(q, k, positions, cos, sin, q_weight, k_weight, grad_q_out.contiguous(),
                                              None if k is None else grad_k_out.contiguous(), ctx.eps,
                                              ctx.interleaved)
        need = ctx.needs_input_grad
        gq, gk, gqw, gkw = (g if need[i] else None for g, i in zip(grads, (0, 1, 5, 6)))
        return gq, gk, None, None, None, gqw, gkw, None, None, None


def qk_norm_rope(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, cos: Optional[torch.Tensor],
                 sin: Optional[torch.Tensor], q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                 err_flag: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RMS norm of every head of q [..., Hq, D] and k [..., Hk, D] (k may be None), then the rotation of their first
    ``rotary_dim`` elements by the angles of each token's position; computed in fp32, rounded once to q's dtype (fp32,
    fp16 or bf16).  Differentiable in q, k and the weights.

    positions: int32 / int64, one for each token (q's leading dimensions); a negative one marks padding, whose rows and
    gradients are zeros, and so does one beyond the tables, which also sets ``err_flag`` (int32, never cleared).
    cos, sin: fp32 [positions, rotary_dim / 2] (:func:`rotary_tables`); None: no rotation.  ``interleaved``: pairs (2i,
    2i + 1) instead of (i, i + rotary_dim / 2).  q_weight, k_weight: [D], fp32 or q's dtype; None: no norm."""
    if (cos is not None and cos.requires_grad) or (sin is not None and sin.requires_grad):
        raise ValueError("cos and sin take no gradient")
    _no_tangent("qk_norm_rope", q, k, cos, sin, q_weight, k_weight)
    lead = q.shape[:-2]
    if positions.shape != lead:
        raise ValueError(f"positions must be {tuple(lead)}, one for each token, got {tuple(positions.shape)}")
    if k is not None and k.shape[:-2] != lead:
        raise ValueError(f"k must hold q's tokens {tuple(lead)}, got {tuple(k.shape)}")
    for n, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and w.dtype not in (torch.float32, q.dtype):
            raise TypeError(f"{n} must be float32 or {q.dtype}, got {w.dtype}")
    q3, k3 = _heads(q), None if k is None else _heads(k)
    pos = positions if len(lead) == 1 and positions.is_contiguous() else positions.reshape(-1).contiguous()
    qw, kw = _fp32(q_weight), _fp32(k_weight)
    if _traced(q, direct=err_flag is not None):
        if err_flag is not None:
            raise ValueError("err_flag is not available in a compiled or traced graph")
        q_out, k_out = torch.ops.pdm.qk_norm_rope(q3, k3, pos, cos, sin, qw, kw, eps, interleaved)
        k_out = None if k is None else k_out
    elif torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q3, k3, qw, kw)):
        q_out, k_out = _QkNormRope.apply(q3, k3, pos, cos, sin, qw, kw, eps, interleaved, err_flag)
    else:
        q_out, k_out = ops.qk_norm_rope_raw(q3, k3, pos, cos, sin, qw, kw, eps, interleaved, err_flag)
    if len(lead) != 1:
        q_out = q_out.view(*lead, *q_out.shape[1:])
        k_out = None if k is None else k_out.view(*lead, *k_out.shape[1:])
    return q_out, k_out


def _no_grad(name: str, *tensors: Optional[torch.Tensor]) -> None:
    _no_tangent(name, *tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() or detach its inputs")


def kv_append(k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor,
              v_scale: torch.Tensor, cu_seqlens: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, *,
              positions: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
              sin: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
              interleaved: bool = False, err_flag: Optional[torch.Tensor] = None) -> None:
    """Writes the new keys and values k, v [T, Hk, D] (fp32, fp16 or bf16) into an 8-bit paged cache, in place.

    k_codes, v_codes: float8_e4m3fn [pages, Hk, page_size, D], k_scale, v_scale: fp32 [pages, Hk] powers of two; a value
    is code * scale.  Sequence b's new tokens are rows ``cu_seqlens[b] : cu_seqlens[b + 1]``; with them it holds
    ``seq_lens[b]`` tokens, token i in slot ``i % page_size`` of page ``page_table[b, i // page_size]`` (all int32).  Rows
    behind ``cu_seqlens[-1]`` are ignored.  The keys are normed first where ``k_weight`` is given and rotated where cos
    and sin are, by ``positions`` [T] or else by each token's index in its sequence, as :func:`qk_norm_rope` does, and are
    rounded once, to their codes.

    A page's scale is the smallest power of two under which none of its values exceeds 448; where it grows, the codes that
    the page holds already are brought to it (exactly, but for the smallest).  NaN and infinities become NaN.  A page that
    is written belongs to one sequence of the call.  ``err_flag`` (int32) is set where spans, lengths, pages or positions
    do not fit; such tokens are left out."""
    _no_grad("kv_append", k, v, k_codes, v_codes, k_scale, v_scale, cos, sin, k_weight)
    kw = k_weight
    if kw is not None:
        if kw.dtype not in (torch.float32, k.dtype):
            raise TypeError(f"k_weight must be float32 or {k.dtype}, got {kw.dtype}")
        kw = _fp32(kw.detach())
    k, v = _heads(k), _heads(v)
    run = torch.ops.pdm.kv_append if _traced(k) else ops.kv_append_raw
    run(k, v, k_codes, v_codes, k_scale, v_scale, cu_seqlens, page_table, seq_lens, positions, cos, sin, kw, eps,
        interleaved, err_flag)


def kv_attention(q: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor,
                 v_scale: torch.Tensor, cu_seqlens: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, *,
                 scale: Optional[float] = None, causal: bool = True, window: int = 0,
                 max_q_len: Optional[int] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None,
                 err_flag: Optional[torch.Tensor] = None):
    """Attention of the new tokens q [T, Hq, D] (bf16 or fp16) over the cache, their own keys and values included (call
    :func:`kv_append` first).  Sequences and cache as there; query head h reads key head ``h // (Hq / Hk)``.  A query at
    index p of its sequence sees the keys up to p (``causal``) and none of ``window`` or more tokens before it (``window``
    > 0); ``scale`` defaults to D^-1/2.  Returns out [T, Hq, D], and with ``return_lse`` the fp32 logarithm of each row's
    sum of exponentials [T, Hq].  Rows that see no key and rows behind the last sequence are zeros, with lse -inf.

    ``max_q_len``: the most new tokens that any sequence has, where the program knows it (1 when decoding); a sequence
    with more is left out and sets ``err_flag``.  Without it the work is laid out for any share of the rows, and a decoding
    batch takes up to half as long again.  Slice ``page_table`` to the columns that the longest sequence needs: its
    width bounds the lengths the work is laid out for."""
    _no_grad("kv_attention", q, k_codes, v_codes, k_scale, v_scale, out)
    q = _heads(q)
    if _traced(q, direct=out is not None):
        if out is not None:
            raise ValueError("out is not available in a compiled or traced graph")
        out, lse = torch.ops.pdm.kv_attention(q, k_codes, v_codes, k_scale, v_scale, cu_seqlens, page_table, seq_lens,
                                              q.shape[-1] ** -0.5 if scale is None else scale, causal, window,
                                              q.shape[0] if max_q_len is None else max_q_len, return_lse, err_flag)
    else:
        out, lse = ops.kv_attention_raw(q, k_codes, v_codes, k_scale, v_scale, cu_seqlens, page_table, seq_lens, scale,
                                        causal, window, max_q_len, return_lse, out, err_flag)
    return (out, lse) if return_lse else out


class QKNormRope(nn.Module):
    """The norms (``q_norm.weight``, ``k_norm.weight``) and the rotation of a layer's queries and keys.

    ``forward(q, k, positions)`` is :func:`qk_norm_rope`; k may be None, where :meth:`PagedKVCache.append` norms and
    rotates the keys on their way into the cache.  The cos / sin tables stay fp32 when the module is cast.

    Before a backward pass is captured into a HIP graph, let go of eager outputs of the same parameters: torch
    accumulates their gradients on the stream that those were made on, which a capture does not survive."""

    def __init__(self, head_dim: int, max_positions: int, rotary_dim: Optional[int] = None, theta: float = 10000.0,
                 eps: float = 1e-6, interleaved: bool = False, norm: bool = True, device=None):
        super().__init__()
        self.head_dim, self.max_positions, self.theta = head_dim, max_positions, theta
        self.rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim % 16 or self.rotary_dim % 16 or not 0 <= self.rotary_dim <= head_dim:
            raise ValueError("head_dim and rotary_dim must be multiples of 16, rotary_dim at most head_dim")
        self.eps, self.interleaved = eps, interleaved
        self.q_norm = RMSNorm(head_dim, eps).to(device) if norm else None
        self.k_norm = RMSNorm(head_dim, eps).to(device) if norm else None
        cos, sin = rotary_tables(max_positions, self.rotary_dim, theta, device) if self.rotary_dim else (None, None)
        self.register_buffer("cos", cos, persistent=False)
        self.register_buffer("sin", sin, persistent=False)

    def _apply(self, fn, *args, **kwargs):
        empty = self.cos is not None and self.cos.is_meta
        super()._apply(fn, *args, **kwargs)
        if self.cos is not None and (self.cos.dtype != torch.float32 or (empty and not self.cos.is_meta)):
            self.cos, self.sin = rotary_tables(self.max_positions, self.rotary_dim, self.theta, self.cos.device)
        return self

    def forward(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                err_flag: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        qw = None if self.q_norm is None else self.q_norm.weight
        kw = None if self.k_norm is None or k is None else self.k_norm.weight
        return qk_norm_rope(q, k, positions, self.cos, self.sin, qw, kw, self.eps, self.interleaved, err_flag)


class PagedKVCache:
    """The pages of one layer's 8-bit keys and values on one device: codes (e4m3) [num_pages, n_kv_heads, page_size,
    head_dim] and a power-of-two scale for each (page, head).  Which page belongs to which sequence is the caller's page
    table.  ``err_flag`` collects what a call had to leave out (:meth:`check`)."""

    def __init__(self, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, device):
        if page_size not in (16, 32, 64, 128):
            raise ValueError(f"page_size must be 16, 32, 64 or 128, got {page_size}")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
        shape = (num_pages, n_kv_heads, page_size, head_dim)
        self.num_pages, self.page_size, self.n_kv_heads, self.head_dim = shape
        self.k_codes = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        self.v_codes = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        self.k_scale = torch.ones(shape[:2], dtype=torch.float32, device=device)
        self.v_scale = torch.ones(shape[:2], dtype=torch.float32, device=device)
        self.err_flag = torch.zeros(1, dtype=torch.int32, device=device)

    def append(self, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, page_table: torch.Tensor,
               seq_lens: torch.Tensor, *, rope: Optional[QKNormRope] = None,
               positions: Optional[torch.Tensor] = None) -> None:
        """:func:`kv_append` into this cache; ``rope`` norms and rotates the keys."""
        extra = {}
        if rope is not None:
            extra = dict(cos=rope.cos, sin=rope.sin, eps=rope.eps, interleaved=rope.interleaved,
                         k_weight=None if rope.k_norm is None else rope.k_norm.weight.detach())
        kv_append(k, v, self.k_codes, self.v_codes, self.k_scale, self.v_scale, cu_seqlens, page_table, seq_lens,
                  positions=positions, err_flag=self.err_flag, **extra)

    def attend(self, q: torch.Tensor, cu_seqlens: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, *,
               scale: Optional[float] = None, causal: bool = True, window: int = 0, max_q_len: Optional[int] = None,
               return_lse: bool = False):
        """:func:`kv_attention` over this cache."""
        return kv_attention(q, self.k_codes, self.v_codes, self.k_scale, self.v_scale, cu_seqlens, page_table, seq_lens,
                            scale=scale, causal=causal, window=window, max_q_len=max_q_len, return_lse=return_lse,
                            err_flag=self.err_flag)

    def values(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """The keys and values that the codes stand for, bf16 (exact) [num_pages, n_kv_heads, page_size, head_dim]."""
        return tuple((c.float() * s[:, :, None, None]).to(torch.bfloat16)
                     for c, s in ((self.k_codes, self.k_scale), (self.v_codes, self.v_scale)))

    def check(self) -> None:
        """Raises RuntimeError if any call had to leave something out (waits for the device), and clears the flag."""
        if int(self.err_flag.item()):
            self.err_flag.zero_()
            raise RuntimeError("a span, length, page id or position did not fit the batch, the page table, the cache or "
                               "the rotation tables: the tokens concerned were left out")

"""64-bit reference of the attention of ragged batches on the CPU, forward and backward, from the definition; and what its
tolerances are made of.  Pairs that are not seen are left out of every sum, not multiplied by zero."""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch


def seen_pairs(n, length, causal, window, sinks):
    """Truth values [n, length]: the keys that each of the last n tokens sees."""
    p, j = torch.arange(length - n, length)[:, None], torch.arange(length)[None]
    seen = torch.ones(n, length, dtype=torch.bool)
    if causal:
        seen &= j <= p
    if window:
        seen &= (j > p - window) | (j < sinks)
    return seen


def columns(n, length, span, start):
    p, j = torch.arange(length - n, length)[:, None], torch.arange(length)[None]
    return (p - j - start).clamp(0, span - 1)


def _mul(w, x, seen):
    """w @ x over seen pairs alone."""
    if torch.isfinite(x).all():
        return torch.where(seen, w, 0.0) @ x
    return torch.stack([w[r, seen[r]] @ x[seen[r]] if seen[r].any() else torch.zeros_like(x[0]) for r in range(len(w))])


def attention(q, k, v, cu_q, cu_k, scale, causal=True, window=0, sinks=0, bias=None, start=0, go=None, gl=None):
    """Values out, lse and, with the gradients go (of out) and gl (of lse, or None), dq, dk, dv, dbias.  For tolerances: per row
    serr (the largest sum of the sizes that a score is made of), mag (sum p |v|); and for the gradients sums of the errors that
    a dS has when its weight is off by a relative 1 (rel), its product by 1 (dp) or delta by 1 (delta), each times the other factor."""
    T, hq, D = q.shape
    g = hq // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    r = SimpleNamespace(out=torch.zeros_like(q), lse=torch.full((T, hq), -math.inf, dtype=torch.float64), mag=torch.zeros_like(q),
                        serr=torch.zeros(T, hq, dtype=torch.float64))
    if go is not None:
        go = go.double()
        r.dq, r.dk, r.dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        r.dbias = None if bias is None else torch.zeros_like(bias, dtype=torch.float64)
        r.t = SimpleNamespace(dv=torch.zeros_like(v), **{n + x: torch.zeros_like(y) for n in ("rel", "dp", "delta", "all", "one")
                                                        for x, y in (("q", q), ("k", k))})
        r.t.dbias = None if bias is None else {n: torch.zeros_like(r.dbias) for n in ("rel", "dp", "delta", "all")}
    for b in range(len(cu_q) - 1):
        a0, a1, b0, b1 = cu_q[b], cu_q[b + 1], cu_k[b], cu_k[b + 1]
        n, length = a1 - a0, b1 - b0
        if n == 0 or length == 0:
            continue
        seen = seen_pairs(n, length, causal, window, sinks)
        col = None if bias is None else columns(n, length, bias.shape[1], start)
        for h in range(hq):
            qh, kh, vh = q[a0:a1, h], k[b0:b1, h // g], v[b0:b1, h // g]
            s = qh @ kh.T * scale
            size = qh.abs() @ kh.nan_to_num(posinf=0, neginf=0).abs().T * abs(scale)
            if bias is not None:
                add = bias[h].double()[col]
                s, size = s + add, size + add.abs()
            s = torch.where(seen, s, -math.inf)
            m = s.amax(-1, keepdim=True)
            m = torch.where(torch.isinf(m) & (m < 0), 0.0, m)
            w = torch.where(seen, torch.exp(s - m), 0.0)
            total = w.sum(-1, keepdim=True)
            some = total != 0
            w = torch.where(some, w / torch.where(some, total, 1.0), 0.0)
            o = _mul(w, vh, seen)
            r.out[a0:a1, h] = o
            r.lse[a0:a1, h] = torch.where(some, m + total.log(), -math.inf)[:, 0]
            vabs = vh.nan_to_num(posinf=0, neginf=0).abs()
            mag = w.nan_to_num() @ vabs
            r.mag[a0:a1, h] = mag
            size = torch.where(seen & torch.isfinite(s), size, 0.0).nan_to_num()
            serr = size.amax(-1)
            r.serr[a0:a1, h] = serr
            if go is None:
                continue
            gh = go[a0:a1, h]
            delta = torch.where(some[:, 0], (gh * o).sum(-1), 0.0)
            if gl is not None:
                delta = delta - torch.where(some[:, 0], gl[a0:a1, h].double(), 0.0)
            dp = gh @ vh.T
            ds = torch.where(seen, w * (dp - delta[:, None]), 0.0)
            r.dv[b0:b1, h // g] += _mul(w.T, gh, seen.T)
            r.dq[a0:a1, h] = scale * _mul(ds, kh, seen)
            r.dk[b0:b1, h // g] += scale * _mul(ds.T, qh, seen.T)
            # the same sums over sizes of errors
            wn, kn, qn, gn = w.nan_to_num(), kh.nan_to_num(posinf=0, neginf=0).abs(), qh.nan_to_num(posinf=0, neginf=0).abs(), gh.nan_to_num(posinf=0, neginf=0).abs()
            dsn = ds.nan_to_num(posinf=0, neginf=0).abs()
            e_dp = torch.where(seen, wn * (gn @ vabs.T), 0.0)
            e_delta = torch.where(seen, wn * (gn * mag).sum(-1, keepdim=True), 0.0)
            if gl is not None:
                e_delta = e_delta + torch.where(seen, wn * gl[a0:a1, h].double().abs()[:, None], 0.0)
            e_rel = dsn * (1 + serr[:, None])
            t, sc = r.t, abs(scale)
            t.dv[b0:b1, h // g] += (wn * (1 + serr[:, None])).T @ gn
            for name, e in (("rel", e_rel), ("dp", e_dp), ("delta", e_delta), ("all", dsn), ("one", seen.double())):
                getattr(t, name + "q")[a0:a1, h] = sc * e @ kn
                getattr(t, name + "k")[b0:b1, h // g] += sc * e.T @ qn
                if bias is not None and name != "one":
                    t.dbias[name][h].index_add_(0, col.flatten(), e.flatten())
            if bias is not None:
                r.dbias[h].index_add_(0, col.flatten(), ds.flatten())
    return r

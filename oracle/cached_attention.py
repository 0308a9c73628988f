"""64-bit references of the cached-attention operators on the CPU: norm + rotation, append to 8-bit pages, attention.

Each works row by row, page by page or sequence by sequence from the definition, on torch float64 tensors; the
quantizer rounds to e4m3 by arithmetic on the value, not by a cast."""
from __future__ import annotations

import math

import torch

E_MIN, E_MAX, E4M3_MAX = -117, 119, 448.0


def norm_rope(x, weight, positions, cos, sin, eps, interleaved):
    """x [T, H, D]; cos, sin [P, R/2] or None.  Rows of a position outside the tables are zeros."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    if cos is None:
        return torch.where((positions >= 0)[:, None, None], x, torch.zeros_like(x))
    ok = (positions >= 0) & (positions < len(cos))
    p = positions.clamp(0, max(len(cos) - 1, 0)).long()
    c, s = cos.double()[p][:, None], sin.double()[p][:, None]
    R = 2 * cos.shape[1]
    y = x.clone()
    ia = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    ib = ia + 1 if interleaved else ia + R // 2
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return torch.where(ok[:, None, None], y, torch.zeros_like(y))


def scale_exponent(amax: float) -> int:
    """Smallest e in [E_MIN, E_MAX] with amax <= 448 * 2^e (E_MAX where none is)."""
    if amax <= 0:
        return E_MIN
    e = math.floor(math.log2(amax / E4M3_MAX)) - 1
    while amax > E4M3_MAX * 2.0 ** e:
        e += 1
    return min(max(e, E_MIN), E_MAX)


def round_e4m3(x):
    """The nearest e4m3 value, ties to even, saturating; NaN and infinities to NaN."""
    bad = ~torch.isfinite(x)
    x = torch.where(bad, torch.zeros_like(x), x).clamp(-E4M3_MAX, E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.where(bad, torch.full_like(x, math.nan), (x / step).round() * step)


def append(x, codes, scale, cu, table, lens):
    """x [T, H, D] float64 (already normed and rotated) into codes [pages, H, page, D] and scale [pages, H] (float64
    values), in place."""
    page = codes.shape[2]
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        start = lens[b] - n
        for i in range(n):
            if i and (start + i) % page:
                continue  # a segment begins with its first token or a page
            slot = (start + i) % page
            m = min(page - slot, n - i)
            p = table[b][(start + i) // page]
            part = x[cu[b] + i:cu[b] + i + m]
            for h in range(x.shape[1]):
                v = part[:, h]
                fin = v[torch.isfinite(v)].abs()
                e = scale_exponent(fin.max().item() if fin.numel() else 0.0)
                if slot:
                    held = int(math.log2(scale[p, h].item()))
                    if e > held:
                        codes[p, h, :slot] = round_e4m3(codes[p, h, :slot] * 2.0 ** (held - e))
                    e = max(e, held)
                scale[p, h] = 2.0 ** e
                codes[p, h, slot:slot + m] = round_e4m3(v * 2.0 ** -e)


def attention(q, k_val, v_val, cu, table, lens, scale, causal, window):
    """q [T, Hq, D]; k_val, v_val [pages, Hk, page, D] (the values that the codes stand for).  Returns out, lse, and for
    tolerances mag = sum_j p_j |v_j| and serr = the largest scale * sum_d |q_d k_jd| of a row."""
    T, hq, D = q.shape
    hk, page = k_val.shape[1], k_val.shape[2]
    out = torch.zeros(T, hq, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64)
    serr = torch.zeros(T, hq, dtype=torch.float64)
    q = q.double()
    for b in range(len(lens)):
        n, length = cu[b + 1] - cu[b], lens[b]
        if n <= 0:
            continue
        ids = [(j, table[b][j // page], j % page) for j in range(length)
               if j // page < len(table[b]) and 0 <= table[b][j // page] < len(k_val)]
        if not ids:
            continue
        j = torch.tensor([i[0] for i in ids])
        at, slot = torch.tensor([i[1] for i in ids]), torch.tensor([i[2] for i in ids])
        p = torch.arange(length - n, length)[:, None]
        seen = torch.ones(n, len(ids), dtype=torch.bool)
        if causal:
            seen &= j[None] <= p
        if window:
            seen &= j[None] > p - window
        for h in range(hk):
            k, v = k_val[at, h, slot].double(), v_val[at, h, slot].double()
            for g in range(h * (hq // hk), (h + 1) * (hq // hk)):
                qr = q[cu[b]:cu[b + 1], g]
                s = torch.where(seen, qr @ k.T * scale, torch.full((), -math.inf, dtype=torch.float64))
                m = s.amax(-1, keepdim=True)
                m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
                w = torch.where(seen, torch.exp(s - m), torch.zeros_like(s))
                total = w.sum(-1, keepdim=True)
                some = seen.any(-1, keepdim=True)
                w = w / torch.where(some, total, torch.ones_like(total))
                # a weight of zero beside a value that is not seen: leave the value out
                if torch.isfinite(v).all() and torch.isfinite(s[seen]).all():
                    o = w @ v
                else:
                    o = torch.stack([w[r, seen[r]] @ v[seen[r]] if seen[r].any() else torch.zeros(D, dtype=torch.float64)
                                     for r in range(n)])
                out[cu[b]:cu[b + 1], g] = o
                mag[cu[b]:cu[b + 1], g] = w.nan_to_num() @ v.nan_to_num().abs()
                lse[cu[b]:cu[b + 1], g] = torch.where(some, m + total.log(), -math.inf)[:, 0]
                sa = torch.where(seen, qr.abs() @ k.nan_to_num().abs().T * abs(scale), 0.0)
                serr[cu[b]:cu[b + 1], g] = sa.amax(-1)
    return out, lse, mag, serr

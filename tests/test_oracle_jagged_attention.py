"""The 64-bit reference of the attention of ragged batches against a dense softmax, and its gradients against differences."""
import math

import pytest
import torch

from oracle import jagged_attention as ref


def _case(seed, hq=4, hk=2, D=8, new=(5, 0, 3), lens=(9, 4, 3), span=4):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    cu_q, cu_k = [0], [0]
    for a, b in zip(new, lens):
        cu_q.append(cu_q[-1] + a)
        cu_k.append(cu_k[-1] + b)
    return rand(cu_q[-1], hq, D), rand(cu_k[-1], hk, D), rand(cu_k[-1], hk, D), rand(hq, span), cu_q, cu_k, rand


MASKS = [dict(causal=True), dict(causal=False), dict(causal=True, window=2), dict(causal=True, window=2, sinks=1),
         dict(causal=False, window=3, sinks=2)]


@pytest.mark.parametrize("mask", MASKS)
def test_against_a_dense_softmax(mask):
    q, k, v, bias, cu_q, cu_k, _ = _case(1)
    start = 0 if mask["causal"] else -2
    got = ref.attention(q, k, v, cu_q, cu_k, 0.3, bias=bias, start=start, **mask)
    for b in range(3):
        n, length = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        for i in range(n):
            p = length - n + i
            keys = [j for j in range(length) if (not mask["causal"] or j <= p)
                    and (not mask.get("window") or j > p - mask["window"] or j < mask.get("sinks", 0))]
            for h in range(4):
                s = torch.stack([0.3 * (q[cu_q[b] + i, h] * k[cu_k[b] + j, h // 2]).sum()
                                 + bias[h, min(max(p - j - start, 0), 3)] for j in keys])
                w = torch.softmax(s, 0)
                want = sum(w[x] * v[cu_k[b] + j, h // 2] for x, j in enumerate(keys))
                assert torch.allclose(got.out[cu_q[b] + i, h], want, atol=1e-13)
                assert abs(float(got.lse[cu_q[b] + i, h] - torch.logsumexp(s, 0))) < 1e-13


@pytest.mark.parametrize("mask", MASKS)
def test_gradients_against_differences(mask):
    """Central differences of step 1e-5 in 64 bits: off by about 1e-10 (their third derivative) and 1e-11 (rounding)."""
    q, k, v, bias, cu_q, cu_k, rand = _case(2)
    start = 0 if mask["causal"] else -2
    go, gl = rand(*q.shape), rand(*q.shape[:2])

    def value(q, k, v, bias):
        r = ref.attention(q, k, v, cu_q, cu_k, 0.3, bias=bias, start=start, **mask)
        return float((r.out * go).sum() + (r.lse * gl).sum())

    r = ref.attention(q, k, v, cu_q, cu_k, 0.3, bias=bias, start=start, go=go, gl=gl, **mask)
    x = [q, k, v, bias]
    for i, grad in enumerate((r.dq, r.dk, r.dv, r.dbias)):
        flat = x[i].reshape(-1)
        for at in range(0, flat.numel(), max(1, flat.numel() // 23)):
            d = torch.zeros_like(flat)
            d[at] = 1e-5
            up, down = list(x), list(x)
            up[i], down[i] = x[i] + d.view_as(x[i]), x[i] - d.view_as(x[i])
            assert abs((value(*up) - value(*down)) / 2e-5 - float(grad.reshape(-1)[at])) < 1e-8


def test_rows_that_see_nothing():
    q, k, v, bias, _, _, rand = _case(3)
    cu_q, cu_k = [0, 5, 8], [0, 2, 2]  # more queries than keys; no keys
    go = rand(8, 4, 8)
    r = ref.attention(q[:8], k[:2], v[:2], cu_q, cu_k, 0.3, bias=bias, go=go)
    assert (r.out[:3] == 0).all() and (r.out[5:] == 0).all() and (r.dq[:3] == 0).all() and (r.out[3:5] != 0).all()
    assert (r.lse[:3] == -math.inf).all() and torch.isfinite(r.lse[3:5]).all()

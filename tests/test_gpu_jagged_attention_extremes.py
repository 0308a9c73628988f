"""jagged_attention at its ends: scores far beyond any softmax's need, spans of a batch without queries."""
import math

import pytest
import torch

from test_gpu_jagged_attention import B, H, HALF, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,power", [(H, 13), (H, 15), (B, 17), (B, 40)])
@pytest.mark.parametrize("span", [0, 1])
def test_scores_of_the_largest_inputs(pdm, dev, D, dtype, power, span):
    """Queries and keys of one size, whose scores are exact: beyond 2^34 in fp16, 2^84 in bf16.  Keys of the largest score share a
    row alike, the others have nothing."""
    c = Case([200], [200], 2, 1, D, dtype, span, seed=power)
    if span:
        c.bias = torch.zeros_like(c.bias)
    c.scale = 0.125
    size = 1.25 * 2.0 ** power  # scores of 25 / 16 of a power of two: times the scale's log2(e) they are not exact
    c.q = torch.full_like(c.q, size)
    for kind in (0, 1, 2):
        part = torch.ones(200)
        if kind:  # every third key, from the first on or not, beside half as large or negative ones
            part = torch.where(torch.arange(200) % 3 == kind - 1, 1.0, -1.0 if kind == 1 else 0.5)
        c.k = (part * size)[:, None, None].expand(-1, 1, D).to(dtype).contiguous()
        sees = torch.arange(200)[:, None] >= torch.arange(200)
        best = torch.where(sees, part, -math.inf).amax(1, keepdim=True)
        p = (sees & (part == best)).double()
        p /= p.sum(1, keepdim=True)
        x = c.inputs(dev, True)
        out, lse = c.call(pdm, dev, x)
        (dv,) = torch.autograd.grad(out, [x[2]], c.go.to(dev))
        v, go = c.v[:, 0].double(), c.go.double()
        # a weight of its type, exponents and sums of fp32, the rounding of the output
        e = HALF[dtype] + 2.0 ** -18
        for h in range(2):
            assert ((out[:, h].detach().cpu().double() - p @ v).abs() <= e * (p @ v.abs()) + HALF[dtype] * (p @ v).abs()).all()
            # (the sum beside the score is less than half a step of it)
            want = best[:, 0].double() * size * size * D * 0.125 + p.count_nonzero(1).double().log()
            assert ((lse[:, h].detach().cpu().double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all()
        want, mag = sum(p.T @ go[:, h] for h in range(2)), sum(p.T @ go[:, h].abs() for h in range(2))
        assert ((dv[:, 0].cpu().double() - want).abs() <= e * mag + HALF[dtype] * want.abs() + 2.0 ** -25).all()


def test_spans_of_a_batch_without_queries(pdm, dev):
    """There is nothing to compute, and spans that do not fit are told all the same."""
    q, k = torch.zeros(0, 2, 64, dtype=B, device=dev), torch.randn(20, 1, 64, device=dev).to(B)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for cu_q, cu_k, bad in (([0, 0, 0], [0, 10, 20], 0), ([0, 0, 0], [0, 10, 21], 1), ([0, 0, 0], [0, 10, 5], 1), ([0, 1, 1], [0, 10, 20], 1), ([0] * 300, [0] * 299 + [21], 1),
                            ([0] * 300, [0] * 300, 0), ([0], [0], 0)):
        flag = torch.zeros(1, dtype=torch.int32, device=dev)
        out = pdm.jagged_attention(q, k, k, t(cu_q), t(cu_k), err_flag=flag)
        assert out.shape == (0, 2, 64) and flag.item() == bad

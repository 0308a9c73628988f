"""kv_attention where scores go far beyond any softmax's need."""
import math

import pytest
import torch

from test_gpu_kv_attention import STEP, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,power", [(torch.float16, 13), (torch.bfloat16, 30)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [5, 70, 900]), ([1], [9000]), ([9, 20], [300, 20]), ([200, 130], [400, 130])])
@pytest.mark.parametrize("mask", [dict(), dict(window=50, sinks=3), dict(bias=1)])
def test_scores_of_the_largest_inputs(pdm, dev, dtype, power, D, new, lens, mask):
    """Queries of one size over keys of one size: all keys of a row have one score, exact, of 2^37 and more, and share the row
    alike.  The product with the scale's log2(e) is not exact, and what rounding leaves of it must not count."""
    c = Case(pdm, dev, new, lens, 4, 2, D, 32, dtype, seed=D)
    c.q = torch.full_like(c.q, 1.25 * 2.0 ** power)
    c.cache.k_codes.copy_(torch.full(c.cache.k_codes.shape, 1.25).to(torch.float8_e4m3fn))
    c.cache.k_scale.fill_(2.0 ** 20)
    kw = dict(mask)
    if "bias" in kw:
        kw["bias"] = torch.zeros(4, 1, device=dev)
    v = c.values()[1]
    for call in (dict(max_q_len=max(new)), {}):
        out, lse = (t.cpu().double() for t in c.run(scale=0.125, **kw, **call))
        for b, (n, length) in enumerate(zip(new, lens)):
            held = torch.stack([v[c.table[b][j // 32], :, j % 32] for j in range(length)]).double()
            for i in {0, n // 2, n - 1}:
                p = length - n + i
                seen = [j for j in range(p + 1) if not mask.get("window") or j > p - 50 or j < 3]
                mean, size = held[seen].mean(0).repeat_interleave(2, 0), held[seen].abs().mean(0).repeat_interleave(2, 0)
                got = out[c.cu[b] + i]
                # a weight of bf16, exponents and sums in fp32, the rounding of the output
                assert ((got - mean).abs() <= (2.0 ** -8 + 2.0 ** -18) * size + STEP[dtype] * mean.abs()).all()
                score = 1.25 ** 2 * 2.0 ** (power + 20) * D * 0.125
                assert ((lse[c.cu[b] + i] - score).abs() <= 4 * 2.0 ** -24 * score).all() and math.isfinite(score)

"""kv_attention with first tokens that stay visible under a window and with a bias by distance, against its definition in 64 bits:
single tokens to prompts, every head width, page size and kind of split; pages given back; what lies where nothing is seen; and
with jagged_attention, whose model it serves.  Tolerances: those of a score without a bias, whose size the bias adds to."""
import math

import pytest
import torch

from oracle import cached_attention as ref
from test_gpu_kv_attention import DECODE, STEP, Case, _t

pytestmark = pytest.mark.gpu


class Biased(Case):
    bias, start = None, 0

    def with_bias(self, span, start=0, seed=1):
        self.start = start
        self.bias = torch.randn(self.q.shape[1], span, generator=torch.Generator().manual_seed(seed)) if span else None
        return self

    def want(self, scale=None, causal=True, window=0, sinks=0):
        k, v = self.values()
        return ref.attention(self.q, k, v, self.cu, self.table, self.lens, self.q.shape[-1] ** -0.5 if scale is None else scale,
                             causal, window, sinks, self.bias, self.start)

    def run(self, **kw):
        bias = None if self.bias is None else self.bias.to(self.dev)
        return super().run(bias=bias, bias_start=self.start, **kw)

    def both(self, **mask):
        """With and without the promise of a largest number of new tokens."""
        want = self.want(**mask)
        self.check(self.run(max_q_len=max(self.new), **mask), want)
        self.check(self.run(**mask), want)


MASKS = [dict(window=1, sinks=1), dict(window=20, sinks=4), dict(window=33, sinks=40), dict(window=100, sinks=130), dict(window=500, sinks=3)]
BIASES = [(0, 0), (1, 0), (30, 0), (129, -5), (800, 0)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page,group", [(16, 1), (32, 4), (64, 7), (128, 16), (16, 24)])
@pytest.mark.parametrize("at", range(len(MASKS)))
def test_single_tokens(pdm, dev, dtype, D, page, group, at):
    c = Biased(pdm, dev, [1] * len(DECODE), DECODE, 2 * group, 2, D, page, dtype, seed=group, extra=1)
    c.with_bias(*BIASES[(at + D // 64 + group) % 5]).both(**MASKS[at])


@pytest.mark.parametrize("span,start", BIASES)
def test_biases_alone(pdm, dev, span, start):
    for new, lens in (([1] * len(DECODE), DECODE), ([5, 0, 1, 64], [5, 7, 300, 64]), ([150], [470])):
        for causal in (True, False):
            c = Biased(pdm, dev, new, lens, 6, 2, 64, 32, seed=3).with_bias(span, start if causal else start - 20)
            c.both(causal=causal)


RAGGED = [([16, 16, 16], [16, 400, 1516]), ([5, 0, 1, 64], [5, 7, 300, 64]), ([33, 1, 130], [33, 1000, 400]), ([300], [300]),
          ([1, 520], [2000, 777])]


@pytest.mark.parametrize("new,lens", RAGGED)
@pytest.mark.parametrize("D,page,hk,group", [(64, 32, 3, 1), (128, 64, 2, 4), (128, 16, 1, 5), (256, 128, 1, 2), (64, 16, 2, 8), (64, 32, 1, 40)])
@pytest.mark.parametrize("mask", [dict(window=100, sinks=4), dict(window=17, sinks=70), dict(causal=False, window=37, sinks=2)])
def test_ragged(pdm, dev, new, lens, D, page, hk, group, mask):
    span, start = BIASES[1:][(len(new) + D // 64 + hk) % 4]
    c = Biased(pdm, dev, new, lens, hk * group, hk, D, page, seed=len(new) + D, extra=2)
    c.with_bias(span, start if mask.get("causal", True) else start - 30).both(**mask)


@pytest.mark.parametrize("mask", [dict(), dict(window=700, sinks=5), dict(window=2500, sinks=300)])
def test_splits(pdm, dev, mask):
    """One long context, whose keys are split; a batch of many, whose keys are dealt; prompts, split and not."""
    for new, lens, hk, group, D, page in (([1], [9001], 1, 4, 128, 16), ([3, 1], [4000, 5], 2, 2, 64, 64), ([40], [3500], 2, 4, 128, 64),
                                          ([1] * 40, [100 * i + 7 for i in range(40)], 8, 1, 64, 32), ([300, 9], [2900, 2000], 16, 4, 64, 32)):
        Biased(pdm, dev, new, lens, hk * group, hk, D, page, seed=len(new)).with_bias(1500).both(**mask)


@pytest.mark.parametrize("dtype,D,hk,group", [(torch.bfloat16, 128, 32, 8), (torch.float16, 64, 64, 1), (torch.bfloat16, 64, 16, 12)])
def test_large_batches(pdm, dev, dtype, D, hk, group):
    for span, mask in ((0, dict(window=200, sinks=70)), (300, dict(window=0)), (90, dict(window=64, sinks=3))):
        Biased(pdm, dev, [300, 260], [700, 300], hk * group, hk, D, 32, dtype, seed=D).with_bias(span).both(**mask)


@pytest.mark.parametrize("new", [[1, 1], [9, 40], [200, 130]])
@pytest.mark.parametrize("page", [16, 64])
def test_pages_given_back(pdm, dev, new, page):
    """Pages between the sinks and the window are not looked at."""
    for window, sinks in ((50, 4), (100, 17), (130, 0)):
        c = Biased(pdm, dev, new, [900, 700], 4, 2, 64, page, seed=page).with_bias(60)
        want = c.want(window=window, sinks=sinks)
        gone = 0
        for row, n, ln in zip(c.table, new, c.lens):
            first = max(0, ln - n - window + 1)
            for i in range(len(row)):
                if i * page >= sinks and (i + 1) * page <= first:
                    row[i], gone = -1, gone + 1
        assert gone
        for kw in (dict(max_q_len=max(new)), {}):
            c.check(c.run(window=window, sinks=sinks, **kw), want)  # (checks that the flag is not set)


@pytest.mark.parametrize("new", [[1], [7], [200]])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_reaches_only_the_rows_that_see_it(pdm, dev, new, D):
    n, length = new[0], 260
    for at in (0, 3, 5, 100, length - 30, length - 1):
        for which in ("k_codes", "v_codes"):
            c = Biased(pdm, dev, new, [length], 4, 2, D, 16, seed=at + D).with_bias(40)
            getattr(c.cache, which).view(torch.uint8)[c.table[0][at // 16], 1, at % 16, 5] = 0x7F
            want = c.want(window=20, sinks=4)
            p = torch.arange(length - n, length)
            hit = (at <= p) & ((at > p - 20) | (at < 4))
            assert torch.equal(want[0].isnan().any(-1)[:, 2:].any(-1), hit)
            c.check(c.run(window=20, sinks=4), want)


@pytest.mark.parametrize("new", [[1], [12], [200]])
def test_biases_that_mask(pdm, dev, new):
    """-inf hides a distance, the type's lowest value hides it from rows that see others; columns that no seen pair has may hold
    anything; rows of -inf alone are zeros, rows of the lowest value alone take all alike."""
    low = torch.finfo(torch.float32).min
    c = Biased(pdm, dev, new, [300], 4, 2, 64, 32, seed=4).with_bias(100)
    c.bias[0, 30:60] = -math.inf
    c.bias[1, 7:] = -1e30
    c.both(window=80, sinks=0)
    want = c.want(window=80)
    for bad in (math.nan, math.inf):
        c.bias[:, 80:] = bad
        c.check(c.run(window=80), want)
    c.bias[2] = -math.inf
    c.bias[3] = low
    out, lse = c.run(window=80)
    assert (out[:, 2] == 0).all() and (lse[:, 2] == -math.inf).all()
    v = c.values()[1]
    held = torch.stack([v[c.table[0][j // 32], 1, j % 32] for j in range(300)]).double()
    for i, p in enumerate(range(300 - new[0], 300)):
        part = held[max(0, p - 79):p + 1]
        assert ((out[i, 3].cpu().double() - part.mean(0)).abs() <= 2 * STEP[torch.bfloat16] * part.abs().mean(0)).all()


def test_nothing_added_changes_nothing(pdm, dev):
    """Sinks without a window: the bits of the plain call; a window that reaches all keys: its values."""
    for new, lens in (([1, 1, 1], [5, 70, 900]), ([40, 3], [500, 3]), ([300], [400])):
        c = Case(pdm, dev, new, lens, 4, 2, 64, 32, seed=5)
        want = c.run()
        assert all(torch.equal(a, b) for a, b in zip(want, c.run(sinks=7)))
        c.check(c.run(sinks=7, window=2000), c.want())


def test_half_precision_bias_and_refusals(pdm, dev):
    c = Biased(pdm, dev, [1, 1], [50, 90], 4, 2, 64, 32, seed=6).with_bias(20)
    c.bias = c.bias.to(torch.bfloat16).float()
    want = c.run()
    bias = c.bias.to(dev).to(torch.bfloat16)
    got = Case.run(c, bias=bias)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="no backward pass"):
        Case.run(c, bias=c.bias.to(dev).requires_grad_(True))
    for match, kw in (("bias must be", dict(bias=c.bias[:3].to(dev))), ("sinks", dict(sinks=-1)),
                      ("bias_start", dict(bias=c.bias.to(dev), bias_start=2 ** 30)), ("columns", dict(bias=c.bias[:, :0].to(dev)))):
        with pytest.raises(ValueError, match=match):
            Case.run(c, **kw)
    with pytest.raises(TypeError, match="bias must be"):
        Case.run(c, bias=bias.half())
    with pytest.raises(RuntimeError, match="GPU only|different devices"):
        Case.run(c, bias=c.bias)


def _bytes(t):
    return t.view(torch.uint8)


def test_graph(pdm, dev):
    """Captured, replayed with other lengths, pages and biases in the same tensors, eager calls in between."""
    for new in ([1, 1], [30, 170]):
        lists = ([900, 400], [170, 950], [300, 300])
        cases = [Biased(pdm, dev, new, lens, 4, 2, 64, 16, seed=i).with_bias(50, seed=i) for i, lens in enumerate(lists)]
        for c in cases:
            c.table = [row + [-1] * (64 - len(row)) for row in c.table]
        mask = dict(window=120, sinks=5, max_q_len=max(new))
        want = [[t.clone() for t in c.run(**mask)] for c in cases]
        cache = pdm.PagedKVCache(max(len(c.cache.k_codes) for c in cases), 16, 2, 64, dev)
        q, cu = cases[0].q.to(dev), _t(cases[0].cu, dev)
        table, lens, bias = _t(cases[0].table, dev), _t(cases[0].lens, dev), cases[0].bias.to(dev)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            got = cache.attend(q, cu, table, lens, return_lse=True, bias=bias, **mask)
        for i in (0, 1, 2, 1):
            c = cases[i]
            for n in ("k_codes", "v_codes", "k_scale", "v_scale"):
                t = getattr(c.cache, n)
                _bytes(getattr(cache, n)[:len(t)]).copy_(_bytes(t))
            q.copy_(c.q), table.copy_(_t(c.table, dev)), lens.copy_(_t(c.lens, dev)), bias.copy_(c.bias)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
            c.run(**mask)


def test_registered_operator(pdm, dev):
    c = Biased(pdm, dev, [1, 3], [40, 9], 4, 2, 64, 16, seed=7).with_bias(9)
    k = c.cache
    args = (c.q.to(dev), _bytes(k.k_codes), _bytes(k.v_codes), k.k_scale, k.v_scale, _t(c.cu, dev), _t(c.table, dev),
            _t(c.lens, dev), 0.125, True, 8, 3, True, None, 2, c.bias.to(dev), 0)
    torch.library.opcheck(torch.ops.pdm.kv_attention.default, args, test_utils=("test_schema", "test_faketensor"))
    f = torch.compile(lambda q: pdm.kv_attention(q, *args[1:8], window=8, sinks=2, max_q_len=3, bias=args[-2]), fullgraph=True)
    assert torch.equal(f(args[0]), c.run(window=8, sinks=2, max_q_len=3)[0])


def test_served_as_trained(pdm, dev):
    """A layer of norm and rotation, bias, window and sinks: tokens appended to a cache in pieces and attended to, the pages behind the
    window given back; and the training form of the same queries over the values that the cache holds at that time."""
    torch.manual_seed(8)
    n, hq, hk, D, page, window, sinks = 150, 4, 2, 64, 16, 40, 3
    rope = pdm.QKNormRope(D, 256, device=dev)
    rel = pdm.RelativeBias(hq, 16, 60, device=dev)
    with torch.no_grad():
        rel.table.normal_()
        q, k, v = (torch.randn(n, h, D, device=dev).to(torch.bfloat16) for h in (hq, hk, hk))
        qr, _ = rope(q, None, torch.arange(n, device=dev))
        bias = rel()
    cache = pdm.PagedKVCache(12, page, hk, D, dev)
    table, at = _t([list(range(10))], dev), 0
    for step in (60, 1, 1, 20, 1, 67):
        cu, lens = _t([0, step], dev), _t([at + step], dev)
        piece = qr[at:at + step]
        with torch.no_grad():
            cache.append(k[at:at + step], v[at:at + step], cu, table, lens, rope=rope)
            got = cache.attend(piece, cu, table, lens, window=window, sinks=sinks, bias=bias, bias_start=rel.start, max_q_len=step)
        at += step
        held = [t[:10].transpose(1, 2).reshape(160, hk, D)[:at].contiguous() for t in cache.values()]
        x = [t.detach().requires_grad_(True) for t in (piece, *held)]
        out = pdm.jagged_attention(*x, cu, lens.new_tensor([0, at]), window=window, sinks=sinks, bias=rel(), bias_start=rel.start)
        grads = torch.autograd.grad(out, [*x, rel.table], torch.ones_like(out))
        assert all(torch.isfinite(g).all() for g in grads)
        # an output off by half a step on either side, and on one side the weights too
        assert float((got - out).float().norm() / out.float().norm()) < 3 * STEP[torch.bfloat16]
        gone = max(0, (at + 1 - window) // page)  # pages that the next token's window has left, but for the first
        if gone > 1:
            table[0, 1:gone] = -1
    cache.check()

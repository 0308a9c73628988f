"""jagged_attention and its backward pass against their definition in 64 bits: lengths from none to long, grouped heads, head
widths, types, masks, biases; what lies where nothing is seen; strides, streams, graphs.

Tolerances.  u = 2^-24; half = half a step of the type, 2^-8 (bf16) or 2^-11 (fp16).  A score is a sum of D exact products in fp32
and a bias, off by e_s <= (D + 8) u sum of sizes; a weight then by the relative e_w = 2 e_s + 2^-20 (exp2 and its argument), and by
half where it meets the values.  fp16 weights below 2^-14 of the row's largest are off by up to 2^-25 of it.  So
  |out - want| <= (half + e_w) sum p |v|  (fp16: + 2^-25 sum |v|)  + half |want|,   |lse - want| <= e_s + 2^-20 + 2 u |want|.
dS = P (dP - delta): off by e_w of itself (P), by P (D + 8) u sum |dO V| (dP), and by P times delta's error, sum |dO| times that of
out: half and e_w of sum p |v| twice over (its weights, its rounding), or 2^-14 + e_w of it where the remainders are kept.  It is
rounded, half of itself, for the products; fp16 dS are off by 2^-25 beside an |dO| of 2^-6 and more, 2^-19 of the largest |dO|.
The bias's gradient is a sum in fp32 of as many as n_k terms: n_k u sum |dS| more, and no rounding of dS."""
import math

import pytest
import torch

from oracle import jagged_attention as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
B, H = torch.bfloat16, torch.float16


def _t(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Case:
    def __init__(self, new, lens, hq, hk, D, dtype=B, span=0, start=0, seed=0, spread=1.5):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.D, self.start = dtype, D, start
        self.cu_q, self.cu_k = [0], [0]
        for a, b in zip(new, lens):
            self.cu_q.append(self.cu_q[-1] + a)
            self.cu_k.append(self.cu_k[-1] + b)
        rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.q, self.k, self.v = (rand(self.cu_q[-1], hq, D) * spread).to(dtype), rand(self.cu_k[-1], hk, D).to(dtype), rand(self.cu_k[-1], hk, D).to(dtype)
        self.bias = rand(hq, span) if span else None
        self.go, self.gl = rand(*self.q.shape).to(dtype), rand(*self.q.shape[:2])
        self.scale = None

    def want(self, grad=False, gl=False, **mask):
        return ref.attention(self.q, self.k, self.v, self.cu_q, self.cu_k, self.D ** -0.5 if self.scale is None else self.scale,
                             bias=self.bias, start=self.start, go=self.go if grad else None, gl=self.gl if gl else None, **mask)

    def inputs(self, dev, grad=False):
        x = [t.to(dev) if t is not None else None for t in (self.q, self.k, self.v, self.bias)]
        return [t.requires_grad_(grad) if t is not None else None for t in x]

    def call(self, pdm, dev, x, **kw):
        q, k, v, bias = x
        return pdm.jagged_attention(q, k, v, _t(self.cu_q, dev), _t(self.cu_k, dev), scale=self.scale, bias=bias,
                                    bias_start=self.start, return_lse=True, **kw)

    def run(self, pdm, dev, **kw):
        return self.call(pdm, dev, self.inputs(dev), **kw)

    def e_w(self, w):
        return 2 * (self.D + 8) * U * w.serr[..., None] + 2.0 ** -20

    def check(self, got, w):
        out, lse = (t.detach().cpu().double() for t in got)
        half, e = HALF[self.dtype], self.e_w(w)
        slack = (half + e) * w.mag + (2.0 ** -25 * self.v.double().nan_to_num().abs().sum(0).max() if self.dtype == H else 0.0)
        assert torch.equal(out.isnan(), w.out.isnan())
        assert torch.equal(out.isinf(), w.out.isinf())
        bad = ((out - w.out).abs() - slack - half * (w.out.abs() + slack) - 2.0 ** -25).nan_to_num(-1, neginf=-1)
        assert bad.numel() == 0 or bad.max().item() <= 0, f"out over by {bad.max().item():.3e}"
        empty = torch.isinf(w.lse) & (w.lse < 0)
        assert torch.equal(torch.isinf(lse) & (lse < 0), empty) and (out[empty] == 0).all()
        assert torch.equal(lse.isnan(), w.lse.isnan())
        bad = ((lse - w.lse).abs() - e[..., 0] - 2.0 ** -20 - 2 * U * w.lse.abs())[~empty].nan_to_num(-1)
        assert bad.numel() == 0 or bad.max().item() <= 0, f"lse over by {bad.max().item():.3e}"

    def grads(self, pdm, dev, gl=False, **kw):
        x = self.inputs(dev, True)
        out, lse = self.call(pdm, dev, x, **kw)
        leaves = [t for t in x if t is not None]
        outs, gs = ([out, lse], [self.go.to(dev), self.gl.to(dev)]) if gl else ([out], [self.go.to(dev)])
        return (out, lse), torch.autograd.grad(outs, leaves, gs)

    def check_grads(self, got, w):
        half, t = HALF[self.dtype], w.t
        e = float((2 * (self.D + 8) * U + 2.0 ** -20))  # of a weight, beside 1 + serr
        rest = self.bias is not None
        d = (2.0 ** -14 if rest else 2 * half) + float(self.e_w(w).max() if w.serr.numel() else 0)
        small = 2.0 ** -19 * float(self.go.double().nan_to_num().abs().max()) if self.dtype == H and self.go.numel() else 0.0
        tol = [e * getattr(t, "rel" + x) + (self.D + 8) * U * getattr(t, "dp" + x) + d * getattr(t, "delta" + x)
               + half * (1 + d) * getattr(t, "all" + x) + small * getattr(t, "one" + x) for x in "qk"]
        tol.append((half + e) * t.dv + (2.0 ** -25 * self.go.double().nan_to_num().abs().sum() if self.dtype == H else 0.0))
        for name, g, want, tl in zip(("dq", "dk", "dv"), got, (w.dq, w.dk, w.dv), tol):
            g = g.cpu().double()
            assert torch.equal(torch.isfinite(g), torch.isfinite(want)), name
            bad = ((g - want).abs() - tl - half * (want.abs() + tl) - 2.0 ** -25).nan_to_num(-1, neginf=-1)
            assert bad.numel() == 0 or bad.max().item() <= 0, f"{name} over by {bad.max().item():.3e}"
        if rest:
            b, most = t.dbias, max(self.cu_k[i + 1] - self.cu_k[i] for i in range(len(self.cu_k) - 1))
            tl = e * b["rel"] + (self.D + 8) * U * b["dp"] + d * b["delta"] + most * U * b["all"] + 2.0 ** -25
            g = got[3].cpu().double()
            assert torch.equal(torch.isfinite(g), torch.isfinite(w.dbias))
            bad = ((g - w.dbias).abs() - tl).nan_to_num(-1, neginf=-1)
            assert bad.max().item() <= 0, f"dbias over by {bad.max().item():.3e}"


RAGGED = [
    ([1], [1]), ([64], [64]), ([200], [200]), ([1, 3, 0, 31, 32, 33], [1, 3, 0, 31, 32, 33]), ([127, 129, 5], [127, 129, 5]),
    ([16, 1, 40], [100, 333, 40]), ([5, 9, 70], [3, 0, 20]), ([300, 1], [513, 400]),
]
MASKS = [dict(causal=True), dict(causal=False), dict(causal=True, window=1), dict(causal=True, window=50, sinks=3),
         dict(causal=True, window=130, sinks=70), dict(causal=False, window=40), dict(causal=False, window=33, sinks=5)]
BIASES = [(0, 0), (1, 0), (20, 0), (129, -64), (600, -300), (40, 17)]


@pytest.mark.parametrize("new,lens", RAGGED)
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("D,hk,group,dtype", [(64, 3, 1, B), (128, 1, 4, B), (64, 2, 2, H), (128, 2, 1, H)])
def test_ragged(pdm, dev, new, lens, mask, D, hk, group, dtype):
    """Forward without and with a bias, one per call of the biases in turn; backward with that bias and without."""
    at = len(new) + sum(new) + len(mask)
    for span, start in ((0, 0), BIASES[1:][at % 5]):
        c = Case(new, lens, hk * group, hk, D, dtype, span, start, seed=at)
        w = c.want(True, **mask)
        c.check(c.run(pdm, dev, **mask), w)
        got, grads = c.grads(pdm, dev, **mask)
        c.check(got, w)
        c.check_grads(grads, w)


@pytest.mark.parametrize("span,start", BIASES)
@pytest.mark.parametrize("mask", [MASKS[0], MASKS[1], MASKS[4]])
def test_biases(pdm, dev, span, start, mask):
    c = Case([150, 70], [150, 300], 4, 2, 64, B, span, start, seed=span)
    w = c.want(True, gl=True, **mask)
    got, grads = c.grads(pdm, dev, gl=True, **mask)
    c.check(got, w)
    c.check_grads(grads, w)


def test_longer(pdm, dev):
    for D, dtype, mask, span in ((64, B, dict(causal=True), 128), (128, H, dict(causal=True, window=300, sinks=4), 301),
                                 (128, B, dict(causal=False), 2000), (64, H, dict(causal=True, window=700, sinks=129), 0)):
        c = Case([1500, 37], [1500, 1111], 2, 1, D, dtype, span, 0 if mask["causal"] else -1000, seed=D)
        w = c.want(True, **mask)
        got, grads = c.grads(pdm, dev, **mask)
        c.check(got, w)
        c.check_grads(grads, w)


@pytest.mark.parametrize("spread,scale", [(60.0, None), (0.0, None), (1.0, -0.3), (1.0, 0.0), (40.0, 0.5)])
def test_scores_of_any_size(pdm, dev, spread, scale):
    for span in (0, 30):
        c = Case([140, 3], [200, 90], 2, 2, 64, B, span, seed=5, spread=spread)
        c.scale = scale
        w = c.want(True)
        got, grads = c.grads(pdm, dev)
        c.check(got, w)
        c.check_grads(grads, w)


def test_small_gradients_in_half_precision(pdm, dev):
    """Gradients near fp16's smallest, and of very unlike sizes along the queries."""
    c = Case([400], [400], 2, 1, 64, H, 16, seed=6)
    c.go = (c.go.float() * torch.logspace(-6, 0, 400)[:, None, None]).to(H)
    w = c.want(True)
    c.check_grads(c.grads(pdm, dev)[1], w)
    c.go = (c.go.float() * 2.0 ** -8).to(H)
    w = c.want(True)
    _, (dq, dk, dv, db) = c.grads(pdm, dev)
    assert float((db.cpu().double() - w.dbias).norm() / w.dbias.norm()) < 1e-4
    c.check_grads((dq, dk, dv, db), w)


def test_gradients_of_lse_in_half_precision(pdm, dev):
    """Of lse alone, and much larger than those of out."""
    for size, mask in ((0.0, dict(causal=True)), (2.0 ** -20, dict(causal=True, window=60, sinks=4))):
        c = Case([150, 20], [150, 70], 2, 1, 64, H, 12, seed=23)
        c.go = (c.go.float() * size).to(H)
        w = c.want(True, gl=True, **mask)
        _, grads = c.grads(pdm, dev, gl=True, **mask)
        # half a step of dS and of the result, each of its own size
        for g, want in zip((grads[0], grads[1], grads[3]), (w.dq, w.dk, w.dbias)):
            assert float((g.cpu().double() - want).norm() / want.norm()) < 2 * HALF[H]
        assert size or (grads[2] == 0).all()


@pytest.mark.parametrize("D,hk,group,dtype", [(64, 1, 4, B), (128, 2, 1, H), (64, 2, 1, H), (128, 1, 2, B)])
def test_more_than_64_sequences(pdm, dev, D, hk, group, dtype):
    g = torch.Generator().manual_seed(24)
    lens = torch.randint(0, 60, (70,), generator=g).tolist()
    lens[40], lens[41] = 400, 0
    new = [min(n, x) for n, x in zip(lens, torch.randint(1, 500, (70,), generator=g).tolist())]
    for span, start, mask in ((0, 0, dict(causal=False)), (30, 0, dict(causal=True, window=45, sinks=33)), (90, -40, dict(causal=False, window=20))):
        c = Case(new, lens, hk * group, hk, D, dtype, span, start, seed=25)
        w = c.want(True, **mask)
        got, grads = c.grads(pdm, dev, **mask)
        c.check(got, w)
        c.check_grads(grads, w)


@pytest.mark.parametrize("D,dtype", [(64, H), (128, B)])
def test_sinks_of_long_sequences(pdm, dev, D, dtype):
    """Queries beyond the window that are dealt to several workgroups; distances between the window and the sinks that no column
    of the bias has, or that it has and no pair."""
    for window, sinks, span, start in ((40, 2, 600, -100), (70, 100, 45, 0), (300, 33, 2600, 0), (40, 2, 100, 1900)):
        c = Case([2600, 3], [2600, 2100], 4, 1, D, dtype, span, start, seed=window)
        mask = dict(causal=True, window=window, sinks=sinks)
        w = c.want(True, **mask)
        got, grads = c.grads(pdm, dev, **mask)
        c.check(got, w)
        c.check_grads(grads, w)


def test_two_graphs_on_two_streams(pdm, dev):
    """Captured steps of different sizes, replayed at once and in turn."""
    cases = [Case([700, 20], [700, 20], 2, 1, 64, H, 40, seed=26), Case([300], [300], 4, 2, 128, B, 90, seed=27)]
    mask = dict(window=50, sinks=5)
    want, graphs, made = [], [], []
    for c in cases:
        (out, _), grads = c.grads(pdm, dev, **mask)
        want.append([out.detach().clone(), *[g.clone() for g in grads]])
    del out, grads
    for c in cases:
        x, go, cu, cu_k = c.inputs(dev, True), c.go.to(dev), _t(c.cu_q, dev), _t(c.cu_k, dev)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = pdm.jagged_attention(*x[:3], cu, cu_k, bias=x[3], **mask)
            grads = torch.autograd.grad(out, x, go)
        graphs.append(graph)
        made.append([x, go, cu, cu_k, out.detach(), *grads])
        del out, grads
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for m in made:
            for t in m[4:]:
                t.fill_(math.nan)
        torch.cuda.synchronize()
        for i in (0, 1) if turn % 2 else (1, 0):
            with torch.cuda.stream(side[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for m, wanted in zip(made, want):
            assert all(torch.equal(a, b) for a, b in zip(wanted, m[4:]))
        cases[0].run(pdm, dev)


def test_values_up_to_the_largest(pdm, dev):
    c = Case([300], [300], 2, 1, 64, B, seed=7)
    c.v = (torch.sign(c.v.float()) * 3.3e38).to(B)
    c.check(c.run(pdm, dev, causal=False), c.want(causal=False))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D,dtype", [(64, B), (128, H)])
def test_what_is_not_seen_does_not_matter(pdm, dev, bad, D, dtype):
    """Keys, values, queries and gradients that are not finite reach the rows alone that see them."""
    mask = dict(causal=True, window=20, sinks=2)
    for which, rows in (("v", [9, 70, 40]), ("k", [30]), ("q", [90]), ("go", [33])):
        c = Case([100, 8], [100, 8], 2, 1, D, dtype, 10, seed=8)
        for r in rows:
            getattr(c, which)[r, 0, r % D] = bad
        w = c.want(True, **mask)
        got, grads = c.grads(pdm, dev, **mask)
        c.check(got, w)
        clean = Case([100, 8], [100, 8], 2, 1, D, dtype, 10, seed=8).want(True, **mask)
        seen = ref.seen_pairs(100, 100, True, 20, 2)
        hit = torch.zeros(108, dtype=torch.bool)   # queries that see a changed key, or are changed
        key = torch.zeros(108, dtype=torch.bool)   # keys that these queries see
        for r in rows:
            hit[:100] |= seen[:, r] if which in "vk" else torch.arange(100) == r
        key[:100] = (seen & hit[:100, None]).any(0)
        dq, dk, dv, _ = (g.cpu().double() for g in grads)
        for g, cl, touched in ((dq, clean.dq, hit), (dk, clean.dk, key), (dv, clean.dv, key)):
            left = ~touched
            assert torch.isfinite(g[left]).all()
            err = float((g[left] - cl[left]).norm() / cl[left].norm())
            assert err < 4 * HALF[dtype], (which, err)
        assert not torch.isfinite(dk[key]).all() or which == "v"


def test_biases_that_mask(pdm, dev):
    """-inf hides a distance; the type's lowest value hides it from rows that see others, and leaves rows of it alone equal."""
    low = torch.finfo(torch.float32).min
    c = Case([40], [40], 2, 1, 64, B, 12, seed=9)
    c.bias[0, 3:] = -math.inf
    c.bias[1, 3:] = low
    w = c.want(True)
    got, grads = c.grads(pdm, dev)
    c.check(got, w)
    w.dbias[0, 3:] = 0.0
    c.check_grads(grads, w)
    c.bias[0] = -math.inf  # nothing is left
    c.bias[1] = low        # all scores are alike
    out, lse = c.run(pdm, dev)
    assert (out[:, 0] == 0).all() and (lse[:, 0] == -math.inf).all()
    mean = c.v[:, 0].double().cumsum(0) / torch.arange(1, 41)[:, None]
    assert ((out[:, 1].cpu().double() - mean).abs() <= 2 * HALF[B] * (c.v[:, 0].double().abs().cumsum(0) / torch.arange(1, 41)[:, None])).all()
    _, (dq, dk, dv, db) = c.grads(pdm, dev)
    assert (dq[:, 0] == 0).all() and (db[0] == 0).all() and all(torch.isfinite(g).all() for g in (dq, dk, dv, db))
    want = torch.zeros(40, 64, dtype=torch.float64)
    for i in range(40):
        want[:i + 1] += c.go[i, 1].double() / (i + 1)
    assert float((dv[:, 0].cpu().double() - want).norm() / want.norm()) < 2 * HALF[B]


def test_rows_that_no_sequence_covers(pdm, dev):
    c = Case([20, 30], [20, 30], 2, 1, 64, B, 5, seed=10)
    w = c.want(True)
    x = c.inputs(dev)
    pad = [torch.cat((torch.full_like(t[:7], math.nan), t, torch.full_like(t[:300 - 57 + 50], math.nan))).requires_grad_() for t in x[:3]]
    cu = _t([7, 27, 57], dev)
    pad.append(x[3].requires_grad_(True))  # (the remainders that the tolerance counts on are kept for its gradient)
    out, lse = pdm.jagged_attention(*pad[:3], cu, bias=pad[3], return_lse=True)
    assert (out[:7] == 0).all() and (out[57:] == 0).all() and (lse[57:] == -math.inf).all()
    c.check((out[7:57], lse[7:57]), w)
    go = torch.full_like(out, math.nan)
    go[7:57] = c.go.to(dev)
    grads = torch.autograd.grad(out, pad, go)
    for g in grads[:3]:
        assert (g[:7] == 0).all() and (g[57:] == 0).all()
    c.check_grads([g[7:57] for g in grads[:3]] + [grads[3]], w)


def test_strides(pdm, dev):
    """Heads as columns of fused rows, keys shared by expansion, transposed batches, rows that are not aligned."""
    c = Case([50, 90], [50, 90], 4, 4, 64, B, 9, seed=11)
    w = c.want(True)
    rows = torch.cat([t.flatten(1) for t in (c.q, c.k, c.v)], 1).to(dev)
    views = [rows[:, i * 256:(i + 1) * 256].view(140, 4, 64) for i in range(3)]
    bias = c.bias.to(dev)
    base = c.call(pdm, dev, [*c.inputs(dev)[:3], bias])
    for make in (lambda t: t, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: torch.cat((t.flatten(), t.flatten()[:1])).roll(1)[1:].view(t.shape),
                 lambda t: torch.nn.functional.pad(t, (0, 3))[..., :64], lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)):
        x = [make(t).detach().requires_grad_(True) for t in views]
        got = c.call(pdm, dev, [*x, bias])
        assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
        grads = torch.autograd.grad(got[0], x, c.go.to(dev).transpose(0, 1).contiguous().transpose(0, 1))
        for g, want in zip(grads, (w.dq, w.dk, w.dv)):
            assert float((g.cpu().double() - want).norm() / want.norm()) < 2 * HALF[B]
    one = Case([50, 90], [50, 90], 4, 1, 64, B, seed=11)
    k, v = one.k.to(dev), one.v.to(dev)
    got = pdm.jagged_attention(one.q.to(dev), k.expand(-1, 4, -1), v.expand(-1, 4, -1), _t(one.cu_q, dev), return_lse=True)
    one.check(got, one.want())
    # a batch [B, S, heads, D] of one length
    q = torch.randn(3, 17, 2, 64, device=dev).to(B)
    out = pdm.jagged_attention(q, q, q, _t([0, 17, 34, 51], dev))
    assert out.shape == q.shape and torch.equal(out.flatten(0, 1), pdm.jagged_attention(*[q.flatten(0, 1)] * 3, _t([0, 17, 34, 51], dev)))


def test_empty_batches(pdm, dev):
    for T, S, cu_q, cu_k in ((0, 0, [0], [0]), (0, 5, [0, 0], [0, 5]), (5, 0, [0, 5], [0, 0]), (4, 4, [0], [0]), (4, 6, [0, 0, 0], [0, 0, 0])):
        x = [torch.randn(n, 2, 64, device=dev).to(B).requires_grad_(True) for n in (T, S, S)]
        bias = torch.randn(2, 7, device=dev, requires_grad=True)
        out, lse = pdm.jagged_attention(*x, _t(cu_q, dev), _t(cu_k, dev), bias=bias, return_lse=True)
        assert out.shape == (T, 2, 64) and (out == 0).all() and (lse == -math.inf).all()
        for g in torch.autograd.grad(out, [*x, bias], torch.ones_like(out)):
            assert (g == 0).all()


def test_the_same_bits(pdm, dev):
    """Two runs, and a batch of two beside its halves."""
    c = Case([700, 300], [900, 300], 4, 2, 64, B, 200, seed=12)
    first = c.grads(pdm, dev)
    for _ in range(2):
        again = c.grads(pdm, dev)
        assert all(torch.equal(a, b) for a, b in zip([*first[0], *first[1]], [*again[0], *again[1]]))


def test_gradients_of_some_inputs(pdm, dev):
    c = Case([60], [60], 2, 1, 64, B, 8, seed=13)
    full = c.grads(pdm, dev)[1]
    for pick in range(4):
        x = c.inputs(dev)
        x[pick].requires_grad_(True)
        out, _ = c.call(pdm, dev, x)
        (g,) = torch.autograd.grad(out, [x[pick]], c.go.to(dev))
        # without the bias's gradient, weights are rounded once and delta is the rounded output's
        assert float((g - full[pick]).float().norm() / full[pick].float().norm()) < 4 * HALF[B]


def test_half_precision_bias(pdm, dev):
    c = Case([60], [60], 2, 1, 64, B, 8, seed=14)
    c.bias = c.bias.to(B).float()
    x = c.inputs(dev, True)
    b16 = x[3].detach().to(B).requires_grad_(True)
    out, _ = c.call(pdm, dev, [*x[:3], b16])
    (g,) = torch.autograd.grad(out, [b16], c.go.to(dev))
    want = c.want(True).dbias
    assert g.dtype == B and float((g.cpu().double() - want).norm() / want.norm()) < 2 * HALF[B]


def test_spans_that_do_not_fit(pdm, dev):
    q = torch.randn(20, 2, 64, device=dev).to(B)
    for cu in ([0, 10, 5], [0, 10, 21], [-1, 10, 20], [0, 25, 30]):
        flag = torch.zeros(1, dtype=torch.int32, device=dev)
        pdm.jagged_attention(q, q, q, _t([0, 10, 20], dev), _t(cu, dev), err_flag=flag)
        assert flag.item() == 1
        flag.zero_()
        pdm.jagged_attention(q, q, q, _t(cu, dev), _t([0, 10, 20], dev), err_flag=flag)
        assert flag.item() == 1
    flag = torch.zeros(1, dtype=torch.int32, device=dev)
    pdm.jagged_attention(q, q, q, _t([0, 10, 20], dev), err_flag=flag)
    assert flag.item() == 0


def test_keys_of_a_sequence_that_does_not_fit(pdm, dev):
    """Its rows are zeros, forward and backward; the others are computed."""
    x = [torch.randn(30, 2, 64, device=dev).to(B).requires_grad_(True) for _ in range(3)]
    cu_q, cu_k = _t([0, 10, 20], dev), _t([0, 10, 31], dev)
    out, lse = pdm.jagged_attention(*x, cu_q, cu_k, return_lse=True)
    assert (out[10:] == 0).all() and (lse[10:] == -math.inf).all() and (out[:10] != 0).any()
    for g in torch.autograd.grad(out, x, torch.ones_like(out)):
        assert (g[10:] == 0).all() and torch.isfinite(g).all()


def test_places_beyond_32_bits(pdm, dev):
    """Rows 18 KB apart, 300,000 of them: the last lie 5.4 GB behind the first."""
    T, wide = 300_000, 9_216
    rows = torch.empty(T, wide, dtype=B, device=dev)
    c = Case([100], [100], 2, 1, 64, B, seed=15)
    rows[-100:, :128] = c.q.to(dev).flatten(1)
    rows[-100:, 128:192] = c.k.to(dev).flatten(1)
    rows[-100:, wide - 64:] = c.v.to(dev).flatten(1)
    x = [rows[:, :128].view(T, 2, 64), rows[:, 128:192].view(T, 1, 64), rows[:, wide - 64:].view(T, 1, 64)]
    cu = _t([T - 100, T], dev)
    out, lse = pdm.jagged_attention(*x, cu, return_lse=True)
    w = c.want(True)
    c.check((out[-100:], lse[-100:]), w)
    x = [t.detach().requires_grad_(True) for t in x]
    out = pdm.jagged_attention(*x, cu)
    go = torch.zeros_like(out)
    go[-100:] = c.go.to(dev)
    c.check_grads([g[-100:] for g in torch.autograd.grad(out, x, go)], w)


def test_many_sequences(pdm, dev):
    """100,000 sequences of none to three tokens."""
    g = torch.Generator().manual_seed(16)
    n = torch.randint(0, 4, (100_000,), generator=g)
    cu = torch.cat((torch.zeros(1, dtype=torch.long), n.cumsum(0))).int().to(dev)
    T = int(n.sum())
    q, k, v = (torch.randn(T, 1, 64, generator=g).to(B).to(dev) for _ in range(3))
    out = pdm.jagged_attention(q, k, v, cu).float()
    first = cu[:-1][n.to(dev) > 0].long()
    assert torch.equal(out[first], v[first].float())
    s = (q[:, 0].float()[1:] * k[:, 0].float()[1:]).sum(-1) / 8, (q[:, 0].float()[1:] * k[:, 0].float()[:-1]).sum(-1) / 8
    w = torch.softmax(torch.stack(s, -1), -1)
    want = w[:, :1] * v[1:, 0].float() + w[:, 1:] * v[:-1, 0].float()
    second = first[n.to(dev)[n.to(dev) > 0] > 1] + 1
    assert float((out[second, 0] - want[second - 1]).norm() / want[second - 1].norm()) < 2 * HALF[B]


def test_another_stream(pdm, dev):
    c = Case([300, 20], [300, 40], 4, 2, 64, B, 50, seed=17)
    want = c.grads(pdm, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.grads(pdm, dev)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip([*want[0], *want[1]], [*got[0], *got[1]]))


def test_graph(pdm, dev):
    """A captured training step replayed with other inputs and lengths in the same tensors, eager work in between."""
    cases = [Case([120, 30], [120, 30], 2, 1, 64, B, 40, seed=18), Case([1, 149], [1, 149], 2, 1, 64, B, 40, seed=19),
             Case([75, 75], [75, 75], 2, 1, 64, B, 40, seed=20)]
    want = []
    for c in cases:
        (out, _), grads = c.grads(pdm, dev)
        want.append([out.detach().clone(), *[g.clone() for g in grads]])
    del out, grads
    x = cases[0].inputs(dev, True)
    go, cu = cases[0].go.to(dev), _t(cases[0].cu_q, dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = pdm.jagged_attention(*x[:3], cu, bias=x[3])
        grads = torch.autograd.grad(out, x, go)
    for i in (0, 1, 2, 0, 1):
        c = cases[i]
        with torch.no_grad():
            for t, n in zip(x, (c.q, c.k, c.v, c.bias)):
                t.copy_(n)
        go.copy_(c.go)
        cu.copy_(_t(c.cu_q, dev))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want[i], [out, *grads]))
        c.run(pdm, dev)  # eager work between the replays


def test_two_layers_train(pdm, dev):
    """Norm and rotation, bias and attention, twice: gradients of all weights against the same in 64 bits on the CPU."""
    torch.manual_seed(21)
    lens, hq, hk, D = [40, 9], 2, 1, 64
    cu = [0, 40, 49]
    rel = pdm.RelativeBias(hq, 8, 20, device=dev)
    with torch.no_grad():
        rel.table.normal_()
    x = torch.randn(49, 64, device=dev).to(B)
    w = [(torch.randn(64, (hq + 2 * hk) * D, device=dev) / 8).to(B).requires_grad_(True) for _ in range(2)]
    o = [(torch.randn(hq * D, 64, device=dev) / 11).to(B).requires_grad_(True) for _ in range(2)]
    y = x
    for i in range(2):
        rows = y @ w[i]
        q, k, v = rows[:, :128].view(49, 2, 64), rows[:, 128:192].view(49, 1, 64), rows[:, 192:].view(49, 1, 64)
        y = y + pdm.jagged_attention(q, k, v, _t(cu, dev), window=15, sinks=2, bias=rel(), bias_start=rel.start).flatten(1) @ o[i]
    grads = torch.autograd.grad(y.float().square().sum(), [*w, *o, rel.table])
    # 64 bits
    wd, od = [t.detach().cpu().double().requires_grad_(True) for t in w], [t.detach().cpu().double().requires_grad_(True) for t in o]
    table = rel.table.detach().cpu().double().requires_grad_(True)
    z = x.cpu().double()
    for i in range(2):
        rows = z @ wd[i]
        outs = []
        for b in range(2):
            r = rows[cu[b]:cu[b + 1]]
            n = lens[b]
            seen = ref.seen_pairs(n, n, True, 15, 2)
            col = ref.columns(n, n, 21, 0)
            heads = []
            for h in range(2):
                s = r[:, h * 64:h * 64 + 64] @ r[:, 128:192].T / 8 + table[rel.buckets.cpu().long(), h][col]
                heads.append(torch.softmax(s.masked_fill(~seen, -math.inf), -1) @ r[:, 192:])
            outs.append(torch.cat(heads, 1))
        z = z + torch.cat(outs) @ od[i]
    want = torch.autograd.grad(z.square().sum(), [*wd, *od, table])
    # bf16 at each of some ten steps between a weight and the loss
    for g, t in zip(grads, want):
        assert float((g.cpu().double() - t).norm() / t.norm()) < 16 * HALF[B]


def test_compiled(pdm, dev):
    c = Case([60, 33], [60, 33], 4, 2, 64, B, seed=22)
    table = torch.randn(6, 4, device=dev, requires_grad=True)
    buckets = pdm.relative_buckets(6, 12, device=dev)
    cu = _t(c.cu_q, dev)

    def f(q, k, v, table):
        bias = pdm.bucket_bias(table, buckets)
        return pdm.jagged_attention(q, k, v, cu, bias=bias, window=30, sinks=1)

    x = c.inputs(dev, True)[:3]
    want = f(*x, table)
    wg = torch.autograd.grad(want, [*x, table], c.go.to(dev))
    got = torch.compile(f, fullgraph=True)(*x, table)
    gg = torch.autograd.grad(got, [*x, table], c.go.to(dev))
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(gg, wg))
    with torch.no_grad():
        assert float((torch.compile(f, fullgraph=True)(*x, table) - want).float().norm() / want.float().norm()) < 2 * HALF[B]


def test_registered_operators(pdm, dev):
    q, k, v = (torch.randn(20, n, 64, device=dev).to(B).requires_grad_(True) for n in (2, 1, 1))
    bias = torch.randn(2, 5, device=dev, requires_grad=True)
    cu = _t([0, 12, 20], dev)
    for b, keep in ((bias, 2), (None, 1)):
        torch.library.opcheck(torch.ops.pdm.jagged_attention.default, (q, k, v, cu, cu, b, 0.125, True, 5, 1, 0, keep))
    table = torch.randn(4, 2, device=dev, requires_grad=True)
    torch.library.opcheck(torch.ops.pdm.bucket_bias.default, (table, pdm.relative_buckets(4, 9, device=dev)))


# ---- the bias by buckets ----------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, B, H])
@pytest.mark.parametrize("n,heads,span", [(1, 1, 1), (7, 5, 300), (32, 16, 1000), (8192, 3, 9000), (3, 130, 64), (64, 6, 70_000)])
def test_bucket_bias(pdm, dev, dtype, n, heads, span):
    """Spread bit for bit; a gradient is a sum in 64 bits, rounded to fp32 and to the table's type."""
    g = torch.Generator().manual_seed(span)
    table = torch.randn(n, heads, generator=g).to(dtype)
    for maps in (torch.randint(-1, n + 1, (span,), generator=g), torch.arange(span) * n // span, torch.full((span,), n - 1)):
        t = table.to(dev).requires_grad_(True)
        out = pdm.bucket_bias(t, maps.int().to(dev))
        ok = (maps >= 0) & (maps < n)
        want = torch.where(ok, table.float()[maps.clamp(0, n - 1)].t(), 0.0)
        assert out.dtype == torch.float32 and torch.equal(out.cpu(), want)
        go = torch.randn(heads, span, generator=g)
        (got,) = torch.autograd.grad(out, [t], go.to(dev))
        sums = torch.zeros(n, heads, dtype=torch.float64).index_add_(0, maps[ok], go.t()[ok].double())
        size = torch.zeros(n, heads, dtype=torch.float64).index_add_(0, maps[ok], go.t()[ok].double().abs())
        step = torch.finfo(dtype).eps / 2
        assert got.dtype == dtype
        assert ((got.cpu().double() - sums).abs() <= (step + U) * sums.abs() + 1e-15 * size + 2.0 ** -25).all()


def test_relative_bias_module(pdm, dev):
    for both in (False, True):
        rel = pdm.RelativeBias(3, 16, 50, both_sides=both, device=dev)
        assert rel().shape == (3, 101 if both else 51) and rel.start == (-50 if both else 0)
        assert list(rel.state_dict()) == ["table"]
        rel().sum().backward()
        assert float(rel.table.grad.sum()) == 3 * (101 if both else 51)
        assert torch.equal(rel.half()().cpu(), torch.zeros(3, 101 if both else 51)) and rel.buckets.dtype == torch.int32

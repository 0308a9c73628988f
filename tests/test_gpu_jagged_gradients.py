"""Gradients of jagged_attention where the definition leaves no room: rows that see one key; rows behind the last query, columns that no
pair has; small weights; sinks of many sequences; very wide biases; columns of nearly all weights."""
import math

import pytest
import torch

from test_gpu_jagged_attention import B, H, HALF, Case

pytestmark = pytest.mark.gpu

KINDS = [(64, 3, 1, B), (128, 1, 4, B), (64, 2, 2, H), (128, 2, 1, H)]


def _new(c, dtype):
    """The case's gradients of a batch of its own seed: of any size, as training has them."""
    c.go = (c.go.float() * 3).to(dtype)
    return c


# ---- rows that see one key ------------------------------------------------------------------
# The softmax of one score is 1 whatever the score, so dS is 0: q, k and the bias get no gradient at all, and v that of the output.

@pytest.mark.parametrize("D,hk,group,dtype", KINDS)
@pytest.mark.parametrize("span,start", [(0, 0), (1, 0), (40, -3)])
@pytest.mark.parametrize("lens,mask", [([1] * 130, dict(causal=True)), ([1] * 9, dict(causal=False)), ([100, 33, 1], dict(causal=True, window=1)),
                                       ([700], dict(causal=True, window=1)), ([1] * 70, dict(causal=True, window=5, sinks=2))])
def test_rows_that_see_one_key(pdm, dev, D, hk, group, dtype, span, start, lens, mask):
    c = _new(Case(lens, lens, hk * group, hk, D, dtype, span, start, seed=len(lens) + D), dtype)
    (out, _), grads = c.grads(pdm, dev, **mask)
    assert torch.equal(out.cpu(), c.v.repeat_interleave(group, 1))
    dq, dk, dv, *db = (g.cpu() for g in grads)
    assert not dq.any() and not dk.any() and not (db and db[0].any())
    want = c.go.double().view(-1, hk, group, D).sum(2)
    # the sum over the group in fp32, rounded once
    assert ((dv.double() - want).abs() <= HALF[dtype] * want.abs() + 4 * 2.0 ** -24 * c.go.double().abs().view(-1, hk, group, D).sum(2)).all()


@pytest.mark.parametrize("D,hk,group,dtype", KINDS)
@pytest.mark.parametrize("span", [0, 25])
def test_rows_that_see_one_key_beside_others(pdm, dev, D, hk, group, dtype, span):
    """The first query of a causal sequence; the first one that has a key at all; queries before their window's sink."""
    for new, lens, mask, rows in (([150, 1, 40], [150, 90, 40], dict(causal=True), [0, 151]), ([70, 5], [30, 5], dict(causal=True), [40, 70]),
                                  ([90], [90], dict(causal=True, window=1, sinks=1), [0])):
        c = _new(Case(new, lens, hk * group, hk, D, dtype, span, seed=D), dtype)
        got, grads = c.grads(pdm, dev, **mask)
        assert not grads[0][rows].any() and grads[0].any()
        w = c.want(True, **mask)
        c.check(got, w)
        c.check_grads(grads, w)


def test_rows_that_see_one_key_through_lse(pdm, dev):
    """lse is the score then, and its gradient the score's."""
    for D, dtype, span in ((64, B, 0), (128, H, 30), (64, H, 0), (128, B, 30)):
        c = Case([90, 1], [90, 1], 2, 1, D, dtype, span, seed=D)
        c.go = torch.zeros_like(c.go)
        _, (dq, dk, dv, *db) = c.grads(pdm, dev, gl=True, window=1)
        gl, scale = c.gl.double()[..., None], D ** -0.5
        for got, want in ((dq, gl * scale * c.k.double()), (dk, (gl * scale * c.q.double()).sum(1, keepdim=True))):
            # half a step of dS, of the result
            slack = 2 * HALF[dtype] * (gl.abs() * scale * (c.k if got is dq else c.q).double().abs())
            slack = slack if got is dq else slack.sum(1, keepdim=True)
            assert ((got.cpu().double() - want).abs() <= slack + 2.0 ** -24).all()
        assert not dv.any()
        if span:
            assert ((db[0].cpu().double()[:, 0] - c.gl.double().sum(0)).abs() <= 91 * 2.0 ** -24 * c.gl.double().abs().sum(0)).all()
            assert not db[0][:, 1:].any()


# ---- rows behind a sequence's last query -------------------------------------------------------
# A block holds 32 queries, of which the last ones may not be there.  What the bias holds at their distances is nobody's.

@pytest.mark.parametrize("D,dtype", [(64, B), (128, H)])
@pytest.mark.parametrize("new,lens", [([100], [300]), ([1, 33], [65, 400]), ([150], [150])])
def test_a_bias_of_any_size(pdm, dev, D, dtype, new, lens):
    """A constant added to a head's bias changes no gradient, however large the weights of it alone would be."""
    for mask, span in ((dict(causal=True), 350), (dict(causal=True), 20), (dict(causal=False), 30), (dict(causal=True, window=70, sinks=3), 350)):
        c = Case(new, lens, 2, 1, D, dtype, span, -100 if not mask["causal"] else 0, seed=span)
        c.bias[0] += 100.0
        c.bias[1] += 1000.0
        w = c.want(True, **mask)
        got, grads = c.grads(pdm, dev, **mask)
        c.check(got, w)
        c.check_grads(grads, w)


@pytest.mark.parametrize("D,dtype", [(64, B), (128, H)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, 3e38])
def test_columns_that_no_seen_pair_has(pdm, dev, D, dtype, bad):
    for new, lens, mask, span, first in (([100], [300], dict(causal=True, window=80), 300, 80), ([33, 70], [33, 300], dict(causal=True), 400, 300),
                                         ([40], [140], dict(causal=False, window=100), 250, 100 + 139)):
        c = Case(new, lens, 2, 1, D, dtype, span, 0 if mask["causal"] else -139, seed=3)
        w = c.want(True, **mask)
        c.bias[:, first:] = bad
        got, grads = c.grads(pdm, dev, **mask)
        c.check(got, w)
        assert not grads[3][:, first:].any()
        c.check_grads(grads, w)


def test_a_key_that_is_not_finite_reaches_seen_columns_alone(pdm, dev):
    for D, dtype in ((64, B), (128, H)):
        c = Case([70], [300], 2, 1, D, dtype, 400, seed=4)
        c.k[200, 0, 3] = math.inf
        _, grads = c.grads(pdm, dev)
        # (a row whose score of that key is -inf does without it)
        finite = torch.isfinite(c.want(True).dbias)
        assert not finite.all() and torch.equal(torch.isfinite(grads[3]).cpu(), finite) and not grads[3][:, 300:].any()


# ---- small weights in fp16 --------------------------------------------------------------------------

@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("gap", [9.0, 13.0, 17.0, 19.5])
@pytest.mark.parametrize("mask", [dict(causal=False), dict(causal=True, window=60, sinks=40)])
def test_small_weights_in_half_precision(pdm, dev, D, gap, mask):
    """One key takes nearly all of every row; the others' gradients, of weights about e^-gap and a scaled gradient of the output,
    are as exact as large ones.  p <= 1 meets dO as p 2^15: half a step of it down to 2^-29, 2^-40 below."""
    n, scale = 200, D ** -0.5
    c = Case([n], [n], 1, 1, D, H, seed=int(gap))
    u = torch.ones(D) / math.sqrt(D)
    c.q = (u + torch.randn(n, 1, D, generator=torch.Generator().manual_seed(1)) * 0.02).to(H)
    c.k = (c.k.float() * 0.02).to(H)
    c.k[0, 0] = (u * gap / scale).to(H)
    c.go = (c.go.float() * 500).to(H)
    q, k, go = c.q[:, 0].double(), c.k[:, 0].double(), c.go[:, 0].double()
    seen = torch.ones(n, n, dtype=torch.bool)
    if mask["causal"]:
        i, j = torch.arange(n)[:, None], torch.arange(n)[None]
        seen = (j <= i) & ((j > i - 60) | (j < 40))
    p = torch.softmax((q @ k.T * scale).masked_fill(~seen, -math.inf), -1)
    assert p[100, 1:][seen[100, 1:]].max() < 2.0 ** -11
    want, size = p.T @ go, p.T @ go.abs()
    serr = float((q.abs() @ k.abs().T * scale).max())
    e_w = 2 * (D + 8) * 2.0 ** -24 * serr + 2.0 ** -20 + n * 2.0 ** -24
    tol = (HALF[H] + e_w) * size + 2.0 ** -40 * go.abs().sum(0)
    _, (_, _, dv) = c.grads(pdm, dev, **mask)
    bad = (dv[:, 0].cpu().double() - want).abs() - tol - HALF[H] * (want.abs() + tol) - 2.0 ** -25
    assert bad.max().item() <= 0, f"dv over by {bad.max().item():.3e}"
    # (a result below 2^-14 is off by 2^-25)
    rest = want[1:]
    assert float((dv[1:, 0].cpu().double() - rest).norm() / rest.norm()) < 2 * HALF[H] + 2.0 ** -25 * math.sqrt(rest.numel()) / float(rest.norm())


# ---- sinks of many sequences ------------------------------------------------------------------------
# Queries beyond the window are those of sequences longer than it, and so are the sums kept for them.

@pytest.mark.parametrize("D,hk,group,dtype", KINDS)
@pytest.mark.parametrize("window,sinks", [(30, 4), (7, 33), (1, 1), (1, 200), (5, 200), (40, 41), (100, 3), (33, 32)])
def test_sinks_of_many_sequences(pdm, dev, D, hk, group, dtype, window, sinks):
    """Mostly short ones, some of about the window's length, a few long; empty ones; with queries for all of the keys or for some."""
    g = torch.Generator().manual_seed(window)
    lens = torch.randint(0, 12, (200,), generator=g).tolist()
    for at, n in ((3, window), (4, window + 1), (5, window), (50, window + 2), (51, window + 1), (52, 2 * window + 2), (120, 150), (121, 0), (122, 129), (199, window + 33)):
        lens[at] = n
    for new in (lens, [min(n, x) for n, x in zip(lens, torch.randint(0, 60, (200,), generator=g).tolist())]):
        c = Case(new, lens, hk * group, hk, D, dtype, 20, seed=sinks)
        mask = dict(causal=True, window=window, sinks=sinks)
        w = c.want(True, **mask)
        got, grads = c.grads(pdm, dev, **mask)
        c.check(got, w)
        c.check_grads(grads, w)


def test_many_short_sequences_with_sinks(pdm, dev):
    """40,000 sequences of 50 tokens, none of which has a query beyond the window, and one that has: the bits that the same
    sequences have without sinks, within memory of the size of the batch's."""
    n, length = 40_000, 50
    g = torch.Generator(device=dev).manual_seed(5)
    cu = torch.cat((torch.arange(n + 1) * length, torch.tensor([n * length + 400]))).int().to(dev)
    T = n * length + 400
    x = [torch.randn(T, 1, 64, generator=g, device=dev).to(B).requires_grad_(True) for _ in range(3)]
    go = torch.randn(T, 1, 64, generator=g, device=dev).to(B)
    torch.cuda.synchronize()
    grads = []
    for sinks in (0, 4):
        out = pdm.jagged_attention(*x, cu, window=300, sinks=sinks)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        grads.append(torch.autograd.grad(out, x, go))
        torch.cuda.synchronize()
        assert torch.cuda.max_memory_allocated() - held < 6 * T * 64 * 2
    for a, b in zip(*grads):
        assert torch.equal(a[:n * length], b[:n * length]) and not torch.equal(a[n * length:], b[n * length:])


# ---- a bias of more columns than a dimension of a launch has threads -------------------------------------

def test_gradient_of_a_very_wide_bias(pdm, dev):
    c = Case([40], [40], 1, 1, 64, B, 50, seed=6)
    w = c.want(True)
    x, span = c.inputs(dev), 2 ** 28 + 100
    wide = torch.zeros(1, span, device=dev)
    wide[:, :50] = x[3]
    held = torch.full_like(wide, math.nan)  # whose memory the gradient gets
    del held
    x = [t.detach().requires_grad_(True) for t in (*x[:3], wide)]
    out, _ = c.call(pdm, dev, x)
    grads = list(torch.autograd.grad(out, x, c.go.to(dev)))
    assert not grads[3][:, 50:].any()
    grads[3] = grads[3][:, :50]
    c.check_grads(grads, w)


# ---- columns of nearly all weights -----------------------------------------------------------------------

@pytest.mark.parametrize("D,dtype", [(64, B), (128, B), (64, H), (128, H)])
@pytest.mark.parametrize("span,start,mask", [(2, 0, dict(causal=True)), (3, 5000, dict(causal=False)), (70, -900, dict(causal=True, window=1000, sinks=4))])
@pytest.mark.parametrize("gl", [False, True])
def test_columns_of_nearly_all_weights(pdm, dev, D, dtype, span, start, mask, gl):
    """The dS of a row add up to the gradient of its lse, and so does what such a column has of it, but for the few others: terms far
    larger than their sum.  What is left of delta's error (2^-19 of |dO| |out|, in every row) would be ten times what fp32 sums
    are off by.  These: an addition by 2^-25 of what has been summed, half of a row's sizes at most; a row's are summed in
    blocks of 32 keys.  As a root mean square over the heads, twice that (another part is the products', of the same size)."""
    n, length, heads = 200, 1200, 16
    c = Case([n], [length], heads, heads, D, dtype, span, start, seed=D, spread=3.0)
    c.bias[:, 0] = -8.0 if span == 2 else 0.0
    if not gl:
        c.gl = torch.zeros_like(c.gl)
    _, (_, _, _, db) = c.grads(pdm, dev, gl=True, **mask)
    i, j = torch.arange(length - n, length)[:, None], torch.arange(length)[None]
    seen = (j <= i) if mask["causal"] else torch.ones(n, length, dtype=torch.bool)
    if "window" in mask:
        seen = seen & ((j > i - mask["window"]) | (j < mask["sinks"]))
    col = (i - j - start).clamp(0, span - 1)
    errors, sizes = [], []
    for h in range(heads):
        q, k, v, go = (t[:, h].double() for t in (c.q, c.k, c.v, c.go))
        s = q @ k.T * D ** -0.5 + c.bias[h].double()[col]
        p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        ds = p * (go @ v.T - (go * (p @ v)).sum(-1, keepdim=True) + c.gl[:, h, None].double())
        mass = torch.zeros(span, dtype=torch.float64).index_add_(0, col.flatten(), p.flatten())
        most = int(mass.argmax())
        assert mass[most] > 0.99 * n and most in (0, span - 1)
        errors.append(float(db[h, most]) - float(ds[col == most].sum()))
        sizes.append(float(ds.abs().sum(-1).square().sum()) * length / 32)
    rms = lambda x: math.sqrt(sum(x) / heads)  # noqa: E731
    assert rms([e * e for e in errors]) <= 2 * 2.0 ** -25 * rms(sizes)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,span", [(100, 128), (500, 128), (300, 400)])
def test_precision_of_the_bias_gradient(pdm, dev, D, n, span):
    """What is left of delta's error in bf16 is that of weights in two parts, outputs being kept whole.  The second part is off by half
    a step of bf16 of the first's error, which lies anywhere in half a step: 2^-19.6 of a weight as a root mean square (2^-18 at most).
    A row's delta is off by the mean of dP that these make, and a column by the rows' by its weights.  Beside it scores and sums of
    fp32, 2^-22 of the result."""
    c = Case([n], [n], 8, 8, D, B, span, seed=n)
    db = c.grads(pdm, dev)[1][3].cpu().double()
    w = c.want(True)
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    col = (i - j).clamp(0, span - 1)
    square = 0.0
    for h in range(8):
        q, k, v, go = (t[:, h].double() for t in (c.q, c.k, c.v, c.go))
        p = torch.softmax((q @ k.T * D ** -0.5 + c.bias[h].double()[col]).masked_fill(j > i, -math.inf), -1)
        of_row = (p * (go @ v.T)).square().sum(-1, keepdim=True)
        in_column = torch.zeros(n, span, dtype=torch.float64).scatter_add_(1, col, p)
        square += float((in_column.square() * of_row).sum())
    assert float((db - w.dbias).norm()) < 2.0 ** -19.6 * math.sqrt(square) + 2.0 ** -22 * float(w.dbias.norm())


@pytest.mark.parametrize("D,hk,group,dtype", KINDS)
def test_a_bias_of_one_column(pdm, dev, D, hk, group, dtype):
    """It moves all scores of a row alike: its gradient is that of the lse, of the rows that see a key."""
    for new, lens, mask, start in (([300, 5], [300, 90], dict(causal=True), 0), ([70, 40], [30, 40], dict(causal=True, window=20, sinks=3), 7),
                                   ([90], [200], dict(causal=False), -50)):
        c = Case(new, lens, hk * group, hk, D, dtype, 1, start, seed=D)
        _, (*_, db) = c.grads(pdm, dev, **mask)
        assert not db.any()
        got, (*_, db) = c.grads(pdm, dev, gl=True, **mask)
        gl = torch.where(torch.isinf(got[1].detach().cpu()), 0.0, c.gl).double()
        # sums of 128 rows in fp32, of those in 64 bits
        assert ((db.cpu().double()[:, 0] - gl.sum(0)).abs() <= 10 * 2.0 ** -24 * gl.abs().sum(0)).all()


def test_one_plane_of_statistics(pdm, dev):
    """Callers of the C entries that keep one plane: the same outputs and gradients, but for the outer columns' correction."""
    import ctypes

    L, ops = pdm._lib, pdm.ops
    c = Case([90, 20], [90, 120], 4, 2, 64, B, 12, seed=9)
    q, k, v, bias = c.inputs(dev)
    cu = [torch.tensor(x, dtype=torch.int32, device=dev) for x in (c.cu_q, c.cu_k)]
    args = (0.125, True, 0, 0, 0)
    out, _, stats, rest = ops.jagged_attention_raw(q, k, v, *cu, bias, *args, keep=2)
    assert stats.shape == (2, 110, 4, 2)
    out1, rest1, stats1 = torch.empty_like(out), torch.empty_like(rest), torch.full((2, 110, 4, 2), 7.0, device=dev)
    desc = ops._jagged_desc(q, k, v, *cu, bias, *args, 1)
    L.check(L.lib().pdm_jagged_attention_fwd(ctypes.byref(desc), q.data_ptr(), k.data_ptr(), v.data_ptr(), cu[0].data_ptr(), cu[1].data_ptr(),
                                             bias.data_ptr(), out1.data_ptr(), rest1.data_ptr(), None, stats1.data_ptr(), None, 0, None,
                                             L.raw_stream(0)), "pdm_jagged_attention_fwd")
    assert torch.equal(out, out1) and torch.equal(rest, rest1) and torch.equal(stats[0], stats1[0]) and (stats1[1] == 7).all()
    both = ops.jagged_attention_backward_raw(q, k, v, *cu, bias, out, stats, rest, c.go.to(dev), None, *args)
    one = ops.jagged_attention_backward_raw(q, k, v, *cu, bias, out, stats[0], rest, c.go.to(dev), None, *args)
    assert all(torch.equal(a, b) for a, b in zip(both[:3], one[:3])) and torch.equal(both[3][:, 1:-1], one[3][:, 1:-1])
    w = c.want(True)
    c.check_grads(both, w)
    c.check_grads(one, w)

"""kv_attention against its definition in 64 bits: single tokens to prompts, grouped heads, every head width, page size and
mask; what lies in masked and unused places; bad pages and lengths; graphs, streams; the three operators together.

Tolerance of an output: scores are sums of D exact products in fp32, in some order, e_s = (D + 8) u max_j scale sum_d |q_d
k_jd| (u = 2^-24), plus the rounding of the exponent's argument and of exp2, 2^-21; a weight is then off by the factor
1 + 2 e_s + 2^-20, and by half a step of bf16, 2^-8, where it meets the values.  So |out - want| <= (2^-8 + 2 e_s + 2^-20) sum
p |v|, and half a step of the output's type.  The sum of the weights, before their rounding, has the first two errors only:
|lse - want| <= e_s + 2^-20 + 2 u |want|."""
import math

import pytest
import torch

from oracle import cached_attention as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _t(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Case:
    def __init__(self, pdm, dev, new, lens, hq, hk, D, page, dtype=torch.bfloat16, seed=0, extra=0, spread=1.5):
        g = torch.Generator().manual_seed(seed)
        self.pdm, self.dev, self.new, self.lens = pdm, dev, new, lens
        counts = [-(-n // page) for n in lens]
        pages = sum(counts) + 2
        order = torch.randperm(pages, generator=g).tolist()
        width = max(counts + [0]) + extra
        self.table = []
        for c in counts:
            self.table.append([order.pop() for _ in range(c)] + [-1] * (width - c))
        self.cu = [0]
        for n in new:
            self.cu.append(self.cu[-1] + n)
        self.cache = pdm.PagedKVCache(pages, page, hk, D, dev)
        c = self.cache
        for codes, scale, e in ((c.k_codes, c.k_scale, -7), (c.v_codes, c.v_scale, -8)):
            # what the sequences do not use is NaN
            vals = torch.full(codes.shape, math.nan)
            for row, n in zip(self.table, lens):
                for i in range(-(-n // page)):
                    m = min(page, n - i * page)
                    vals[row[i], :, :m] = torch.randn(hk, m, D, generator=g) * 100
            codes.copy_(vals.clamp(-448, 448).to(torch.float8_e4m3fn))
            scale.copy_(torch.exp2(torch.randint(e - 2, e + 2, scale.shape, generator=g).float()))
        self.q = (torch.randn(self.cu[-1], hq, D, generator=g) * spread).to(dtype)

    def values(self):
        return [t.cpu() for t in self.cache.values()]

    def want(self, scale=None, causal=True, window=0):
        k, v = self.values()
        return ref.attention(self.q, k, v, self.cu, self.table, self.lens,
                             self.q.shape[-1] ** -0.5 if scale is None else scale, causal, window)

    def run(self, q=None, table=None, **kw):
        B = len(self.lens)
        table = torch.tensor(self.table if table is None else table, dtype=torch.int32).view(B, -1).to(self.dev)
        return self.cache.attend((self.q if q is None else q).to(self.dev), _t(self.cu, self.dev), table,
                                 _t(self.lens, self.dev), return_lse=True, **kw)

    def check(self, got, want):
        out, lse = got
        w_out, w_lse, mag, sabs = want
        D = self.q.shape[-1]
        e = (D + 8) * U * sabs[..., None]
        slack = (2.0 ** -8 + 2 * e + 2.0 ** -20) * mag
        out, lse = out.cpu().double(), lse.cpu().double()
        assert torch.equal(out.isnan(), w_out.isnan())
        bad = ((out - w_out).abs() - slack - STEP[self.q.dtype] * (w_out.abs() + slack) - 2.0 ** -25).nan_to_num(-1)
        assert bad.max().item() <= 0 if bad.numel() else True, f"out over by {bad.max().item():.3e}"
        empty = torch.isinf(w_lse)
        assert torch.equal(torch.isinf(lse), empty) and (lse[empty] < 0).all() and (out[empty] == 0).all()
        assert torch.equal(lse.isnan(), w_lse.isnan())
        bad = ((lse - w_lse).abs() - e[..., 0] - 2.0 ** -20 - 2 * U * w_lse.abs())[~empty].nan_to_num(-1)
        assert bad.max().item() <= 0 if bad.numel() else True, f"lse over by {bad.max().item():.3e}"
        assert self.cache.err_flag.item() == 0


DECODE = [1, 15, 16, 17, 33, 64, 100, 129, 250, 700]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("group", [1, 4, 7, 16, 24])
def test_single_tokens(pdm, dev, dtype, D, page, group):
    c = Case(pdm, dev, [1] * len(DECODE), DECODE, 2 * group, 2, D, page, dtype, seed=group, extra=1)
    want = c.want()
    c.check(c.run(max_q_len=1), want)
    c.check(c.run(), want)


@pytest.mark.parametrize("hk,group", [(1, 1), (1, 40), (8, 4)])
@pytest.mark.parametrize("length", [3000, 9001])
def test_long_contexts(pdm, dev, hk, group, length):
    """One sequence alone: its keys are split over many workgroups and joined."""
    c = Case(pdm, dev, [1], [length], hk * group, hk, 128, 16, seed=length)
    c.check(c.run(max_q_len=1), c.want())
    c = Case(pdm, dev, [3, 1], [length, 5], hk * group, hk, 64, 64, seed=length)
    c.check(c.run(max_q_len=3), c.want())


RAGGED = [
    ([16, 16, 16], [16, 400, 1516]), ([5, 0, 1, 64], [5, 7, 300, 64]), ([33, 1, 130], [33, 1000, 400]),
    ([257, 2, 0], [500, 90, 0]), ([300], [300]), ([1, 520], [2000, 777]),
]


@pytest.mark.parametrize("new,lens", RAGGED)
@pytest.mark.parametrize("D,page,hk,group", [(64, 32, 3, 1), (128, 64, 2, 4), (128, 16, 1, 5), (256, 128, 1, 2), (64, 16, 2, 8)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 100), (False, 37)])
def test_ragged(pdm, dev, new, lens, D, page, hk, group, causal, window):
    c = Case(pdm, dev, new, lens, hk * group, hk, D, page, seed=len(new) + D, extra=2)
    kw = dict(causal=causal, window=window)
    want = c.want(**kw)
    c.check(c.run(max_q_len=max(new), **kw), want)
    c.check(c.run(**kw), want)


@pytest.mark.parametrize("new,lens", [([4, 2], [40, 300]), ([150], [470])])
def test_fp16_queries(pdm, dev, new, lens):
    for D in (64, 128, 256):
        c = Case(pdm, dev, new, lens, 6, 2, D, 32, torch.float16, seed=D)
        c.check(c.run(), c.want())


def test_scores_of_any_size(pdm, dev):
    """Sharp and flat softmaxes, negative and zero scales, sizes that a plain exponential would not hold, scores that grow
    along the keys so that the running maximum moves all the time."""
    for spread, scale in ((60.0, None), (0.0, None), (1.0, -0.3), (1.0, 0.0), (400.0, 0.5)):
        for new, lens in (([1, 3], [300, 90]), ([140], [500])):
            c = Case(pdm, dev, new, lens, 4, 2, 64, 16, seed=3, spread=spread)
            c.check(c.run(scale=scale), c.want(scale=scale))
    for D in (64, 128):
        for new in (1, 200):
            c = Case(pdm, dev, [new], [600], 2, 1, D, 32, seed=4)
            grow = torch.zeros(c.cache.k_codes.shape)
            for i, p in enumerate(c.table[0]):
                at = torch.arange(32)[:, None] + 32.0 * i
                grow[p, 0] = at / 600 * 300 + torch.randn(32, D)
            c.cache.k_codes.copy_(grow.clamp(-448, 448).to(torch.float8_e4m3fn))
            c.cache.k_scale.fill_(2.0 ** -4)
            c.q = c.q.abs()
            c.check(c.run(), c.want())


@pytest.mark.parametrize("new,lens", [([1], [70]), ([7], [70]), ([200], [260])])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_reaches_only_the_rows_that_see_it(pdm, dev, new, lens, D):
    """A NaN key or value of one token: rows before it (causal), and rows whose window has left it, stay as they are."""
    n, length = new[0], lens[0]
    for at in (length - 1, length - 3, length // 2, 0):
        for which in ("k_codes", "v_codes"):
            for window in (0, 20):
                c = Case(pdm, dev, new, lens, 4, 2, D, 16, seed=at + D)
                codes = getattr(c.cache, which).view(torch.uint8)
                codes[c.table[0][at // 16], 1, at % 16, 5] = 0x7F
                want = c.want(window=window)
                got = c.run(window=window)
                hit = torch.arange(length - n, length) >= at
                if window:
                    hit &= torch.arange(length - n, length) < at + window
                assert torch.equal(want[0].isnan().any(-1)[:, 2:].any(-1), hit)
                c.check(got, want)


def test_infinite_queries_stay_in_their_rows(pdm, dev):
    for new, lens in (([3], [50]), ([140], [200])):
        c = Case(pdm, dev, new, lens, 4, 2, 64, 16, seed=1)
        want = c.run()
        c.q[1, 2] = math.inf
        got = c.run()
        keep = torch.ones(c.q.shape[:2], dtype=torch.bool)
        keep[1, 2] = False
        assert torch.equal(got[0].cpu()[keep], want[0].cpu()[keep]) and got[0][1, 2].isnan().all()


def test_padding_rows_and_given_output(pdm, dev):
    """Rows behind the last sequence come out as zeros, whatever they hold; `out` is written completely."""
    for n_pad in (1, 50, 300):
        c = Case(pdm, dev, [3, 1], [20, 90], 4, 2, 64, 16, seed=2)
        want = c.want()
        q = torch.cat((c.q, torch.full((n_pad, 4, 64), math.nan, dtype=c.q.dtype)))
        for kw in (dict(max_q_len=3), {}):
            out, lse = c.run(q=q, **kw)
            assert (out[4:] == 0).all() and (lse[4:] == -math.inf).all()
            c.check((out[:4], lse[:4]), want)
        given = torch.full_like(q, 7).to(dev)
        k = c.cache
        got = pdm.kv_attention(q.to(dev), k.k_codes, k.v_codes, k.k_scale, k.v_scale, _t(c.cu, dev), _t(c.table, dev),
                               _t(c.lens, dev), out=given)
        assert got.data_ptr() == given.data_ptr() and torch.equal(got, out)
    for T, B in ((0, 0), (0, 2), (5, 0), (5, 2)):
        out, lse = pdm.kv_attention(torch.ones(T, 4, 64, dtype=torch.bfloat16, device=dev), k.k_codes, k.v_codes, k.k_scale,
                                    k.v_scale, _t([0] * (B + 1), dev), torch.zeros(B, 1, dtype=torch.int32, device=dev),
                                    _t([5] * B, dev), return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all() and out.shape == (T, 4, 64)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 40, 40], [140, 3, 140]])
def test_bad_pages_and_lengths(pdm, dev, new):
    """Keys on pages that do not exist, and beyond the table, are left out; so are sequences whose spans do not fit; the
    flag says so; the sequence beside them has its result."""
    lens = [200, 180, 190]
    base = Case(pdm, dev, new, lens, 4, 2, 64, 16, seed=6)
    for bad in (-1, -(2 ** 31), 10_000, 2 ** 31 - 1):
        c = Case(pdm, dev, new, lens, 4, 2, 64, 16, seed=6)
        c.table[0][3] = bad
        c.table[2][0] = bad
        got, want = c.run(), c.want()
        assert c.cache.err_flag.item() == 1
        c.cache.err_flag.zero_()
        c.check(got, want)
    want = base.want()
    for change in (dict(lens=[200, 180, new[2] - 1]), dict(lens=[200, 180, -5]), dict(cu=base.cu[:3] + [base.cu[3] + 1])):
        c = Case(pdm, dev, new, lens, 4, 2, 64, 16, seed=6)
        for n, v in change.items():
            setattr(c, n, v)
        out, lse = c.run()
        assert c.cache.err_flag.item() == 1
        last = slice(base.cu[2], base.cu[3])
        assert (out[last] == 0).all() and (lse[last] == -math.inf).all()
        c.cache.err_flag.zero_()
        keep = slice(0, base.cu[2])
        c.check((out[keep], lse[keep]), [w[keep] for w in want])
    # more new tokens than promised
    if max(new) > 2:
        out, lse = base.run(max_q_len=2)
        assert base.cache.err_flag.item() == 1 and (out == 0).all() and (lse == -math.inf).all()
        base.cache.err_flag.zero_()
    # a table that is too narrow: the first 96 tokens are all that there is
    c = Case(pdm, dev, new, lens, 4, 2, 64, 16, seed=6)
    c.table = [row[:6] for row in c.table]
    got, want = c.run(), c.want()
    assert c.cache.err_flag.item() == 1
    c.cache.err_flag.zero_()
    c.check(got, want)


def test_every_key_of_a_row_on_a_bad_page(pdm, dev):
    for new in (2, 150):
        c = Case(pdm, dev, [new], [170], 4, 2, 64, 32, seed=1)
        c.table = [[-1] * 6]
        out, lse = c.run()
        assert (out == 0).all() and (lse == -math.inf).all() and c.cache.err_flag.item() == 1


def test_shared_pages_strides_and_tables(pdm, dev):
    """Candidates that share a history's pages; q as columns of wider rows, at an odd address, heads outermost; a page table
    that is a slice of a wider one."""
    c = Case(pdm, dev, [4, 4, 4], [100, 100, 100], 4, 2, 64, 16, seed=9)
    for row in c.table[1:]:
        row[:6] = c.table[0][:6]
    want = c.want()
    c.check(c.run(), want)
    base = c.run()
    wide = torch.zeros(12, 1001, dtype=c.q.dtype, device=dev)
    odd = wide[:, 3:259].view(12, 4, 64).copy_(c.q)
    turned = c.q.to(dev).transpose(0, 1).contiguous().transpose(0, 1)
    table = torch.full((3, 40), -1, dtype=torch.int32, device=dev)
    table[:, 5:12] = _t(c.table, dev)
    k = c.cache
    for q in (odd, turned, c.q.to(dev).view(3, 4, 4, 64)):
        got = pdm.kv_attention(q, k.k_codes, k.v_codes, k.k_scale, k.v_scale, _t(c.cu, dev), table[:, 5:12],
                               _t(c.lens, dev), return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(got, base))
    # the bytes of the codes as uint8
    got = pdm.kv_attention(c.q.to(dev), k.k_codes.view(torch.uint8), k.v_codes.view(torch.uint8), k.k_scale, k.v_scale,
                           _t(c.cu, dev), table[:, 5:12], _t(c.lens, dev), return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(got, base))


def test_many_sequences(pdm, dev):
    g = torch.Generator().manual_seed(2)
    new = torch.randint(0, 4, (4500,), generator=g).tolist()
    lens = [max(1, n + p) for n, p in zip(new, torch.randint(0, 20, (4500,), generator=g).tolist())]
    c = Case(pdm, dev, new, lens, 2, 1, 64, 16, seed=2)
    want = c.want()
    c.check(c.run(max_q_len=3), want)
    c.check(c.run(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,lens,D,page,hk,group", [
    ([150, 110], [500, 700], 128, 16, 32, 8), ([260, 0, 1, 600], [260, 9, 130, 901], 64, 64, 16, 5),
    ([1100, 950], [1100, 1000], 64, 128, 32, 1), ([700], [700], 128, 32, 24, 4), ([33, 400], [33, 64], 128, 64, 32, 8)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 70), (False, 333)])
def test_large_batches(pdm, dev, dtype, new, lens, D, page, hk, group, causal, window):
    """Rows enough that workgroups take 256 of them; blocks that end inside a sequence, a page, a tile."""
    lens = [max(n, x) for n, x in zip(new, lens)]
    c = Case(pdm, dev, new, lens, hk * group, hk, D, page, dtype, seed=D + hk)
    c.check(c.run(causal=causal, window=window), c.want(causal=causal, window=window))


@pytest.mark.parametrize("D", [64, 128])
def test_large_batches_with_bad_places(pdm, dev, D):
    """The same with a NaN value and a NaN key of one head, seen by some rows only, pages that do not exist, lengths that do
    not fit, padding; and the same bits from a second run."""
    new, lens = [500, 300, 600], [800, 350, 600]
    for which in ("k_codes", "v_codes"):
        for at in (40, 333, 799):
            c = Case(pdm, dev, new, lens, 64, 64, D, 32, seed=at)
            getattr(c.cache, which).view(torch.uint8)[c.table[0][at // 32], 5, at % 32, 7] = 0x7F
            got = c.run(window=250)
            c.check(got, c.want(window=250))
            assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(got, c.run(window=250)))
    c = Case(pdm, dev, new, lens, 64, 64, D, 32, seed=1)
    for b, i, bad in ((0, 3, -1), (0, 4, 2 ** 31 - 1), (2, 0, 10_000)):
        c.table[b][i] = bad
    want = c.want()
    q = torch.cat((c.q, torch.full((300, 64, D), math.nan, dtype=c.q.dtype)))
    out, lse = c.run(q=q)
    assert c.cache.err_flag.item() == 1 and (out[1400:] == 0).all() and (lse[1400:] == -math.inf).all()
    c.cache.err_flag.zero_()
    c.check((out[:1400], lse[:1400]), want)
    c.lens[1] = 299
    out, lse = c.run()
    assert c.cache.err_flag.item() == 1 and (out[500:800] == 0).all() and (lse[500:800] == -math.inf).all()
    c.cache.err_flag.zero_()
    keep = torch.cat((torch.arange(500), torch.arange(800, 1400)))
    c.check((out[keep], lse[keep]), [w[keep] for w in want])


@pytest.mark.parametrize("dtype,D,page", [(torch.bfloat16, 128, 32), (torch.float16, 64, 16), (torch.bfloat16, 256, 64)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 700)])
def test_prompts_among_single_tokens(pdm, dev, dtype, D, page, causal, window):
    """Keys of the sequences with many rows are split, those of the others too; some have no new tokens, one a page that does
    not exist in one of its splits, one a NaN value that some of its rows see; rows behind the last sequence."""
    new = [1, 60, 0, 1, 150, 2, 1, 0, 1, 33]
    lens = [900, 2500, 70, 5, 1800, 640, 3000, 40, 1, 33]
    c = Case(pdm, dev, new, lens, 8, 2, D, page, dtype, seed=D, extra=3)
    c.cache.v_codes.view(torch.uint8)[c.table[4][1700 // page], 1, 1700 % page, 9] = 0x7F
    c.table[1][1200 // page] = -1
    kw = dict(causal=causal, window=window)
    want = c.want(**kw)
    q = torch.cat((c.q, torch.full((7, 8, D), math.nan, dtype=dtype)))
    T = len(c.q)
    first = None
    for _ in range(2):
        out, lse = c.run(q=q, max_q_len=150, **kw)
        # (pages that no row's window reaches are not looked at: the lost one ends 1,200 tokens before the first row)
        assert c.cache.err_flag.item() == (window == 0) and (out[T:] == 0).all() and (lse[T:] == -math.inf).all()
        c.cache.err_flag.zero_()
        c.check((out[:T], lse[:T]), want)
        assert first is None or torch.equal(out.view(torch.int16), first.view(torch.int16))
        first = out


def _uneven(seed, n, most, longest):
    g = torch.Generator().manual_seed(seed)
    new = torch.randint(0, most + 1, (n,), generator=g).tolist()
    lens = torch.randint(1, 400, (n,), generator=g).tolist()
    lens[n // 3], lens[n - 1], lens[0] = longest, 2000, 1
    return new, [max(a, b) for a, b in zip(new, lens)]


@pytest.mark.parametrize("D,page,n,hk,group,most,longest", [
    (64, 16, 40, 8, 4, 2, 5000), (128, 32, 33, 8, 1, 8, 9000), (256, 64, 64, 4, 2, 2, 3500), (128, 128, 256, 4, 3, 1, 6001),
    (64, 64, 255, 2, 5, 1, 20000), (128, 16, 9, 40, 8, 1, 2500)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 150), (False, 1000)])
def test_many_uneven_contexts(pdm, dev, D, page, n, hk, group, most, longest, causal, window):
    """Batches whose keys are dealt to the workgroups: parts of a (sequence, head), several in a workgroup, one over many
    workgroups; sequences without new tokens."""
    new, lens = _uneven(D + n, n, most, longest)
    c = Case(pdm, dev, new, lens, hk * group, hk, D, page, torch.float16 if n == 64 else torch.bfloat16, seed=n, extra=1)
    kw = dict(causal=causal, window=window)
    want = c.want(**kw)
    c.check(c.run(max_q_len=most, **kw), want)
    c.check(c.run(max_q_len=8 // group, **kw), want)


@pytest.mark.parametrize("D,page,n,hk,group,most", [
    (64, 16, 32, 8, 4, 2), (128, 32, 33, 8, 1, 8), (128, 64, 90, 8, 2, 4), (256, 128, 64, 8, 3, 1), (64, 128, 255, 2, 8, 1)])
@pytest.mark.parametrize("lo,hi", [(700, 840), (150, 250), (130, 1000)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 140)])
def test_many_even_contexts(pdm, dev, D, page, n, hk, group, most, lo, hi, causal, window):
    """About equal contexts (the last range is not): parts of their own for each (sequence, head), one to four of them, some
    of which come out empty; sequences without new tokens among them."""
    g = torch.Generator().manual_seed(n)
    new = torch.randint(0, most + 1, (n,), generator=g).tolist()
    lens = torch.randint(lo, hi, (n,), generator=g).tolist()
    c = Case(pdm, dev, new, lens, hk * group, hk, D, page, torch.float16 if n == 64 else torch.bfloat16, seed=n, extra=9)
    kw = dict(causal=causal, window=window)
    got = c.run(max_q_len=most, **kw)
    c.check(got, c.want(**kw))
    assert all(torch.equal(a, b) for a, b in zip(got, c.run(max_q_len=most, **kw)))


def test_many_uneven_contexts_with_bad_places(pdm, dev):
    """NaN keys and values, infinite queries, pages that do not exist, sequences that do not fit, padding, in turn."""
    new, lens = _uneven(3, 40, 2, 4000)
    new[13], new[20] = 2, 1
    for which in ("k_codes", "v_codes"):
        c = Case(pdm, dev, new, lens, 16, 8, 128, 32, seed=1)
        for at in (0, 1500, lens[13] - 1):
            getattr(c.cache, which).view(torch.uint8)[c.table[13][at // 32], 3, at % 32, 64] = 0x7F
            for window in (0, 300):
                c.check(c.run(max_q_len=2, window=window), c.want(window=window))
    c = Case(pdm, dev, new, lens, 16, 8, 128, 32, seed=2)
    base = c.run(max_q_len=2)
    r = c.cu[13]
    c.q[r, 5] = math.inf
    got = c.run(max_q_len=2)
    keep = torch.ones(c.q.shape[:2], dtype=torch.bool)
    keep[r, 5] = False
    assert torch.equal(got[0].cpu()[keep], base[0].cpu()[keep]) and got[0][r, 5].isnan().all()
    c = Case(pdm, dev, new, lens, 16, 8, 128, 32, seed=2)
    for i in (0, 30, 31, 90):
        c.table[13][i] = -1
    c.table[20] = [-1] * len(c.table[20])
    want = c.want()
    q = torch.cat((c.q, torch.full((5, 16, 128), math.nan, dtype=c.q.dtype)))
    T = len(c.q)
    out, lse = c.run(q=q, max_q_len=2)
    assert c.cache.err_flag.item() == 1 and (out[T:] == 0).all() and (lse[T:] == -math.inf).all()
    c.cache.err_flag.zero_()
    c.check((out[:T], lse[:T]), want)
    fit = list(c.lens)
    c.lens[13] = 1  # below its two new tokens
    out, lse = c.run(max_q_len=2)
    assert c.cache.err_flag.item() == 1 and (out[r:r + 2] == 0).all() and (lse[r:r + 2] == -math.inf).all()
    c.cache.err_flag.zero_()
    keep = torch.tensor([t for t in range(T) if not r <= t < r + 2])
    c.check((out[keep], lse[keep]), [w[keep] for w in want])
    c.lens = fit
    out, lse = c.run(max_q_len=1)  # more new tokens than promised
    assert c.cache.err_flag.item() == 1
    c.cache.err_flag.zero_()
    one = torch.tensor([t for b in range(40) for t in range(c.cu[b], c.cu[b + 1]) if new[b] == 1])
    assert (out[r:r + 2] == 0).all() and (lse[r:r + 2] == -math.inf).all()
    c.check((out[one], lse[one]), [w[one] for w in want])


UNEVEN = _uneven(5, 140, 1, 2500)


@pytest.mark.parametrize("new,lens", [([1, 1], [900, 30]), ([40, 2, 200], [700, 90, 260]), UNEVEN, ([9000, 7400], [9000, 7400])])
def test_repeats_streams_and_graphs(pdm, dev, new, lens):
    """The same bits every time; two captured graphs and eager calls in turn, with lengths that change in place."""
    cs = [Case(pdm, dev, new, lens, 4, 2, 128, 32, seed=s, extra=2) for s in (0, 1)]
    dq = [c.q.to(dev) for c in cs]
    cu, table = _t(cs[0].cu, dev), [_t(c.table, dev) for c in cs]
    ln = _t(lens, dev)

    def step(i):
        k = cs[i].cache
        return pdm.kv_attention(dq[i], k.k_codes, k.v_codes, k.k_scale, k.v_scale, cu, table[i], ln, max_q_len=max(new),
                                return_lse=True)

    first = [step(0), step(1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(0)
    other = step(1)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*first[0], *first[1]), (*again, *other)))
    graphs, held = [], []
    for i in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(step(i))
        graphs.append(g)
    for r in range(4):
        ln.copy_(_t([max(n, x - 7 * r) for n, x in zip(new, lens)], dev))
        for i in (0, 1):
            graphs[i].replay()
        eager = [step(0), step(1)]
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(held[i], eager[i])), (r, i)


def test_compiled(pdm, dev):
    c = Case(pdm, dev, [3, 1], [40, 9], 4, 2, 64, 16, seed=2)
    k = c.cache
    args = (k.k_codes, k.v_codes, k.k_scale, k.v_scale, _t(c.cu, dev), _t(c.table, dev), _t(c.lens, dev))

    def f(q):
        out, lse = pdm.kv_attention(q * 1, *args, return_lse=True, err_flag=k.err_flag)
        return out * 2, lse, pdm.kv_attention(q, *args)

    want = f(c.q.to(dev))
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(c.q.to(dev))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_pages_beyond_32_bit_offsets(pdm, dev):
    """The last pages of a cache of more than 2^32 bytes, by single tokens and by a prompt."""
    D, page, hk = 128, 128, 4
    pages = 2 ** 32 // (D * page * hk) + 3
    c = Case(pdm, dev, [1, 140], [130, 200], 8, hk, D, page, seed=2)
    big = pdm.PagedKVCache(pages, page, hk, D, dev)
    n = c.cache.num_pages
    want = c.run()
    for name in ("k_codes", "v_codes", "k_scale", "v_scale"):
        a, b = getattr(big, name), getattr(c.cache, name)
        a.view(torch.uint8)[-n:] = b.view(torch.uint8)
    c.cache = big
    got = c.run(table=[[p + pages - n if p >= 0 else -1 for p in row] for row in c.table])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_layer_as_it_is_served(pdm, dev):
    """Histories arrive, grow by events, and candidates' tokens attend to them: the three operators in turn against one
    causal attention over all tokens in 64 bits.  An 8-bit key or value is off by 2^-4 of itself at most, the products'
    inputs by a bf16 rounding: outputs agree to a fraction of the values' size, and with the cache's own values exactly as
    in the tests above."""
    hq, hk, D, page, width = 6, 2, 64, 32, 128
    g = torch.Generator().manual_seed(1)
    w = (torch.randn(width, (hq + 2 * hk) * D, generator=g) / width ** 0.5).to(torch.bfloat16).to(dev)
    rope = pdm.QKNormRope(D, 512, device=dev)
    with torch.no_grad():
        rope.q_norm.weight.uniform_(0.8, 1.2)
        rope.k_norm.weight.uniform_(0.8, 1.2)
    cache = pdm.PagedKVCache(40, page, hk, D, dev)
    steps = [[200, 31, 64], [1, 1, 1], [7, 0, 20], [16, 16, 16]]
    table = _t(torch.randperm(40, generator=g)[:36].view(3, 12).tolist(), dev)
    lens, seen = [0, 0, 0], [[], [], []]
    for more in steps:
        start, lens = lens, [a + b for a, b in zip(lens, more)]
        x = torch.randn(sum(more), width, generator=g).to(torch.bfloat16).to(dev)
        pos = torch.cat([torch.arange(s, s + m) for s, m in zip(start, more)]).to(dev)
        cu = _t([0, more[0], more[0] + more[1], sum(more)], dev)
        with torch.no_grad():
            q, k, v = (t.view(len(x), -1, D) for t in (x @ w).split([hq * D, hk * D, hk * D], 1))
            qr, kr = rope(q, k, pos)
            q1, none = rope(q, None, pos)
            assert none is None and torch.equal(q1, qr)
            cache.append(k, v, cu, table, _t(lens, dev), rope=rope)
            out, lse = cache.attend(qr, cu, table, _t(lens, dev), max_q_len=max(more), return_lse=True)
        cache.check()
        # the cache holds the rotated keys and the values, within the quantizer's half step (and that of the bf16 keys)
        kc, vc = cache.values()
        for b in range(3):
            rows = slice(int(cu[b]), int(cu[b + 1]))
            seen[b].append((kr[rows].double().cpu(), v[rows].double().cpu()))
            at = torch.arange(lens[b])
            pg = table[b].cpu()[at // page].long()
            for held, i in ((kc.cpu(), 0), (vc.cpu(), 1)):
                true = torch.cat([s[i] for s in seen[b]])
                got = held[pg, :, at % page].double()
                top = true.abs().amax()
                assert ((got - true).abs() <= true.abs() * (2.0 ** -4 + 2.0 ** -8) + top * 2.0 ** -16).all()
            kt, vt = (torch.cat([s[i] for s in seen[b]]).repeat_interleave(hq // hk, 1) for i in (0, 1))
            if more[b]:
                s = torch.einsum("thd,jhd->htj", qr[rows].double().cpu(), kt) / D ** 0.5
                p = torch.arange(start[b], lens[b])
                s.masked_fill_(torch.arange(lens[b])[None] > p[:, None], -math.inf)
                true = torch.einsum("htj,jhd->thd", s.softmax(-1), vt)
                err = (out[rows].double().cpu() - true).norm() / true.norm()
                assert err < 2.0 ** -4, err
        # and exactly what the cache's own values give
        want = ref.attention(qr.cpu(), kc.cpu(), vc.cpu(), cu.tolist(), table.tolist(), lens, D ** -0.5, True, 0)
        c = Case.__new__(Case)
        c.q, c.cache = qr.cpu(), cache
        c.check((out, lse), want)


@pytest.mark.parametrize("T", [5, 40, 300])
@pytest.mark.parametrize("width", [0, 1, 64])
@pytest.mark.parametrize("D,hq,hk", [(64, 4, 2), (128, 40, 1), (256, 8, 8)])
def test_no_sequences(pdm, dev, T, width, D, hq, hk):
    """A batch of padding rows alone, few and many of them, with tables of any width: zeros."""
    cache = pdm.PagedKVCache(3, 16, hk, D, dev)
    q = torch.full((T, hq, D), math.nan, dtype=torch.bfloat16, device=dev)
    for most in (None, 1):
        out, lse = cache.attend(q, _t([0], dev), torch.zeros(0, width, dtype=torch.int32, device=dev), _t([], dev),
                                max_q_len=most, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
    cache.check()


@pytest.mark.parametrize("group", [2, 24, 40])
@pytest.mark.parametrize("cu", [[1000, 1003], [2 ** 31 - 4, 2 ** 31 - 1], [1000, 1003, 1003, 1003], [-3, 0], [6, 5]])
def test_spans_outside_the_batch_set_the_flag(pdm, dev, group, cu):
    """Also where no row of the batch leads to them, by either kernel."""
    cache = pdm.PagedKVCache(3, 16, 1, 64, dev)
    B = len(cu) - 1
    for most in (None, 3):
        out, lse = cache.attend(torch.ones(5, group, 64, dtype=torch.bfloat16, device=dev), _t(cu, dev),
                                torch.zeros(B, 1, dtype=torch.int32, device=dev), _t([9] * B, dev), max_q_len=most,
                                return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
        assert cache.err_flag.item() == 1
        cache.err_flag.zero_()


def test_traced(pdm, dev):
    """torch.jit.trace keeps the three operators: a traced step gives new results for new inputs."""
    c = Case(pdm, dev, [3, 1], [40, 9], 4, 2, 64, 16, seed=2)
    k, other = c.cache, Case(pdm, dev, [3, 1], [40, 9], 4, 2, 64, 16, seed=3)
    batch = (_t(c.cu, dev), _t(c.table, dev), _t(c.lens, dev))
    cos, sin = pdm.rotary_tables(50, 64, device=dev)
    pos = torch.tensor([37, 38, 39, 8], device=dev)
    held = (k.k_codes.view(torch.uint8), k.v_codes.view(torch.uint8), k.k_scale, k.v_scale)

    def f(q, kv):
        yq, yk = pdm.qk_norm_rope(q, kv, pos, cos, sin)
        codes = [t.clone() for t in held]
        pdm.kv_append(yk, kv, *codes, *batch)
        return pdm.kv_attention(yq, *codes, *batch, return_lse=True)

    kv = [torch.randn(4, 2, 64, device=dev).to(torch.bfloat16) for _ in range(2)]
    q = [x.q.to(dev) for x in (c, other)]
    traced = torch.jit.trace(f, (q[0], kv[0]), check_trace=False)
    for i in (0, 1):
        want, got = f(q[i], kv[i]), traced(q[i], kv[i])
        assert all(torch.equal(a, b) for a, b in zip(want, got)), i


HUGE = {  # new tokens, lengths, query heads per key head, key heads, max_q_len
    "alone": ([1], [100], 2, 2, 1), "split": ([3, 1], [2500, 700], 2, 1, 3), "two tiles of rows": ([7], [900], 4, 1, 7),
    "dealt": ([1] * 40, [130 + 40 * i for i in range(40)], 2, 8, 1), "even": ([1] * 40, [500] * 40, 2, 8, 1),
    "many": ([150, 40], [470, 900], 2, 2, 150), "many, split": ([60, 1], [2500, 30], 4, 1, 60),
    "two groups": ([500, 300, 600], [800, 350, 600], 1, 64, 600),
}


@pytest.mark.parametrize("which", HUGE)
@pytest.mark.parametrize("D,e", [(64, 81), (64, 119), (128, 113), (128, 119), (256, 119)])
def test_values_near_the_top_of_the_range(pdm, dev, which, D, e):
    """Values of up to 448 * 2^119, one step below what bf16 holds, behind scores that grow by 7.5 (a weight of 2^7.5 before the
    maximum moves) or move it with every tile: every output is a mean of the values, so it is finite, whatever sums it comes
    from.  The other places of the cache hold values of ordinary size."""
    new, lens, group, hk, most = HUGE[which]
    if len(new) == 3 and D == 256:
        hk = 8
    c = Case(pdm, dev, new, lens, group * hk, hk, D, 32, seed=e + D)
    c.q.zero_()
    c.q[..., 0] = 1.0
    for grow in (lambda j: torch.where(j < 40, 0.0, 7.5), lambda j: 6.5 * (j // 32).clamp(max=60), lambda j: 0.0 * j):
        k = torch.zeros(c.cache.k_codes.shape)
        for row, n in zip(c.table, lens):
            for i, p in enumerate(row):
                if p >= 0:
                    k[p, :, :, 0] = grow(torch.arange(32) + 32 * i)
        c.cache.k_codes.copy_(k.to(torch.float8_e4m3fn))
        c.cache.k_scale.fill_(1.0)
        v = c.cache.v_codes.float()
        v[:, 0] = 448.0
        if grow(torch.tensor([41])) == 0:  # with equal scores, the first pages of ordinary size
            c.cache.v_scale.fill_(2.0 ** e)
            c.cache.v_scale[[row[0] for row in c.table]] = 2.0 ** -6
        else:
            c.cache.v_scale.fill_(2.0 ** e)
        c.cache.v_codes.copy_(v.to(torch.float8_e4m3fn))
        got, want = c.run(scale=math.log(2), max_q_len=most), c.want(scale=math.log(2))
        assert torch.isfinite(got[0]).all()
        c.check(got, want)


@pytest.mark.parametrize("dtype,which", [(t, n) for n in HUGE for t in STEP if t == torch.float16 or HUGE[n][4] <= 16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_weights_are_finer_than_the_output(pdm, dev, dtype, which, D):
    """Weights reach the second product as a bf16 number and the bf16 remainder (all but many rows of bf16 outputs, whose own
    half step is a weight's): each rounding leaves 2^-8 of what it rounds, so a weight is off by 2^-16 of itself.  Sums of N
    products, N weights and up to N / 32 changes of the maximum are within (3 N + 16) u of their terms' sizes."""
    new, lens, group, hk, most = HUGE[which]
    if len(new) == 3 and D == 256:
        hk = 8
    c = Case(pdm, dev, new, lens, group * hk, hk, D, 32, dtype, seed=D)
    (out, lse), want = c.run(max_q_len=most), c.want()
    c.check((out, lse), want)
    w_out, _, mag, sabs = want
    slack = (2.0 ** -16 + 2 * (D + 8) * U * sabs[..., None] + 2.0 ** -20 + (3 * max(lens) + 16) * U) * mag
    bad = (out.cpu().double() - w_out).abs() - slack - STEP[dtype] * (w_out.abs() + slack) - 2.0 ** -25
    assert bad.max().item() <= 0, f"over by {bad.max().item():.3e}"


def test_under_a_dispatch_mode(pdm, dev):
    """A mode that watches operators sees the calls that are registered operators and leaves the others (a flag of
    qk_norm_rope, a given output) as they are."""
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    c = Case(pdm, dev, [3, 1], [40, 9], 4, 2, 64, 16, seed=2)
    k = c.cache
    args = (k.k_codes, k.v_codes, k.k_scale, k.v_scale, _t(c.cu, dev), _t(c.table, dev), _t(c.lens, dev))
    q, pos, err = c.q.to(dev), torch.arange(4, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    cos, sin = pdm.rotary_tables(50, 64, device=dev)
    want = pdm.kv_attention(q, *args), pdm.qk_norm_rope(q, None, pos, cos, sin)[0]
    given = torch.empty_like(q)
    with Watch():
        got = pdm.kv_attention(q, *args), pdm.qk_norm_rope(q, None, pos, cos, sin)[0]
        flagged = pdm.qk_norm_rope(q, None, pos, cos, sin, err_flag=err)[0]
        pdm.kv_attention(q, *args, out=given)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(flagged, want[1]) and torch.equal(given, want[0])
    assert [s for s in seen if s.startswith("pdm.")] == ["pdm.kv_attention.default", "pdm.qk_norm_rope.default"]


def test_registered_operators(pdm, dev):
    """Schemas, shapes without memory, autograd registration and dispatch of the three operators."""
    c = Case(pdm, dev, [3, 1], [40, 9], 4, 2, 64, 16, seed=2)
    k = c.cache
    held = [k.k_codes.view(torch.uint8).clone(), k.v_codes.view(torch.uint8).clone(), k.k_scale.clone(), k.v_scale.clone()]
    batch = (_t(c.cu, dev), _t(c.table, dev), _t(c.lens, dev))
    cos, sin = pdm.rotary_tables(50, 64, device=dev)
    pos, err = torch.arange(4, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    q, kv = c.q.to(dev), torch.randn(4, 2, 64, device=dev).to(torch.bfloat16)
    w = [torch.ones(64, device=dev) for _ in range(2)]
    grad = lambda t: t.detach().clone().requires_grad_(True)  # noqa: E731
    check = torch.library.opcheck
    ops = torch.ops.pdm
    check(ops.qk_norm_rope.default, (grad(q), grad(kv), pos, cos, sin, grad(w[0]), grad(w[1]), 1e-6, False))
    check(ops.qk_norm_rope.default, (grad(q), None, pos, cos, sin, grad(w[0]), None, 1e-6, True))
    check(ops.qk_norm_rope.default, (q, None, pos, None, None, None, None, 1e-6, False))
    check(ops.qk_norm_rope_backward.default, (q, kv, pos, cos, sin, *w, q, kv, 1e-6, False))
    for flag in (err, None):
        check(ops.kv_append.default, (kv, kv, *held, *batch, None, cos, sin, w[0], 1e-6, False, flag))
        for lse in (True, False):
            check(ops.kv_attention.default, (q, *held, *batch, 0.125, True, 0, 3, lse, flag))

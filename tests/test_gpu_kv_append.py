"""kv_append against its definition in 64 bits: codes, scales, untouched slots; every dtype, head width, page size; pages
filled at once and token by token; scales that grow; NaN and infinities; bad spans, lengths, pages and positions.

Every code is the reference's, bit for bit: keys that are computed on the way are computed in 64 bits and rounded to odd
before their code, so that only a value within about 2^-50 of the middle of two codes could get the other one.
"""
import pytest
import torch

from oracle import cached_attention as ref

pytestmark = pytest.mark.gpu

class Pool:
    """A cache on both sides, and sequences that own pages of it."""

    def __init__(self, pdm, dev, pages, page, hk, D, seed=0):
        self.pdm, self.dev, self.page = pdm, dev, page
        g = torch.Generator().manual_seed(seed)
        self.cache = pdm.PagedKVCache(pages, page, hk, D, dev)
        self.codes, self.scale = [], []
        for c, s in ((self.cache.k_codes, self.cache.k_scale), (self.cache.v_codes, self.cache.v_scale)):
            # what an earlier owner left: any codes (NaN among them), any scale
            c.view(torch.uint8).copy_(torch.randint(0, 256, c.shape, generator=g, dtype=torch.uint8))
            s.copy_(torch.exp2(torch.randint(-20, 20, s.shape, generator=g).float()))
            self.codes.append(c.cpu().double())
            self.scale.append(s.cpu().double())

    def append(self, k, v, cu, table, lens, k64, v64, **kw):
        t = lambda x: torch.tensor(x, dtype=torch.int32, device=self.dev)  # noqa: E731
        c = self.cache
        self.pdm.kv_append(k.to(self.dev), v.to(self.dev), c.k_codes, c.v_codes, c.k_scale, c.v_scale, t(cu), t(table),
                           t(lens), err_flag=c.err_flag, **kw)
        for x, codes, scale in ((k64, self.codes[0], self.scale[0]), (v64, self.codes[1], self.scale[1])):
            ref.append(x, codes, scale, cu, table, lens)

    def check(self):
        for i, (c, s) in enumerate(((self.cache.k_codes, self.cache.k_scale), (self.cache.v_codes, self.cache.v_scale))):
            assert torch.equal(s.cpu().double(), self.scale[i])
            assert torch.equal(torch.nan_to_num(c.cpu().double(), 1e6), torch.nan_to_num(self.codes[i], 1e6))


def _deal(lens, page, pages, seed):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    table, width = [], max(-(-n // page) for n in lens) + 1
    for n in lens:
        own = [order.pop() for _ in range(-(-n // page))]
        table.append(own + [-1] * (width - len(own)))
    return table


def _rows(T, hk, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    mag = torch.exp2(torch.randint(-6, 7, (T, hk, 1), generator=g).float())
    return [(torch.randn(T, hk, D, generator=g) * mag).to(dtype) for _ in range(2)]


def _cu(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_prompts_then_tokens(pdm, dev, dtype, D, page):
    """Ragged prompts from an empty cache, more tokens behind them, then single tokens: scales grow on held pages."""
    hk = 3
    new = [1, page, page + 1, 0, 3 * page - 5, 2]
    lens = [0] * len(new)
    final = [n + 20 + 9 for n in new]
    table = _deal(final, page, sum(-(-n // page) for n in final) + 2, 1)
    pool = Pool(pdm, dev, sum(-(-n // page) for n in final) + 2, page, hk, D)
    for step, more in enumerate([new, [5, 0, 20, 1, 7, 3]] + [[1] * 6] * 4 + [[1, 0, 0, 1, 0, 1]]):
        lens = [a + b for a, b in zip(lens, more)]
        k, v = _rows(sum(more), hk, D, dtype, 10 * step + D)
        pool.append(k, v, _cu(more), table, lens, k.double(), v.double())
        pool.check()
    assert pool.cache.err_flag.item() == 0


@pytest.mark.parametrize("D,R,inter", [(64, 64, False), (128, 64, True), (128, 128, False), (256, 128, False)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("explicit", [False, True])
def test_rotated_and_normed_keys(pdm, dev, D, R, inter, norm, explicit):
    hk, page = 2, 32
    g = torch.Generator().manual_seed(4)
    ang = torch.rand(300, R // 2, generator=g, dtype=torch.float64) * 50
    cos, sin = ang.cos().float(), ang.sin().float()
    w = 1 + 0.3 * torch.randn(D, generator=g)
    final = [140, 33, 90]
    table = _deal(final, page, 12, 2)
    pool = Pool(pdm, dev, 12, page, hk, D)
    lens = [0, 0, 0]
    for step, more in enumerate(([100, 32, 0], [1, 1, 1], [39, 0, 89])):
        start, lens = lens, [a + b for a, b in zip(lens, more)]
        k, v = _rows(sum(more), hk, D, torch.bfloat16, step)
        pos = torch.cat([torch.arange(s, s + m) for s, m in zip(start, more)])
        kw = {}
        if explicit:
            pos = torch.randint(0, 300, pos.shape, generator=g)
            kw["positions"] = pos.to(dev)
        if norm:
            kw["k_weight"] = w.to(dev)
        k64 = ref.norm_rope(k, w if norm else None, pos, cos, sin, 1e-6, inter)
        pool.append(k, v, _cu(more), table, lens, k64, v.double(), cos=cos.to(dev), sin=sin.to(dev), interleaved=inter, **kw)
        pool.check()
    pool.cache.check()


@pytest.mark.parametrize("tokens", [1, 40])
def test_keys_beside_the_middle_of_two_codes(pdm, dev, tokens):
    """17 + 2^-30 and 17 - 2^-30 lie on either side of the middle of 16 and 18, and are 17 in fp32."""
    D, page = 64, 64
    k = torch.ones(tokens, 1, D, dtype=torch.bfloat16)
    k[..., :D // 2] = 17.0
    k[..., 0] = 448.0
    cos, sin = torch.ones(64, D // 2), torch.full((64, D // 2), 2.0 ** -30)
    sin[:, 8:] *= -1
    k64 = ref.norm_rope(k, None, torch.arange(tokens), cos, sin, 0.0, False)
    pool = Pool(pdm, dev, 1, page, 1, D)
    pool.append(k, k, [0, tokens], [[0]], [tokens], k64, k.double(), cos=cos.to(dev), sin=sin.to(dev))
    pool.check()
    codes = pool.cache.k_codes[0, 0, :tokens].float().cpu()
    assert (codes[:, 1:8] == 16.0).all() and (codes[:, 8:32] == 18.0).all()


def test_token_by_token_is_as_good_as_at_once(pdm, dev):
    """One page per sequence, filled by single tokens whose size grows: the same scale as in one call, codes off by
    no more than the roundings of subnormal codes."""
    D, page, hk = 64, 64, 2
    k, v = _rows(page, hk, D, torch.float32, 3)
    k *= torch.exp2(torch.arange(page) / 6)[:, None, None]
    once, each = (Pool(pdm, dev, 1, page, hk, D) for _ in range(2))
    once.append(k, v, [0, page], [[0]], [page], k.double(), v.double())
    for i in range(page):
        each.append(k[i:i + 1], v[i:i + 1], [0, 1], [[0]], [i + 1], k[i:i + 1].double(), v[i:i + 1].double())
        each.check()
    assert torch.equal(once.cache.k_scale, each.cache.k_scale) and torch.equal(once.cache.v_scale, each.cache.v_scale)
    a, b = (p.cache.k_codes.double() for p in (once, each))
    # a subnormal code is rounded again at each of up to 23 changes of scale, by at most half a step of 2^-9, halved at
    # each later change: at most one step in all
    assert ((a - b).abs() <= 2.0 ** -9).all()
    kb, _ = each.cache.values()
    assert torch.equal(kb.double(), each.cache.k_codes.double() * each.cache.k_scale.double()[:, :, None, None])


def test_same_tokens_again(pdm, dev):
    D, page, hk = 128, 16, 2
    table = _deal([50, 3], page, 6, 5)
    pool = Pool(pdm, dev, 6, page, hk, D)
    k, v = _rows(43, hk, D, torch.bfloat16, 1)
    pool.append(k, v, [0, 40, 43], table, [40, 3], k.double(), v.double())
    k, v = _rows(10, hk, D, torch.bfloat16, 2)
    for _ in range(3):
        pool.append(k, v, [0, 10, 10], table, [50, 3], k.double(), v.double())
        pool.check()


def test_special_values(pdm, dev):
    """NaN, infinities, zeros, denormals, the largest numbers, ties."""
    D, page, hk = 64, 16, 1
    big = torch.finfo(torch.bfloat16).max
    rows = [
        torch.zeros(D), torch.full((D,), 1e-40), torch.full((D,), big), torch.full((D,), -big),
        torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0] * 16), torch.full((D,), float("nan")),
        torch.tensor([448.0] * 63 + [17.0]), torch.tensor([450.0] * 63 + [17.0]), torch.tensor([0.0, -0.0, 2.0 ** -9, 2.0 ** -10] * 16),
        torch.arange(64).float() + 0.5, 2.0 ** torch.arange(-60, 4).float(),
    ]
    for dtype in (torch.float32, torch.bfloat16):
        for i, r in enumerate(rows):
            r = r.to(dtype)
            pool = Pool(pdm, dev, 1, page, hk, D, seed=i)
            x = r.view(1, 1, D)
            pool.append(x, x.flip(-1), [0, 1], [[0]], [1], x.double(), x.flip(-1).double())
            pool.check()
            # behind it a token of ones: what was there is brought to a larger scale or stays
            y = torch.ones(1, 1, D, dtype=dtype)
            pool.append(y, y, [0, 1], [[0]], [2], y.double(), y.double())
            pool.check()
    assert torch.isfinite(pool.cache.values()[0][0, 0, :2].float()).all()


def test_strides_and_alignment(pdm, dev):
    D, page, hk = 64, 32, 3
    k, v = _rows(70, hk, D, torch.bfloat16, 7)
    kw = dict(cu=[0, 70], table=[[2, 0, 1]], lens=[70], k64=k.double(), v64=v.double())
    wide = torch.zeros(70, 7 * hk * D + 1, dtype=torch.bfloat16, device=dev)
    a = wide[:, 1:1 + hk * D].view(70, hk, D).copy_(k)  # rows at odd addresses
    b = v.to(dev).transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    pool = Pool(pdm, dev, 3, page, hk, D)
    pool.append(a, b, **kw)
    pool.check()
    pool = Pool(pdm, dev, 3, page, hk, D)
    pool.append(k.view(7, 10, hk, D), v.view(7, 10, hk, D), **kw)
    pool.check()


def test_what_does_not_fit_is_left_out(pdm, dev):
    """Each bad sequence stands beside a good one, whose tokens arrive; nothing else changes."""
    D, page, hk = 64, 16, 2
    k, v = _rows(24, hk, D, torch.bfloat16, 9)
    good = dict(cu=[0, 4, 24], table=[[0, 1], [2, 3]], lens=[4, 20])
    bad = [
        dict(table=[[0, 1], [2, 9]]), dict(table=[[0, 1], [-1, 3]]), dict(table=[[0], [2]]), dict(lens=[4, 19]),
        dict(lens=[4, -1]), dict(cu=[0, 4, 25]), dict(lens=[4, 2 ** 31 - 1]),
    ]
    for change in bad:
        pool = Pool(pdm, dev, 4, page, hk, D)
        a = {**good, **change}
        t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        c = pool.cache
        pdm.kv_append(k.to(dev), v.to(dev), c.k_codes, c.v_codes, c.k_scale, c.v_scale, t(a["cu"]), t(a["table"]),
                      t(a["lens"]), err_flag=c.err_flag)
        assert c.err_flag.item() == 1, change
        with pytest.raises(RuntimeError, match="did not fit"):
            c.check()
        cu, lens, table = [0, 4, 4], [4, 0], a["table"]
        if "table" in change and change["table"][0] == [0]:  # a table too narrow: the first 16 tokens fit
            cu, lens = [0, 4, 20], [4, 16]
        elif change.get("table") == [[0, 1], [2, 9]]:
            cu, lens = [0, 4, 20], [4, 16]
        for x, codes, scale in ((k, pool.codes[0], pool.scale[0]), (v, pool.codes[1], pool.scale[1])):
            ref.append(x.double(), codes, scale, cu, table, lens)
            if change.get("table") == [[0, 1], [-1, 3]]:  # its second page is good
                ref.append(x.double()[20:], codes, scale, [0, 0, 4], [[0, 1], [0, 3]], [0, 20])
        pool.check()


def test_bad_positions_and_rows_behind_the_last_sequence(pdm, dev):
    D, page, hk = 64, 16, 2
    cos, sin = torch.ones(4, 32), torch.zeros(4, 32)
    k, v = _rows(8, hk, D, torch.bfloat16, 9)
    k[6:] = float("nan")  # rows 6 and 7 belong to no sequence
    pool = Pool(pdm, dev, 2, page, hk, D)
    pos = torch.tensor([0, 3, 4, -1, 2, 1, 0, 0])
    k64 = k.double().clone()
    k64[2:4] = 0
    pool.append(k, v, [0, 6], [[1]], [6], k64, v.double(), cos=cos.to(dev), sin=sin.to(dev), positions=pos.to(dev))
    pool.check()
    assert pool.cache.err_flag.item() == 1
    # nothing to do: no rows, no sequences, no new tokens
    t = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    c = pool.cache
    for T, B in ((0, 0), (0, 1), (3, 1), (3, 0)):
        c.append(k[:T].to(dev), v[:T].to(dev), t(B + 1), t(B, 1), t(B) + 6)
    pool.check()


@pytest.mark.parametrize("D,page", [(64, 128), (128, 16), (256, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_busy_sequence_among_idle_ones(pdm, dev, D, page, dtype):
    """No more new tokens than sequences, but most of them one sequence's: several rows for each lane group."""
    hk, R = 3, D // 2
    g = torch.Generator().manual_seed(D)
    ang = torch.rand(400, R // 2, generator=g, dtype=torch.float64) * 50
    cos, sin = ang.cos().float(), ang.sin().float()
    w = 1 + 0.3 * torch.randn(D, generator=g)
    lens = [0] * 160
    final = [3] * 160
    final[7], final[100] = 300, 40
    pages = sum(-(-n // page) for n in final) + 2
    table = _deal(final, page, pages, 2)
    pool = Pool(pdm, dev, pages, page, hk, D)
    for step, some in enumerate(({7: 150, 100: 5}, {7: 1, 100: 2, 8: 1, 159: 3}, {7: 149, 100: 6}, {100: 27, 0: 3})):
        more = [some.get(i, 0) for i in range(160)]
        start, lens = lens, [a + b for a, b in zip(lens, more)]
        k, v = _rows(sum(more), hk, D, dtype, step)
        pos = torch.cat([torch.arange(s, s + m) for s, m in zip(start, more)])
        pool.append(k, v, _cu(more), table, lens, ref.norm_rope(k, w, pos, cos, sin, 1e-6, False), v.double(),
                    cos=cos.to(dev), sin=sin.to(dev), k_weight=w.to(dev))
        pool.check()
    pool.cache.check()


@pytest.mark.parametrize("page,D", [(16, 64), (64, 128)])
def test_busy_sequences_among_many(pdm, dev, page, D):
    """The same over more than 256 sequences, several of them busy, single tokens beside them; a busy one that holds fewer
    tokens than it brings, and one with a page that does not exist, are left out."""
    hk, B = 2, 700
    some = {0: 40, 7: 1, 255: 130, 256: 3, 300: 90, 301: 2, 302: 33, 650: 1, 699: 70}
    more = [some.get(i, 0) for i in range(B)]
    past = [i % 23 for i in range(B)]
    lens = [n + p for n, p in zip(more, past)]
    pages = sum(-(-n // page) for n in lens) + 2
    table = _deal(lens, page, pages, 3)
    pool = Pool(pdm, dev, pages, page, hk, D)
    k, v = _rows(B, hk, D, torch.bfloat16, 1)  # rows behind the last sequence too
    pool.append(k, v, _cu(more), table, lens, k.double(), v.double())
    pool.check()
    assert pool.cache.err_flag.item() == 0
    pool = Pool(pdm, dev, pages, page, hk, D)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    short = list(lens)
    short[255] = 129
    holed = [list(r) for r in table]
    holed[300][(past[300] + 60) // page] = pages
    c = pool.cache
    pdm.kv_append(k.to(dev), v.to(dev), c.k_codes, c.v_codes, c.k_scale, c.v_scale, t(_cu(more)), t(holed), t(short),
                  err_flag=c.err_flag)
    assert c.err_flag.item() == 1
    # the reference, on the host, for what is left: whole sequences but 255, and 300 without its lost page
    cu = _cu(more)
    for x, codes, scale in ((k.double(), pool.codes[0], pool.scale[0]), (v.double(), pool.codes[1], pool.scale[1])):
        lost = table[300][(past[300] + 60) // page]
        keep = codes[lost].clone(), scale[lost].clone()
        for b in some:
            if b != 255:
                ref.append(x[cu[b]:cu[b + 1]], codes, scale, [0, more[b]], [table[b]], [lens[b]])
        codes[lost], scale[lost] = keep
    pool.check()


def test_many_sequences(pdm, dev):
    """More sequences than two rounds of the search over 64 entries hold, empty ones among them."""
    D, page, hk = 64, 16, 1
    g = torch.Generator().manual_seed(2)
    new = torch.randint(0, 4, (5000,), generator=g).tolist()
    lens = [n + p for n, p in zip(new, torch.randint(0, 30, (5000,), generator=g).tolist())]
    table = _deal([max(n, 1) for n in lens], page, 12000, 3)
    pool = Pool(pdm, dev, 12000, page, hk, D)
    k, v = _rows(sum(new), hk, D, torch.bfloat16, 1)
    pool.append(k, v, _cu(new), table, lens, k.double(), v.double())
    pool.check()
    assert pool.cache.err_flag.item() == 0


def test_graph_replays_and_streams(pdm, dev):
    D, page, hk = 128, 32, 2
    cos, sin = (t.to(dev) for t in pdm.rotary_tables(200, D))
    k, v = (t.to(dev) for t in _rows(4, hk, D, torch.bfloat16, 0))
    a, b = (Pool(pdm, dev, 16, page, hk, D) for _ in range(2))
    cu = torch.arange(5, dtype=torch.int32, device=dev)
    table = torch.randperm(16, device=dev).to(torch.int32).view(4, 4)
    lens = torch.tensor([1, 33, 64, 97], dtype=torch.int32, device=dev)

    def step(c):
        pdm.kv_append(k, v, c.k_codes, c.v_codes, c.k_scale, c.v_scale, cu, table, lens, cos=cos, sin=sin)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a.cache)
    side = torch.cuda.Stream()
    for i in range(5):
        for t, x in zip((k, v), _rows(4, hk, D, torch.bfloat16, i)):
            t.copy_(x)
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(b.cache)
        torch.cuda.current_stream().wait_stream(side)
        for n in ("k_codes", "v_codes", "k_scale", "v_scale"):
            x, y = getattr(a.cache, n), getattr(b.cache, n)
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), (i, n)
        lens += 1


def test_compiled(pdm, dev):
    D, page, hk = 64, 16, 2
    k, v = (t.to(dev) for t in _rows(5, hk, D, torch.bfloat16, 0))
    a, b = (Pool(pdm, dev, 2, page, hk, D).cache for _ in range(2))
    cu, table, lens = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 5], [[1]], [9]))

    def f(c, k, v):
        pdm.kv_append(k * 2, v, c.k_codes, c.v_codes, c.k_scale, c.v_scale, cu, table, lens)
        return k + 1

    f(a, k, v)
    torch.compile(f, fullgraph=True, backend="aot_eager")(b, k, v)
    assert torch.equal(a.k_codes.view(torch.uint8), b.k_codes.view(torch.uint8)) and torch.equal(a.v_scale, b.v_scale)


def test_pages_beyond_32_bit_offsets(pdm, dev):
    D, page, hk = 128, 128, 4
    pages = 2 ** 32 // (D * page * hk) + 3
    c = pdm.PagedKVCache(pages, page, hk, D, dev)
    k, v = _rows(140, hk, D, torch.bfloat16, 0)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    c.append(k.to(dev), v.to(dev), t([0, 140]), t([[pages - 1, pages - 2]]), t([140]))
    c.check()
    for x, codes, scale in ((k, c.k_codes, c.k_scale), (v, c.v_codes, c.v_scale)):
        want, ws = torch.zeros(2, hk, page, D, dtype=torch.float64), torch.ones(2, hk, dtype=torch.float64)
        ref.append(x.double(), want, ws, [0, 140], [[1, 0]], [140])
        assert torch.equal(codes[-2:].cpu().double(), want) and torch.equal(scale[-2:].cpu().double(), ws)
        assert not codes[:4].view(torch.uint8).any()


@pytest.mark.parametrize("D,R,inter", [(64, 16, False), (128, 64, True), (256, 128, False), (128, 128, False)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("bits", [None, torch.int32, torch.int64])
def test_positions_outside_the_tables_of_partly_rotated_keys(pdm, dev, D, R, inter, norm, bits):
    """A key whose position the tables do not hold is zero in all of its elements, the ones behind the rotated part too, and
    counts as zero for its page's scale; by prompts and by single tokens, positions given or not."""
    hk, page, rows = 2, 16, 24
    g = torch.Generator().manual_seed(D + R)
    ang = torch.rand(rows, R // 2, generator=g, dtype=torch.float64) * 50
    cos, sin = ang.cos().float(), ang.sin().float()
    w = 1 + 0.3 * torch.randn(D, generator=g)
    kw = dict(cos=cos.to(dev), sin=sin.to(dev), interleaved=inter)
    if norm:
        kw["k_weight"] = w.to(dev)
    final = [45, 20, 27, 1]
    table = _deal(final, page, 12, 2)
    pool = Pool(pdm, dev, 12, page, hk, D)
    lens = [0] * 4
    for step, more in enumerate(([40, 19, 25, 0], [1, 0, 1, 1], [1, 1, 1, 0], [3, 0, 0, 0])):
        start, lens = lens, [a + b for a, b in zip(lens, more)]
        k, v = _rows(sum(more), hk, D, torch.bfloat16, step)
        pos = torch.cat([torch.arange(s, s + m) for s, m in zip(start, more)])
        if bits is not None:
            pos = torch.randint(-rows, 2 * rows, pos.shape, generator=g).to(bits)
            if bits == torch.int64:
                pos[0] = 2 ** 40
            kw["positions"] = pos.to(dev)
        # (one sequence's largest keys lie outside)
        outside = (pos < 0) | (pos >= rows)
        k[outside] *= 64
        pool.cache.err_flag.zero_()
        pool.append(k, v, _cu(more), table, lens, ref.norm_rope(k, w if norm else None, pos, cos, sin, 1e-6, inter),
                    v.double(), **kw)
        pool.check()
        assert pool.cache.err_flag.item() == int(outside.any())


@pytest.mark.parametrize("cu,lens", [
    ([1000, 1003], [3]), ([1000, 1003, 1003, 1003, 1003, 1003, 1003], [3] * 6), ([2 ** 31 - 4, 2 ** 31 - 1], [3]),
    ([0, 4, 0, 4], [4, 9, 4]), ([0, 4, 0, 4, 4, 4], [4, 9, 4, 0, 0]), ([-3, 0], [3]), ([-1000, 0] + [0] * 5, [1000] * 6)])
def test_spans_outside_the_batch_set_the_flag(pdm, dev, cu, lens):
    """Also where no row or page of the batch leads to them: a first span behind the batch, one that runs backwards; in batches
    of more and of no more tokens than sequences.  Nothing of them is written."""
    D, page, hk, T = 64, 16, 2, 5
    k, v = _rows(T, hk, D, torch.bfloat16, 9)
    B = len(lens)
    pool = Pool(pdm, dev, 2 * B, page, hk, D)
    c = pool.cache
    table = [[2 * b, 2 * b + 1] for b in range(B)]
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    c.append(k.to(dev), v.to(dev), t(cu), t(table), t(lens))
    assert c.err_flag.item() == 1
    for b in range(B):
        if 0 <= cu[b] < cu[b + 1] <= T:
            for x, codes, scale in ((k, pool.codes[0], pool.scale[0]), (v, pool.codes[1], pool.scale[1])):
                n = cu[b + 1] - cu[b]
                ref.append(x[cu[b]:cu[b + 1]].double(), codes, scale, [0, n], [table[b]], [lens[b]])
    pool.check()


@pytest.mark.parametrize("D,page,hk", [(128, 64, 3), (64, 16, 1), (128, 16, 2), (256, 128, 1)])
def test_a_third_of_the_sequences_busy(pdm, dev, D, page, hk):
    """Many sequences with a few tokens each beside many with none, more of them than workgroups that share them out; pages
    begun in earlier calls, tokens that pass on to another page, a single token and a longer run between them."""
    B = 600
    final = [100 if i % 3 == 0 else 5 for i in range(B)]
    pages = sum(-(-n // page) for n in final) + 2
    table = _deal(final, page, pages, 4)
    pool = Pool(pdm, dev, pages, page, hk, D)
    lens = [0] * B
    for step in range(3):
        more = [(3 if i < 500 else 0) if i % 3 == 0 else 0 for i in range(B)]
        more[1], more[300] = 1, 3 + 17 * step
        if step == 1:
            more[0], more[597] = 0, 29
        start, lens = lens, [a + b for a, b in zip(lens, more)]
        assert sum(more) <= B
        k, v = _rows(sum(more), hk, D, torch.bfloat16, step)
        pool.append(k, v, _cu(more), table, lens, k.double(), v.double())
        pool.check()
    assert pool.cache.err_flag.item() == 0


def test_autograd_notices_what_is_written(pdm, dev):
    """A backward pass that saved a scale, codes, the flag or a given output before a call wrote it raises; inference tensors,
    which have no versions, are written all the same."""
    D, page, hk = 64, 16, 2
    k, v = (t.to(dev) for t in _rows(5, hk, D, torch.bfloat16, 0))
    cu, table, lens = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 5], [[1]], [9]))
    c = pdm.PagedKVCache(2, page, hk, D, dev)
    a = torch.ones((), device=dev, requires_grad=True)
    for name in ("k_scale", "v_scale"):
        y = (a * getattr(c, name)).sum()
        c.append(k, v, cu, table, lens)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.backward()
    tensors = (c.k_codes, c.v_codes, c.k_scale, c.v_scale, c.err_flag)
    held = [t._version for t in tensors]
    c.append(k, v, cu, table, lens)
    assert all(t._version > x for t, x in zip(tensors, held))
    q, out = torch.ones(5, 4, D, dtype=torch.bfloat16, device=dev), torch.zeros(5, 4, D, dtype=torch.bfloat16, device=dev)
    y = (a * out).sum()
    held = c.err_flag._version
    pdm.kv_attention(q, *tensors[:4], cu, table, lens, out=out, err_flag=c.err_flag)
    assert c.err_flag._version > held
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    held = c.err_flag._version
    pdm.qk_norm_rope(q, None, torch.arange(5, device=dev), None, None, err_flag=c.err_flag)
    assert c.err_flag._version > held
    with torch.inference_mode():
        d = pdm.PagedKVCache(2, page, hk, D, dev)
        d.append(k, v, cu, table, lens)
        d.attend(q, cu, table, lens)
    e = pdm.PagedKVCache(2, page, hk, D, dev)
    e.append(k, v, cu, table, lens)
    assert torch.equal(d.k_codes.view(torch.uint8), e.k_codes.view(torch.uint8)) and torch.equal(d.v_scale, e.v_scale)
    d.append(k, v, cu, table, lens)  # inference tensors outside the mode
    d.check()

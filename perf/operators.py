"""Cases of the operators around a cached attention: what each is timed on, its plain form, and its definition in 64 bits.

* ``rope``    ``qk_norm_rope``: RMS norm of every query and key head and the position rotation, forward
* ``train``   the same with its backward pass: outputs, gradients of q and k and of both norm weights
* ``append``  ``kv_append``: new keys (rotated on the way) and values into 8-bit pages with a scale per (page, head)
* ``attend``  ``kv_attention``: ragged queries over those pages, from one token to long prompts

Sequences: sequence b has n_b new tokens, the rows cu_seqlens[b] .. cu_seqlens[b+1] of the batch, and holds
seq_lens[b] tokens with them.  Lengths are log-spaced between a case's bounds and dealt to the sequences by the seed, so
that a case's work does not depend on the seed.  Pages are dealt by the seed too.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
THETA = 10000.0
FP8_MAX = 448.0
E_MIN, E_MAX = -117, 119  # exponents of a page's scale


def listed():
    return [
        # the queries of one decoding step of 16 sequences: latency
        dict(name="rope_decode_t16", path="rope", tokens=16, hq=32, hk=8, dim=128, rot=128, dtype="bf16", norm=True,
             interleaved=False, max_pos=32_768),
        # a prompt of 8,192 tokens, q and k as columns of the fused projection's rows
        dict(name="rope_prompt_t8192", path="rope", tokens=8_192, hq=32, hk=8, dim=128, rot=128, dtype="bf16",
             norm=True, interleaved=False, max_pos=32_768),
        # training of a 6-head layer of 64 on a user batch of odd size
        dict(name="train_h6_d64", path="train", tokens=24_259, hq=6, hk=6, dim=64, rot=64, dtype="bf16", norm=True,
             interleaved=False, max_pos=4_096),
        # training on long rows, half of each head rotated in neighbouring pairs
        dict(name="train_partial_fp16", path="train", tokens=16_384, hq=24, hk=6, dim=128, rot=64, dtype="fp16",
             norm=True, interleaved=True, max_pos=16_384),
        # one new token for each of 64 sequences
        dict(name="append_decode_b64", path="append", batch=64, q_lo=1, q_hi=1, past_lo=100, past_hi=2_000, hk=8,
             dim=128, rot=128, page=64, dtype="bf16", norm=True, interleaved=False),
        # new events of 512 users: 1 to 60 each, 6 heads of 64
        dict(name="append_events_b512", path="append", batch=512, q_lo=1, q_hi=60, past_lo=1, past_hi=1_500, hk=6,
             dim=64, rot=64, page=32, dtype="bf16", norm=False, interleaved=False),
        # prompts: five ragged ones from an empty cache
        dict(name="append_prompts_b5", path="append", batch=5, q_lo=1_001, q_hi=7_777, past_lo=0, past_hi=0, hk=8,
             dim=128, rot=128, page=16, dtype="bf16", norm=True, interleaved=False),
        # one sequence decoding alone: latency
        dict(name="attend_decode_b1", path="attend", batch=1, q_lo=1, q_hi=1, past_lo=999, past_hi=999, hq=32, hk=8,
             dim=128, page=64, dtype="bf16", causal=True, window=0, lse=False),
        # a decoding batch of ragged contexts
        dict(name="attend_decode_b64", path="attend", batch=64, q_lo=1, q_hi=1, past_lo=127, past_hi=8_191, hq=32,
             hk=8, dim=128, page=64, dtype="bf16", causal=True, window=0, lse=False),
        # four sequences decoding far into long contexts, small pages
        dict(name="attend_decode_long", path="attend", batch=4, q_lo=1, q_hi=1, past_lo=60_000, past_hi=120_000,
             hq=32, hk=8, dim=128, page=16, dtype="bf16", causal=True, window=0, lse=True),
        # scoring: 16 NS tokens of each of 256 requests over their cached histories, 6 heads of 64
        dict(name="attend_ns_b256", path="attend", batch=256, q_lo=16, q_hi=16, past_lo=300, past_hi=1_500, hq=6,
             hk=6, dim=64, page=32, dtype="bf16", causal=True, window=0, lse=False),
        # prompts continued over a cached prefix; the largest case
        dict(name="attend_prompts_b2", path="attend", batch=2, q_lo=3_500, q_hi=4_500, past_lo=3_001, past_hi=5_001,
             hq=32, hk=8, dim=128, page=64, dtype="bf16", causal=True, window=0, lse=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["rope", "train", "append", "append", "attend", "attend", "attend"])
    dim = rng.choice([64, 64, 128, 128, 128, 256])
    hk = rng.choice([1, 2, 4, 6, 8])
    group = rng.choice([1, 1, 2, 4, 7, 8, 16])
    rot = rng.choice([dim, dim, dim // 2])
    if path in ("rope", "train"):
        tokens = _log(rng, 1, 16_384)
        while tokens * hk * (group + 1) * dim > 16_384 * 40 * 128:
            tokens = max(1, tokens // 2)
        return dict(path=path, tokens=tokens, hq=hk * group, hk=hk, dim=dim, rot=rot,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), norm=rng.random() < 0.8,
                    interleaved=rng.random() < 0.3, max_pos=_log(rng, 512, 131_072))
    page = rng.choice([16, 32, 64, 128])
    batch = _log(rng, 1, 512)
    q_lo = rng.choice([1, 1, _log(rng, 1, 2_000)])
    q_hi = rng.choice([q_lo, q_lo, _log(rng, q_lo, 5_000)])
    past_lo = rng.choice([0, _log(rng, 1, 8_000)])
    past_hi = max(past_lo, _log(rng, 16, 60_000))
    if path == "append":
        while batch > 1 and batch * (q_hi + past_hi + page) * hk * dim > 3e8:
            batch //= 2
        return dict(path=path, batch=batch, q_lo=q_lo, q_hi=q_hi, past_lo=past_lo, past_hi=past_hi, hk=hk, dim=dim,
                    rot=rng.choice([0, rot, rot]), page=page, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    norm=rng.random() < 0.5, interleaved=rng.random() < 0.3)
    while batch > 1 and (batch * (q_hi + past_hi) * hk * dim > 3e8
                         or batch * q_hi * (q_hi + past_hi) * hk * group > 1e9
                         or batch * q_hi * (q_hi + past_hi) * hk * group * dim > 1.3e11):
        batch //= 2
    while q_hi * (q_hi + past_hi) * hk * group > 1e9 or q_hi * (q_hi + past_hi) * hk * group * dim > 1.3e11:
        q_lo, q_hi = max(1, q_lo // 2), max(1, q_hi // 2)
    return dict(path=path, batch=batch, q_lo=q_lo, q_hi=q_hi, past_lo=past_lo, past_hi=past_hi, hq=hk * group, hk=hk,
                dim=dim, page=page, dtype=rng.choice(["bf16", "bf16", "fp16"]), causal=rng.random() < 0.8,
                window=rng.choice([0, 0, 0, _log(rng, 1, 4_096)]), lse=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _lengths(n, lo, hi):
    """n lengths from lo to hi, log-spaced (the same list for every seed)."""
    if lo >= hi:
        return [lo] * n
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [int(round(math.exp(a + (b - a) * (i + 0.5) / n))) - 1 for i in range(n)]


def _sequences(case, seed):
    """(n_b, length after the call) of every sequence: the lists of the case, dealt by the seed."""
    new = [max(1, v) for v in _lengths(case["batch"], case["q_lo"], case["q_hi"])]
    past = _lengths(case["batch"], case["past_lo"], case["past_hi"])
    rng = random.Random(seed)
    rng.shuffle(new)
    rng.shuffle(past)
    return new, [n + p for n, p in zip(new, past)]


def _tables(rot, rows, dev):
    """cos and sin of position * theta^(-2i/rot), angles in 64 bits."""
    freq = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    angle = torch.arange(rows, dtype=torch.float64, device=dev)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _paged(case, seed, dev, gen):
    """Cumulative new lengths, lengths, page table (-1 behind a sequence's pages), and the number of pages."""
    new, lens = _sequences(case, seed)
    page = case["page"]
    counts = [(n + page - 1) // page for n in lens]
    # a pool of one size for every seed, with pages to spare
    total = sum((n + page - 1) // page for n in new) + sum((ln - n + page - 1) // page for n, ln in zip(new, lens))
    width = max(counts)
    order = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    cnt = torch.tensor(counts, device=dev)
    col = torch.arange(width, device=dev)[None, :]
    first = (torch.cumsum(cnt, 0) - cnt)[:, None]
    table = torch.where(col < cnt[:, None], order[(first + col).clamp(max=total - 1)], -1).to(torch.int32)
    cu = torch.zeros(len(new) + 1, dtype=torch.int32, device=dev)
    cu[1:] = torch.cumsum(torch.tensor(new, device=dev), 0)
    return new, lens, cu, torch.tensor(lens, dtype=torch.int32, device=dev), table.contiguous(), total


def _weight(dim, gen, dev):
    return 1 + 0.2 * torch.randn(dim, generator=gen, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, dim = _TORCH[case["dtype"]], case["dim"]
    st = dict(case=dict(case))
    rand = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    if case["path"] in ("rope", "train"):
        T, hq, hk = case["tokens"], case["hq"], case["hk"]
        # rows of the fused projection: q, k and v beside each other, channels of unlike sizes
        rows = (rand(T, (hq + 2 * hk) * dim) * (0.5 + rand((hq + 2 * hk) * dim).abs())).to(dt)
        st["q"] = rows[:, :hq * dim].view(T, hq, dim)
        st["k"] = rows[:, hq * dim:(hq + hk) * dim].view(T, hk, dim)
        st["positions"] = torch.randint(0, case["max_pos"], (T,), generator=gen, device=dev)
        st["cos"], st["sin"] = _tables(case["rot"], case["max_pos"], dev)
        st["qw"] = _weight(dim, gen, dev) if case["norm"] else None
        st["kw"] = _weight(dim, gen, dev) if case["norm"] else None
        if case["path"] == "train":
            st["gq"], st["gk"] = rand(T, hq, dim).to(dt), rand(T, hk, dim).to(dt)
            for n in ("q", "k", "qw", "kw"):
                if st[n] is not None:
                    st[n] = st[n].detach().requires_grad_(True)
        return st
    hk, page = case["hk"], case["page"]
    new, lens, cu, st["seq_lens"], st["page_table"], pages = _paged(case, seed, dev, gen)
    st["cu"], st["max_new"] = cu, max(new)
    T = sum(new)
    # a cache that holds something: codes of normal values, scales around 2^-7 (keys) and 2^-8 (values)
    for n, e in (("k", -7), ("v", -8)):
        codes = torch.empty(pages, hk, page, dim, dtype=torch.float8_e4m3fn, device=dev)
        for i in range(0, pages, 4096):
            part = codes[i:i + 4096]
            part.copy_((rand(*part.shape) * 100).clamp_(-FP8_MAX, FP8_MAX))
        st[n + "_codes"] = codes
        st[n + "_scale"] = torch.exp2(torch.randint(e - 1, e + 2, (pages, hk), generator=gen, device=dev).float())
    if case["path"] == "append":
        rows = (rand(T, 3 * hk * dim) * (0.5 + rand(3 * hk * dim).abs())).to(dt)
        st["k"] = rows[:, hk * dim:2 * hk * dim].view(T, hk, dim)
        st["v"] = rows[:, 2 * hk * dim:].view(T, hk, dim)
        st["kw"] = _weight(dim, gen, dev) if case["norm"] else None
        st["cos"], st["sin"] = _tables(case["rot"], max(lens), dev) if case["rot"] else (None, None)
    else:
        st["q"] = (rand(T, case["hq"] * dim) * 1.5).to(dt).view(T, case["hq"], dim)
    return st


# ---------------------------------------------------------------------------
# Plain forms (fp32, elementary operations)
# ---------------------------------------------------------------------------

def _norm_rope(x, weight, cos, sin, interleaved):
    """x [T, H, D] fp32; cos, sin [T, R/2] or None."""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    if cos is None:
        return x
    c, s, R = cos[:, None, :], sin[:, None, :], 2 * cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        r = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        r = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((r, x[..., R:]), -1)


def _plain_rope(st):
    c, s, i = st["cos"][st["positions"]], st["sin"][st["positions"]], st["case"]["interleaved"]
    return (_norm_rope(st["q"].float(), st["qw"], c, s, i).to(st["q"].dtype),
            _norm_rope(st["k"].float(), st["kw"], c, s, i).to(st["k"].dtype))


def _exponent(amax):
    """Smallest e with amax <= 448 * 2^e, within the scale's range."""
    m, e = torch.frexp(amax / FP8_MAX)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.where(amax > 0, e, E_MIN).clamp(E_MIN, E_MAX)


def _plain_append(st):
    case, table, cu, lens = st["case"], st["page_table"], st["cu"].long(), st["seq_lens"].long()
    page, T = case["page"], st["k"].shape[0]
    rows = torch.arange(T, device=cu.device)
    seq = torch.searchsorted(cu[1:], rows, right=True)
    start = lens - (cu[1:] - cu[:-1])
    index = start[seq] + rows - cu[seq]
    cos = sin = None
    if st["cos"] is not None:
        cos, sin = st["cos"][index], st["sin"][index]
    slot, entry = index % page, seq * table.shape[1] + index // page
    pages = table.reshape(-1)[entry].long()
    held = start % page  # tokens of the sequence on the first page that is written
    first = table.gather(1, (start // page).clamp(max=table.shape[1] - 1)[:, None])[:, 0].long()
    first_entry = torch.arange(len(lens), device=cu.device) * table.shape[1] + start // page
    keep = held > 0
    for name, x in (("k", _norm_rope(st["k"].float(), st["kw"], cos, sin, case["interleaved"])),
                    ("v", st["v"].float())):
        codes, scale = st[name + "_codes"], st[name + "_scale"]
        most = torch.zeros(table.numel(), x.shape[1], device=x.device)
        most.scatter_reduce_(0, entry[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
        e = _exponent(most)
        old = scale[first[keep]]
        e[first_entry[keep]] = torch.maximum(e[first_entry[keep]], torch.frexp(old)[1] - 1)
        new = torch.ldexp(torch.ones_like(most), e)
        # the codes that the first page already holds, brought to its new scale
        at = first[keep]
        was = codes.view(torch.uint8)[at].view(torch.float8_e4m3fn)
        now = (was.float() * (old / new[first_entry[keep]])[:, :, None, None]).to(torch.float8_e4m3fn)
        mine = (torch.arange(page, device=x.device) < held[keep][:, None])[:, None, :, None]
        codes.view(torch.uint8)[at] = torch.where(mine, now.view(torch.uint8), was.view(torch.uint8))
        scale[pages] = new[entry]
        codes.view(torch.uint8)[pages, :, slot] = (x / new[entry][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"]


def _plain_attend(st):
    case, table, cu, lens = st["case"], st["page_table"].long(), st["cu"].long(), st["seq_lens"].long()
    q, page, B = st["q"], case["page"], len(st["seq_lens"])
    T, hq, D = q.shape
    hk, n = case["hk"], st["max_new"]
    g, L, dev = hq // hk, table.shape[1] * page, q.device

    def held(name):  # [B, hk, L, D]
        at = table.clamp(min=0)
        codes = st[name + "_codes"].view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
        x = codes * st[name + "_scale"][at][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(B, hk, L, D)

    new = cu[1:] - cu[:-1]
    i = torch.arange(n, device=dev)
    rows = (cu[:-1, None] + i).clamp(max=T - 1)
    qs = q.float()[rows].view(B, n, hk, g, D).permute(0, 2, 3, 1, 4).reshape(B, hk, g * n, D)
    s = torch.matmul(qs, held("k").transpose(-1, -2)) * (1 / math.sqrt(D))
    j, at = torch.arange(L, device=dev), (lens - new)[:, None] + i
    seen = (j < lens[:, None, None]).expand(B, n, L)
    if case["causal"]:
        seen = seen & (j <= at[..., None])
    if case["window"]:
        seen = seen & (j > at[..., None] - case["window"])
    s = s.view(B, hk, g, n, L).masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0, m)
    p = (s - m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hk, g * n, L), held("v")).view(B, hk, g, n, D)
    o = torch.where(total > 0, o / total, 0)
    back = (i < new[:, None]).reshape(-1).nonzero()[:, 0]
    out = o.permute(0, 3, 1, 2, 4).reshape(B * n, hq, D)[back].to(q.dtype)
    if not case["lse"]:
        return out
    lse = (m + total.log()).permute(0, 3, 1, 2, 4).reshape(B * n, hq)[back]
    return out, lse


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _package():
    from __graft_entry__ import pdm_import

    return pdm_import()


def run(st):
    case = st["case"]
    path = case["path"]
    if path in ("rope", "train"):
        if own:
            yq, yk = _package().qk_norm_rope(st["q"], st["k"], st["positions"], st["cos"], st["sin"],
                                             q_weight=st["qw"], k_weight=st["kw"], eps=EPS,
                                             interleaved=case["interleaved"])
        else:
            yq, yk = _plain_rope(st)
        if path == "rope":
            return yq, yk
        leaves = [st[n] for n in ("q", "k", "qw", "kw") if st[n] is not None]
        return (yq.detach(), yk.detach(), *torch.autograd.grad((yq, yk), leaves, (st["gq"], st["gk"])))
    cache = (st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"])
    if path == "append":
        if not own:
            return _plain_append(st)
        _package().kv_append(st["k"], st["v"], *cache, st["cu"], st["page_table"], st["seq_lens"], cos=st["cos"],
                             sin=st["sin"], k_weight=st["kw"], eps=EPS, interleaved=case["interleaved"])
        return cache
    if not own:
        return _plain_attend(st)
    return _package().kv_attention(st["q"], *cache, st["cu"], st["page_table"], st["seq_lens"],
                                   causal=case["causal"], window=case["window"], max_q_len=st["max_new"],
                                   return_lse=case["lse"])


# ---------------------------------------------------------------------------
# Work and the definition in 64 bits
# ---------------------------------------------------------------------------

def _visible(n, length, causal, window):
    """(query, key) pairs that are seen, and the keys that any query sees, of one sequence."""
    pairs, low, high = 0, length, 0
    for i in range(n):
        p = length - n + i
        hi = p + 1 if causal else length
        lo = max(0, p - window + 1) if window else 0
        pairs += max(0, hi - lo)
        low, high = min(low, lo), max(high, hi)
    return pairs, max(0, high - low)


def work(case):
    dim, b = case["dim"], _BYTES[case["dtype"]]
    if case["path"] in ("rope", "train"):
        T, heads = case["tokens"], case["hq"] + case["hk"]
        tables = min(T, case["max_pos"]) * case["rot"] * 4 + 8 * T
        x = T * heads * dim
        if case["path"] == "rope":
            return {"bytes": 2 * x * b + tables, "flops": 8 * x}
        return {"bytes": 4 * x * b + tables, "flops": 24 * x}
    new, lens = _sequences(case, 0)
    ints = 4 * (2 * case["batch"] + 1) + 4 * sum((n + case["page"] - 1) // case["page"] for n in lens)
    if case["path"] == "append":
        x = 2 * sum(new) * case["hk"] * dim
        return {"bytes": x * (b + 1) + sum(new) * case["rot"] * 4 + ints, "flops": 8 * x}
    seen = [_visible(n, ln, case["causal"], case["window"]) for n, ln in zip(new, lens)]
    pairs, keys = sum(s[0] for s in seen), sum(s[1] for s in seen)
    return {"bytes": 2 * keys * case["hk"] * dim + 2 * sum(new) * case["hq"] * dim * b
            + (4 * sum(new) * case["hq"] if case["lse"] else 0) + ints,
            "flops": 4 * dim * case["hq"] * pairs}


def _turn64(x, weight, angle_cos, angle_sin, interleaved):
    """x [T, H, D] in 64 bits, normed and turned: each pair as a complex number."""
    if weight is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    if angle_cos is None:
        return x
    half = angle_cos.shape[-1]
    turn = torch.complex(angle_cos.double(), angle_sin.double())[:, None]
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    pairs = head.unflatten(-1, (half, 2)) if interleaved else head.unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return torch.cat((z, rest), -1)


def _exact_rope(st):
    case = st["case"]
    out, grads, wgrads = [], [], []
    cos, sin = st["cos"][st["positions"]], st["sin"][st["positions"]]
    for x, w, g in ((st["q"], st["qw"], st.get("gq")), (st["k"], st["kw"], st.get("gk"))):
        x = x.detach().double()
        w = None if w is None else w.detach().double()
        out.append(_turn64(x, w, cos, sin, case["interleaved"]))
        if g is None:
            continue
        back = _turn64(g.double(), None, cos, -sin, case["interleaved"])  # the inverse rotation
        if w is None:
            grads.append(back)
            continue
        r = 1 / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
        h = back * w
        grads.append(r * h - x * r ** 3 * (h * x).mean(-1, keepdim=True))
        wgrads.append((back * x * r).sum((0, 1)))
    return (*out, *grads, *wgrads)


def _round_e4m3(x):
    """To the nearest e4m3 value, ties to even; steps of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (x / step).round() * step


def _exact_append(st):
    """Page by page."""
    case, page = st["case"], st["case"]["page"]
    cu, lens, table = st["cu"].tolist(), st["seq_lens"].tolist(), st["page_table"].tolist()
    steps = sum((lens[b] - 1) // page - (lens[b] - cu[b + 1] + cu[b]) // page + 1 for b in range(len(lens)))
    if steps > 6000 or st["k_codes"].numel() > 4e8:
        return None
    index = torch.cat([torch.arange(lens[b] - cu[b + 1] + cu[b], lens[b]) for b in range(len(lens))]).cuda()
    cos, sin = (None, None) if st["cos"] is None else (st["cos"][index], st["sin"][index])
    values = []
    scales = []
    for name in ("k", "v"):
        x = st[name].double()
        if name == "k":
            x = _turn64(x, st["kw"], cos, sin, case["interleaved"])
        codes, scale = st[name + "_codes"].double(), st[name + "_scale"].double()
        for b in range(len(lens)):
            at, row = lens[b] - (cu[b + 1] - cu[b]), cu[b]
            while at < lens[b]:
                slot = at % page
                n = min(page - slot, lens[b] - at)
                part, p = x[row:row + n], table[b][at // page]
                e = torch.ceil(torch.log2(part.abs().amax((0, 2)).clamp(min=1e-300) / FP8_MAX)).clamp(E_MIN, E_MAX)
                if slot:
                    e = torch.maximum(e, torch.log2(scale[p]))
                    codes[p, :, :slot] = _round_e4m3(codes[p, :, :slot] * (scale[p] / torch.exp2(e))[:, None, None])
                scale[p] = torch.exp2(e)
                codes[p, :, slot:slot + n] = _round_e4m3(part / scale[p][:, None]).transpose(0, 1)
                at, row = at + n, row + n
        values.append(codes)
        scales.append(scale)
    return (*values, *scales)


def _exact_attend(st):
    """Sequence by sequence, head by head."""
    case, page = st["case"], st["case"]["page"]
    cu, lens = st["cu"].tolist(), st["seq_lens"].tolist()
    q, hk = st["q"].double(), case["hk"]
    g = case["hq"] // hk
    if len(lens) * hk > 4096:
        return None
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        pages = st["page_table"][b, :(length + page - 1) // page].long()
        i = torch.arange(length - n, length, device=q.device)[:, None]
        j = torch.arange(length, device=q.device)[None, :]
        hidden = (j > i) if case["causal"] else torch.zeros_like(j > i)
        if case["window"]:
            hidden = hidden | (j <= i - case["window"])
        for h in range(hk):
            k, v = ((st[c + "_codes"].view(torch.uint8)[pages, h].view(torch.float8_e4m3fn).double()
                     * st[c + "_scale"][pages, h].double()[:, None, None]).reshape(-1, case["dim"])[:length]
                    for c in "kv")
            for head in range(h * g, h * g + g):
                s = (q[cu[b]:cu[b + 1], head] @ k.T / math.sqrt(case["dim"])).masked_fill_(hidden, -math.inf)
                total = torch.logsumexp(s, -1)
                w = torch.exp(s - total.clamp(min=-1e300)[:, None])
                out[cu[b]:cu[b + 1], head] = w @ v
                lse[cu[b]:cu[b + 1], head] = total
    return (out, lse) if case["lse"] else out


def exact(case, seed):
    st = prepare(case, seed)
    if case["path"] in ("rope", "train"):
        return _exact_rope(st)
    return _exact_append(st) if case["path"] == "append" else _exact_attend(st)

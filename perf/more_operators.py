"""Cases of windowed attention with a relative position bias: what each is timed on, its plain form, its definition in 64 bits.

* ``forward``  ``jagged_attention`` of a ragged batch: causal or not, a window, first tokens that stay visible (sinks), a bias by
               distance; outputs and the logarithms of the rows' sums
* ``train``    ``bucket_bias`` and ``jagged_attention`` with their backward passes: outputs, gradients of q, k, v and of the
               table of buckets
* ``bias``     ``bucket_bias`` and its backward pass alone
* ``cached``   ``kv_attention`` over 8-bit pages with sinks and the bias, from one token to long prompts

Query i of a sequence of n_q queries and n_k keys stands at position p = n_k - n_q + i and sees the keys j with j <= p (causal)
and, where there is a window, j > p - window or j < sinks.  Its score of key j has bias[head, p - j - start] added, where the
column is held within the bias's.  Lengths are log-spaced between a case's bounds and dealt to the sequences by the seed, so that
a case's work does not depend on the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
FP8_MAX = 448.0


def listed():
    return [
        # one user's history of 200 events, 6 heads of 64: latency
        dict(name="forward_user", path="forward", batch=1, q_lo=200, q_hi=200, past_lo=0, past_hi=0, hq=6, hk=6, dim=64,
             dtype="bf16", causal=True, window=0, sinks=0, span=128, buckets=32),
        # the last 1 to 60 events of 512 users over their whole histories
        dict(name="forward_events_b512", path="forward", batch=512, q_lo=1, q_hi=60, past_lo=1, past_hi=700, hq=6, hk=6,
             dim=64, dtype="bf16", causal=True, window=0, sinks=0, span=512, buckets=64),
        # a prompt of 8,192 tokens under a window of 1,024, its first 4 tokens visible throughout
        dict(name="forward_window_t8192", path="forward", batch=1, q_lo=8_192, q_hi=8_192, past_lo=0, past_hi=0, hq=32,
             hk=8, dim=128, dtype="bf16", causal=True, window=1_024, sinks=4, span=0, buckets=0),
        # training on 64 users of 32 to 500 events, 6 heads of 64
        dict(name="train_users_b64", path="train", batch=64, q_lo=32, q_hi=500, past_lo=0, past_hi=0, hq=6, hk=6, dim=64,
             dtype="bf16", causal=True, window=0, sinks=0, span=128, buckets=32, table="fp32"),
        # training on long rows: grouped heads, a window with sinks, a bias over the window
        dict(name="train_window_fp16", path="train", batch=2, q_lo=3_500, q_hi=4_700, past_lo=0, past_hi=0, hq=24, hk=6,
             dim=128, dtype="fp16", causal=True, window=512, sinks=4, span=513, buckets=64, table="fp32"),
        # training on both sides of a token, ragged rows of odd lengths; no window: the most products
        dict(name="train_both_sides", path="train", batch=8, q_lo=1_001, q_hi=2_777, past_lo=0, past_hi=0, hq=8, hk=8,
             dim=64, dtype="bf16", causal=False, window=0, sinks=0, span=2_001, buckets=64, table="bf16"),
        # the table of 16 heads spread over 4,096 distances, and back
        dict(name="bias_h16_s4096", path="bias", hq=16, span=4_096, buckets=128, causal=True, table="fp32"),
        # a large one: 64 heads, 65,536 distances on both sides
        dict(name="bias_h64_s65536", path="bias", hq=64, span=65_536, buckets=320, causal=False, table="bf16"),
        # one sequence decoding alone under a window with sinks: latency
        dict(name="cached_decode_b1", path="cached", batch=1, q_lo=1, q_hi=1, past_lo=2_999, past_hi=2_999, hq=32, hk=8,
             dim=128, page=64, dtype="bf16", causal=True, window=512, sinks=4, span=512, buckets=32, lse=False),
        # a decoding batch of ragged contexts, no window, bias of the nearest 1,024 distances
        dict(name="cached_decode_b64", path="cached", batch=64, q_lo=1, q_hi=1, past_lo=127, past_hi=8_191, hq=32, hk=8,
             dim=128, page=64, dtype="bf16", causal=True, window=0, sinks=0, span=1_024, buckets=32, lse=False),
        # scoring: 16 NS tokens of each of 256 requests over their cached histories, 6 heads of 64
        dict(name="cached_ns_b256", path="cached", batch=256, q_lo=16, q_hi=16, past_lo=300, past_hi=1_500, hq=6, hk=6,
             dim=64, page=32, dtype="bf16", causal=True, window=0, sinks=0, span=256, buckets=32, lse=False),
        # prompts continued over a cached prefix, window with sinks and bias; the largest case
        dict(name="cached_prompts_b2", path="cached", batch=2, q_lo=3_500, q_hi=4_500, past_lo=3_001, past_hi=5_001,
             hq=32, hk=8, dim=128, page=64, dtype="bf16", causal=True, window=2_048, sinks=64, span=2_048, buckets=64,
             lse=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["forward", "forward", "train", "train", "train", "bias", "cached", "cached", "cached"])
    causal = rng.random() < 0.75
    span = rng.choice([0, _log(rng, 1, 4_096), _log(rng, 1, 4_096)])
    if path == "bias":
        span = _log(rng, 1, 65_536)
        return dict(path=path, hq=_log(rng, 1, 64), span=span, buckets=min(span, _log(rng, 1, 512)), causal=causal,
                    table=rng.choice(["fp32", "bf16", "fp16"]))
    dim = rng.choice([64, 128])
    hk = rng.choice([1, 2, 4, 6, 8])
    group = rng.choice([1, 1, 2, 4, 7])
    window = rng.choice([0, 0, _log(rng, 1, 4_096)])
    case = dict(path=path, batch=_log(rng, 1, 512), hq=hk * group, hk=hk, dim=dim, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                causal=causal, window=window, sinks=rng.choice([0, 4, _log(rng, 1, 200)]) if window else 0, span=span,
                buckets=min(span, _log(rng, 1, 128)))
    case["q_lo"] = rng.choice([1, 1, _log(rng, 1, 2_000)])
    case["q_hi"] = rng.choice([case["q_lo"], _log(rng, case["q_lo"], 5_000)])
    if path == "cached":
        case.update(dim=rng.choice([64, 128, 128, 256]), page=rng.choice([16, 32, 64, 128]), lse=rng.random() < 0.5,
                    past_lo=rng.choice([0, _log(rng, 1, 8_000)]))
        case["past_hi"] = max(case["past_lo"], _log(rng, 16, 40_000))
        pairs, keys = 5e8, 2e8
    else:
        case["past_lo"] = rng.choice([0, 0, _log(rng, 1, 500)])
        case["past_hi"] = max(case["past_lo"], rng.choice([0, 0, _log(rng, 1, 5_000)]))
        pairs, keys = (3e8, 2e8) if path == "forward" else (1.5e8, 1e8)
        if path == "train":
            case["table"] = rng.choice(["fp32", "bf16"])

    def cost():
        per = case["batch"] * (case["q_hi"] + case["past_hi"])
        return max(per * case["hk"] * case["dim"] / keys, per * case["q_hi"] * case["hq"] / pairs)

    while case["batch"] > 1 and cost() > 1:
        case["batch"] //= 2
    while cost() > 1:
        for n in ("q_lo", "q_hi", "past_lo", "past_hi"):
            case[n] = max(1 if n[0] == "q" else 0, case[n] // 2)
    return case


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
    """(queries, keys) of every sequence: the lists of the case, dealt by the seed."""
    new = [max(1, v) for v in _lengths(case["batch"], case["q_lo"], case["q_hi"])]
    past = _lengths(case["batch"], case["past_lo"], case["past_hi"])
    rng = random.Random(seed)
    rng.shuffle(new)
    rng.shuffle(past)
    return new, [n + p for n, p in zip(new, past)]


def _start(case):
    """The distance of the bias's first column."""
    return 0 if case["causal"] else -(case["span"] // 2)


def _bucket_map(case):
    """The bucket of every column: exact near a token, in logarithmic steps farther off, sides apart."""
    span, n, start = case["span"], case["buckets"], _start(case)
    sides = 2 if start < 0 and n > 1 else 1
    per = n // sides
    far = max(span + start, 2)
    out = []
    for c in range(span):
        d = abs(c + start)
        side = per if sides == 2 and c + start < 0 else 0
        near = (per + 1) // 2
        b = d if d < near else near + int((per - near) * math.log((d + 1) / (near + 1)) / math.log((far + 1) / (near + 1))
                                          if far > near else 0)
        out.append(side + min(b, per - 1))
    return out


def _cumulative(lengths, dev):
    return torch.tensor([0] + lengths, device=dev).cumsum(0).to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    st = dict(case=dict(case), start=_start(case) if case["span"] else 0)
    rand = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    if case["span"]:
        st["map"] = torch.tensor(_bucket_map(case), dtype=torch.int32, device=dev)
        table = rand(case["buckets"], case["hq"]) * 0.7 - torch.linspace(0, 1, case["buckets"], device=dev)[:, None]
        st["table"] = table.to(_TORCH[case.get("table", "fp32")])
        if case["path"] in ("forward", "cached"):  # a serving program spreads its table once
            st["bias"] = st["table"].float()[st["map"].long()].t().contiguous()
    if case["path"] == "bias":
        st["table"].requires_grad_(True)
        st["grad"] = rand(case["hq"], case["span"])
        return st
    dt, dim, hq, hk = _TORCH[case["dtype"]], case["dim"], case["hq"], case["hk"]
    new, lens = _sequences(case, seed)
    T, st["n_q"], st["n_k"] = sum(new), max(new), max(lens)
    st["cu"] = _cumulative(new, dev)
    if case["path"] != "cached":
        st["cu_k"] = st["cu"] if new == lens else _cumulative(lens, dev)
        st["new"], st["lens"] = new, lens
        # heads as columns of the fused projections' rows
        rows = rand(sum(lens), 2 * hk * dim).to(dt)
        st["q"] = (rand(T, hq * dim) * 1.5).to(dt).view(T, hq, dim)
        st["k"] = rows[:, :hk * dim].view(-1, hk, dim)
        st["v"] = rows[:, hk * dim:].view(-1, hk, dim)
        if case["path"] == "train":
            st["grad"] = rand(T, hq, dim).to(dt)
            for n in ("q", "k", "v", "table"):
                if n in st:
                    st[n] = st[n].detach().requires_grad_(True)
        return st
    page = case["page"]
    counts = [(n + page - 1) // page for n in lens]
    # a pool of one size for every seed, with pages to spare
    total = sum((n + page - 1) // page for n in new) + sum((ln - n + page - 1) // page for n, ln in zip(new, lens))
    order = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    cnt = torch.tensor(counts, device=dev)
    col = torch.arange(max(counts), device=dev)[None, :]
    first = (torch.cumsum(cnt, 0) - cnt)[:, None]
    st["page_table"] = torch.where(col < cnt[:, None], order[(first + col).clamp(max=total - 1)], -1).to(torch.int32)
    st["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    # codes of normal values, scales around 2^-7 (keys) and 2^-8 (values)
    for n, e in (("k", -7), ("v", -8)):
        codes = torch.empty(total, hk, page, dim, dtype=torch.float8_e4m3fn, device=dev)
        for i in range(0, total, 4096):
            part = codes[i:i + 4096]
            part.copy_((rand(*part.shape) * 100).clamp_(-FP8_MAX, FP8_MAX))
        st[n + "_codes"] = codes
        st[n + "_scale"] = torch.exp2(torch.randint(e - 1, e + 2, (total, hk), generator=gen, device=dev).float())
    st["q"] = (rand(T, hq * dim) * 1.5).to(dt).view(T, hq, dim)
    return st


# ---------------------------------------------------------------------------
# Plain forms (fp32, elementary operations, padded to the longest sequence)
# ---------------------------------------------------------------------------

def _pad_rows(x, cu, n):
    """[T, H, D] to fp32 [B, H, n, D]; what lies behind a sequence is zero."""
    i = torch.arange(n, device=x.device)
    rows = cu[:-1, None] + i
    there = i < (cu[1:] - cu[:-1])[:, None]
    y = x.detach()[rows.clamp(max=x.shape[0] - 1)].float()
    return torch.where(there[..., None, None], y, 0).permute(0, 2, 1, 3), there


def _unpad_rows(x, there):
    """[B, H, n, D] to [T, H, D]."""
    return x.permute(0, 2, 1, 3)[there]


def _seen(case, n, nk, new, lens, dev):
    """[B, n, nk]: which keys each query sees; and the distances [n, nk] but for a sequence's offset lens - new."""
    j = torch.arange(nk, device=dev)
    at = (lens - new)[:, None] + torch.arange(n, device=dev)
    seen = (j < lens[:, None, None]).expand(len(lens), n, nk)
    if case["causal"]:
        seen = seen & (j <= at[..., None])
    if case["window"]:
        near = j > at[..., None] - case["window"]
        seen = seen & ((near | (j < case["sinks"])) if case["sinks"] else near)
    return seen, at


def _columns(st, at, nk):
    """The bias's column of every (sequence, query, key)."""
    j = torch.arange(nk, device=at.device)
    return (at[..., None] - j - st["start"]).clamp_(0, st["case"]["span"] - 1)


def _softmax(st, s, seen, at, bias):
    """s [B, hk, g, n, nk] scores; returns weights before their division, sums, maxima."""
    B, hk, g, n, nk = s.shape
    if bias is not None:
        s = s + bias[:, _columns(st, at, nk)].view(hk, g, B, n, nk).permute(2, 0, 1, 3, 4)
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0, m)
    p = (s - m).exp_()
    return p, p.sum(-1, keepdim=True), m


def _plain_table_grad(st, by_column, dtype):
    """[hq, span] in 64 bits to [buckets, hq]."""
    out = torch.zeros(st["case"]["buckets"], by_column.shape[0], dtype=torch.float64, device=by_column.device)
    return out.index_add_(0, st["map"].long(), by_column.t().double()).to(dtype)


def _plain_jagged(st):
    case, dt = st["case"], st["q"].dtype
    hk, D = case["hk"], case["dim"]
    g, scale = case["hq"] // hk, 1 / math.sqrt(case["dim"])
    cu, cu_k = st["cu"].long(), st["cu_k"].long()
    new, lens = cu[1:] - cu[:-1], cu_k[1:] - cu_k[:-1]
    q, there = _pad_rows(st["q"], cu, st["n_q"])
    k, there_k = _pad_rows(st["k"], cu_k, st["n_k"])
    v, _ = _pad_rows(st["v"], cu_k, st["n_k"])
    B, _, n, _ = q.shape
    nk = k.shape[2]
    seen, at = _seen(case, n, nk, new, lens, q.device)
    q = q.reshape(B, hk, g * n, D)
    bias = None
    if case["span"]:
        bias = st["bias"] if case["path"] == "forward" else st["table"].detach().float()[st["map"].long()].t()
    p, total, m = _softmax(st, (torch.matmul(q, k.transpose(-1, -2)) * scale).view(B, hk, g, n, nk), seen, at, bias)
    o = torch.matmul(p.view(B, hk, g * n, nk), v).view(B, hk, g, n, D)
    o = torch.where(total > 0, o / total, 0)
    out = _unpad_rows(o.reshape(B, hk * g, n, D), there).to(dt)
    if case["path"] == "forward":
        return out, _unpad_rows((m + total.log()).view(B, hk * g, n, 1), there)[..., 0]
    p = torch.where(total > 0, p / total, 0).view(B, hk, g * n, nk)
    do = _pad_rows(st["grad"], cu, n)[0].reshape(B, hk, g * n, D)
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds = (ds - (do * o.reshape(B, hk, g * n, D)).sum(-1, keepdim=True)).mul_(p)
    del p
    dq = torch.matmul(ds, k).mul_(scale).view(B, hk * g, n, D)
    dk = torch.matmul(ds.transpose(-1, -2), q).mul_(scale)
    grads = [_unpad_rows(x, w).to(dt) for x, w in ((dq, there), (dk, there_k), (dv, there_k))]
    if bias is not None:
        # diagonals as columns: with rows one longer than they are, row i lies i places further right
        ds = ds.view(B, hk * g, n, nk).flip(-1)
        ds = torch.nn.functional.pad(ds, (0, n)).view(B, hk * g, -1)[..., :n * (nk + n - 1)]
        ds = ds.view(B, hk * g, n, nk + n - 1).sum(-2, dtype=torch.float64)  # column c: i - j = c - nk + 1
        d = (lens - new)[:, None] + torch.arange(nk + n - 1, device=q.device) - (nk - 1)
        col = (d - st["start"]).clamp(0, case["span"] - 1)
        by = torch.zeros(hk * g, case["span"], dtype=torch.float64, device=q.device)
        by.scatter_add_(1, col.reshape(1, -1).expand(hk * g, -1), ds.transpose(0, 1).reshape(hk * g, -1))
        grads.append(_plain_table_grad(st, by, st["table"].dtype))
    return (out, *grads)


def _plain_cached(st):
    case, table, cu, lens = st["case"], st["page_table"].long(), st["cu"].long(), st["seq_lens"].long()
    q, page, B = st["q"], case["page"], len(st["seq_lens"])
    hk, D, n = case["hk"], case["dim"], st["n_q"]
    g, L = case["hq"] // hk, table.shape[1] * page

    def held(name):  # [B, hk, L, D]
        at = table.clamp(min=0)
        codes = st[name + "_codes"].view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
        x = codes * st[name + "_scale"][at][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(B, hk, L, D)

    qs, there = _pad_rows(q, cu, n)
    seen, at = _seen(case, n, L, cu[1:] - cu[:-1], lens, q.device)
    s = torch.matmul(qs.reshape(B, hk, g * n, D), held("k").transpose(-1, -2)) * (1 / math.sqrt(D))
    p, total, m = _softmax(st, s.view(B, hk, g, n, L), seen, at, st.get("bias"))
    o = torch.matmul(p.view(B, hk, g * n, L), held("v")).view(B, hk, g, n, D)
    o = torch.where(total > 0, o / total, 0)
    out = _unpad_rows(o.view(B, hk * g, n, D), there).to(q.dtype)
    if not case["lse"]:
        return out
    return out, _unpad_rows((m + total.log()).view(B, hk * g, n, 1), there)[..., 0]


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _package():
    from __graft_entry__ import pdm_import

    return pdm_import()


def _own(st):
    case, pdm = st["case"], _package()
    if case["path"] == "bias":
        bias = pdm.bucket_bias(st["table"], st["map"])
        return bias.detach(), *torch.autograd.grad(bias, [st["table"]], st["grad"])
    mask = dict(causal=case["causal"], window=case["window"], sinks=case["sinks"], bias_start=st["start"])
    if case["path"] == "cached":
        return pdm.kv_attention(st["q"], st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"], st["cu"],
                                st["page_table"], st["seq_lens"], max_q_len=st["n_q"], return_lse=case["lse"],
                                bias=st.get("bias"), **mask)
    if case["path"] == "forward":
        return pdm.jagged_attention(st["q"], st["k"], st["v"], st["cu"], st["cu_k"], bias=st.get("bias"),
                                    return_lse=True, **mask)
    bias = pdm.bucket_bias(st["table"], st["map"]) if case["span"] else None
    out = pdm.jagged_attention(st["q"], st["k"], st["v"], st["cu"], st["cu_k"], bias=bias, **mask)
    leaves = [st[n] for n in ("q", "k", "v", "table") if n in st]
    return (out.detach(), *torch.autograd.grad(out, leaves, st["grad"]))


def run(st):
    if own:
        return _own(st)
    if st["case"]["path"] == "bias":
        return (st["table"].detach().float()[st["map"].long()].t().contiguous(),
                _plain_table_grad(st, st["grad"], st["table"].dtype))
    return _plain_cached(st) if st["case"]["path"] == "cached" else _plain_jagged(st)


# ---------------------------------------------------------------------------
# Work and the definition in 64 bits
# ---------------------------------------------------------------------------

def _visible(case, n, length):
    """(query, key) pairs that are seen, and the keys that any query sees, of one sequence."""
    window, first = case["window"], case["sinks"]
    pairs, low, high = 0, length, 0
    for i in range(n):
        p = length - n + i
        hi = p + 1 if case["causal"] else length
        lo = max(0, p - window + 1) if window else 0
        pairs += max(0, hi - lo) + (min(first, lo, hi) if lo else 0)
        low, high = min(low, lo), max(high, hi)
    return pairs, max(0, high - low) + min(first, low)


def work(case):
    if case["path"] == "bias":
        cells, held = case["hq"] * case["span"], case["hq"] * case["buckets"] * _BYTES[case["table"]]
        return {"bytes": 8 * cells + 2 * held + 4 * case["span"], "flops": cells}
    dim, b = case["dim"], _BYTES[case["dtype"]]
    new, lens = _sequences(case, 0)
    seen = [_visible(case, n, ln) for n, ln in zip(new, lens)]
    pairs, keys = sum(s[0] for s in seen), sum(s[1] for s in seen)
    queries, ints = sum(new) * case["hq"], 4 * (2 * case["batch"] + 1)
    bias = 4 * case["hq"] * case["span"]
    if case["path"] == "cached":
        ints += 4 * sum((n + case["page"] - 1) // case["page"] for n in lens)
        return {"bytes": 2 * keys * case["hk"] * dim + 2 * queries * dim * b + (4 * queries if case["lse"] else 0) + bias + ints,
                "flops": 4 * dim * case["hq"] * pairs}
    held = 2 * keys * case["hk"] * dim * b
    if case["path"] == "forward":
        return {"bytes": held + 2 * queries * dim * b + 4 * queries + bias + ints, "flops": 4 * dim * case["hq"] * pairs}
    table = 2 * case["hq"] * case["buckets"] * _BYTES[case["table"]] + 4 * case["span"]
    # inputs, the output's gradient; the output and four gradients; two products forward, five back
    return {"bytes": 2 * held + 4 * queries * dim * b + table + ints, "flops": 14 * dim * case["hq"] * pairs}


def _mask64(case, p, j):
    """Truth values [queries, keys] of positions p and keys j."""
    p, j = p[:, None], j[None, :]
    hidden = (j > p) if case["causal"] else torch.zeros_like(j > p)
    if case["window"]:
        hidden = hidden | ((j <= p - case["window"]) & (j >= case["sinks"]))
    return hidden


def _exact_bias(st):
    table = st["table"].detach().double()
    where = torch.nn.functional.one_hot(st["map"].long(), st["case"]["buckets"])
    back = torch.zeros_like(table)
    for at in range(0, st["case"]["span"], 4096):
        part = where[at:at + 4096].double()
        back += part.t() @ st["grad"][:, at:at + 4096].double().t()
    return torch.stack([table[b] for b in st["map"].tolist()], 1), back


def _exact_jagged(st):
    """Sequence by sequence, head by head."""
    case = st["case"]
    new, lens = st["new"], st["lens"]
    g, D, dev = case["hq"] // case["hk"], case["dim"], st["q"].device
    pairs = sum(n * ln for n, ln in zip(new, lens)) * case["hq"]
    if len(new) * case["hq"] > 6000 or pairs > 4e9:
        return None
    train = case["path"] == "train"
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=dev)
    dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v))
    cells, start = case["span"], st["start"]
    dtable = torch.zeros(max(case["buckets"], 1), case["hq"], dtype=torch.float64, device=dev)
    row = key = 0
    for n, length in zip(new, lens):
        p, j = torch.arange(length - n, length, device=dev), torch.arange(length, device=dev)
        hidden = _mask64(case, p, j)
        if cells:
            bucket = st["map"].long()[(p[:, None] - j[None, :] - start).clamp(0, cells - 1)]
        for h in range(case["hq"]):
            at = h // g
            qh, kh, vh = q[row:row + n, h], k[key:key + length, at], v[key:key + length, at]
            s = qh @ kh.T / math.sqrt(D)
            if cells:
                s += st["table"].detach().double()[:, h][bucket]
            s.masked_fill_(hidden, -math.inf)
            total = torch.logsumexp(s, -1)
            w = torch.exp(s - total.clamp(min=-1e300)[:, None])
            o = w @ vh
            out[row:row + n, h], lse[row:row + n, h] = o, total
            if not train:
                continue
            go = st["grad"][row:row + n, h].double()
            ds = w * (go @ vh.T - (go * o).sum(-1, keepdim=True))
            dv[key:key + length, at] += w.T @ go
            dq[row:row + n, h] = ds @ kh / math.sqrt(D)
            dk[key:key + length, at] += ds.T @ qh / math.sqrt(D)
            if cells:
                dtable[:, h] += torch.bincount(bucket.flatten(), weights=ds.flatten(), minlength=case["buckets"])
        row, key = row + n, key + length
    if not train:
        return out, lse
    return (out, dq, dk, dv, dtable) if cells else (out, dq, dk, dv)


def _exact_cached(st):
    """Sequence by sequence, head by head."""
    case, page = st["case"], st["case"]["page"]
    cu, lens = st["cu"].tolist(), st["seq_lens"].tolist()
    q, hk = st["q"].double(), case["hk"]
    g, cells = case["hq"] // hk, case["span"]
    pairs = sum((cu[b + 1] - cu[b]) * lens[b] for b in range(len(lens))) * case["hq"]
    if len(lens) * case["hq"] > 6000 or pairs > 4e9:
        return None
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    for b, length in enumerate(lens):
        p = torch.arange(length - (cu[b + 1] - cu[b]), length, device=q.device)
        j = torch.arange(length, device=q.device)
        pages = st["page_table"][b, :(length + page - 1) // page].long()
        hidden = _mask64(case, p, j)
        if cells:
            bucket = st["map"].long()[(p[:, None] - j[None, :] - st["start"]).clamp(0, cells - 1)]
        for h in range(hk):
            k, v = ((st[c + "_codes"].view(torch.uint8)[pages, h].view(torch.float8_e4m3fn).double()
                     * st[c + "_scale"][pages, h].double()[:, None, None]).reshape(-1, case["dim"])[:length]
                    for c in "kv")
            for head in range(h * g, h * g + g):
                s = q[cu[b]:cu[b + 1], head] @ k.T / math.sqrt(case["dim"])
                if cells:
                    s += st["table"].double()[:, head][bucket]
                s.masked_fill_(hidden, -math.inf)
                total = torch.logsumexp(s, -1)
                out[cu[b]:cu[b + 1], head] = torch.exp(s - total.clamp(min=-1e300)[:, None]) @ v
                lse[cu[b]:cu[b + 1], head] = total
    return (out, lse) if case["lse"] else out


def exact(case, seed):
    st = prepare(case, seed)
    if case["path"] == "bias":
        return _exact_bias(st)
    return _exact_cached(st) if case["path"] == "cached" else _exact_jagged(st)

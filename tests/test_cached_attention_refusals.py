"""What the cached-attention operators refuse, before any device work: shapes, types, sizes, gradients, CPU tensors; and
the argument checks of their C entry points."""
import ctypes

import pytest
import torch


def _rope(**kw):
    a = dict(q=torch.zeros(4, 2, 64), k=torch.zeros(4, 1, 64), positions=torch.zeros(4, dtype=torch.int64),
             cos=torch.zeros(8, 32), sin=torch.zeros(8, 32), q_weight=torch.ones(64), k_weight=torch.ones(64))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error,text", [
    (dict(q=torch.zeros(4, 2, 60), k=None, k_weight=None, q_weight=None), ValueError, "multiple of 16"),
    (dict(q=torch.zeros(4, 64)), ValueError, "positions"),
    (dict(q=torch.zeros(4, 2, 64, dtype=torch.float64)), (TypeError, ValueError), "float"),
    (dict(k=torch.zeros(4, 1, 32)), ValueError, "beside q"),
    (dict(k=torch.zeros(3, 1, 64)), ValueError, "tokens"),
    (dict(k=torch.zeros(4, 1, 64, dtype=torch.bfloat16)), ValueError, "beside q"),
    (dict(positions=torch.zeros(4)), TypeError, "positions"),
    (dict(positions=torch.zeros(5, dtype=torch.int64)), ValueError, "positions"),
    (dict(cos=None), ValueError, "together"),
    (dict(cos=torch.zeros(8, 40), sin=torch.zeros(8, 40)), ValueError, "rotary_dim"),
    (dict(cos=torch.zeros(8, 20), sin=torch.zeros(8, 20)), ValueError, "rotary_dim"),
    (dict(cos=torch.zeros(8, 32).double(), sin=torch.zeros(8, 32).double()), TypeError, "float32"),
    (dict(cos=torch.zeros(8, 32, requires_grad=True)), ValueError, "gradient"),
    (dict(q_weight=None), ValueError, "together"),
    (dict(q_weight=torch.ones(32)), ValueError, "q_weight"),
    (dict(q_weight=torch.ones(64, dtype=torch.float16)), TypeError, "q_weight"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(err_flag=torch.zeros(1)), ValueError, "err_flag"),
    (dict(), RuntimeError, "GPU only"),
])
def test_qk_norm_rope(pdm, kw, error, text):
    with pytest.raises(error, match=text):
        pdm.qk_norm_rope(**_rope(**kw))


def _cache(pages=3, heads=2, page=16, D=64):
    codes = [torch.zeros(pages, heads, page, D, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]
    return dict(k_codes=codes[0], v_codes=codes[1], k_scale=torch.ones(pages, heads), v_scale=torch.ones(pages, heads))


def _batch(B=2):
    return dict(cu_seqlens=torch.tensor([0, 1, 3][:B + 1], dtype=torch.int32),
                page_table=torch.zeros(B, 2, dtype=torch.int32), seq_lens=torch.tensor([1, 2][:B], dtype=torch.int32))


SHARED = [
    (_cache(D=96), ValueError, "head_dim"),
    (_cache(page=24), ValueError, "page_size"),
    (dict(k_codes=torch.zeros(3, 2, 16, 64)), TypeError, "k_codes"),
    (dict(k_scale=torch.ones(3, 1)), ValueError, "k_scale"),
    (dict(v_scale=torch.ones(3, 2).double()), ValueError, "v_scale"),
    (dict(v_codes=_cache(pages=4)["v_codes"]), ValueError, "one shape"),
    (dict(cu_seqlens=torch.tensor([0, 1, 3])), TypeError, "cu_seqlens"),
    (dict(cu_seqlens=torch.tensor([0, 3], dtype=torch.int32)), ValueError, "cu_seqlens"),
    (dict(seq_lens=torch.ones(2, 1, dtype=torch.int32)), ValueError, "seq_lens"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int32)), ValueError, "page_table"),
    (dict(page_table=torch.zeros(2, 4, dtype=torch.int32)[:, ::2]), ValueError, "page_table"),
    (dict(err_flag=torch.zeros(1)), ValueError, "err_flag"),
    (dict(), RuntimeError, "GPU only"),
]


@pytest.mark.parametrize("kw,error,text", SHARED + [
    (dict(k=torch.zeros(3, 1, 64)), ValueError, "as k is"),
    (dict(k=torch.zeros(3, 1, 64), v=torch.zeros(3, 1, 64)), ValueError, "heads"),
    (dict(k=torch.zeros(3, 2, 64).int()), TypeError, "k must be"),
    (dict(positions=torch.zeros(2, dtype=torch.int64)), ValueError, "positions"),
    (dict(cos=torch.zeros(8, 32)), ValueError, "together"),
    (dict(k_weight=torch.ones(128)), ValueError, "k_weight"),
    (dict(k=torch.zeros(3, 2, 64, requires_grad=True)), RuntimeError, "no backward"),
    (dict(eps=float("nan")), ValueError, "eps"),
])
def test_kv_append(pdm, kw, error, text):
    a = dict(k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), **_cache(), **_batch())
    a.update(kw)
    if a["k_codes"].dim() == 4 and a["k_codes"].shape[-1] == 96:
        a.update(k=torch.zeros(3, 2, 96), v=torch.zeros(3, 2, 96))
    with pytest.raises(error, match=text):
        pdm.kv_append(**a)


@pytest.mark.parametrize("kw,error,text", SHARED + [
    (dict(q=torch.zeros(3, 4, 64)), TypeError, "float16 or bfloat16"),
    (dict(q=torch.zeros(3, 3, 64, dtype=torch.bfloat16)), ValueError, "multiple"),
    (dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16)), ValueError, "head_dim"),
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16, requires_grad=True)), RuntimeError, "no backward"),
    (dict(scale=float("inf")), ValueError, "scale"),
    (dict(window=-1), ValueError, "window"),
    (dict(max_q_len=-1), ValueError, "max_q_len"),
    (dict(out=torch.zeros(3, 4, 64)), ValueError, "out"),
])
def test_kv_attention(pdm, kw, error, text):
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), **_cache(), **_batch())
    a.update(kw)
    with pytest.raises(error, match=text):
        pdm.kv_attention(**a)


def test_modules(pdm):
    with pytest.raises(ValueError):
        pdm.QKNormRope(60, 10)
    with pytest.raises(ValueError):
        pdm.QKNormRope(64, 10, rotary_dim=72)
    with pytest.raises(ValueError):
        pdm.PagedKVCache(4, 24, 2, 64, "cpu")
    with pytest.raises(ValueError):
        pdm.PagedKVCache(4, 16, 2, 80, "cpu")
    m = pdm.QKNormRope(64, 10, norm=False)
    assert not list(m.parameters()) and not m.state_dict()
    assert set(pdm.QKNormRope(64, 10).state_dict()) == {"q_norm.weight", "k_norm.weight"}


def test_c_entry_points(pdm):
    L = pdm._lib
    lib = L.lib()
    assert ctypes.sizeof(L.QkRopeDesc) == 80 and ctypes.sizeof(L.KvCacheDesc) == 56
    assert ctypes.sizeof(L.KvBatchDesc) == 48 and ctypes.sizeof(L.KvAppendDesc) == 64
    assert ctypes.sizeof(L.KvAttentionDesc) == 40
    none = [None] * 11
    assert lib.pdm_qk_norm_rope_fwd(None, *none) == L.PDM_ERR_INVALID and "null" in L.last_error()
    for change, text in (("head_dim", "head_dim"), ("rotary_dim", "rotary_dim"), ("dtype", "dtype"),
                         ("position_bits", "position_bits")):
        d = L.QkRopeDesc(4, 2, 1, 64, 64, L.PDM_BF16, 64, 0, 1e-6, 8, 128, 64, 64, 64)
        setattr(d, change, 9)
        assert lib.pdm_qk_norm_rope_fwd(ctypes.byref(d), *none) == L.PDM_ERR_INVALID and text in L.last_error()
        assert lib.pdm_qk_norm_rope_bwd_workspace_size(ctypes.byref(d)) == L.PDM_ERR_INVALID
    d = L.QkRopeDesc(1 << 30, 2, 1, 64, 64, L.PDM_BF16, 64, 0, 1e-6, 8, 128, 64, 64, 64)
    assert lib.pdm_qk_norm_rope_fwd(ctypes.byref(d), *none) == L.PDM_ERR_INVALID and "2^31" in L.last_error()
    d = L.QkRopeDesc(4, 2, 1, 64, 64, L.PDM_BF16, 64, 0, 1e-6, 8, 128, 64, 64, 64)
    assert lib.pdm_qk_norm_rope_fwd(ctypes.byref(d), *none) == L.PDM_ERR_INVALID and "null q" in L.last_error()
    assert lib.pdm_qk_norm_rope_bwd(ctypes.byref(d), 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 8,
                                    None) == L.PDM_ERR_WORKSPACE
    assert lib.pdm_qk_norm_rope_fwd(ctypes.byref(d), 16, 16, 16, 8, 16, 16, 16, 16, 16, None,
                                    None) == L.PDM_ERR_INVALID and "aligned" in L.last_error()
    cache, batch = L.KvCacheDesc(16, 16, 16, 16, 4, 2, 16, 64, 0), L.KvBatchDesc(16, 16, 16, 2, 4, 2, 2)
    att = L.KvAttentionDesc(L.PDM_BF16, 4, 1, 0, 0.1, 4, 256, 64)
    app = L.KvAppendDesc(L.PDM_BF16, 64, 64, 0, 1e-6, 0, 8, 128, 64, 128, 64)
    by = ctypes.byref
    assert lib.pdm_kv_append(None, None, None, *([None] * 8)) == L.PDM_ERR_INVALID
    assert lib.pdm_kv_append(by(app), by(cache), by(batch), *([None] * 8)) == L.PDM_ERR_INVALID
    assert "null k / v" in L.last_error()
    assert lib.pdm_kv_attention_fwd(None, None, None, None, None, None, None, 0, None, None) == L.PDM_ERR_INVALID
    assert lib.pdm_kv_attention_fwd(by(att), by(cache), by(batch), None, None, None, None, 0, None,
                                    None) == L.PDM_ERR_INVALID
    for obj, field, value, text in ((cache, "page_size", 48, "page_size"), (cache, "head_dim", 32, "head_dim"),
                                    (cache, "num_pages", 1 << 31, "num_pages"), (batch, "tokens", 1 << 31, "tokens"),
                                    (batch, "table_width", 1 << 28, "table_width"), (att, "n_q_heads", 5, "n_q_heads"),
                                    (att, "dtype", 0, "dtype"), (att, "window", -1, "window")):
        held = getattr(obj, field)
        setattr(obj, field, value)
        assert lib.pdm_kv_attention_workspace_size(by(att), by(cache), by(batch)) == L.PDM_ERR_INVALID, field
        assert text in L.last_error()
        setattr(obj, field, held)
    assert lib.pdm_kv_attention_workspace_size(by(att), by(cache), by(batch)) >= 0


def test_ops_are_registered(pdm):
    for name in ("qk_norm_rope", "qk_norm_rope_backward", "kv_append", "kv_attention"):
        assert hasattr(torch.ops.pdm, name)


def test_reference_quantizer_matches_the_cast():
    """The tests' own rounding to e4m3 against torch's cast, over every pair of neighbouring codes, their middle and the
    values beside it."""
    from oracle import cached_attention as ref

    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    x = torch.cat((codes, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)))
    x = torch.cat((x, -x))
    assert torch.equal(ref.round_e4m3(x), x.float().to(torch.float8_e4m3fn).double())
    assert [ref.scale_exponent(v) for v in (448.0, 448.0000001, 224.0, 1.75, 1.76, 0.0)] == [0, 1, -1, -8, -7, -117]


NO_SEQUENCES = """
import ctypes, sys
sys.path.insert(0, {root!r})
import __graft_entry__
L = __graft_entry__.pdm_import()._lib
lib, by = L.lib(), ctypes.byref
cache = L.KvCacheDesc(16, 16, 16, 16, 4, 2, 64, 64, 0)
for group, tokens, width, most in {cases!r}:
    batch = L.KvBatchDesc(16, 16, 16, width, tokens, 0, width)
    att = L.KvAttentionDesc(L.PDM_BF16, 2 * group, 1, 0, 0.1, min(most, tokens), 2 * group * 64, 64)
    size = lib.pdm_kv_attention_workspace_size(by(att), by(cache), by(batch))
    lib.pdm_kv_attention_fwd(by(att), by(cache), by(batch), 256, 256, None, 256, 1 << 40, None, None)
    print(size, flush=True)
"""


def test_attention_without_sequences(pdm):
    """A batch of padding alone is laid out without keys: no split, no join, no workspace, whatever the width of its table and
    the number of its rows.  The process has no GPU: it may not launch anything, and has to come back."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cases = [(2, 5, 1, 5), (2, 5, 10, 5), (2, 40, 1, 40), (2, 40, 10, 40), (2, 300, 1, 300), (2, 300, 64, 1), (24, 3, 10, 3),
             (40, 300, 10, 300)]
    env = {**os.environ, "HIP_VISIBLE_DEVICES": "-1", "ROCR_VISIBLE_DEVICES": "-1", "CUDA_VISIBLE_DEVICES": "-1"}
    r = subprocess.run([sys.executable, "-c", NO_SEQUENCES.format(root=root, cases=cases)], env=env, capture_output=True,
                       text=True)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr[-500:])
    assert r.stdout.split() == ["0"] * len(cases)


@pytest.mark.parametrize("how", ["fake", "meta"])
def test_tensors_without_memory(pdm, how):
    """Shapes and dtypes come out where no kernel can run, as from the framework's other operators; the cache is left alone."""
    import contextlib

    from torch._subclasses.fake_tensor import FakeTensorMode

    where = "meta" if how == "meta" else "cpu"
    with FakeTensorMode() if how == "fake" else contextlib.nullcontext():
        e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device=where)  # noqa: E731
        i = lambda *s: torch.empty(*s, dtype=torch.int32, device=where)  # noqa: E731
        q, k = e(3, 4, 64), e(3, 2, 64)
        f32 = lambda *s: e(*s, dtype=torch.float32)  # noqa: E731
        yq, yk = pdm.qk_norm_rope(q, k, e(3, dtype=torch.int64), f32(8, 32), f32(8, 32), f32(64), f32(64))
        assert yq.shape == q.shape and yk.shape == k.shape and yq.dtype == q.dtype
        yq, none = pdm.qk_norm_rope(q.view(1, 3, 4, 64), None, e(1, 3, dtype=torch.int64), None, None)
        assert yq.shape == (1, 3, 4, 64) and none is None
        cache = [e(5, 2, 16, 64, dtype=torch.float8_e4m3fn) for _ in range(2)] + [f32(5, 2) for _ in range(2)]
        batch = (i(2), i(1, 4), i(1))
        assert pdm.kv_append(k, k, *cache, *batch, err_flag=i(1)) is None
        out = pdm.kv_attention(q, *cache, *batch)
        assert out.shape == q.shape and out.dtype == q.dtype
        out, lse = pdm.kv_attention(q, *cache, *batch, return_lse=True)
        assert lse.shape == (3, 4) and lse.dtype == torch.float32
        assert all(t.device.type == where for t in (yq, out, lse))


@pytest.mark.parametrize("which", ["q", "k", "q_weight", "k_weight", "cos"])
def test_forward_mode_is_refused_by_qk_norm_rope(pdm, which):
    from torch.autograd import forward_ad

    a = _rope()
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="GPU only"):
            pdm.qk_norm_rope(**a)
        a[which] = forward_ad.make_dual(a[which], torch.ones_like(a[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            pdm.qk_norm_rope(**a)


@pytest.mark.parametrize("how", ["tangent", "gradient"])
@pytest.mark.parametrize("which", ["k", "v", "q", "k_codes", "v_codes", "k_scale", "v_scale", "k_weight", "cos", "sin", "out"])
def test_derivatives_of_the_cache_are_refused(pdm, how, which):
    """A derivative that nothing would carry on is refused, by whichever input it comes."""
    from torch.autograd import forward_ad

    app = dict(k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), k_weight=torch.ones(64), cos=torch.zeros(8, 32),
               sin=torch.zeros(8, 32), **_cache(), **_batch())
    att = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), out=torch.zeros(3, 4, 64, dtype=torch.bfloat16), **_cache(),
               **_batch())
    for f, a in ((pdm.kv_append, app), (pdm.kv_attention, att)):
        if which not in a:
            continue
        with forward_ad.dual_level():
            if how == "tangent":
                a[which] = forward_ad.make_dual(a[which], torch.ones_like(a[which]))
            else:
                a[which] = a[which].requires_grad_(True)
            with pytest.raises(RuntimeError, match="forward-mode" if how == "tangent" else "no backward"):
                f(**a)
            if how == "gradient":
                with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
                    f(**a)


def test_sizes_whose_product_passes_64_bits(pdm):
    """(Where the product overflows, the sanitized build stops.)"""
    L = pdm._lib
    d = L.QkRopeDesc(1 << 62, 4, 1, 64, 64, L.PDM_BF16, 64, 0, 1e-6, 8, 128, 64, 64, 64)
    assert L.lib().pdm_qk_norm_rope_fwd(ctypes.byref(d), *[None] * 11) == L.PDM_ERR_INVALID and "2^31" in L.last_error()
    assert L.lib().pdm_qk_norm_rope_bwd_workspace_size(ctypes.byref(d)) == L.PDM_ERR_INVALID


def test_module_that_was_made_without_memory(pdm):
    """The tables are in no state dict: they are there once the module has memory, whatever that held."""
    want = pdm.rotary_tables(10, 32)
    for dtype in (torch.float32, torch.bfloat16):
        with torch.device("meta"):
            m = pdm.QKNormRope(64, 10, rotary_dim=32)
        m = m.to(dtype).to_empty(device="cpu")
        assert m.cos.device.type == "cpu" and torch.equal(m.cos, want[0]) and torch.equal(m.sin, want[1])
        m.load_state_dict(pdm.QKNormRope(64, 10, rotary_dim=32).state_dict())
        assert m.q_norm.weight.dtype == dtype and torch.equal(m.to(torch.float64).cos, want[0])


@pytest.mark.parametrize("mode", ["real", "fake"])
def test_arguments_that_a_recorded_graph_would_lose(pdm, mode):
    """A given output and the flag of qk_norm_rope are not arguments of the registered operators: a graph that is being recorded
    refuses them, where it would come out without the call."""
    from torch.fx.experimental.proxy_tensor import make_fx

    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), **_cache(), **_batch())
    out, r = torch.zeros(3, 4, 64, dtype=torch.bfloat16), _rope()
    flag = torch.zeros(1, dtype=torch.int32)

    def attend(q, out):
        return pdm.kv_attention(**{**a, "q": q}, out=out)

    def turn(q, flag):
        return pdm.qk_norm_rope(**{**r, "q": q}, err_flag=flag)

    with pytest.raises(ValueError, match="traced graph"):
        make_fx(attend, tracing_mode=mode)(a["q"], out)
    with pytest.raises(ValueError, match="traced graph"):
        make_fx(turn, tracing_mode=mode)(r["q"], flag)

"""jagged_attention, bucket_bias and what belongs to them refuse what they cannot take, before anything touches a GPU; the
bucket maps; the C entries' checks."""
import ctypes

import pytest
import torch

B, I = torch.bfloat16, torch.int32
CU = torch.tensor([0, 3, 8], dtype=I)


def _qkv(T=8, hq=4, hk=2, D=64, dtype=B):
    return torch.zeros(T, hq, D, dtype=dtype), torch.zeros(T, hk, D, dtype=dtype), torch.zeros(T, hk, D, dtype=dtype)


def _refuses(pdm, error, match, q=None, k=None, v=None, cu=CU, cu_k=None, **kw):
    a, b, c = _qkv()
    with pytest.raises(error, match=match):
        pdm.jagged_attention(a if q is None else q, b if k is None else k, c if v is None else v, cu, cu_k, **kw)


def test_tensors_on_the_cpu(pdm):
    _refuses(pdm, RuntimeError, "GPU only")
    with pytest.raises(RuntimeError, match="GPU only"):
        pdm.bucket_bias(torch.zeros(2, 3), torch.zeros(4, dtype=I))


@pytest.fixture
def as_gpu(pdm, monkeypatch):
    """The checks behind the one of the device."""
    monkeypatch.setattr(pdm.ops, "_gpu_index", lambda *t: 0)


def test_arguments(pdm, as_gpu):
    f = lambda *a, **kw: _refuses(pdm, *a, **kw)  # noqa: E731
    f(TypeError, "float16 or bfloat16", *[t.float() for t in _qkv()])
    f(TypeError, "one dtype", k=_qkv()[1].half(), v=_qkv()[1].half())
    f(TypeError, "one dtype", v=_qkv()[1].half())
    f(ValueError, "head_dim must be 64 or 128", *_qkv(D=96))
    f(ValueError, "head_dim must be 64 or 128", *_qkv(D=256))
    f(ValueError, "the same for q, k and v", k=_qkv(D=128)[1], v=_qkv(D=128)[2])
    f(ValueError, "multiple of the key heads", *_qkv(hq=3))
    f(ValueError, "v must be", v=_qkv(T=7)[2])
    f(ValueError, "expected", q=torch.zeros(8, 64, dtype=B))
    f(TypeError, "int32", cu=CU.long())
    f(ValueError, "sequences \\+ 1", cu=torch.zeros(2, 2, dtype=I))
    f(ValueError, "sequences \\+ 1", cu=torch.zeros(0, dtype=I))
    f(ValueError, "as many entries", cu_k=torch.zeros(2, dtype=I))
    f(ValueError, "window", window=-1)
    f(ValueError, "window", window=2 ** 31)
    f(ValueError, "sinks", sinks=-1)
    f(ValueError, "scale", scale=float("inf"))
    f(ValueError, "scale", scale=float("nan"))
    f(ValueError, "bias must be", bias=torch.zeros(3, 5))
    f(ValueError, "bias must be", bias=torch.zeros(4))
    f(ValueError, "1 to 2\\^30 columns", bias=torch.zeros(4, 0))
    f(TypeError, "bias must be float32", bias=torch.zeros(4, 5, dtype=torch.float16))
    f(ValueError, "bias_start", bias=torch.zeros(4, 5), bias_start=2 ** 30)
    f(ValueError, "err_flag", err_flag=torch.zeros(1))


def test_sinks_of_a_backward_pass(pdm, as_gpu):
    q, k, v = (t.requires_grad_() for t in _qkv(T=1030))
    with pytest.raises(ValueError, match="1024 sinks"):
        pdm.jagged_attention(q, k, v, CU, window=5, sinks=1025)


def test_gradients_that_do_not_fit(pdm, as_gpu):
    q, k, v = _qkv()
    out, stats = torch.zeros_like(q), torch.zeros(8, 4, 2)
    back = lambda go, gl=None: pdm.ops.jagged_attention_backward_raw(q, k, v, CU, CU, None, out, stats, None, go, gl, 0.125,  # noqa: E731
                                                                     True, 0, 0, 0)
    with pytest.raises(ValueError, match="grad_out"):
        back(out.half())
    with pytest.raises(ValueError, match="grad_out"):
        back(out[:5])
    with pytest.raises(ValueError, match="grad_lse"):
        back(out, torch.zeros(8, 3))


def test_bucket_bias_arguments(pdm, as_gpu):
    t, m = torch.zeros(3, 2), torch.zeros(5, dtype=I)
    for error, match, table, maps in ((TypeError, "table must be float32", t.double(), m), (ValueError, "table must be", t[0], m),
                                      (ValueError, "table must be", torch.zeros(8193, 1), m), (TypeError, "int32", t, m.long()),
                                      (ValueError, "table must be", torch.zeros(0, 1), m), (ValueError, "buckets must be", t, m[:0]),
                                      (ValueError, "buckets must be", t, m.view(1, 5))):
        with pytest.raises(error, match=match):
            pdm.bucket_bias(table, maps)
    with pytest.raises(ValueError, match="grad_out"):
        pdm.ops.bucket_bias_backward_raw(torch.zeros(2, 4), m, 3, torch.float32)


def test_no_forward_mode(pdm):
    q, k, v = _qkv()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(RuntimeError, match="forward-mode"):
            pdm.jagged_attention(dual, k, v, CU)


def test_traced_without_a_gpu(pdm):
    """Shapes under fake tensors, forward and backward."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q, k, v = (torch.empty(8, n, 64, dtype=B, requires_grad=True) for n in (4, 2, 2))
        table = torch.empty(3, 4, requires_grad=True)
        cu = torch.empty(3, dtype=I)
        bias = pdm.bucket_bias(table, torch.empty(9, dtype=I))
        out, lse = pdm.jagged_attention(q, k, v, cu, bias=bias, return_lse=True)
        assert bias.shape == (4, 9) and out.shape == q.shape and lse.shape == (8, 4) and lse.dtype == torch.float32
        grads = torch.autograd.grad(out, [q, k, v, table], torch.empty_like(out))
        assert [g.shape for g in grads] == [q.shape, k.shape, v.shape, table.shape]
        with pytest.raises(ValueError, match="err_flag"):
            pdm.jagged_attention(q, k, v, cu, err_flag=torch.empty(1, dtype=I))


def test_bucket_maps(pdm):
    f = pdm.relative_buckets
    assert f(4, 3).tolist() == [0, 1, 2, 3] and f(8, 3).tolist() == [0, 1, 2, 3] and f(1, 5).tolist() == [0] * 6
    one = f(32, 128).tolist()
    assert one[:17] == list(range(17)) and one[-1] == 31 and one == sorted(one) and len(one) == 129 and len(set(one)) == 32
    two = f(32, 128, both_sides=True).tolist()
    assert len(two) == 257 and two[128:] == f(16, 128).tolist() and min(two[:128]) == 16 and max(two) == 31
    assert two[127] == 16 and two[:128] == sorted(two[:128], reverse=True)
    for bad in ((0, 5), (3, -1)):
        with pytest.raises(ValueError):
            f(*bad)
    with pytest.raises(ValueError):
        f(1, 5, both_sides=True)


def test_module_on_the_meta_device(pdm):
    rel = pdm.RelativeBias(3, 16, 50, device="meta")
    rel.to_empty(device="cpu")
    assert torch.equal(rel.buckets, pdm.relative_buckets(16, 50))


def test_c_entries(pdm):
    L = pdm._lib
    lib = L.lib()
    assert ctypes.sizeof(L.JaggedAttentionDesc) == 12 * 4 + 8 * 8

    def desc(**kw):
        base = dict(dtype=L.PDM_BF16, n_q_heads=4, n_kv_heads=2, head_dim=64, num_seqs=2, causal=1, scale=0.125, q_tokens=8,
                    k_tokens=8, q_stride_t=256, q_stride_h=64, k_stride_t=128, k_stride_h=64, v_stride_t=128, v_stride_h=64)
        d = L.JaggedAttentionDesc()
        for n, x in {**base, **kw}.items():
            setattr(d, n, x)
        return ctypes.byref(d)

    size = lib.pdm_jagged_attention_bwd_workspace_size
    assert size(desc(), 0) > 0 and lib.pdm_jagged_attention_workspace_size(desc()) >= 0
    for kw, text in ((dict(dtype=L.PDM_F32), "dtype"), (dict(head_dim=256), "head_dim"), (dict(n_q_heads=3), "multiple"),
                     (dict(n_kv_heads=0), "multiple"), (dict(num_seqs=-1), "num_seqs"), (dict(q_tokens=-1), "tokens"),
                     (dict(k_tokens=1 << 30), "tokens"), (dict(q_tokens=1 << 29, n_q_heads=64), "2^31"), (dict(window=-1), "window"),
                     (dict(sinks=-1), "window"), (dict(scale=float("nan")), "scale"), (dict(bias_span=-1), "bias_span"),
                     (dict(k_stride_t=1 << 24), "strides"), (dict(bias_start=1 << 30), "bias_start"), (dict(n_q_heads=65536 * 2), "65535")):
        assert lib.pdm_jagged_attention_workspace_size(desc(**kw)) == L.PDM_ERR_INVALID and text in L.last_error(), kw
        assert size(desc(**kw), 0) == L.PDM_ERR_INVALID
    sinks = dict(k_tokens=5000, window=10, sinks=1025)
    assert lib.pdm_jagged_attention_workspace_size(desc(**sinks)) == 0 and size(desc(**sinks), 0) == L.PDM_ERR_INVALID
    assert "1024 sinks" in L.last_error() and size(desc(**{**sinks, "window": 5000}), 0) > 0
    assert size(desc(scale=3e38), 0) == L.PDM_ERR_INVALID and "scale" in L.last_error()
    assert size(desc(), 1) == L.PDM_ERR_INVALID and "without a bias" in L.last_error()
    assert size(None, 0) == L.PDM_ERR_INVALID and "null" in L.last_error()
    fwd, bwd = lib.pdm_jagged_attention_fwd, lib.pdm_jagged_attention_bwd
    p = 1 << 20  # never read: every call below is refused
    assert fwd(desc(), None, p, p, p, p, None, p, None, None, None, None, 0, None, None) == L.PDM_ERR_INVALID
    assert fwd(desc(), p, p, p, p, None, None, p, None, None, None, None, 0, None, None) == L.PDM_ERR_INVALID
    assert fwd(desc(), p + 2, p, p, p, p, None, p, None, None, None, None, 0, None, None) == L.PDM_ERR_INVALID and "aligned" in L.last_error()
    assert fwd(desc(q_stride_h=68), p, p, p, p, p, None, p, None, None, None, None, 0, None, None) == L.PDM_ERR_INVALID
    assert fwd(desc(), p, p, p, p, p, p, p, None, None, None, None, 0, None, None) == L.PDM_ERR_INVALID and "together" in L.last_error()
    assert fwd(desc(), p, p, p, p, p, None, p, p, None, None, None, 0, None, None) == L.PDM_ERR_INVALID and "out_rest" in L.last_error()
    assert fwd(desc(), p, p, p, p, p, None, p + 4, None, None, None, None, 0, None, None) == L.PDM_ERR_INVALID
    assert bwd(desc(), p, p, p, p, p, None, p, None, p, p, None, p, p, p, None, None, 0, None) == L.PDM_ERR_WORKSPACE
    assert bwd(desc(), p, p, p, p, p, None, p, None, p, p, None, p, p, p, p, p, 1 << 30, None) == L.PDM_ERR_INVALID
    assert bwd(desc(), p, p, p, p, p, None, p, None, p, p, None, p, p, p, None, p + 8, 1 << 30, None) == L.PDM_ERR_INVALID
    f, g = lib.pdm_bucket_bias_fwd, lib.pdm_bucket_bias_bwd
    assert f(p, 9, 4, 2, p, 5, p, None) == L.PDM_ERR_INVALID and f(p, 0, 8193, 2, p, 5, p, None) == L.PDM_ERR_INVALID
    assert f(None, 0, 4, 2, p, 5, p, None) == L.PDM_ERR_INVALID and f(p, 0, 4, 2, p, 0, p, None) == L.PDM_ERR_INVALID
    assert g(p, p, 5, 4, 2, 0, p, p, 31, None) == L.PDM_ERR_WORKSPACE and g(p, p, 5, 4, 70000, 0, p, p, 32, None) == L.PDM_ERR_INVALID

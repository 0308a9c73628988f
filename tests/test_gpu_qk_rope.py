"""qk_norm_rope against its definition in 64 bits: outputs and gradients, every dtype, head width, pairing, part of a
head rotated, stride and alignment; padding and out-of-table positions; graphs, streams, the compiled op.

Tolerances, with u = 2^-24 (half a step of fp32): the sum of D squares is a chain of 16 FMAs and at most 6 tree sums,
then a division, an addition, a square root and a division: 24 u on the sum of squares, 14 u on r; x r w adds 2 u and
the rotation 2 u, so an output is off by at most 24 u (|n1| + |n2|) before its rounding, half a step of its type.
A gradient r (h - x m) adds the mean of h x (24 u of the mean of |h x|) and three products: 48 u of the sum of the
magnitudes.  A weight's gradient is a sum of N terms of 24 u each in some order: (24 + N) u sum |terms|."""
import pytest
import torch

from oracle import cached_attention as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def _near(got, want, slack, dtype):
    got = got.double().cpu()
    bad = (got - want).abs() - (slack + STEP[dtype] * (want.abs() + slack) + TINY[dtype])
    assert bad.max().item() <= 0 if bad.numel() else True, f"over by {bad.max().item():.3e}"


def _case(dev, T, hq, hk, D, R, dtype, norm, seed=0, max_pos=97, positions=None, bits=torch.int64):
    g = torch.Generator().manual_seed(seed)
    rows = (torch.randn(T, (hq + 2 * hk) * D, generator=g) * 1.7).to(dtype)
    q, k = rows[:, :hq * D].view(T, hq, D), rows[:, hq * D:(hq + hk) * D].view(T, hk, D)
    pos = torch.randint(0, max_pos, (T,), generator=g).to(bits) if positions is None else positions
    ang = torch.rand(max_pos, R // 2, generator=g, dtype=torch.float64) * 50
    cos, sin = (ang.cos().float(), ang.sin().float()) if R else (None, None)
    w = [1 + 0.3 * torch.randn(D, generator=g) for _ in range(2)] if norm else [None, None]
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    drows = rows.to(dev)
    dq, dk = drows[:, :hq * D].view(T, hq, D), drows[:, hq * D:(hq + hk) * D].view(T, hk, D)
    return (q, k, pos, cos, sin, *w), (dq, dk, pos.to(dev), to(cos), to(sin), to(w[0]), to(w[1]))


def _slack(x, w, pos, cos, sin, eps, inter):
    """24 u (|n1| + |n2|) of each output."""
    n = ref.norm_rope(x, w, torch.zeros_like(pos), None, None, eps, inter).abs()
    if cos is None:
        return 24 * U * n
    mixed = n.clone()
    R = 2 * cos.shape[1]
    ia = torch.arange(0, R, 2) if inter else torch.arange(R // 2)
    ib = ia + 1 if inter else ia + R // 2
    mixed[..., ia] = n[..., ia] + n[..., ib]
    mixed[..., ib] = mixed[..., ia]
    return 24 * U * mixed


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,R", [(64, 64), (128, 128), (128, 64), (128, 0), (256, 256), (16, 16), (80, 48), (96, 96),
                                 (192, 64), (1024, 512)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norm", [True, False])
def test_forward(pdm, dev, dtype, D, R, inter, norm):
    for T, hq, hk in ((1, 1, 1), (7, 6, 6), (33, 8, 2), (130, 7, 1)):
        host, args = _case(dev, T, hq, hk, D, R, dtype, norm, seed=D + T)
        yq, yk = pdm.qk_norm_rope(*args, eps=1e-5, interleaved=inter)
        q, k, pos, cos, sin, qw, kw = host
        for y, x, w in ((yq, q, qw), (yk, k, kw)):
            assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
            _near(y, ref.norm_rope(x, w, pos, cos, sin, 1e-5, inter), _slack(x, w, pos, cos, sin, 1e-5, inter), dtype)


def _formula_grads(x, w, pos, cos, sin, eps, inter, g):
    x = x.double().requires_grad_(True)
    w = None if w is None else w.double().requires_grad_(True)
    y = ref.norm_rope(x, w, pos, cos, sin, eps, inter)
    grads = torch.autograd.grad(y, [x] if w is None else [x, w], g.double())
    return grads


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,R,inter", [(64, 64, False), (128, 128, False), (128, 64, True), (96, 32, False), (256, 256, True),
                                       (128, 0, False)])
@pytest.mark.parametrize("norm", [True, False])
def test_gradients(pdm, dev, dtype, D, R, inter, norm):
    eps = 1e-5
    for T, hq, hk in ((1, 1, 1), (45, 6, 2), (259, 4, 4)):
        host, args = _case(dev, T, hq, hk, D, R, dtype, norm, seed=D + T)
        q, k, pos, cos, sin, qw, kw = host
        gen = torch.Generator().manual_seed(5)
        gq, gk = (torch.randn(x.shape, generator=gen).to(dtype) for x in (q, k))
        leaves = [t.detach().requires_grad_(True) for t in (args[0], args[1], args[5], args[6]) if t is not None]
        ins = list(args)
        ins[0], ins[1] = leaves[:2]
        if norm:
            ins[5], ins[6] = leaves[2:]
        out = pdm.qk_norm_rope(*ins, eps=eps, interleaved=inter)
        got = torch.autograd.grad(out, leaves, (gq.to(dev), gk.to(dev)))
        for i, (x, w, g) in enumerate(((q, qw, gq), (k, kw, gk))):
            want = _formula_grads(x, w, pos, cos, sin, eps, inter, g)
            gabs = _slack(g, None, pos, cos, sin, eps, inter) / (24 * U)
            if norm:
                x64 = x.double()
                r = 1 / (x64.square().mean(-1, keepdim=True) + eps).sqrt()
                h = gabs * w.double().abs()
                slack = 48 * U * (r * h + x64.abs() * r ** 3 * (h * x64.abs()).mean(-1, keepdim=True))
                terms = (gabs * (x64 * r).abs()).sum((0, 1))
                dw = got[2 + i].double().cpu()
                assert ((dw - want[1]).abs() <= (24 + T * x.shape[1]) * U * terms + 1e-30).all()
            else:
                slack = 48 * U * gabs
            _near(got[i], want[0], slack, dtype)


def test_gradients_against_differences(pdm, dev):
    """fp32, central differences of the forward pass itself: (f(x + e) - f(x - e)) / 2e, f a random weighting of the
    outputs.  Outputs that do not depend on the moved element are the same bits on both sides; the at most 64 that do
    are off by 24 u (|n1| + |n2|) each, 64 * 24 u * 6 = 5.5e-4 in f with weights and values of order one, over 2e = 2^-5
    1.8e-2.  The curvature adds e^2 / 6 = 4e-5 times a third derivative of order |gradient| / |x|^2."""
    host, args = _case(dev, 5, 2, 1, 64, 64, torch.float32, True, seed=3)
    gen = torch.Generator().manual_seed(8)
    gq, gk = torch.randn(5, 2, 64, generator=gen).to(dev), torch.randn(5, 1, 64, generator=gen).to(dev)
    leaves = [args[i].detach().clone().requires_grad_(True) for i in (0, 1, 5, 6)]

    def f(q, k, qw, kw):
        yq, yk = pdm.qk_norm_rope(q, k, *args[2:5], qw, kw)
        return (yq.double() * gq.double()).sum() + (yk.double() * gk.double()).sum()

    grads = torch.autograd.grad(f(*leaves), leaves)
    e = 2.0 ** -6
    with torch.no_grad():
        for i, leaf in enumerate(leaves):
            for _ in range(6):
                at = torch.randint(0, leaf.numel(), (1,), generator=gen).item()
                side = []
                for s in (e, -e):
                    moved = [t.clone() for t in leaves]
                    moved[i].view(-1)[at] += s
                    side.append(f(*moved).item())
                got = grads[i].reshape(-1)[at].item()
                assert abs((side[0] - side[1]) / (2 * e) - got) <= 2e-2 + 2e-3 * abs(got)


@pytest.mark.parametrize("bits", [torch.int32, torch.int64])
def test_padding_and_positions_beyond_the_tables(pdm, dev, bits):
    pos = torch.tensor([3, -1, 96, 97, -(2 ** 31), 2 ** 31 - 1, 0], dtype=bits)
    host, args = _case(dev, 7, 3, 2, 64, 64, torch.bfloat16, True, positions=pos)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    rows = args[0]._base
    rows[[1, 3, 4, 5]] = float("nan")  # padding rows may hold anything
    leaves = [args[i].detach().requires_grad_(True) for i in (0, 1, 5, 6)]
    yq, yk = pdm.qk_norm_rope(*leaves[:2], *args[2:5], *leaves[2:], err_flag=err)
    assert err.item() == 1
    grads = torch.autograd.grad((yq.float().sum() + yk.float().sum()), leaves)
    for t in (yq, yk, *grads[:2]):
        assert (t[[1, 3, 4, 5]] == 0).all() and torch.isfinite(t).all() and (t[[0, 2, 6]] != 0).any()
    assert torch.isfinite(grads[2]).all() and torch.isfinite(grads[3]).all()
    # padding alone is no error
    err.zero_()
    with torch.no_grad():
        pdm.qk_norm_rope(args[0], args[1], torch.full_like(args[2], -5), *args[3:], err_flag=err)
    assert err.item() == 0


def test_strides_alignment_and_shapes(pdm, dev):
    """Unaligned bases, token-major and head-major strides, 4-d inputs, broadcast rows and gradients: the same bits as the
    contiguous call."""
    host, args = _case(dev, 12, 4, 4, 64, 64, torch.bfloat16, True)
    q, k = args[0].contiguous(), args[1].contiguous()
    want = pdm.qk_norm_rope(q, k, *args[2:])
    flat = torch.zeros(q.numel() + 3, dtype=q.dtype, device=dev)
    odd = flat[3:].view(q.shape).copy_(q)
    assert odd.data_ptr() % 16
    head_major = k.transpose(0, 1).contiguous().transpose(0, 1)
    got = pdm.qk_norm_rope(odd, head_major, *args[2:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = pdm.qk_norm_rope(q.view(3, 4, 4, 64), k.view(3, 4, 4, 64), args[2].view(3, 4), *args[3:])
    assert got[0].shape == (3, 4, 4, 64) and all(torch.equal(a.flatten(0, 1), b) for a, b in zip(got, want))
    got = pdm.qk_norm_rope(q, None, *args[2:5], args[5])
    assert got[1] is None and torch.equal(got[0], want[0])
    # elements of a head with a stride: copied
    wide = torch.empty(12, 4, 128, dtype=q.dtype, device=dev)
    wide[..., ::2] = q
    assert torch.equal(pdm.qk_norm_rope(wide[..., ::2], k, *args[2:])[0], want[0])
    # one head expanded to all, an expanded gradient
    one = q[:, :1].detach().clone().requires_grad_(True)
    y, _ = pdm.qk_norm_rope(one.expand(12, 4, 64), None, *args[2:5], args[5])
    y.sum().backward()
    ref1 = q[:, :1].detach().clone().requires_grad_(True)
    y1, _ = pdm.qk_norm_rope(ref1, None, *args[2:5], args[5])
    y1.sum().backward()
    assert torch.allclose(one.grad.float(), 4 * ref1.grad.float(), rtol=2 ** -6, atol=1e-3)


def test_empty_and_only_one_output_used(pdm, dev):
    host, args = _case(dev, 6, 2, 2, 64, 64, torch.bfloat16, True)
    yq, yk = pdm.qk_norm_rope(args[0][:0], args[1][:0], args[2][:0], *args[3:])
    assert yq.shape == (0, 2, 64) and yk.shape == (0, 2, 64)
    leaves = [args[i].detach().requires_grad_(True) for i in (0, 1, 5, 6)]
    e = [leaves[0][:0], leaves[1][:0]]
    grads = torch.autograd.grad(sum(y.sum() for y in pdm.qk_norm_rope(*e, args[2][:0], *args[3:5], *leaves[2:])), leaves)
    assert all((g == 0).all() for g in grads)
    yq, _ = pdm.qk_norm_rope(leaves[0], leaves[1], *args[2:5], *leaves[2:])
    grads = torch.autograd.grad(yq.sum(), leaves, allow_unused=True)
    assert (grads[1] == 0).all() and (grads[3] == 0).all() and (grads[0] != 0).any()


def test_weights_of_the_inputs_type_and_module(pdm, dev):
    m = pdm.QKNormRope(64, 97, rotary_dim=32, device=dev)
    with torch.no_grad():
        m.q_norm.weight.uniform_(0.5, 1.5)
        m.k_norm.weight.uniform_(0.5, 1.5)
    host, args = _case(dev, 9, 4, 2, 64, 32, torch.bfloat16, True)
    want = pdm.qk_norm_rope(*args[:3], m.cos, m.sin, m.q_norm.weight, m.k_norm.weight)
    got = m(*args[:3])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got[0].sum().backward()
    assert m.q_norm.weight.grad is not None and m.k_norm.weight.grad is not None
    m.bfloat16()
    assert m.cos.dtype == torch.float32 and m.q_norm.weight.dtype == torch.bfloat16
    m.zero_grad(set_to_none=True)
    y, _ = m(*args[:3])
    y.sum().backward()
    assert m.q_norm.weight.grad.dtype == torch.bfloat16
    c, s = pdm.rotary_tables(200_000, 8, device=dev)
    far = 199_999 * 10000.0 ** (-torch.arange(4, dtype=torch.float64) / 4)
    assert (c[-1].cpu().double() - far.cos()).abs().max() < 1e-6 and (s[-1].cpu().double() - far.sin()).abs().max() < 1e-6


def test_repeated_runs_are_equal_and_other_streams(pdm, dev):
    host, args = _case(dev, 5000, 6, 6, 64, 64, torch.bfloat16, True)
    leaves = [args[i].detach().requires_grad_(True) for i in (0, 1, 5, 6)]

    def step():
        y = pdm.qk_norm_rope(*leaves[:2], *args[2:5], *leaves[2:])
        return (*y, *torch.autograd.grad((y[0].float().square().sum() + y[1].float().sum()), leaves))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_graph_replays(pdm, dev):
    """Forward and backward captured; replays with new inputs in the same tensors, eager work between them."""
    host, args = _case(dev, 300, 6, 2, 128, 128, torch.bfloat16, True)
    leaves = [args[i].detach().clone().requires_grad_(True) for i in (0, 1, 5, 6)]
    gq = torch.randn(300, 6, 128, device=dev).to(torch.bfloat16)
    gk = torch.randn(300, 2, 128, device=dev).to(torch.bfloat16)

    def step():
        y = pdm.qk_norm_rope(*leaves[:2], *args[2:5], *leaves[2:])
        return (*(t.detach() for t in y), *torch.autograd.grad(y, leaves, (gq, gk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            for t in (leaves[0], leaves[1], gq, gk):
                t.copy_(torch.randn_like(t))
            args[2].copy_(torch.randint(0, 97, (300,), device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), i


def test_compiled(pdm, dev):
    host, args = _case(dev, 20, 4, 2, 64, 64, torch.bfloat16, True)
    leaves = [args[i].detach().clone().requires_grad_(True) for i in (0, 1, 5, 6)]

    def f(q, k, qw, kw):
        yq, yk = pdm.qk_norm_rope(q, k, *args[2:5], qw, kw)
        return yq.float().square().sum() + yk.float().sum()

    want = torch.autograd.grad(f(*leaves), leaves)
    got = torch.autograd.grad(torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_beyond_32_bit_offsets(pdm, dev):
    """The last rows of q lie more than 2^32 bytes behind its first."""
    T, stride = 9, 300_000_000
    base = torch.empty(8 * stride + 128, dtype=torch.bfloat16, device=dev)
    q = base.as_strided((T, 2, 64), (stride, 64, 1))
    host, args = _case(dev, T, 2, 2, 64, 64, torch.bfloat16, True)
    q.copy_(args[0])
    got, _ = pdm.qk_norm_rope(q, None, *args[2:5], args[5])
    want, _ = pdm.qk_norm_rope(args[0], None, *args[2:5], args[5])
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_weight_gradients_without_tokens(pdm, dev, dtype, D):
    """No tokens, with and without k: the weights' gradients are zeros, not what their memory held."""
    w = [torch.ones(D, device=dev, requires_grad=True) for _ in range(2)]
    cos, sin = torch.ones(4, D // 2, device=dev), torch.zeros(4, D // 2, device=dev)
    pos = torch.zeros(0, dtype=torch.int64, device=dev)
    x = torch.zeros(0, 2, D, dtype=dtype, device=dev, requires_grad=True)
    for k, kw in ((None, None), (x, w[1])):
        # the gradients' memory is of this size
        held = [torch.full((D,), float("nan"), device=dev) for _ in range(8)]
        del held
        y = pdm.qk_norm_rope(x, k, pos, cos, sin, w[0], kw)
        grads = torch.autograd.grad(sum(t.sum() for t in y if t is not None), [w[0]] if kw is None else w)
        assert all((g == 0).all() for g in grads)

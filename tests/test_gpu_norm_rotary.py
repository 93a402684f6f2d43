"""qk_norm_rotary and its gradients against the definition in 64 bits (tests/_cache_util.py: norm_rotary)."""
import pytest
import torch

import flashmask_b200 as fm
import _cache_util as ref

pytestmark = pytest.mark.gpu


def tables(n_pos, half):
    angle = torch.arange(n_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))[None]
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def problem(B, S, Hq, Hk, d, n, dtype, w_dtype=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, gq, gk = (torch.randn(B, S, h, d, generator=g).to(dtype).cuda() for h in (Hq, Hk, Hq, Hk))
    w = [None, None] if w_dtype is None else [(1 + 0.3 * torch.randn(d, generator=g)).to(w_dtype).cuda() for _ in range(2)]
    cos, sin = tables(100, n)
    pos = torch.randint(0, 100, (B, S), generator=g).cuda()
    return q, k, gq, gk, w, cos, sin, pos


def check(q, k, gq, gk, w, cos, sin, pos, interleaved=False, eps=1e-6):
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (q, k, *w)]
    got = fm.qk_norm_rotary(*leaves, cos, sin, pos, eps=eps, interleaved=interleaved)
    wrt = [t for t in leaves if t is not None]
    grads = list(torch.autograd.grad(got, wrt, [gq, gk]))
    for at in (2, 3):
        if leaves[at] is None:
            grads.insert(at, None)
    half = torch.finfo(q.dtype).eps / 2
    p64 = (torch.arange(q.shape[1], device="cuda").expand(q.shape[:2]) if pos is None else pos.expand(q.shape[:2])).long()
    for i, (x, g) in enumerate(((q, gq), (k, gk))):
        x64 = x.double().requires_grad_(True)
        w64 = None if w[i] is None else w[i].double().requires_grad_(True)
        y = ref.norm_rotary(x64, w64, cos.double(), sin.double(), p64, eps, interleaved)
        # a pair's two products each carry the roundings of r, of x r w and their own: under 8 steps of 2^-24 of either
        mag = ref.norm_rotary(x.double().abs(), None if w64 is None else w64.detach().abs(), cos.double().abs(), -sin.double().abs(), p64, eps, interleaved).abs()
        mag = torch.maximum(mag, ref.norm_rotary(x.double().abs(), None if w64 is None else w64.detach().abs(), cos.double().abs(), sin.double().abs(), p64, eps, interleaved).abs())
        tiny = torch.finfo(q.dtype).tiny * half * 4
        assert ((got[i].double() - y).abs() <= half * y.abs() + 2.0 ** -20 * mag + tiny).all(), (got[i].double() - y).abs().max()
        want = torch.autograd.grad(y, [x64] + ([w64] if w64 is not None else []), g.double())
        r = 1 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + eps)
        # |h| <= |w| (|g_a| + |g_b|), the two terms of dx are each within 2^-20 of their magnitudes
        wmax = 1.0 if w64 is None else float(w64.detach().abs().max())
        h = wmax * g.double().abs().amax(-1, keepdim=True) * 2
        scale = r * (h + (x.double() * r).abs() * h * (x.double() * r).abs().mean(-1, keepdim=True))
        dx = grads[i].double()
        assert ((dx - want[0]).abs() <= half * want[0].abs() + 2.0 ** -20 * scale + tiny).all(), (dx - want[0]).abs().max()
        if w64 is not None:
            dw = grads[2 + i].double()
            total = (2 * g.double().abs().amax(-1, keepdim=True) * (x.double() * r).abs()).sum((0, 1, 2))
            whalf = torch.finfo(w[i].dtype).eps / 2
            # sums of up to B S H terms in fp32, in parts
            assert ((dw - want[1]).abs() <= whalf * want[1].abs() + 2.0 ** -18 * total + 1e-30).all(), (dw - want[1]).abs().max()
    return got, grads


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,Hq,Hk,d,n", [(1, 1, 1, 1, 16, 8), (2, 5, 3, 1, 64, 32), (1, 33, 8, 2, 80, 40), (2, 17, 5, 5, 96, 24), (1, 70, 32, 8, 128, 64),
                                           (3, 9, 4, 4, 128, 0), (1, 20, 3, 2, 192, 96), (1, 12, 6, 1, 256, 64), (1, 7, 2, 2, 512, 256)])
def test_forward_and_gradients(dtype, interleaved, B, S, Hq, Hk, d, n):
    check(*problem(B, S, Hq, Hk, d, n, dtype, dtype, seed=1), interleaved=interleaved)


@pytest.mark.parametrize("w_dtype", [None, torch.float32, torch.bfloat16])
def test_weights(w_dtype):
    q, k, gq, gk, w, cos, sin, pos = problem(2, 40, 8, 2, 128, 64, torch.bfloat16, w_dtype, seed=2)
    check(q, k, gq, gk, w, cos, sin, pos)
    if w_dtype is not None:
        check(q, k, gq, gk, [w[0], None], cos, sin, pos)
        check(q, k, gq, gk, [None, w[1]], cos, sin, pos)


def test_many_tokens_and_positions():
    """More jobs than warps of the grid; int32, int64, shared and no positions; documents that start over."""
    q, k, gq, gk, w, cos, sin, pos = problem(2, 3000, 4, 1, 64, 32, torch.bfloat16, torch.float32, seed=3)
    cos, sin = tables(3000, 32)
    a, _ = check(q, k, gq, gk, w, cos, sin, None)
    b, _ = check(q, k, gq, gk, w, cos, sin, torch.arange(3000, device="cuda"))
    c, _ = check(q, k, gq, gk, w, cos, sin, torch.arange(3000, device="cuda", dtype=torch.int32)[None])
    for x, y in zip(b + c, a + a):
        assert torch.equal(x, y)
    docs = torch.cat([torch.arange(1000), torch.arange(1500), torch.arange(500)]).cuda()
    check(q, k, gq, gk, w, cos, sin, torch.stack([docs, docs.flip(0)]).int())


def test_views_of_a_fused_projection():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 30, 12, 128, generator=g).bfloat16().cuda().requires_grad_(True)
    w = [torch.ones(128, device="cuda").requires_grad_(True) for _ in range(2)]
    cos, sin = tables(30, 64)
    q, k = fm.qk_norm_rotary(x[:, :, :8], x[:, :, 8:10], *w, cos, sin)
    dx, = torch.autograd.grad([q, k], [x], [torch.ones_like(q), torch.ones_like(k)], retain_graph=True)
    q2, k2 = fm.qk_norm_rotary(x[:, :, :8].contiguous(), x[:, :, 8:10].contiguous(), *w, cos, sin)
    dx2, = torch.autograd.grad([q2, k2], [x], [torch.ones_like(q), torch.ones_like(k)])
    assert torch.equal(q, q2) and torch.equal(k, k2) and torch.equal(dx, dx2) and not dx[:, :, 10:].any()
    # a transposed layout, rows that 16-byte vectors cannot read, an expanded key, an expanded gradient
    t = x.detach()[:, :, :8].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(fm.qk_norm_rotary(t, t, *w, cos, sin)[0], q)
    odd = torch.empty(2, 30, 8, 129, dtype=torch.bfloat16, device="cuda")[..., 1:]
    odd.copy_(t)
    assert torch.equal(fm.qk_norm_rotary(odd, odd, *w, cos, sin)[0], q)
    one = x.detach()[:, :, :1].clone().requires_grad_(True)
    ke = one.expand(2, 30, 4, 128)
    q3, k3 = fm.qk_norm_rotary(t, ke, *w, cos, sin)
    assert all(torch.equal(k3[:, :, i], k3[:, :, 0]) for i in range(4))
    k3.sum().backward()
    ref_one = one.detach().clone().requires_grad_(True)
    fm.qk_norm_rotary(t, ref_one, *w, cos, sin)[1].sum().backward()
    assert torch.allclose(one.grad.float(), 4 * ref_one.grad.float(), rtol=2e-2, atol=1e-3)


def test_only_one_output_used_and_some_inputs_frozen():
    q, k, gq, gk, w, cos, sin, pos = problem(1, 10, 4, 2, 64, 32, torch.float16, torch.float32, seed=5)
    ql, wl = q.clone().requires_grad_(True), w[0].clone().requires_grad_(True)
    a, b = fm.qk_norm_rotary(ql, k, wl, w[1], cos, sin, pos)
    dq, dw = torch.autograd.grad(a, [ql, wl], gq)
    full = check(q, k, gq, gk, w, cos, sin, pos)[1]
    assert torch.equal(dq, full[0]) and torch.equal(dw, full[2])
    kl = k.clone().requires_grad_(True)
    _, b = fm.qk_norm_rotary(q, kl, None, None, cos, sin, pos)
    torch.autograd.grad(b, [kl], gk)


def test_gradient_against_differences():
    """Directional derivatives in 64 bits of the definition at the inputs, against the kernel's gradient."""
    q, k, gq, gk, w, cos, sin, pos = problem(1, 6, 3, 2, 32, 16, torch.float16, torch.float32, seed=6)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, *w)]
    out = fm.qk_norm_rotary(*leaves, cos, sin, pos)
    grads = torch.autograd.grad(out, leaves, [gq, gk])
    f = lambda a, b, c, e: sum((ref.norm_rotary(x, ww, cos.double(), sin.double(), pos, 1e-6, False) * gg.double()).sum()
                               for x, ww, gg in ((a, c, gq), (b, e, gk)))
    base = [t.double() for t in (q, k, *w)]
    for i in range(4):
        g = torch.Generator().manual_seed(10 + i)
        v = torch.randn(base[i].shape, generator=g).double().cuda()
        step = 1e-5
        up, down = ([t + s * step * v if j == i else t for j, t in enumerate(base)] for s in (1, -1))
        num = (f(*up) - f(*down)) / (2 * step)
        got = (grads[i].double() * v).sum()
        # every entry of the kernel's gradient is off by at most half a step of its type and 2^-18 of its terms
        tol = (grads[i].double().abs() * v.abs()).sum() * 2.0 ** -11 + 1e-4 * (1 + num.abs())
        assert (num - got).abs() <= tol, (i, num, got)


def test_zero_rows_empty_tensors_and_positions_outside():
    cos, sin = tables(10, 32)
    q = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16, device="cuda").requires_grad_(True)
    a, b = fm.qk_norm_rotary(q, q, None, None, cos, sin)
    assert not a.any() and not b.any()
    (dq,) = torch.autograd.grad(a, q, torch.ones_like(a))
    assert torch.isfinite(dq).all()
    for shape in ((0, 3, 2, 64), (1, 0, 2, 64), (1, 3, 0, 64)):
        z = torch.zeros(shape, dtype=torch.bfloat16, device="cuda").requires_grad_(True)
        w = torch.ones(64, device="cuda").requires_grad_(True)
        a, b = fm.qk_norm_rotary(z, z, w, w, cos, sin)
        assert a.shape == shape
        gz, gw = torch.autograd.grad([a, b], [z, w], [torch.ones_like(a), torch.ones_like(b)])
        assert gz.shape == shape and not gw.any()
    x = torch.randn(1, 4, 2, 64, device="cuda").bfloat16()
    y, _ = fm.qk_norm_rotary(x, x, None, None, cos, sin, torch.tensor([[0, 9, 10, -1]], device="cuda"))
    assert torch.isfinite(y[:, :2]).all() and torch.isnan(y[:, 2:]).all()


def test_bitwise_reproducible_on_streams():
    args = problem(2, 500, 8, 2, 128, 64, torch.bfloat16, torch.bfloat16, seed=7)
    first = check(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = check(*args)
    torch.cuda.synchronize()
    for a, b in zip((*first[0], *first[1]), (*second[0], *second[1])):
        assert torch.equal(a, b)


def test_before_the_attention_of_a_training_step():
    """qk_norm_rotary and flashmask_attention in one graph: gradients reach the projection's output and the weights."""
    g = torch.Generator().manual_seed(8)
    B, S, Hq, Hk, d = 1, 256, 4, 2, 128
    x = torch.randn(B, S, Hq + 2 * Hk, d, generator=g).bfloat16().cuda().requires_grad_(True)
    w = [torch.ones(d, device="cuda").requires_grad_(True) for _ in range(2)]
    cos, sin = tables(S, d // 2)
    q, k = fm.qk_norm_rotary(x[:, :, :Hq], x[:, :, Hq:Hq + Hk], *w, cos, sin)
    out = fm.flashmask_attention(q, k, x[:, :, Hq + Hk:], causal=True)
    go = torch.randn(out.shape, generator=g).bfloat16().cuda()
    got = torch.autograd.grad(out, [x, *w], go)
    x64, w64 = x.detach().double().requires_grad_(True), [t.detach().double().requires_grad_(True) for t in w]
    pos = torch.arange(S, device="cuda")[None]
    q64, k64 = (ref.norm_rotary(t, ww, cos.double(), sin.double(), pos, 1e-6, False) for t, ww in
                ((x64[:, :, :Hq], w64[0]), (x64[:, :, Hq:Hq + Hk], w64[1])))
    k64, v64 = (t.repeat_interleave(Hq // Hk, dim=2) for t in (k64, x64[:, :, Hq + Hk:]))
    s = torch.einsum("bihd,bjhd->bhij", q64, k64) / d ** 0.5
    s = s.masked_fill(torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
    want = torch.autograd.grad(torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v64), [x64, *w64], go.double())
    for a, b in zip(got, want):
        # q, k, p, dS, dq, dk and the results each are rounded to bf16 once: 2^-9 each, in the 2-norm of what they make up
        assert (a.double() - b).norm() <= 8 * 2.0 ** -9 * b.norm(), ((a.double() - b).norm() / b.norm())


def test_forward_and_gradients_replay_from_a_cuda_graph():
    """Replays with new inputs give the bits of eager calls.  (No eager graph of the same leaves may live at the capture: torch ties a
    leaf to the stream of its first graph.)"""
    q, k, gq, gk, w, cos, sin, pos = problem(2, 300, 8, 2, 128, 64, torch.bfloat16, torch.float32, seed=11)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, *w)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = fm.qk_norm_rotary(*leaves, cos, sin, pos)
        torch.autograd.grad(out, leaves, [gq, gk])
        del out
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fm.qk_norm_rotary(*leaves, cos, sin, pos)
        grads = torch.autograd.grad(out, leaves, [gq, gk])
    for seed in (12, 13):
        q2, k2, gq2, gk2, w2, _, _, pos2 = problem(2, 300, 8, 2, 128, 64, torch.bfloat16, torch.float32, seed=seed)
        with torch.no_grad():
            for a, b in zip((*leaves, gq, gk, pos), (q2, k2, *w2, gq2, gk2, pos2)):
                a.copy_(b)
        graph.replay()
        want, wgrads = check(q2, k2, gq2, gk2, w2, cos, sin, pos2)
        for a, b in zip((*out, *grads), (*want, *wgrads)):
            assert torch.equal(a, b)


def test_refusals():
    q, k, _, _, w, cos, sin, pos = problem(1, 4, 4, 2, 64, 32, torch.bfloat16, torch.float32, seed=9)
    ok = lambda q=q, k=k, w=w, cos=cos, sin=sin, pos=pos, **kw: fm.qk_norm_rotary(q, k, *w, cos, sin, pos, **kw)
    ok()
    for bad in (dict(k=k[:, :2]), dict(k=k.half()), dict(cos=cos.half()), dict(sin=sin[:5]), dict(cos=cos.cpu()), dict(w=[w[0][:32], w[1]]),
                dict(w=[w[0], w[1].bfloat16()]), dict(pos=pos.float()), dict(pos=pos[:, :2]), dict(cos=torch.zeros(10, 64).cuda(), sin=torch.zeros(10, 64).cuda())):
        with pytest.raises(AssertionError):
            ok(**bad)
    with pytest.raises(TypeError):
        ok(q=q.float(), k=k.float())
    with pytest.raises(RuntimeError):
        ok(q=q.cpu())
    with pytest.raises(NotImplementedError):
        fm.qk_norm_rotary(q[..., :24], k[..., :24], None, None, cos[:, :8].contiguous(), sin[:, :8].contiguous())
    with pytest.raises(NotImplementedError):
        ok(cos=cos[:, :4].contiguous(), sin=sin[:, :4].contiguous())
    with pytest.raises(ValueError):
        ok(cos=cos[:2], sin=sin[:2], pos=None)
    with pytest.raises(ValueError):
        ok(eps=-1.0)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,n", [(48, 16), (64, 32), (112, 56), (128, 32), (192, 96), (256, 128), (320, 64), (512, 256)])
def test_several_tokens_a_warp(interleaved, d, n):
    """Rows of every number of lanes, full ones and not, and heads that fill no group; what a kernel before left in shared memory
    (here NaN) is no part of a row."""
    full = 64 if d <= 64 else 128 if d <= 128 else 256 if d <= 256 else 512
    bad = problem(1, 700, 9, 3, full, full // 2, torch.bfloat16, torch.float32, seed=7)
    leaves = [torch.full_like(t, float("nan")).requires_grad_(True) for t in bad[:2]]
    torch.autograd.grad(fm.qk_norm_rotary(*leaves, *bad[4], *bad[5:]), leaves, bad[2:4])
    check(*problem(3, 1500, 9, 3, d, n, torch.bfloat16, torch.float32, seed=8), interleaved=interleaved)


def test_no_second_derivative():
    q, k, gq, gk, w, cos, sin, pos = problem(1, 6, 3, 2, 64, 32, torch.bfloat16, torch.float32, seed=9)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, *w)]
    out = fm.qk_norm_rotary(*leaves, cos, sin, pos)
    want = torch.autograd.grad(out, leaves, [gq, gk], retain_graph=True)
    got = torch.autograd.grad(out, leaves, [gq, gk], create_graph=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
        with pytest.raises(NotImplementedError, match="no gradient"):
            a.float().square().sum().backward(retain_graph=True)


def test_tangents_are_refused():
    """The operator has no forward-mode derivative: a dual tensor is refused, under no_grad too, and not taken for a constant."""
    import torch.autograd.forward_ad as ad
    q, k, _, _, w, cos, sin, pos = problem(1, 4, 2, 1, 64, 32, torch.bfloat16, torch.bfloat16, seed=12)
    args = [q, k, *w, cos, sin]
    with ad.dual_level():
        for i in range(6):
            dual = [ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises((RuntimeError, AssertionError)):
                fm.qk_norm_rotary(*dual, pos)
            with torch.no_grad(), pytest.raises((RuntimeError, AssertionError)):
                fm.qk_norm_rotary(*dual, pos)
        fm.qk_norm_rotary(*args, pos)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,n", [(64, 16), (128, 32), (96, 24), (256, 64), (512, 8)])
def test_a_position_outside_takes_the_whole_row(interleaved, d, n):
    """NaN in what does not turn as well, and in the gradients of the same rows; the others keep their bits.  Without a
    rotated part positions say nothing."""
    cos, sin = tables(10, n)
    g = torch.Generator().manual_seed(11)
    x, gy = (torch.randn(1, 5, 3, d, generator=g).bfloat16().cuda() for _ in range(2))
    pos = torch.tensor([[0, 10, 9, -1, 2 ** 40]], device="cuda")
    bad = torch.tensor([False, True, False, True, True], device="cuda")
    runs = []
    for p in (pos, pos.clamp(0, 9)):
        leaf, w = x.clone().requires_grad_(True), torch.ones(d, device="cuda").requires_grad_(True)
        y, _ = fm.qk_norm_rotary(leaf, x, w, None, cos, sin, p, interleaved=interleaved)
        runs.append((y, *torch.autograd.grad(y, [leaf, w], gy)))
    for a, b in zip(runs[0][:2], runs[1][:2]):
        assert torch.isnan(a[:, bad]).all() and torch.equal(a[:, ~bad], b[:, ~bad])
    assert torch.isnan(runs[0][2]).all()
    none = torch.zeros(10, 0, device="cuda")
    y, _ = fm.qk_norm_rotary(x, x, None, None, none, none, pos)
    assert torch.isfinite(y).all()

"""qk_norm_rope and its gradients on the GPU against 64 bits (tolerances: tests/_operators64.py)."""
import pytest
import torch

import tbf16

from _operators64 import norm_rope64

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def tables(dev, n, R):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return a.cos().float().to(dev), a.sin().float().to(dev)


def inputs(dev, B, S, H, Hkv, D, R, wide=False, pad=0, far=300, seed=0):
    """(q, k, wq, wk, cos, sin, pos): q and k views of one projection's output."""
    g = gen(seed + D + H)
    lead = (S,) if B is None else (B, S)
    qkv = torch.randn(*lead, H + 2 * Hkv, D, generator=g) * torch.exp2(torch.randint(-6, 7, (*lead, H + 2 * Hkv, 1), generator=g))
    qkv = qkv.to(BF).to(dev)
    pos = torch.randint(0, far, lead, generator=g, dtype=torch.int32)
    if pad:
        pos.view(-1)[-pad:] = -1
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(torch.float32 if wide else BF).to(dev) for _ in "qk"]
    return (qkv[..., :H, :], qkv[..., H:H + Hkv, :], *w, *tables(dev, far, R), pos.to(dev))


def close(got, want, bound, why):
    assert got.shape == want.shape and torch.isfinite(got).all(), why
    err = (got.cpu().double() - want).abs()
    assert (err <= bound).all(), (why, (err - bound).max())


def check(a, eps=1e-6, near=False, dys=None):
    q, k, wq, wk, cos, sin, pos = a
    pos64 = pos.expand(q.shape[:-2])
    out = tbf16.qk_norm_rope(*a, eps=eps, interleaved=near)
    for y, x, w in ((out[0], q, wq), (out[1], k, wk)):
        assert y.dtype == BF and y.is_contiguous()
        close(y, *norm_rope64(x, w, cos, sin, pos64, eps, near), "y")
    if dys is None:
        return out
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    y = tbf16.autograd.qk_norm_rope(*leaves, cos, sin, pos, eps, near)
    assert torch.equal(y[0], out[0]) and torch.equal(y[1], out[1])
    grads = torch.autograd.grad(y, leaves, dys)
    for x, w, dy, dx, dw in ((q, wq, dys[0], grads[0], grads[2]), (k, wk, dys[1], grads[1], grads[3])):
        _, _, dx64, dx_bound, dw64, dw_bound = norm_rope64(x, w, cos, sin, pos64, eps, near, dy)
        assert dx.dtype == BF and dw.dtype == w.dtype
        close(dx, dx64, dx_bound, "dx")
        if dw.dtype == BF:
            dw_bound = dw_bound * (1 + 2.0 ** -8) + 2.0 ** -8 * dw64.abs()
        close(dw, dw64, dw_bound, "dw")
    return out, grads


SHAPES = [  # B, S, H, Hkv, D, R, near, wide, padding
    (None, 1, 1, 1, 16, 16, False, False, 0),
    (None, 1, 32, 8, 128, 128, False, False, 0),
    (None, 5, 3, 1, 64, 64, True, False, 0),
    (None, 17, 20, 4, 80, 32, True, True, 3),
    (None, 33, 20, 4, 80, 80, False, False, 0),
    (2, 9, 12, 4, 96, 64, False, True, 4),
    (3, 7, 6, 6, 48, 16, False, False, 21),
    (1, 300, 16, 16, 128, 128, False, False, 5),
    (2, 130, 8, 1, 256, 256, False, False, 0),
    (2, 64, 5, 2, 240, 96, True, True, 1),
    (1, 10, 40, 9, 112, 112, True, False, 0),
    (2, 2500, 2, 1, 32, 32, False, False, 9),
    (1, 6001, 4, 2, 128, 64, True, False, 0),
]


@pytest.mark.parametrize("B,S,H,Hkv,D,R,near,wide,pad", SHAPES)
def test_shapes(dev, B, S, H, Hkv, D, R, near, wide, pad):
    a = inputs(dev, B, S, H, Hkv, D, R, wide, pad)
    g = gen(7)
    lead = (S,) if B is None else (B, S)
    dys = [torch.randn(*lead, h, D, generator=g).to(BF).to(dev) for h in (H, Hkv)]
    check(a, near=near, dys=dys)


def test_layouts(dev):
    """Heads outside positions, misaligned or spread rows, positions of one sequence for all, tables and
    weights that are views, gradients as attention leaves them or of a broadcast sum."""
    B, S, H, Hkv, D, R = 2, 37, 4, 2, 64, 32
    q, k, wq, wk, cos, sin, pos = inputs(dev, B, S, H, Hkv, D, R)
    swap = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    odd = torch.empty(B, S, H, D + 1, dtype=BF, device=dev)[..., 1:].copy_(q)
    thin = torch.empty(B, S, Hkv, 2 * D, dtype=BF, device=dev)[..., ::2].copy_(k)
    w2 = torch.empty(D, 2, dtype=BF, device=dev)[:, 0].copy_(wq)
    c2 = torch.empty(cos.shape[0], R, device=dev)[:, ::2].copy_(cos)
    s2 = torch.empty(cos.numel() + 1, device=dev)[1:].view_as(sin).copy_(sin)
    dq = torch.randn(B, H, S, D, generator=gen(1)).to(BF).to(dev).transpose(1, 2)
    dk = torch.ones((), dtype=BF, device=dev).expand(B, S, Hkv, D)
    want = check((q, k, wq, wk, cos, sin, pos), dys=(dq, dk))
    for a in ((swap(q), swap(k), wq, wk, cos, sin, pos), (odd, thin, w2, torch.cat((wk[:1], wk))[1:], c2, s2, pos),
              (q, k, wq, wk, cos, sin, pos.t().contiguous().t())):
        got = check(a, dys=(dq, dk))
        assert all(torch.equal(x, y) for u, v in zip(got, want) for x, y in zip(u, v))
    check((q, k, wq, wk, cos, sin, pos[0]), dys=(dq, dk))
    check((q, k, wq, wk, cos, sin, torch.tensor(5, dtype=torch.int32, device=dev).expand(B, S)), dys=(dq, dk))
    check((q[:0], k[:0], wq, wk, cos, sin, pos[:0]))


def test_leaves_inputs_alone(dev):
    a = inputs(dev, 2, 20, 4, 2, 64, 64, pad=3)
    before = [t.clone() for t in a]
    dys = [torch.ones_like(a[0]), torch.ones_like(a[1])]
    check(a, dys=dys)
    assert all(torch.equal(x, y) for x, y in zip(a, before))


@pytest.mark.parametrize("scale,eps", [(2.0 ** 100, 1e-6), (2.0 ** 62, 1e-6), (2.0 ** -60, 0.0), (2.0 ** -100, 0.0),
                                       (2.0 ** -20, 1e-6), (1.0, 100.0), (2.0 ** -70, 1e-38)])
def test_far_sizes(dev, scale, eps):
    """Squares outside fp32's range, beside heads of ordinary size."""
    q, k, wq, wk, cos, sin, pos = inputs(dev, 1, 9, 8, 4, 128, 64, seed=4)
    q, k = q.clone(), k.clone()
    q[:, ::2] *= scale
    k[:, 1::2] *= scale
    dys = [torch.randn(t.shape, generator=gen(5)).to(dev) * 2.0 ** -10 for t in (q, k)]
    dys = [(d * min(1.0, scale) * 2.0 ** 10).to(BF) if scale < 1 else d.to(BF) for d in dys]
    check((q, k, wq, wk, cos, sin, pos), eps=eps, dys=dys)


def test_values_that_are_none(dev):
    """A head with a NaN or an infinity concerns itself alone; a position past the tables gives NaN;
    a head of zeros without an eps too; padding gives zeros whatever lies there."""
    a = list(inputs(dev, None, 8, 4, 2, 64, 64))
    q = a[0] = a[0].clone()
    clean = tbf16.qk_norm_rope(*a)
    q[1, 2, 5] = float("nan")
    q[3, 1, 7] = float("inf")
    yq, yk = tbf16.qk_norm_rope(*a)
    assert torch.isnan(yq[1, 2]).all() and torch.isnan(yq[3, 1, 7]) and torch.equal(yk, clean[1])
    same = torch.ones(8, 4, dtype=torch.bool)
    same[1, 2] = same[3, 1] = False
    assert torch.equal(yq[same], clean[0][same])
    a[6] = a[6].clone()
    a[6][1] = a[6][3] = -5
    a[6][0] = a[4].shape[0]
    yq, yk = tbf16.qk_norm_rope(*a)
    assert (yq[1] == 0).all() and (yq[3] == 0).all() and (yk[1] == 0).all()
    assert torch.isnan(yq[0]).all() and torch.isnan(yk[0]).all()
    assert torch.equal(yq[4:], clean[0][4:]) and torch.equal(yq[2], clean[0][2])
    a[6][0] = 0
    leaves = [t.detach().requires_grad_() for t in a[:4]]
    grads = torch.autograd.grad(tbf16.autograd.qk_norm_rope(*leaves, *a[4:]), leaves,
                                (torch.ones_like(a[0]), torch.ones_like(a[1])))
    assert all(torch.isfinite(g).all() for g in grads) and (grads[0][1] == 0).all() and (grads[0][3] == 0).all()
    q[4, 0] = 0
    assert torch.isnan(tbf16.qk_norm_rope(*a, eps=0.0)[0][4, 0]).all() and (tbf16.qk_norm_rope(*a)[0][4, 0] == 0).all()


def test_wanted_gradients_only(dev):
    a = inputs(dev, 2, 40, 4, 2, 64, 64)
    dys = (torch.ones_like(a[0]), torch.ones_like(a[1]))
    leaves = [t.detach().requires_grad_() for t in a[:4]]
    want = torch.autograd.grad(tbf16.autograd.qk_norm_rope(*leaves, *a[4:]), leaves, dys)
    for on in range(1, 16):
        some = [t.detach().requires_grad_(bool(on >> i & 1)) for i, t in enumerate(a[:4])]
        y = tbf16.autograd.qk_norm_rope(*some, *a[4:])
        got = torch.autograd.grad(y, [t for t in some if t.requires_grad], dys)
        assert all(torch.equal(x, w) for x, w in zip(got, [w for i, w in enumerate(want) if on >> i & 1]))
    # one output alone
    y = tbf16.autograd.qk_norm_rope(*leaves, *a[4:])
    got = torch.autograd.grad(y[1], leaves, dys[1])
    assert torch.equal(got[1], want[1]) and torch.equal(got[3], want[3]) and not got[0].any() and not got[2].any()


def test_no_tokens_no_gradient(dev):
    a = inputs(dev, 0, 5, 4, 2, 64, 64)
    leaves = [t.detach().requires_grad_() for t in a[:4]]
    got = torch.autograd.grad(tbf16.autograd.qk_norm_rope(*leaves, *a[4:]), leaves, (leaves[0].detach(), leaves[1].detach()))
    assert got[0].shape == a[0].shape and not got[2].any() and not got[3].any()


def test_twice_the_same_and_other_streams(dev):
    a = inputs(dev, 1, 3000, 8, 4, 128, 128)
    dys = (torch.randn(a[0].shape, generator=gen(1)).to(BF).to(dev), torch.randn(a[1].shape, generator=gen(2)).to(BF).to(dev))
    leaves = [t.detach().requires_grad_() for t in a[:4]]

    def step():
        y = tbf16.autograd.qk_norm_rope(*leaves, *a[4:])
        return (*(t.detach() for t in y), *torch.autograd.grad(y, leaves, dys))
    want = step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = step()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(step(), want)) and all(torch.equal(x, y) for x, y in zip(other, want))


def test_graph(dev):
    """Forward and backward captured once, replayed on other inputs."""
    a = inputs(dev, 2, 100, 4, 2, 64, 32, pad=2)
    static = [t.clone() for t in a]
    dys = [torch.ones_like(a[0]), torch.ones_like(a[1])]

    def step(x, dys):
        leaves = [t.detach().requires_grad_() for t in x[:4]]
        y = tbf16.autograd.qk_norm_rope(*leaves, *x[4:])
        return (*(t.detach() for t in y), *torch.autograd.grad(y, leaves, dys))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(static, dys)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = step(static, dys)
    for seed in range(3):
        b = inputs(dev, 2, 100, 4, 2, 64, 32, pad=seed, seed=seed)
        for x, y in zip(static, b):
            x.copy_(y)
        g.replay()
        want = step(b, dys)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_no_second_derivatives(dev):
    """create_graph gives the same gradients; differentiating them raises."""
    a = inputs(dev, 1, 9, 4, 2, 64, 32)
    leaves = [t.detach().requires_grad_() for t in a[:4]]
    dys = (torch.ones_like(a[0]), torch.ones_like(a[1]))
    want = torch.autograd.grad(tbf16.autograd.qk_norm_rope(*leaves, *a[4:]), leaves, dys)
    got = torch.autograd.grad(tbf16.autograd.qk_norm_rope(*leaves, *a[4:]), leaves, dys, create_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    with pytest.raises(RuntimeError):
        got[0].sum().backward()


def test_saved_tensors_moved_by_hooks(dev):
    """Saved inputs that come back from the host in another layout."""
    a = inputs(dev, 2, 30, 4, 2, 64, 32)
    dys = (torch.ones_like(a[0]), torch.ones_like(a[1]))
    leaves = [t.detach().requires_grad_() for t in a[:4]]
    want = torch.autograd.grad(tbf16.autograd.qk_norm_rope(*leaves, *a[4:]), leaves, dys)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(dev)):
        y = tbf16.autograd.qk_norm_rope(*leaves, *a[4:])
    got = torch.autograd.grad(y, leaves, dys)
    assert all(torch.equal(x, w) for x, w in zip(got, want))

"""Norm and rotation of query / key heads against the formula in 64 bits.

Tolerances: u = eps / 2 of the output's type (one rounding of the result), and
for the fp32 arithmetic before it at most 16 roundings a component: 2^-19 of
the pair's magnitude.  dw is a sum of fp32 products; with the sizes here a
chain is below 64 additions of terms good to 2^-19: 2^-17 of sum |t n|.
"""

import pytest
import torch

from blocksparsefa_reorder_b200 import qk_norm_rope, qk_norm_rope_autograd, qk_norm_rope_backward, rope_table

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _u(t):
    return torch.finfo(t).eps / 2


def _turn(y, c, s, R, il):
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if il else (y[..., :R // 2], y[..., R // 2:R])
    y0, y1 = a * c - b * s, a * s + b * c
    t = torch.stack((y0, y1), -1).flatten(-2) if il else torch.cat((y0, y1), -1)
    return torch.cat((t, y[..., R:]), -1)


def _tables(pos, cos, sin, N):
    at = torch.arange(N, device="cuda") if pos is None else pos.long()
    c, s = cos.double()[at], sin.double()[at]
    return (c[:, None], s[:, None]) if at.dim() == 2 else (c, s)


def _forward(x, w, pos, cos, sin, eps, il):
    """(y, bound of its fp32 error)"""
    xd = x.double()
    n = xd / (xd.square().mean(-1, keepdim=True) + eps).sqrt()
    y = n * w.double() if w is not None else n
    tol = 2.0 ** -18 * y.abs().amax(-1, keepdim=True)
    if cos is not None:
        c, s = _tables(pos, cos, sin, x.shape[2])
        y = _turn(y, c, s, 2 * cos.shape[1], il)
    return y, tol


def _backward(x, w, dy, pos, cos, sin, eps, il):
    xd, t = x.double(), dy.double()
    if cos is not None:
        c, s = _tables(pos, cos, sin, x.shape[2])
        t = _turn(t, c, -s, 2 * cos.shape[1], il)
    r = (xd.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = xd * r
    u = t * w.double() if w is not None else t
    dx = r * (u - n * (u * n).mean(-1, keepdim=True))
    tol = 2.0 ** -17 * r * (u.abs().amax(-1, keepdim=True) + n.abs() * (u * n).abs().mean(-1, keepdim=True))
    return dx, tol, (t * n).sum((0, 1, 2)), 2.0 ** -17 * (t * n).abs().sum((0, 1, 2))


def _near(got, ref, tol, what):
    bound = _u(got.dtype) * ref.abs() * (1 + 2.0 ** -7) + tol + torch.finfo(got.dtype).tiny
    bad = ((got.double() - ref).abs() > bound).sum().item()
    assert bad == 0, f"{what}: {bad} of {ref.numel()} off, worst {((got.double() - ref).abs() / bound).max().item():.2f}x"


def _inputs(B, H, Hk, N, D, dtype, seed, fused=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if fused:
        x = torch.randn(B, N, (H + 2 * Hk) * D, generator=g, device="cuda").to(dtype)
        q = x[..., :H * D].view(B, N, H, D).transpose(1, 2)
        k = x[..., H * D:(H + Hk) * D].view(B, N, Hk, D).transpose(1, 2)
    else:
        q = torch.randn(B, H, N, D, generator=g, device="cuda").to(dtype)
        k = torch.randn(B, Hk, N, D, generator=g, device="cuda").to(dtype)
    w = [1 + 0.3 * torch.randn(D, generator=g, device="cuda") for _ in range(2)]
    d = [torch.randn(t.shape, generator=g, device="cuda").to(dtype) for t in (q, k)]
    return q, k, *w, *d, g


CASES = [
    # B, H, Hk, N, D, R, il, fused, weights, positions
    (1, 1, 1, 1, 64, 64, False, False, "f32", None),
    (2, 4, 2, 5, 128, 128, False, True, "f32", "BN32"),
    (3, 5, 1, 33, 128, 64, True, False, "same", "N64"),
    (1, 17, 3, 100, 64, 32, False, True, None, "BN64"),
    (2, 3, 2, 9, 96, 96, False, False, "f32", "N32"),
    (2, 2, 2, 7, 96, 48, True, False, "same", "BN32"),
    (1, 8, 1, 300, 256, 256, True, False, "f32", "N32"),
    (2, 2, 1, 11, 256, 128, False, True, "f32", "BN64"),
    (1, 3, 2, 13, 8, 0, False, False, "f32", None),
    (2, 3, 1, 6, 24, 16, False, False, "same", "N32"),
    (1, 2, 2, 21, 16, 16, True, False, "f32", "N64"),
    (4, 33, 9, 3, 32, 32, False, False, "f32", "BN32"),
]


def _case(c, dtype, seed=1):
    B, H, Hk, N, D, R, il, fused, wt, pt = c
    q, k, wq, wk, dq, dk, g = _inputs(B, H, Hk, N, D, dtype, seed, fused)
    wq, wk = (None, None) if wt is None else (wq, wk) if wt == "f32" else (wq.to(dtype), wk.to(dtype))
    cos, sin = rope_table(4096, R, device="cuda") if R else (None, None)
    pos = None
    if pt:
        shape = (B, N) if pt.startswith("BN") else (N,)
        pos = torch.randint(0, 4096, shape, generator=g, device="cuda").to(torch.int32 if pt.endswith("32") else torch.int64)
    return q, k, wq, wk, dq, dk, dict(positions=pos, cos=cos, sin=sin, eps=1e-6, interleaved=il)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("c", CASES)
def test_forward_and_gradient_match_the_formula(c, dtype):
    q, k, wq, wk, dq, dk, kw = _case(c, DT[dtype])
    oq, ok = qk_norm_rope(q, k, wq, wk, check_errors=True, **kw)
    gq, gk, gwq, gwk = qk_norm_rope_backward(dq, dk, q, k, wq, wk, check_errors=True, **kw)
    args = (kw["positions"], kw["cos"], kw["sin"], kw["eps"], kw["interleaved"])
    for x, w, o, dy, gx, gw, name in ((q, wq, oq, dq, gq, gwq, "q"), (k, wk, ok, dk, gk, gwk, "k")):
        ref, tol = _forward(x, w, *args)
        _near(o, ref, tol, f"{name} out")
        dx, tol, dw, wtol = _backward(x, w, dy, *args)
        _near(gx, dx, tol, f"d{name}")
        if w is None:
            assert gw is None
        else:
            assert gw.dtype == w.dtype
            _near(gw, dw, wtol, f"d{name} weight")


def test_gradient_matches_differences():
    """Central differences of the 64-bit formula along random directions."""
    q, k, wq, wk, dq, dk, kw = _case(CASES[1], torch.float32, 3)
    gq, _, gwq, _ = qk_norm_rope_backward(dq, dk, q, k, wq, wk, **kw)
    args = (kw["positions"], kw["cos"], kw["sin"], kw["eps"], kw["interleaved"])
    g = torch.Generator(device="cuda").manual_seed(9)
    h = 1e-5
    for which in ("x", "w"):
        d = torch.randn((q if which == "x" else wq).shape, generator=g, device="cuda", dtype=torch.float64)

        def f(t):
            x, w = (q.double() + t * d, wq) if which == "x" else (q, wq.double() + t * d)
            return (_forward(x, w, *args)[0] * dq.double()).sum()

        diff = (f(h) - f(-h)) / (2 * h)
        got = (d * (gq if which == "x" else gwq).double()).sum()
        # differences: h^2 f''' and 1e-16 |f| / h; kernel: 2^-17 of the sum's terms
        bound = 1e-6 * (1 + diff.abs()) + 2.0 ** -17 * (d * (gq if which == "x" else gwq)).abs().sum()
        assert (diff - got).abs() <= bound, (which, diff.item(), got.item())


def test_one_side_in_place_and_into_a_cache():
    q, k, wq, wk, _, _, kw = _case(CASES[1], torch.bfloat16)
    oq, ok = qk_norm_rope(q, k, wq, wk, **kw)
    only, none = qk_norm_rope(q, None, wq, None, **kw)
    assert none is None and torch.equal(only, oq)
    none, only = qk_norm_rope(None, k, None, wk, **kw)
    assert none is None and torch.equal(only, ok)
    # into rows 3 .. 3 + N of a key cache; the rest of the cache stays
    cache = torch.full((k.shape[0], k.shape[1], 20, k.shape[3]), 7.0, dtype=k.dtype, device="cuda")
    view = cache[:, :, 3:3 + k.shape[2]]
    qk_norm_rope(q, k, wq, wk, out=(torch.empty_like(oq), view), **kw)
    assert torch.equal(view, ok)
    assert (cache[:, :, :3] == 7).all() and (cache[:, :, 3 + k.shape[2]:] == 7).all()
    a, b = q.clone(), k.clone()
    qk_norm_rope(a, b, wq, wk, out=(a, b), **kw)
    assert torch.equal(a, oq) and torch.equal(b, ok)


def test_positions_outside_the_table():
    q, k, wq, wk, dq, dk, kw = _case(CASES[1], torch.float16)
    good = qk_norm_rope(q, k, wq, wk, **kw)
    for bad in (-1, 4096, 2 ** 31 - 1):
        pos = kw["positions"].clone()
        pos[1, 2] = bad
        o = qk_norm_rope(q, k, wq, wk, **{**kw, "positions": pos})
        for x, y in zip(o, good):
            assert x[1, :, 2].isnan().all()
            keep = torch.ones(x.shape[0], x.shape[2], dtype=torch.bool, device="cuda")
            keep[1, 2] = False
            assert torch.equal(x.transpose(1, 2)[keep], y.transpose(1, 2)[keep])
        with pytest.raises(RuntimeError, match="coordinate out of range"):
            qk_norm_rope(q, k, wq, wk, check_errors=True, **{**kw, "positions": pos})
        with pytest.raises(RuntimeError, match="coordinate out of range"):
            qk_norm_rope_backward(dq, dk, q, k, wq, wk, check_errors=True, **{**kw, "positions": pos})


def test_zero_row_and_far_positions():
    """A row of zeros stays zero (eps keeps the norm finite) and its gradient
    finite; positions in the hundreds of thousands keep their angle."""
    cos, sin = rope_table(300000, 64, device="cuda")
    x = torch.zeros(1, 1, 2, 64, device="cuda")
    x[0, 0, 1] = torch.arange(64, device="cuda").float() - 30
    pos = torch.tensor([5, 299999], device="cuda")
    kw = dict(positions=pos, cos=cos, sin=sin, eps=1e-6)
    o, _ = qk_norm_rope(x, None, None, None, **kw)
    assert (o[0, 0, 0] == 0).all()
    ang = 299999.0 * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64, device="cuda") / 64)
    y = x[0, 0, 1].double() / (x[0, 0, 1].double().square().mean() + 1e-6).sqrt()
    ref = torch.cat((y[:32] * ang.cos() - y[32:] * ang.sin(), y[:32] * ang.sin() + y[32:] * ang.cos()))
    assert (o[0, 0, 1].double() - ref).abs().max() <= 2.0 ** -18 * y.abs().max()
    dx, _, _, _ = qk_norm_rope_backward(torch.ones_like(x), None, x, None, **kw)
    assert dx.isfinite().all()


def test_autograd_shares_and_skips():
    """A weight used for q and k gets both gradients; expanded and transposed
    output gradients are taken; an unused side has none."""
    q, k, wq, _, dq, dk, kw = _case(CASES[1], torch.float32)
    q, k = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    w = wq.clone().requires_grad_(True)
    oq, ok = qk_norm_rope_autograd(q, k, w, w, **kw)
    (oq.sum() + (ok * dk).sum()).backward()
    ones = torch.ones_like(dq)
    gq, gk, gw1, gw2 = qk_norm_rope_backward(ones, dk, q.detach(), k.detach(), w.detach(), w.detach(), **kw)
    assert torch.equal(q.grad, gq) and torch.equal(k.grad, gk)
    assert torch.equal(w.grad, gw1 + gw2)
    q.grad = None
    oq, ok = qk_norm_rope_autograd(q, k.detach(), w, w, **kw)
    (oq.transpose(1, 2) * dq.transpose(1, 2)).sum().backward()
    assert torch.equal(q.grad, qk_norm_rope_backward(dq, None, q.detach(), None, w.detach(), None, **kw)[0])


def test_repeatable_streams_and_graphs():
    q, k, wq, wk, dq, dk, kw = _case(CASES[3], torch.bfloat16)
    wq = torch.ones(64, device="cuda")
    one = qk_norm_rope_backward(dq, dk, q, k, wq, wq, **kw)
    fwd = qk_norm_rope(q, k, wq, wq, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(5):
            two = qk_norm_rope_backward(dq, dk, q, k, wq, wq, **kw)
            assert all(torch.equal(a, b) for a, b in zip(one, two))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = qk_norm_rope(q, k, wq, wq, **kw)
            back = qk_norm_rope_backward(dq, dk, q, k, wq, wq, **kw)
    for t in (*got, *back):
        t.fill_(3)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*got, *back), (*fwd, *one)))


def test_many_rows():
    """More blocks than the backward keeps sums for, and more heads than one walk."""
    q, k, wq, wk, dq, dk, kw = _case((2, 40, 7, 3001, 64, 64, False, True, "f32", "BN32"), torch.bfloat16)
    oq, ok = qk_norm_rope(q, k, wq, wk, **kw)
    gq, gk, gwq, gwk = qk_norm_rope_backward(dq, dk, q, k, wq, wk, **kw)
    args = (kw["positions"], kw["cos"], kw["sin"], kw["eps"], kw["interleaved"])
    for x, w, o, dy, gx, gw, name in ((q, wq, oq, dq, gq, gwq, "q"), (k, wk, ok, dk, gk, gwk, "k")):
        ref, tol = _forward(x, w, *args)
        _near(o, ref, tol, f"{name} out")
        dx, tol, dw, wtol = _backward(x, w, dy, *args)
        _near(gx, dx, tol, f"d{name}")
        _near(gw, dw, wtol, f"d{name} weight")

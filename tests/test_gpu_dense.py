"""Cross attention, its gradient, and shared-prefix attention against the
definitions in 64 bits.

Tolerances, with u = eps / 2 of the 16-bit type and A = sum_j p_j |v_j|:
P is rounded once on its way into the tensor cores (u A), the result once
(u |o|); the scores are fp32 sums of D products, off by at most
D 2^-24 sum |q k| scale <= 2^-12 at these sizes, which moves every p by that
much relatively: |o - ref| <= (u + 2^-12) A + u |o|, |lse - ref| <= 2^-11.
Gradients count the same errors through their formulas (``_grad_bounds``).
"""

import math

import pytest
import torch

from blocksparsefa_reorder_b200 import (cross_attention, cross_attention_autograd, cross_attention_backward,
                                        shared_prefix_attention)

pytestmark = pytest.mark.gpu

E = 2.0 ** -12
BF, HF = torch.bfloat16, torch.float16


def _u(t):
    return torch.finfo(t).eps / 2


def _attend(q, k, v, seen, scale):
    """64-bit (o, lse, A, p) of q [.., M, D] over k [.., N, D]; `seen` [.., M, N]
    bool.  What no row sees is replaced before the products (it may be NaN)."""
    q, k, v = q.double(), k.double(), v.double()
    any_seen = seen.any(-2).unsqueeze(-1)
    k, v = k.masked_fill(~any_seen, 0), v.masked_fill(~any_seen, 0)
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    lse = s.logsumexp(-1)
    p = torch.where(lse.unsqueeze(-1) == -math.inf, torch.zeros_like(s), (s - lse.unsqueeze(-1)).exp())
    return p @ v, lse / math.log(2), p @ v.abs(), p


def _heads(t, H):
    return t.repeat_interleave(H // t.shape[1], 1)


def _cross_ref(q, k, v, lens, scale):
    B, H, M, D = q.shape
    N = k.shape[2]
    ln = torch.full((B,), N, device="cuda") if lens is None else lens.long().clamp(0, N)
    seen = (torch.arange(N, device="cuda") < ln[:, None])[:, None, None].expand(B, H, M, N)
    return _attend(q, _heads(k, H), _heads(v, H), seen, scale)


def _check_o(o, lse, ref, what=""):
    ro, rl, A, _ = ref
    u = _u(o.dtype)
    bound = (u + E) * A + u * ro.abs() * (1 + 2.0 ** -7) + 2.0 ** -24
    off = (o.double() - ro).abs()
    assert o.isfinite().all(), what
    assert (off <= bound).all(), f"{what}: worst {(off / bound).max().item():.2f}x, {(off > bound).sum().item()} off"
    if lse is not None:
        fin = rl.isfinite()
        assert torch.equal(lse.isfinite(), fin) and (lse[~fin] == -math.inf).all(), what
        assert ((lse.double() - rl).abs()[fin] <= 2 * E).all(), what


def _rand(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _poison(t, lens):
    """NaN and infinities behind each sequence's length."""
    for b, n in enumerate(lens.tolist()):
        t[b, :, n:] = math.nan
        t[b, :, n + 1::3] = math.inf
        t[b, :, n + 2::3] = -math.inf
    return t


CROSS = [
    # B, H, Hk, M, N, lens
    (1, 1, 1, 1, 1, None),
    (1, 4, 4, 1, 300, None),
    (2, 8, 2, 1, 129, [129, 1]),
    (3, 6, 2, 3, 257, [0, 128, 200]),
    (2, 4, 1, 17, 1000, [999, 513]),
    (1, 2, 2, 127, 128, [128]),
    (2, 2, 1, 128, 127, [127, 64]),
    (1, 3, 3, 129, 384, [255]),
    (2, 6, 3, 256, 130, [130, 129]),
    (2, 4, 2, 257, 640, [640, 385]),
    (1, 2, 1, 700, 1531, [1400]),
    (3, 2, 2, 200, 260, [0, 260, 2]),
    (1, 2, 2, 1, 9000, None),
    (2, 16, 2, 40, 5000, [5000, 77]),
    (1, 1, 1, 300, 2, None),
    (2, 40, 40, 5, 333, [300, 333]),
]


@pytest.mark.parametrize("D,dtype", [(64, HF), (64, BF), (128, HF), (128, BF)])
@pytest.mark.parametrize("c", CROSS)
def test_cross_matches_definition(c, D, dtype):
    B, H, Hk, M, N, lens = c
    g = torch.Generator(device="cuda").manual_seed(B * 1000 + M + N + D)
    q, k, v = _rand((B, H, M, D), dtype, g), _rand((B, Hk, N, D), dtype, g), _rand((B, Hk, N, D), dtype, g)
    ln = None if lens is None else torch.tensor(lens, device="cuda", dtype=torch.int32 if M % 2 else torch.int64)
    if ln is not None:
        _poison(k, ln), _poison(v, ln)
    o = torch.full_like(q, math.nan)
    o, lse = cross_attention(q, k, v, k_lens=ln, return_lse=True, out=o, check_errors=True)
    ref = _cross_ref(q, k, v, ln, 1 / math.sqrt(D))
    _check_o(o, lse, ref)
    again = cross_attention(q, k, v, k_lens=ln)
    assert torch.equal(again, o)
    if lens is not None and 0 in lens:
        assert (o[lens.index(0)] == 0).all()


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("M", [3, 300])
def test_cross_growing_scores(dtype, M):
    """Scores that grow along the keys by far more than the slack of the
    softmax's reference point, and a few -inf-like ones: the redo path."""
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.zeros(1, 2, M, 64, dtype=dtype, device="cuda")
    q[..., 0] = 8
    q[..., 1:] = _rand((1, 2, M, 63), dtype, g, 0.1)
    k, v = _rand((1, 2, 1100, 64), dtype, g, 0.1), _rand((1, 2, 1100, 64), dtype, g)
    k[0, 0, :, 0] = torch.linspace(-60, 60, 1100, device="cuda").to(dtype)
    k[0, 1, :, 0] = torch.linspace(60, -60, 1100, device="cuda").to(dtype)
    o, lse = cross_attention(q, k, v, return_lse=True, sm_scale=0.5, check_errors=True)
    ro, rl, A, _ = _cross_ref(q, k, v, None, 0.5)
    # |q . k| scale reaches 240: D 2^-24 x 240 = 2^-10 in the scores
    u = _u(dtype)
    assert ((o.double() - ro).abs() <= (u + 2.0 ** -10) * A + u * ro.abs() * 1.01 + 2.0 ** -24).all()
    assert ((lse.double() - rl).abs() <= 2.0 ** -9 + 2.0 ** -23 * rl.abs()).all()


GAPS = (100, 129, 130, 140, 150, 200, 256, 290, 300, 384, 400)


def _far_keys(heads, N, tile, D, dtype, g):
    """One strong key a head in 128-key tile `tile`, at each of 8 neighbouring
    columns and each gap in turn: with q = e_0 and sm_scale = ln 2 it scores its
    gap in log2 units, all others 0."""
    k = torch.zeros(heads, N, D, dtype=dtype, device="cuda")
    at = torch.tensor([tile * 128 + 40 + i % 8 for i in range(heads)], device="cuda")
    gap = torch.tensor([float(GAPS[i // 8 % len(GAPS)]) for i in range(heads)], device="cuda")
    k[torch.arange(heads, device="cuda"), at, 0] = gap.to(dtype)  # (8 bits hold each of them)
    return k, _rand((heads, N, D), dtype, g), at, gap


def _check_far(o, lse, v, at, gap):
    """The strong key takes the whole weight: the others hold 2^-100 of it each.
    Its score is off by four roundings (scale, scale log2 e, product, lse)."""
    own = v[torch.arange(v.shape[0], device="cuda"), at].view(1, -1, 1, v.shape[-1]).expand_as(o)
    assert torch.equal(o, own)
    assert ((lse - gap.view(1, -1, 1)).abs() <= 4 * 2.0 ** -24 * 400).all()


@pytest.mark.parametrize("D,dtype", [(64, HF), (64, BF), (128, HF), (128, BF)])
@pytest.mark.parametrize("tile", [2, 3])
@pytest.mark.parametrize("M", [32, 128, 256, 300])
def test_cross_one_key_far_above_the_first(M, tile, D, dtype):
    """A score far above the row's first keys, in a later tile of either stream, at
    whichever column: its exponential passes the range of the first reference
    point, which has to move."""
    g = torch.Generator(device="cuda").manual_seed(M + D)
    heads = 8 * len(GAPS)
    k, v, at, gap = _far_keys(heads, 640, tile, D, dtype, g)
    q = torch.zeros(1, heads, M, D, dtype=dtype, device="cuda")
    q[..., 0] = 1
    o, lse = cross_attention(q, k[None], v[None], sm_scale=math.log(2), return_lse=True, check_errors=True)
    _check_far(o, lse, v, at, gap)
    # two heads alone: the keys are split over the SMs
    for h in (6, 55):
        a, al = cross_attention(q[:, h:h + 1], k[None, h:h + 1], v[None, h:h + 1], sm_scale=math.log(2), return_lse=True)
        _check_far(a, al, v[h:h + 1], at[h:h + 1], gap[h:h + 1])
    # its gradient: P is 1 at that key, so that dv there is the sum of dout (fp32, rounded once) and dS is rounding alone
    do = _rand(q.shape, dtype, g)
    dq, dk, dv = cross_attention_backward(q, k[None], v[None], o, lse, do, sm_scale=math.log(2))
    ref = do.double().sum(2)
    got = dv[0, torch.arange(heads, device="cuda"), at].double()[None]
    assert ((got - ref).abs() <= (_u(dtype) * 1.01) * ref.abs() + (2.0 ** -11 + _u(dtype)) * do.double().abs().sum(2)).all()
    assert dq.isfinite().all() and dk.isfinite().all()


@pytest.mark.parametrize("D,dtype", [(64, HF), (64, BF), (128, HF), (128, BF)])
@pytest.mark.parametrize("B,T", [(32, 1), (130, 1), (40, 7)])
def test_prefix_one_key_far_above_the_first(B, T, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(B + D)
    heads = 8 * len(GAPS)
    kp, vp, at, gap = _far_keys(heads, 768, 3, D, dtype, g)
    q = torch.zeros(B, heads, T, D, dtype=dtype, device="cuda")
    q[..., 0] = 1
    k, v = torch.zeros(B, heads, T + 2, D, dtype=dtype, device="cuda"), _rand((B, heads, T + 2, D), dtype, g)
    o, lse = shared_prefix_attention(q, kp, vp, k, v, sm_scale=math.log(2), return_lse=True, check_errors=True)
    _check_far(o, lse, vp, at, gap)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,N", [(1, 300), (3, 9000), (40, 200), (128, 1500), (300, 257)])
def test_cross_one_heavy_key_and_many_light_ones(M, N, D):
    """fp16: one key holds nearly all of the weight, with small values; the others
    have about 2^-25 each.  The reference point lies 2^4 below the maximum, so that
    a weight is off by u, or by half of 2^-24 / 2^4 where it is subnormal."""
    g = torch.Generator(device="cuda").manual_seed(M + N)
    q = torch.zeros(1, 2, M, D, dtype=HF, device="cuda")
    q[..., 0] = 1
    k, v = torch.zeros(1, 2, N, D, dtype=HF, device="cuda"), 1 + _rand((1, 2, N, D), HF, g).abs()
    k[..., 0] = -25 - torch.rand(1, 2, N, generator=g, device="cuda").to(HF)
    for h, at in enumerate((0, N - 1)):
        k[0, h, at, 0] = 0
        v[0, h, at] *= 2.0 ** -14
    o, lse = cross_attention(q, k, v, sm_scale=math.log(2), return_lse=True)
    ro, rl, A, _ = _cross_ref(q, k, v, None, math.log(2))
    u = _u(HF)
    bound = (u + E) * A + u * ro.abs() * 1.01 + 2.0 ** -25 + 2.0 ** -29 * _heads(v, 2).double().sum(2, keepdim=True)
    off = (o.double() - ro).abs()
    assert (off <= bound).all(), (off / bound).max()
    assert ((lse.double() - rl).abs() <= 2 * E).all()
    none = torch.empty(1, 2, 0, D, dtype=HF, device="cuda")
    o = shared_prefix_attention(q, k[0], v[0], none, none, sm_scale=math.log(2))
    assert ((o.double() - ro).abs() <= bound).all()


def test_cross_layouts_and_expanded_batch():
    """[B, N, H, D] memory, a slice of a wider projection, k / v shared by the
    batch (expanded) and by the heads, an output view."""
    g = torch.Generator(device="cuda").manual_seed(5)
    B, H, Hk, M, N, D = 3, 4, 2, 130, 200, 64
    q = _rand((B, M, H, D), BF, g).transpose(1, 2)
    kv = _rand((B, N, 2 * Hk * D), BF, g)
    k = kv[..., :Hk * D].view(B, N, Hk, D).transpose(1, 2)
    v = kv[..., Hk * D:].view(B, N, Hk, D).transpose(1, 2)
    out = torch.empty(B, M, H, D, dtype=BF, device="cuda").transpose(1, 2)
    o, lse = cross_attention(q, k, v, out=out, return_lse=True)
    assert o.data_ptr() == out.data_ptr()
    _check_o(o, lse, _cross_ref(q, k, v, None, 1 / 8))
    one_k, one_v = _rand((1, Hk, N, D), BF, g).expand(B, -1, -1, -1), _rand((1, Hk, N, D), BF, g).expand(B, -1, -1, -1)
    ln = torch.tensor([200, 3, 131], device="cuda")
    for m in (1, M):
        o, lse = cross_attention(q[:, :, :m], one_k, one_v, k_lens=ln, return_lse=True)
        _check_o(o, lse, _cross_ref(q[:, :, :m], one_k, one_v, ln, 1 / 8))
    wide_k, wide_v = one_k[:, :1].expand(B, H, N, D), one_v[:, :1].expand(B, H, N, D)
    _check_o(cross_attention(q, wide_k, wide_v), None, _cross_ref(q, wide_k, wide_v, None, 1 / 8))


@pytest.mark.parametrize("M,G", [(1, 24), (3, 50), (40, 6), (65, 8), (100, 4), (129, 4), (43, 3)])
def test_cross_tiles_of_tokens_heads_and_sequences(M, G):
    """Row tiles that hold several heads, some of them cut; queries expanded over
    the batch."""
    g = torch.Generator(device="cuda").manual_seed(M + G)
    B, Hk, N, D = 2, 2, 300, 64
    k, v = _rand((B, Hk, N, D), BF, g), _rand((B, Hk, N, D), BF, g)
    for q in (_rand((B, Hk * G, M, D), BF, g), _rand((1, Hk * G, M, D), BF, g).expand(B, -1, -1, -1)):
        o, lse = cross_attention(q, k, v, return_lse=True)
        _check_o(o, lse, _cross_ref(q, k, v, None, 1 / 8))


@pytest.mark.parametrize("B,T,G", [(37, 1, 8), (13, 5, 3), (9, 30, 2), (5, 50, 3), (3, 129, 2)])
def test_prefix_tiles_of_tokens_heads_and_sequences(B, T, G):
    g = torch.Generator(device="cuda").manual_seed(B + T + G)
    Hk, P, C, D = 2, 333, T + 3, 64
    q = _rand((B, Hk * G, T, D), HF, g)
    kp, vp = _rand((Hk, P, D), HF, g), _rand((Hk, P, D), HF, g)
    k, v = _rand((B, Hk, C, D), HF, g), _rand((B, Hk, C, D), HF, g)
    o, lse = shared_prefix_attention(q, kp, vp, k, v, return_lse=True)
    t = torch.arange(T, device="cuda")
    own = (torch.arange(C, device="cuda") < (C - (T - 1 - t)[:, None])).expand(B, T, C)
    seen = torch.cat((torch.ones(B, T, P, dtype=torch.bool, device="cuda"), own), -1)[:, None].expand(B, Hk * G, T, P + C)
    kk, vv = torch.cat((kp.expand(B, -1, -1, -1), k), 2), torch.cat((vp.expand(B, -1, -1, -1), v), 2)
    _check_o(o, lse, _attend(q, _heads(kk, Hk * G), _heads(vv, Hk * G), seen, 1 / 8))


def test_cross_empty_and_out_of_range_lengths():
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k, v = _rand((2, 2, 5, 64), BF, g), _rand((2, 2, 70, 64), BF, g), _rand((2, 2, 70, 64), BF, g)
    o, lse = cross_attention(q, k[:, :, :0], v[:, :, :0], return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()
    bad = torch.tensor([71, -3], device="cuda")
    o = cross_attention(q, k, v, k_lens=bad)
    assert torch.equal(o, cross_attention(q, k, v, k_lens=bad.clamp(0, 70)))
    with pytest.raises(RuntimeError, match="coordinate out of range"):
        cross_attention(q, k, v, k_lens=bad, check_errors=True)


def _grads_ref(q, k, v, do, lens, scale):
    B, H, M, D = q.shape
    Hk, N = k.shape[1], k.shape[2]
    ln = torch.full((B,), N, device="cuda") if lens is None else lens.long()
    gone = ~(torch.arange(N, device="cuda") < ln[:, None])[:, None, :, None]
    qd, kd, vd, dd = q.double(), k.double().masked_fill(gone, 0), v.double().masked_fill(gone, 0), do.double()
    kh, vh = _heads(kd, H), _heads(vd, H)
    ro, _, A, p = _cross_ref(q, k, v, lens, scale)
    dp = dd @ vh.transpose(-1, -2)
    delta = (dd * ro).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    fold = lambda t: t.view(B, Hk, H // Hk, N, -1).sum(2)  # noqa: E731
    u = _u(q.dtype)
    # errors: o's rounding and P's through Delta; p itself (scores, lse) 4 E; dS's rounding
    e_o = (u + E) * A + u * ro.abs() + 2.0 ** -24
    e_delta = (dd.abs() * e_o).sum(-1, keepdim=True)
    e_ds = (u + 4 * E) * ds.abs() + p * (e_delta + 2.0 ** -16 * (dd.abs() @ vh.abs().transpose(-1, -2)))
    dq, dk, dv = scale * ds @ kh, fold(scale * ds.transpose(-1, -2) @ qd), fold(p.transpose(-1, -2) @ dd)
    b = (scale * e_ds @ kh.abs(), fold(scale * e_ds.transpose(-1, -2) @ qd.abs()),
         fold((u + 4 * E) * p.transpose(-1, -2) @ dd.abs()))
    return (dq, dk, dv), tuple(x + u * g.abs() * 1.01 + torch.finfo(q.dtype).tiny for x, g in zip(b, (dq, dk, dv)))


BWD = [
    (1, 1, 1, 1, 1, None), (2, 4, 2, 5, 130, [130, 1]), (3, 6, 2, 129, 257, [0, 128, 200]),
    (1, 4, 1, 300, 1000, [999]), (2, 2, 2, 256, 128, None), (2, 6, 3, 257, 385, [385, 384]),
    (1, 8, 2, 640, 64, [33]), (1, 2, 2, 1000, 1531, None), (2, 12, 1, 3, 200, [200, 7]), (1, 12, 2, 40, 300, None),
    (2, 8, 1, 65, 150, [150, 129]), (1, 5, 1, 129, 130, None),
]


@pytest.mark.parametrize("D,dtype", [(64, HF), (64, BF), (128, HF), (128, BF)])
@pytest.mark.parametrize("c", BWD)
def test_cross_gradient_matches_formula(c, D, dtype):
    B, H, Hk, M, N, lens = c
    g = torch.Generator(device="cuda").manual_seed(B * 100 + M + N + D)
    q, do = _rand((B, H, M, D), dtype, g), _rand((B, H, M, D), dtype, g)
    k, v = _rand((B, Hk, N, D), dtype, g), _rand((B, Hk, N, D), dtype, g)
    ln = None if lens is None else torch.tensor(lens, device="cuda")
    if ln is not None:
        _poison(k, ln), _poison(v, ln)
    o, lse = cross_attention(q, k, v, k_lens=ln, return_lse=True)
    got = cross_attention_backward(q, k, v, o, lse, do, k_lens=ln, check_errors=True)
    ref, bound = _grads_ref(q, k, v, do, ln, 1 / math.sqrt(D))
    for name, x, r, t in zip(("dq", "dk", "dv"), got, ref, bound):
        assert x.isfinite().all(), name
        off = (x.double() - r).abs()
        assert (off <= t).all(), f"{name}: worst {(off / t).max().item():.2f}x, {(off > t).sum().item()} off"
    if ln is not None:
        for b, n in enumerate(lens):
            assert (got[1][b, :, n:] == 0).all() and (got[2][b, :, n:] == 0).all()
            if n == 0:
                assert (got[0][b] == 0).all()
    again = cross_attention_backward(q, k, v, o, lse, do, k_lens=ln)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("M,N,G", [(3, 20, 2), (40, 20, 2), (40, 5000, 2), (200, 300, 1), (3, 9000, 1)])
def test_cross_rounding_rest(M, N, G, dtype):
    """o + o_rest is the result to twice the bits (rounding left u^2 |o|), whichever
    kernel writes it, and the gradient holds its bound with it."""
    g = torch.Generator(device="cuda").manual_seed(M + N)
    q, do = _rand((2, 2 * G, M, 64), dtype, g), _rand((2, 2 * G, M, 64), dtype, g)
    k, v = _rand((2, 2, N, 64), dtype, g), _rand((2, 2, N, 64), dtype, g)
    rest = torch.full_like(q, math.nan)
    o, lse = cross_attention(q, k, v, return_lse=True, o_rest=rest)
    assert torch.equal(o, cross_attention(q, k, v))
    ro, _, A, _ = _cross_ref(q, k, v, None, 1 / 8)
    u = _u(dtype)
    assert (rest.double().abs() <= u * o.double().abs() * 1.01 + 2.0 ** -24).all()
    assert ((o.double() + rest.double() - ro).abs() <= (u + E) * A + 2 * u * u * ro.abs() + 2.0 ** -24).all()
    got = cross_attention_backward(q, k, v, o, lse, do, o_rest=rest)
    ref, bound = _grads_ref(q, k, v, do, None, 1 / 8)
    assert all(((x.double() - r).abs() <= t).all() for x, r, t in zip(got, ref, bound))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,N,G,e", [(300, 4096, 2, -17), (40, 5000, 1, -12), (2000, 700, 1, -20), (130, 300, 3, 9),
                                     (1, 9000, 1, -16)])
def test_cross_gradient_of_small_and_large_output_gradients(M, N, G, e, D):
    """fp16, dout around 2^e, a second sequence's at 2^0: dS is held relative to the
    largest dout of its key / value head (which comes to lie in [4, 8)), so that it
    is rounded by at most half of 2^-24 in that measure, or relatively by u.  The
    result itself may be subnormal: half of 2^-24."""
    g = torch.Generator(device="cuda").manual_seed(M + N)
    B, Hk, u = 2, 2, _u(HF)
    q, k, v = _rand((B, Hk * G, M, D), HF, g), _rand((B, Hk, N, D), HF, g), _rand((B, Hk, N, D), HF, g)
    do = _rand(q.shape, HF, g)
    do[0] = (do[0].float() * 2.0 ** e).to(HF)
    ln = torch.tensor([N, N - 5], device="cuda")
    rest, scale = torch.empty_like(q), 1 / math.sqrt(D)
    o, lse = cross_attention(q, k, v, k_lens=ln, return_lse=True, o_rest=rest)
    got = cross_attention_backward(q, k, v, o, lse, do, k_lens=ln, o_rest=rest, check_errors=True)
    ro, _, A, p = _cross_ref(q, k, v, ln, scale)
    gone = ~(torch.arange(N, device="cuda") < ln[:, None])[:, None, :, None]
    kh, vh = (_heads(t.double().masked_fill(gone, 0), Hk * G) for t in (k, v))
    d, qd = do.double(), q.double()
    ds = p * (d @ vh.transpose(-1, -2) - (d * ro).sum(-1, keepdim=True))
    # Delta from o + rest: P's and the scores' errors through A, and fp32 sums of D terms
    e_delta = (d.abs() * ((u + E) * A + 2 * u * u * ro.abs())).sum(-1, keepdim=True)
    sums = 2.0 ** -16 * (d.abs() @ vh.abs().transpose(-1, -2) + (d * ro).abs().sum(-1, keepdim=True))
    top = do.double().abs().view(B, Hk, -1).amax(-1).log2().floor().exp2() / 4  # 1 where dout is N(0, 1)
    quantum = top.repeat_interleave(G, 1)[..., None, None] * 2.0 ** -25
    e_ds = (u + 4 * E) * ds.abs() + p * (e_delta + sums) + quantum
    fold = lambda t: t.view(B, Hk, G, N, -1).sum(2)  # noqa: E731
    ref = (scale * ds @ kh, fold(scale * ds.transpose(-1, -2) @ qd), fold(p.transpose(-1, -2) @ d))
    # P is off by u and the scores' error, and by half of 2^-24 where it is subnormal
    bound = (scale * e_ds @ kh.abs(), fold(scale * e_ds.transpose(-1, -2) @ qd.abs()),
             fold(((u + 4 * E) * p + 2.0 ** -25).transpose(-1, -2) @ d.abs()))
    for name, x, r, t in zip(("dq", "dk", "dv"), got, ref, bound):
        assert x.isfinite().all(), name
        off, t = (x.double() - r).abs(), t + u * r.abs() * 1.01 + 2.0 ** -25
        assert (off <= t).all(), f"{name}: worst {(off / t).max().item():.2f}x, {(off > t).sum().item()} off"
    again = cross_attention_backward(q, k, v, o, lse, do, k_lens=ln, o_rest=rest)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("D,dtype", [(64, HF), (128, HF), (64, BF)])
def test_cross_gradient_of_keys_of_little_weight(D, dtype):
    """Keys whose weight is about 2^-26 in every row get their sum over many rows:
    fp16's P is held times 2^12, so it is rounded by at most half of 2^-36."""
    g = torch.Generator(device="cuda").manual_seed(22)
    M, N = 2000, 4096
    q = _rand((1, 2, M, D), dtype, g, 0.1)
    q[..., 0] = 1
    k, v = _rand((1, 2, N, D), dtype, g, 0.1), _rand((1, 2, N, D), dtype, g)
    k[..., 0] = -10.0
    k[:, :, ::64, 0] = 10.0
    do = (1 + _rand(q.shape, dtype, g, 0.1).abs()).to(dtype)
    scale = math.log(2)
    o, lse = cross_attention(q, k, v, sm_scale=scale, return_lse=True)
    dv = cross_attention_backward(q, k, v, o, lse, do, sm_scale=scale)[2]
    p = _cross_ref(q, k, v, None, scale)[3]
    u, d = _u(dtype), do.double()
    ref = p.transpose(-1, -2) @ d
    tiny = 2.0 ** -37 if dtype == HF else 0
    bound = ((u + 4 * E) * p + tiny).transpose(-1, -2) @ d + u * ref * 1.01 + (2.0 ** -25 if dtype == HF else 0)
    assert ((dv.double() - ref).abs() <= bound).all(), ((dv.double() - ref).abs() / bound).max()


def test_cross_gradient_of_degenerate_output_gradients():
    """All zero: zero gradients.  Infinite or NaN in one head: its own group's alone."""
    g = torch.Generator(device="cuda").manual_seed(21)
    q, k, v = _rand((1, 4, 140, 64), HF, g), _rand((1, 2, 200, 64), HF, g), _rand((1, 2, 200, 64), HF, g)
    o, lse = cross_attention(q, k, v, return_lse=True)
    assert all((x == 0).all() for x in cross_attention_backward(q, k, v, o, lse, torch.zeros_like(q)))
    do = _rand(q.shape, HF, g, 2.0 ** -10)
    want = cross_attention_backward(q, k, v, o, lse, do)
    for bad in (math.inf, math.nan):
        spoilt = do.clone()
        spoilt[0, 1, 7, 3] = bad
        got = cross_attention_backward(q, k, v, o, lse, spoilt)
        assert not got[0][0, 1, 7].isfinite().any() and not got[2][0, 0].isfinite().all()
        assert torch.equal(got[0][:, 2:], want[0][:, 2:]) and torch.equal(got[1][:, 1], want[1][:, 1])
        assert torch.equal(got[2][:, 1], want[2][:, 1])


def test_cross_gradient_matches_differences():
    """Central differences of the 64-bit definition along random directions."""
    g = torch.Generator(device="cuda").manual_seed(8)
    B, H, Hk, M, N, D = 2, 4, 2, 140, 150, 64
    q, do = _rand((B, H, M, D), HF, g), _rand((B, H, M, D), HF, g)
    k, v = _rand((B, Hk, N, D), HF, g), _rand((B, Hk, N, D), HF, g)
    ln = torch.tensor([150, 70], device="cuda")
    o, lse = cross_attention(q, k, v, k_lens=ln, return_lse=True)
    got = cross_attention_backward(q, k, v, o, lse, do, k_lens=ln)
    _, bound = _grads_ref(q, k, v, do, ln, 1 / 8)
    for i, x in enumerate((q, k, v)):
        d = torch.randn(x.shape, generator=g, device="cuda", dtype=torch.float64)

        def f(t):
            a = [y.double() for y in (q, k, v)]
            a[i] = a[i] + t * d
            return (_cross_ref(*a, ln, 1 / 8)[0] * do.double()).sum()

        diff = (f(1e-5) - f(-1e-5)) / 2e-5
        val = (d * got[i].double()).sum()
        assert (diff - val).abs() <= (d.abs() * bound[i]).sum() + 1e-5 * (1 + diff.abs()), i


def test_cross_autograd_expanded_and_shared():
    """k / v of one sequence expanded over the batch get the batch's sum; an
    expanded output gradient (a sum's) is taken; no gradient for lengths."""
    g = torch.Generator(device="cuda").manual_seed(10)
    B, H, Hk, M, N, D = 3, 4, 2, 60, 140, 64
    q = _rand((B, H, M, D), BF, g).requires_grad_(True)
    k, v = (_rand((1, Hk, N, D), BF, g).requires_grad_(True) for _ in range(2))
    ln = torch.tensor([140, 5, 100], device="cuda", dtype=torch.int32)
    o = cross_attention_autograd(q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), k_lens=ln)
    o.sum().backward()
    ones = torch.ones_like(q)
    kd, vd = (t.detach().expand(B, -1, -1, -1).contiguous() for t in (k, v))
    with torch.no_grad():
        rest = torch.empty_like(q)
        ob, lb = cross_attention(q, kd, vd, k_lens=ln, return_lse=True, o_rest=rest)
        dq, dk, dv = cross_attention_backward(q, kd, vd, ob, lb, ones, k_lens=ln, o_rest=rest)
    assert torch.equal(o, ob) and torch.equal(q.grad, dq)
    for got, parts in ((k.grad, dk), (v.grad, dv)):
        assert got.shape == (1, Hk, N, D)
        ref = parts.double().sum(0, keepdim=True)
        # bf16 sum of three: at most three roundings
        assert ((got.double() - ref).abs() <= 3 * _u(BF) * parts.double().abs().sum(0, keepdim=True) + 1e-30).all()


PREFIX = [
    # B, H, Hk, T, P, C, lens
    (1, 1, 1, 1, 1, 1, None),
    (3, 4, 2, 1, 200, 40, [1, 40, 17]),
    (4, 8, 2, 1, 1000, 200, [200, 129, 128, 0]),
    (2, 4, 4, 3, 130, 10, [3, 10]),
    (2, 4, 1, 7, 64, 300, [2, 300]),
    (20, 8, 2, 4, 500, 150, list(range(4, 144, 7))),
    (40, 8, 1, 1, 3000, 33, None),
    (5, 2, 2, 1, 0, 60, [1, 60, 0, 5, 6]),
    (3, 2, 1, 2, 77, 0, None),
    (2, 4, 2, 130, 300, 200, [130, 200]),
    (1, 2, 2, 260, 129, 400, [300]),
    (70, 2, 1, 2, 20, 4, None),
]


@pytest.mark.parametrize("D,dtype", [(64, HF), (64, BF), (128, HF), (128, BF)])
@pytest.mark.parametrize("c", PREFIX)
def test_prefix_matches_definition(c, D, dtype):
    B, H, Hk, T, P, C, lens = c
    g = torch.Generator(device="cuda").manual_seed(B + T * 10 + P + C + D)
    q = _rand((B, H, T, D), dtype, g)
    kp, vp = _rand((Hk, P, D), dtype, g), _rand((Hk, P, D), dtype, g)
    k, v = _rand((B, Hk, C, D), dtype, g), _rand((B, Hk, C, D), dtype, g)
    ln = None if lens is None else torch.tensor(lens, device="cuda", dtype=torch.int32 if P % 2 else torch.int64)
    if ln is not None:
        _poison(k, ln), _poison(v, ln)
    o, lse = shared_prefix_attention(q, kp, vp, k, v, lens=ln, return_lse=True, out=torch.full_like(q, math.nan),
                                     check_errors=True)
    n = torch.full((B,), C, device="cuda") if ln is None else ln.long()
    t = torch.arange(T, device="cuda")
    own = torch.arange(C, device="cuda") < (n[:, None, None] - (T - 1 - t)[:, None])
    seen = torch.cat((torch.ones(B, T, P, dtype=torch.bool, device="cuda"), own), -1)[:, None].expand(B, H, T, P + C)
    kk = torch.cat((kp.expand(B, -1, -1, -1), k), 2)
    vv = torch.cat((vp.expand(B, -1, -1, -1), v), 2)
    _check_o(o, lse, _attend(q, _heads(kk, H), _heads(vv, H), seen, 1 / math.sqrt(D)))
    assert torch.equal(shared_prefix_attention(q, kp, vp, k, v, lens=ln), o)


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, HF)])
@pytest.mark.parametrize("B,H,Hk,T,P", [(2, 2, 1, 1, 300), (2, 2, 1, 1, 8192), (2, 2, 1, 1, 8500), (1, 8, 1, 1, 8500),
                                        (3, 4, 2, 4, 8192), (9, 12, 3, 4, 4000), (1, 1, 1, 16, 5000)])
def test_prefix_partial_results_on_both_sides_of_the_joining_rule(B, H, Hk, T, P, D, dtype):
    """Few own rows: up to 32 ranges of the prefix are joined by the own keys'
    kernel, more by one of its own; a NaN query stays in its own rows."""
    g = torch.Generator(device="cuda").manual_seed(P + B)
    C = 40
    q = _rand((B, H, T, D), dtype, g)
    kp, vp = _rand((Hk, P, D), dtype, g), _rand((Hk, P, D), dtype, g)
    k, v = _rand((B, Hk, C, D), dtype, g), _rand((B, Hk, C, D), dtype, g)
    ln = torch.tensor([T if b % 2 else 0 for b in range(B)], device="cuda")
    _poison(k, ln), _poison(v, ln)
    t = torch.arange(T, device="cuda")
    own = torch.arange(C, device="cuda") < (ln[:, None, None] - (T - 1 - t)[:, None])
    seen = torch.cat((torch.ones(B, T, P, dtype=torch.bool, device="cuda"), own), -1)[:, None].expand(B, H, T, P + C)
    kk = torch.cat((kp.expand(B, -1, -1, -1), k), 2)
    vv = torch.cat((vp.expand(B, -1, -1, -1), v), 2)
    o, lse = shared_prefix_attention(q, kp, vp, k, v, lens=ln, return_lse=True, out=torch.full_like(q, math.nan))
    _check_o(o, lse, _attend(q, _heads(kk, H), _heads(vv, H), seen, 1 / math.sqrt(D)))
    q[B - 1, H - 1, T - 1] = math.nan
    p, lse = shared_prefix_attention(q, kp, vp, k, v, lens=ln, return_lse=True)
    assert p[B - 1, H - 1, T - 1].isnan().all() and lse[B - 1, H - 1, T - 1].isnan()
    o[B - 1, H - 1, T - 1] = p[B - 1, H - 1, T - 1] = 0
    assert torch.equal(o, p)


@pytest.mark.parametrize("D,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("B,T,C", [(3, 40, 50), (2, 20, 20), (30, 1, 9), (2, 140, 0), (3, 1, 0), (60, 1, 0)])
def test_prefix_of_no_keys(B, T, C, D, dtype):
    """An empty prefix in front of own keys, or of none: more rows than the
    few-rows kernel takes (T or the batch), and fewer."""
    g = torch.Generator(device="cuda").manual_seed(B + T + C)
    H, Hk = 4, 2
    q, k, v = _rand((B, H, T, D), dtype, g), _rand((B, Hk, C, D), dtype, g), _rand((B, Hk, C, D), dtype, g)
    none = torch.empty(Hk, 0, D, dtype=dtype, device="cuda")
    o, lse = shared_prefix_attention(q, none, none, k, v, return_lse=True, out=torch.full_like(q, math.nan),
                                     check_errors=True)
    if C == 0:
        assert (o == 0).all() and (lse == -math.inf).all()
        return
    t = torch.arange(T, device="cuda")
    seen = (torch.arange(C, device="cuda") < (C - (T - 1 - t)[:, None])).expand(B, H, T, C)
    _check_o(o, lse, _attend(q, _heads(k, H), _heads(v, H), seen, 1 / math.sqrt(D)))


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, HF)])
@pytest.mark.parametrize("B,H,Hk,M", [(2, 4, 2, 100), (1, 3, 3, 300), (2, 8, 1, 5), (1, 2, 2, 1)])
def test_cross_of_no_keys(B, H, Hk, M, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(M)
    q, do = _rand((B, H, M, D), dtype, g), _rand((B, H, M, D), dtype, g)
    none = torch.empty(B, Hk, 0, D, dtype=dtype, device="cuda")
    for lens in (None, torch.zeros(B, dtype=torch.int32, device="cuda")):
        o, lse = cross_attention(q, none, none, k_lens=lens, return_lse=True, out=torch.full_like(q, math.nan),
                                 check_errors=True)
        assert (o == 0).all() and (lse == -math.inf).all()
        dq, dk, dv = cross_attention_backward(q, none, none, o, lse, do, k_lens=lens, check_errors=True)
        assert (dq == 0).all() and dk.shape == dv.shape == none.shape


def test_prefix_equals_cross_attention_without_own_keys():
    """No own keys: the prefix alone, the same for every sequence."""
    g = torch.Generator(device="cuda").manual_seed(12)
    q = _rand((6, 4, 1, 64), BF, g)
    kp, vp = _rand((2, 700, 64), BF, g), _rand((2, 700, 64), BF, g)
    none = torch.empty(6, 2, 0, 64, dtype=BF, device="cuda")
    a = shared_prefix_attention(q, kp, vp, none, none)
    b = cross_attention(q, kp.expand(6, -1, -1, -1), vp.expand(6, -1, -1, -1))
    ref = _cross_ref(q, kp.expand(6, -1, -1, -1), vp.expand(6, -1, -1, -1), None, 1 / 8)
    _check_o(a, None, ref)
    _check_o(b, None, ref)


def test_prefix_cache_views_and_lengths():
    """Slices of longer caches; lengths outside the cache are clamped or refused."""
    g = torch.Generator(device="cuda").manual_seed(13)
    pool_k, pool_v = _rand((2, 900, 64), HF, g), _rand((2, 900, 64), HF, g)
    cache_k, cache_v = _rand((3, 50, 2, 64), HF, g).transpose(1, 2), _rand((3, 50, 2, 64), HF, g).transpose(1, 2)
    q = _rand((3, 4, 1, 64), HF, g)
    ln = torch.tensor([51, -1, 20], device="cuda")
    o = shared_prefix_attention(q, pool_k[:, 100:431], pool_v[:, 100:431], cache_k, cache_v, lens=ln)
    same = shared_prefix_attention(q, pool_k[:, 100:431].contiguous(), pool_v[:, 100:431].contiguous(),
                                   cache_k.contiguous(), cache_v.contiguous(), lens=ln.clamp(0, 50))
    assert torch.equal(o, same)
    with pytest.raises(RuntimeError, match="coordinate out of range"):
        shared_prefix_attention(q, pool_k, pool_v, cache_k, cache_v, lens=ln, check_errors=True)


def test_streams_and_graphs():
    """Two streams at once, and captured graphs replayed with new inputs in place
    (each captured call holds a workspace of its own)."""
    g = torch.Generator(device="cuda").manual_seed(14)
    q, k, v = _rand((2, 8, 1, 128), BF, g), _rand((2, 2, 4000, 128), BF, g), _rand((2, 2, 4000, 128), BF, g)
    q2, kp, vp = _rand((9, 8, 2, 128), BF, g), _rand((2, 3000, 128), BF, g), _rand((2, 3000, 128), BF, g)
    ck, cv = _rand((9, 2, 100, 128), BF, g), _rand((9, 2, 100, 128), BF, g)
    ref1, ref2 = cross_attention(q, k, v), shared_prefix_attention(q2, kp, vp, ck, cv)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(s1):
            a = cross_attention(q, k, v)
        with torch.cuda.stream(s2):
            b = shared_prefix_attention(q2, kp, vp, ck, cv)
        torch.cuda.synchronize()
        assert torch.equal(a, ref1) and torch.equal(b, ref2)
    graphs, outs = [], []
    for f in (lambda: cross_attention(q, k, v), lambda: shared_prefix_attention(q2, kp, vp, ck, cv)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(f())
        graphs.append(gr)
    for _ in range(3):
        for o in outs:
            o.zero_()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], ref1) and torch.equal(outs[1], ref2)
    q.copy_(_rand(q.shape, BF, g))
    graphs[0].replay()
    assert torch.equal(outs[0], cross_attention(q, k, v))


def test_captured_training_step():
    """Forward and gradient captured together, replayed with new inputs."""
    g = torch.Generator(device="cuda").manual_seed(15)
    q, k, v, do = (_rand((1, 2, 200, 64), HF, g) for _ in range(4))
    ln = torch.tensor([150], device="cuda")

    def step():
        o, lse = cross_attention(q, k, v, k_lens=ln, return_lse=True)
        return (o, *cross_attention_backward(q, k, v, o, lse, do, k_lens=ln))

    step()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        outs = step()
    for t in (q, k, v, do):
        t.copy_(_rand(t.shape, HF, g))
    ln.fill_(77)
    gr.replay()
    assert all(torch.equal(a, b) for a, b in zip(outs, step()))


def test_rows_around_the_output_stay():
    """Outputs are views between guard rows."""
    g = torch.Generator(device="cuda").manual_seed(16)
    for M in (1, 129, 300):
        q, k, v = _rand((2, 3, M, 64), BF, g), _rand((2, 3, 200, 64), BF, g), _rand((2, 3, 200, 64), BF, g)
        wide = torch.full((2, 3, M + 2, 64), 5.0, dtype=BF, device="cuda")
        cross_attention(q, k, v, out=wide[:, :, 1:M + 1])
        assert (wide[:, :, 0] == 5).all() and (wide[:, :, M + 1] == 5).all()
        assert torch.equal(wide[:, :, 1:M + 1], cross_attention(q, k, v))


@pytest.mark.parametrize("G,M", [(2, 3), (3, 40)])
def test_offsets_beyond_32_bits(G, M):
    """2 x 64 x (2^24 + 1000) elements: the last keys lie behind 2^31 of them.  All
    other keys are zero (score 0, value 0), so 100 keys give the 64-bit result.
    Gradients: P and dS are rounded once and off by the scores' E; Delta holds the
    output's error (u + E) |dO| A."""
    g = torch.Generator(device="cuda").manual_seed(G)
    Hk, D, N, L = 2, 64, 2 ** 24 + 1000, 100
    n = N - 30
    k, v = (torch.zeros(1, Hk, N, D, dtype=BF, device="cuda") for _ in range(2))
    for t in (k, v):
        t[:, :, N - L:] = _rand((1, Hk, L, D), BF, g)
        t[:, :, n:] = math.nan
    q, do = _rand((1, Hk * G, M, D), BF, g, 8.0), _rand((1, Hk * G, M, D), BF, g)
    ln = torch.tensor([n], device="cuda")
    rest = torch.empty_like(q)
    o, lse = cross_attention(q, k, v, k_lens=ln, return_lse=True, o_rest=rest)
    kk, vv = _heads(k[:, :, N - L:n], Hk * G).double(), _heads(v[:, :, N - L:n], Hk * G).double()
    s = q.double() @ kk.transpose(-1, -2) / 8
    rl = torch.cat((s, torch.full_like(s[..., :1], math.log(N - L))), -1).logsumexp(-1)
    p = (s - rl.unsqueeze(-1)).exp()
    ro, A = p @ vv, p @ vv.abs()
    _check_o(o, lse, (ro, rl / math.log(2), A, p))
    dq, dk, dv = cross_attention_backward(q, k, v, o, lse, do, k_lens=ln, o_rest=rest)
    assert not dk[:, :, n:].any() and not dv[:, :, n:].any() and not dk[:, :, ::4096].isnan().any()
    d, u = do.double(), _u(BF)

    def group(x):
        return x.view(1, Hk, G, *x.shape[2:]).sum(2)

    ds = p * (d @ vv.transpose(-1, -2) - (d * ro).sum(-1, keepdim=True))
    da = p * (d.abs() @ vv.abs().transpose(-1, -2) + (d.abs() * A).sum(-1, keepdim=True)) * (u + 2 * E)
    for got, ref, bound in ((dv, group(p.transpose(-1, -2) @ d), group(p.transpose(-1, -2) @ d.abs()) * (u + E)),
                            (dk, group(ds.transpose(-1, -2) @ q.double() / 8),
                             group(da.transpose(-1, -2) @ q.double().abs() / 8))):
        off = (got[:, :, N - L:n].double() - ref).abs()
        assert (off <= bound + u * ref.abs() * (1 + 2.0 ** -7) + 2.0 ** -24).all()

"""What the operators of cross attention, shared prefixes and query / key norm
refuse: on the host through the C ABI (no GPU work is issued, the addresses are
never read) and through the Python entry points."""

import ctypes
import struct

import pytest
import torch

import blocksparsefa_reorder_b200 as lib
from blocksparsefa_reorder_b200 import _lib

T4 = "Pqqq"
ROPE = struct.Struct("@8i" + 6 * T4 + "4Pq2iPqfi3P")
CROSS = struct.Struct("@8i" + 4 * T4 + "4Pf0q")
CROSS_BWD = struct.Struct("@8i" + 8 * T4 + "5Pf0q")
PREFIX = struct.Struct("@9i" + 6 * T4 + "3Pf0q")
P = 0x10000
F16, BF16, F32 = _lib.DTYPE_F16, _lib.DTYPE_BF16, _lib.DTYPE_F32


def t4(data=P, n=64, h=6400, b=64000):
    return data, b, h, n


def _call(fn, packed):
    n = ctypes.c_size_t()
    return getattr(_lib.lib(), fn)(packed, ctypes.byref(n)), n.value


def _cross(B=2, H=4, Hk=2, M=3, N=100, D=64, dtype=F16, lens_dtype=0, q=t4(), o=t4(), k=t4(), v=t4(), lens=0, lse=0,
           rest=0, err=0, scale=0.125):
    return CROSS.pack(B, H, Hk, M, N, D, dtype, lens_dtype, *q, *o, *k, *v, lens, lse, rest, err, scale)


@pytest.mark.parametrize("kw,status", [
    ({}, 0), ({"B": 0}, 1), ({"H": 0}, 1), ({"Hk": 0}, 1), ({"M": 0}, 1), ({"N": -1}, 1), ({"N": 0}, 0),
    ({"dtype": F32}, 3), ({"dtype": 9}, 3), ({"H": 5}, 2), ({"D": 96}, 5), ({"scale": 0.0}, 5), ({"scale": -1.0}, 5),
    ({"scale": float("nan")}, 5), ({"scale": float("inf")}, 5), ({"q": t4(0)}, 1), ({"k": t4(0)}, 1), ({"v": t4(0)}, 1),
    ({"q": t4(P + 8)}, 4), ({"k": t4(n=68)}, 4), ({"v": t4(b=-64)}, 1), ({"o": t4(h=6404)}, 4), ({"rest": P + 4}, 4),
    ({"lens": P, "lens_dtype": 7}, 3), ({"B": 1 << 16, "H": 1 << 10, "M": 1 << 10}, 5), ({"N": 2 ** 31 - 1}, 5),
    ({"N": 2 ** 30 + 5, "k": t4(n=0), "v": t4(n=0)}, 5),
    ({"k": t4(b=0), "v": t4(b=0)}, 0),
])
def test_cross_forward_abi(kw, status):
    assert _call("bsa_cross_fwd_workspace_bytes", _cross(**kw))[0] == status


def test_cross_forward_workspace():
    rc, n = _call("bsa_cross_fwd_workspace_bytes", _cross(B=1, N=65536))
    assert rc == 0 and n > 0
    assert _lib.lib().bsa_cross_fwd(_cross(B=1, N=65536), None, 0, None) == 9
    assert _lib.lib().bsa_cross_fwd(_cross(B=1, N=65536), P, n - 1, None) == 9
    assert _lib.lib().bsa_cross_fwd_workspace_bytes(None, ctypes.byref(ctypes.c_size_t())) == 1
    assert _lib.lib().bsa_cross_fwd_workspace_bytes(_cross(), None) == 1


def _bwd(B=2, H=4, Hk=2, M=3, N=100, D=64, dtype=F16, lens_dtype=0, lens=0, lse=P, delta=P, rest=0, scale=0.125, **ts):
    names = ("q", "k", "v", "o", "dout", "dq", "dk", "dv")
    vals = [x for n in names for x in ts.get(n, t4())]
    return CROSS_BWD.pack(B, H, Hk, M, N, D, dtype, lens_dtype, *vals, lens, lse, rest, delta, 0, scale)


@pytest.mark.parametrize("kw,status", [
    ({"M": 0}, 1), ({"dtype": F32}, 3), ({"H": 3}, 2), ({"D": 32}, 5), ({"scale": -1.0}, 5), ({"lse": 0}, 1),
    ({"delta": 0}, 1), ({"rest": P + 2}, 4), ({"dout": t4(0)}, 1), ({"dk": t4(P + 2)}, 4), ({"dq": t4(n=65)}, 4),
    ({"v": t4(b=-8)}, 1), ({"lens": P, "lens_dtype": 5}, 3), ({"N": 2 ** 30 + 5}, 5),
])
def test_cross_backward_abi(kw, status):
    assert _lib.lib().bsa_cross_bwd(_bwd(**kw), None) == status


def test_scaled_cross_backward_abi():
    assert _lib.lib().bsa_cross_bwd_scaled(_bwd(dtype=F32), P, None) == 3
    assert _lib.lib().bsa_cross_bwd_scaled(_bwd(), None, None) == 9
    assert _lib.lib().bsa_cross_bwd_scaled(None, P, None) == 1


def _prefix(B=2, H=4, Hk=2, T=1, Pn=100, C=10, D=64, dtype=F16, lens_dtype=0, lens=0, scale=0.125, **ts):
    vals = [x for n in ("q", "o", "kp", "vp", "k", "v") for x in ts.get(n, t4())]
    return PREFIX.pack(B, H, Hk, T, Pn, C, D, dtype, lens_dtype, *vals, lens, 0, 0, scale)


@pytest.mark.parametrize("kw,status", [
    ({}, 0), ({"Pn": 0}, 0), ({"C": 0}, 0), ({"Pn": 0, "C": 0}, 0), ({"T": 0}, 1), ({"C": -1}, 1), ({"dtype": F32}, 3),
    ({"H": 3}, 2), ({"D": 128 + 64}, 5), ({"kp": t4(0)}, 1), ({"vp": t4(P + 8)}, 4), ({"k": t4(n=66)}, 4),
    ({"lens": P, "lens_dtype": 3}, 3), ({"scale": float("nan")}, 5), ({"Pn": 2 ** 30 + 5}, 5), ({"C": 2 ** 30 + 5}, 5),
])
def test_prefix_abi(kw, status):
    assert _call("bsa_prefix_fwd_workspace_bytes", _prefix(**kw))[0] == status


def _rope(B=2, H=4, Hk=2, N=3, D=64, R=64, dtype=F16, wdtype=F32, qw=P, kw=P, cos=P, sin=P, stride=32, length=100, pdt=0,
          pos=0, eps=1e-6, dqw=0, **ts):
    vals = [x for n in ("q", "k", "qo", "ko", "dq", "dk") for x in ts.get(n, t4())]
    return ROPE.pack(B, H, Hk, N, D, R, dtype, wdtype, *vals, qw, kw, cos, sin, stride, length, pdt, pos, 0, eps, 0, dqw, 0,
                     0)


@pytest.mark.parametrize("kw,status", [
    ({"B": 0}, 1), ({"H": 0, "Hk": 0}, 1), ({"H": 2 ** 31 - 1, "Hk": 2 ** 31 - 1}, 5), ({"N": 0}, 1), ({"D": 60}, 5), ({"D": 264}, 5), ({"R": 24}, 5), ({"R": 80}, 5),
    ({"dtype": 7}, 3), ({"wdtype": BF16}, 3), ({"cos": 0}, 1), ({"sin": 0}, 1), ({"length": 0}, 1), ({"stride": 16}, 2),
    ({"stride": 33}, 4), ({"cos": P + 4}, 4), ({"pos": P, "pdt": 9}, 3), ({"eps": -1.0}, 1), ({"eps": float("nan")}, 1),
    ({"q": t4(0)}, 1), ({"ko": t4(P + 2)}, 4), ({"k": t4(n=68)}, 4),
])
def test_rope_abi(kw, status):
    assert _lib.lib().bsa_qk_norm_rope(_rope(**kw), None) == status


def test_rope_backward_abi():
    assert _call("bsa_qk_norm_rope_bwd_workspace_bytes", _rope()) == (0, 0)
    rc, n = _call("bsa_qk_norm_rope_bwd_workspace_bytes", _rope(dqw=P))
    assert rc == 0 and n > 0
    assert _call("bsa_qk_norm_rope_bwd_workspace_bytes", _rope(dq=t4(0)))[0] == 1
    assert _lib.lib().bsa_qk_norm_rope_bwd(_rope(dqw=P), P, n - 1, None) == 9


def test_structures_have_the_compiled_sizes(tmp_path):
    """The packed layouts above are the header's."""
    import shutil
    import subprocess
    from pathlib import Path

    src = tmp_path / "s.c"
    inc = Path(__file__).resolve().parent.parent / "include" / "bsattn_b200.h"
    src.write_text(f'#include <stdio.h>\n#include "{inc}"\nint main(void){{printf("%zu %zu %zu %zu", sizeof(bsa_rope_args), '
                   "sizeof(bsa_cross_args), sizeof(bsa_cross_bwd_args), sizeof(bsa_prefix_args));}\n")
    exe = tmp_path / "s"
    subprocess.run([shutil.which("gcc") or "cc", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    assert got == [ROPE.size, CROSS.size, CROSS_BWD.size, PREFIX.size]


def test_python_refuses_cpu_tensors():
    x = torch.zeros(1, 2, 3, 64, dtype=torch.float16)
    for call in (lambda: lib.cross_attention(x, x, x), lambda: lib.cross_attention_autograd(x, x, x),
                 lambda: lib.cross_attention_backward(x, x, x, x, torch.zeros(1, 2, 3), x),
                 lambda: lib.shared_prefix_attention(x, x[0], x[0], x, x), lambda: lib.qk_norm_rope(x, x),
                 lambda: lib.qk_norm_rope_autograd(x, None)):
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            call()
    with pytest.raises(ValueError, match="pass q or k"):
        lib.qk_norm_rope(None, None)
    with pytest.raises(TypeError):
        lib.cross_attention([1], x, x)
    with pytest.raises(ValueError):
        lib.rope_table(0, 64, device="cpu")
    with pytest.raises(ValueError):
        lib.rope_table(8, 63, device="cpu")


@pytest.mark.parametrize("dim,ok", [("60", False), ("264", False), ("8", True), ("256", True)])
def test_command_line_refuses_head_dims_the_norm_and_rotation_does_not_take(dim, ok, capsys):
    from blocksparsefa_reorder_b200.__main__ import parse_args

    args = ["pattern.mtx", "--head-dim", dim]
    assert parse_args(args).head_dim == int(dim)
    if ok:
        assert parse_args([*args, "--qk-norm-rope"]).qk_norm_rope
        return
    with pytest.raises(SystemExit):
        parse_args([*args, "--qk-norm-rope"])
    assert "multiple of 8" in capsys.readouterr().err


def test_rope_table_angles():
    cos, sin = lib.rope_table(200001, 64, base=1e6, device="cpu")
    assert cos.shape == sin.shape == (200001, 32) and cos.dtype == torch.float32
    ang = 200000.0 * 1e6 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert (cos[-1].double() - ang.cos()).abs().max() <= 2 ** -24 and (sin[-1].double() - ang.sin()).abs().max() <= 2 ** -24


def _places(t):
    """The byte addresses of every element, by enumeration."""
    at = torch.full(t.shape, t.data_ptr(), dtype=torch.int64)
    for i, (n, s) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * s * t.element_size()).view([n if j == i else 1 for j in range(t.dim())])
    return at.flatten().tolist()


def test_overlap_of_strided_views_matches_enumeration():
    """Random strided views of one buffer, dense, nested, interleaved and
    overlapping: the answers are those of their elements' addresses."""
    import random

    rng = random.Random(5)
    buf = torch.zeros(4000, dtype=torch.float16)
    seen = {0: 0, 1: 0, 2: 0}
    rows = {True: 0, False: 0}

    def view():
        t = buf
        size = [rng.choice((1, 2, 3, 4, 5)) for _ in range(4)]
        size[3] = rng.choice((1, 2, 4, 8))
        if rng.random() < 0.7:  # nested, in some order, with gaps
            order, stride, reach = rng.sample(range(3), 3), [0, 0, 0, 1], size[3]
            for i in order:
                stride[i] = reach + rng.choice((0, 0, 4, 8))
                reach = stride[i] * (size[i] - 1) + reach
        else:
            stride = [rng.choice((0, 1, 2, 4, 6, 8, 12, 20, 64, 100)) for _ in range(3)] + [1]
        span = sum(s * (n - 1) for s, n in zip(stride, size)) + 1
        at = rng.randrange(0, min(400, buf.numel() - span), 4)
        if rng.random() < 0.2 and all(s % 2 == 0 for s in stride[:3]) and size[3] > 1:
            t, size, stride = buf.view(torch.float32), size[:3] + [size[3] // 2], [s // 2 for s in stride[:3]] + [1]
            at //= 2
        return t.as_strided(size, stride, at)

    native = _lib.native()
    last = view()
    for _ in range(4000):
        a, b = view(), last if rng.random() < 0.5 else view()
        if rng.random() < 0.1:
            b = a.as_strided(a.shape, a.stride(), a.storage_offset())
        pa, pb = _places(a), _places(b)
        assert native.rows_overlap(a) == (len(set(pa)) < len(pa))
        rows[len(set(pa)) < len(pa)] += 1
        ba = {x + i for x in pa for i in range(a.element_size())}
        bb = {x + i for x in pb for i in range(b.element_size())}
        want = 1 if pa == pb and a.dtype == b.dtype and a.shape == b.shape else 2 if ba & bb else 0
        got = native.overlap(a, b)
        # (equal places with other strides, all of them stride 0 or of one element, are told as overlapping)
        assert got == want or (want == 1 and got == 2 and a.stride() != b.stride()), (a.shape, a.stride(), b.shape, b.stride())
        assert native.overlap(b, a) == got
        seen[got] += 1
        last = b
    assert min(seen.values()) > 100 and min(rows.values()) > 100


def test_overlap_of_the_operators_layouts():
    """Views of a fused projection and of a key cache: neighbours lie apart."""
    native = _lib.native()
    qkv = torch.zeros(2, 5, 12 * 64, dtype=torch.float16)

    def heads(h0, n):
        return qkv[..., h0 * 64:(h0 + n) * 64].view(2, 5, n, 64).transpose(1, 2)

    q, k, v = heads(0, 4), heads(4, 4), heads(8, 4)
    assert [native.overlap(q, k), native.overlap(k, v), native.overlap(q, heads(0, 4))] == [0, 0, 1]
    assert native.overlap(q, heads(1, 4)) == native.overlap(k, heads(3, 2)) == 2
    assert native.overlap(q, q[:, :, 1:]) == 2 and native.overlap(q[:, :, :2], q[:, :, 2:]) == 0
    cache = torch.zeros(2, 4, 100, 64, dtype=torch.float16)
    assert native.overlap(cache[:, :, 7:9], cache[:, :, 9:20]) == 0 and native.overlap(cache[:, :, 7:9], cache[:, :, 8:9]) == 2
    assert not any(native.rows_overlap(t) for t in (q, k, cache[:, :, 3:7], cache[:, :, :0], q[:, :, :1]))
    assert native.rows_overlap(q[:1].expand(2, -1, -1, -1)) and native.rows_overlap(cache.as_strided((1, 4, 5, 64), (0, 32, 128, 1)))


@pytest.mark.gpu
def test_outputs_over_other_memory_of_the_call(dev):
    """Outputs that are views of the buffers the call reads or of each other:
    refused where they meet, taken where they lie apart."""
    h = torch.float16
    qkv = torch.randn(2, 3, 14 * 64, dtype=h, device=dev)

    def heads(h0, n):
        return qkv[..., h0 * 64:(h0 + n) * 64].view(2, 3, n, 64).transpose(1, 2)

    q, k = heads(0, 4), heads(4, 2)
    lse = torch.zeros(2 * 4 * 3 + 8, device=dev)
    ln = torch.tensor([1, 2], device=dev, dtype=torch.int32)
    both = torch.zeros(2, 3, 6 * 64, dtype=h, device=dev)
    new = [both[..., a * 64:(a + n) * 64].view(2, 3, n, 64).transpose(1, 2) for a, n in ((0, 4), (2, 2), (4, 2))]
    kl = torch.zeros(2 * 4 * 3 * 64, dtype=h, device=dev)
    own_lens = kl.view(torch.int32)[:2]
    tab = torch.ones(48, 32, device=dev)
    bad = [
        lambda: lib.qk_norm_rope(q, None, cos=tab, sin=tab, out=(tab.view(h)[:24].view(2, 4, 3, 64), None)),
        lambda: lib.qk_norm_rope(q, k, out=(heads(1, 4), None)),
        lambda: lib.qk_norm_rope(q, None, out=(heads(1, 4), None)),
        lambda: lib.qk_norm_rope(q, k, out=(None, heads(3, 2))),
        lambda: lib.qk_norm_rope(q, k, out=(new[0], new[1])),
        lambda: lib.qk_norm_rope(q, None, out=(both.as_strided((2, 4, 3, 64), (3 * 384, 32, 384, 1)), None)),
        lambda: lib.cross_attention(q, k, k, out=heads(2, 4)),
        lambda: lib.cross_attention(q, heads(6, 2), heads(8, 2), out=heads(8, 4)),
        lambda: lib.cross_attention(q, k, k, out=heads(0, 4)),
        lambda: lib.cross_attention(q, k, k, out=heads(6, 4), o_rest=heads(8, 4)),
        lambda: lib.cross_attention(q, k, k, k_lens=own_lens, out=kl.view(2, 4, 3, 64)),
        lambda: lib.cross_attention(q, k, k, lse_out=qkv.view(-1).view(torch.float32)[:24].view(2, 4, 3)),
        lambda: lib.cross_attention(q, k, k, out=kl.view(2, 4, 3, 64), lse_out=kl.view(torch.float32)[-24:].view(2, 4, 3)),
        lambda: lib.shared_prefix_attention(q, k[0], k[0], k, k, out=heads(3, 4)),
        lambda: lib.shared_prefix_attention(q, k[0], k[0], k, k, lse_out=qkv.view(-1).view(torch.float32)[:24].view(2, 4, 3)),
        lambda: lib.shared_prefix_attention(q, k[0], k[0], k, k, lens=own_lens, out=kl.view(2, 4, 3, 64)),
    ]
    before = qkv.clone()
    for call in bad:
        with pytest.raises(ValueError, match="overlap|wrong shape"):
            call()
    torch.cuda.synchronize()
    assert torch.equal(qkv, before)
    # in place, and into other heads of the same buffer
    ref = lib.qk_norm_rope(q, k)
    o = lib.cross_attention(q, k, heads(6, 2), k_lens=ln)
    got = lib.cross_attention(q, k, heads(6, 2), k_lens=ln, out=heads(8, 4), lse_out=lse[:24].view(2, 4, 3))
    assert torch.equal(got, o)
    lib.qk_norm_rope(q, k, out=(heads(8, 4), heads(12, 2)))
    assert torch.equal(heads(8, 4), ref[0]) and torch.equal(heads(12, 2), ref[1])
    lib.qk_norm_rope(q, k, out=(heads(0, 4), heads(4, 2)))
    assert torch.equal(q, ref[0]) and torch.equal(k, ref[1]) and torch.equal(heads(6, 2), before[..., 384:512].view(2, 3, 2, 64).transpose(1, 2))


@pytest.mark.gpu
def test_python_refusals_on_the_gpu(dev):
    h = torch.float16
    q, k = torch.zeros(2, 4, 3, 64, dtype=h, device=dev), torch.zeros(2, 2, 9, 64, dtype=h, device=dev)
    ln = torch.tensor([1, 2], device=dev)
    flat = torch.zeros(q.numel() + 64, dtype=h, device=dev)
    bad = [
        (TypeError, lambda: lib.cross_attention(q.float(), k.float(), k.float())),
        (TypeError, lambda: lib.cross_attention(q, k.bfloat16(), k)),
        (ValueError, lambda: lib.cross_attention(q, k, k[:, :, :5])),
        (ValueError, lambda: lib.cross_attention(q, k[:1], k[:1])),
        (ValueError, lambda: lib.cross_attention(q[:, :3], k, k)),
        (ValueError, lambda: lib.cross_attention(q[0], k, k)),
        (ValueError, lambda: lib.cross_attention(q, k, k, sm_scale=0.0)),
        (ValueError, lambda: lib.cross_attention(q, k, k, k_lens=ln[:1])),
        (TypeError, lambda: lib.cross_attention(q, k, k, k_lens=ln.float())),
        (ValueError, lambda: lib.cross_attention(q, k, k, k_lens=ln.cpu())),
        (ValueError, lambda: lib.cross_attention(q, k, k, out=torch.zeros(2, 4, 3, 32, dtype=h, device=dev))),
        (ValueError, lambda: lib.cross_attention(q, k, k, lse_out=torch.zeros(2, 4, 4, device=dev))),
        (ValueError, lambda: lib.cross_attention(q.transpose(2, 3), k.transpose(2, 3), k.transpose(2, 3))),
        (_lib.BsaError, lambda: lib.cross_attention(q[..., :32].contiguous(), k[..., :32].contiguous(),
                                                    k[..., :32].contiguous())),
        (_lib.BsaError, lambda: lib.cross_attention(torch.zeros(2 * 4 * 3 * 64 + 1, dtype=h, device=dev)[1:].view(q.shape),
                                                    k, k)),
        (ValueError, lambda: lib.shared_prefix_attention(q, k[0, :1], k[0, :1], k, k)),
        (ValueError, lambda: lib.shared_prefix_attention(q, k, k, k, k)),
        (ValueError, lambda: lib.shared_prefix_attention(q, k[0], k[0], k, k, lens=ln[:1])),
        (ValueError, lambda: lib.qk_norm_rope(q, k)),
        (TypeError, lambda: lib.qk_norm_rope(q.int(), None)),
        (TypeError, lambda: lib.qk_norm_rope(q, None, torch.ones(64, device=dev, dtype=torch.bfloat16))),
        (ValueError, lambda: lib.qk_norm_rope(q, None, torch.ones(32, device=dev))),
        (ValueError, lambda: lib.qk_norm_rope(q, None, positions=ln)),
        (ValueError, lambda: lib.qk_norm_rope(q, None, cos=torch.ones(8, 32, device=dev))),
        (ValueError, lambda: lib.qk_norm_rope(q, None, cos=torch.ones(8, 32, device=dev), sin=torch.ones(8, 32, device=dev),
                                              positions=ln)),
        (ValueError, lambda: lib.qk_norm_rope(q, None, cos=torch.ones(1, 32, device=dev).expand(8, 32),
                                              sin=torch.ones(1, 32, device=dev).expand(8, 32))),
        (ValueError, lambda: lib.qk_norm_rope(q, None, eps=-1.0)),
        (ValueError, lambda: lib.qk_norm_rope(q, None, out=(q[:1], None))),
        # outputs whose rows overlap, lie over an input, or need a gradient
        (ValueError, lambda: lib.qk_norm_rope(q, None, out=(q[:1].expand(2, 4, 3, 64), None))),
        (ValueError, lambda: lib.qk_norm_rope(flat[:-64].view(q.shape), None, out=(flat[64:].view(q.shape), None))),
        (ValueError, lambda: lib.qk_norm_rope(q, q.clone(), out=(None, q))),
        (ValueError, lambda: lib.qk_norm_rope(q, None, out=(torch.zeros_like(q).requires_grad_(True), None))),
        (ValueError, lambda: lib.cross_attention(q, k, k, out=q[:1].expand(2, 4, 3, 64))),
        (ValueError, lambda: lib.cross_attention(q, k, k, out=q)),
        (ValueError, lambda: lib.cross_attention(q, q, q, out=q)),
        (ValueError, lambda: lib.cross_attention(q, k, k, o_rest=q)),
        (ValueError, lambda: lib.shared_prefix_attention(k, k[0], k[0], k, k, out=k)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    # the gradient of a gradient is refused, not silently wrong
    a, b = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    for o in (lib.cross_attention_autograd(a, b, b), lib.qk_norm_rope_autograd(a, None)[0]):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(o.float().sum(), a, create_graph=True)
    # a changed input is noticed, one that an output went into too
    c = q.clone().requires_grad_(True)
    x = c * 2
    y = x * x
    with torch.no_grad():
        lib.qk_norm_rope(x, None, out=(x, None))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    o = lib.cross_attention_autograd(a, b, b)
    with torch.no_grad():
        b.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["cross", "rope"])
def test_captured_backward_and_an_eager_graph_of_the_same_leaves(dev, op):
    """A capture whose gradient would go to the eager graph's (default) stream is
    refused; without that graph it is captured."""
    g = torch.Generator(device=dev).manual_seed(4)
    q = torch.randn(1, 2, 5, 64, device=dev, dtype=torch.float16, generator=g).requires_grad_(True)
    k = torch.randn(1, 2, 9, 64, device=dev, dtype=torch.float16, generator=g).requires_grad_(True)

    def forward():
        return lib.cross_attention_autograd(q, k, k) if op == "cross" else lib.qk_norm_rope_autograd(q, None)[0]

    def capture(step):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        return graph, out

    want, = torch.autograd.grad(forward().sum(), q)
    eager = forward()
    for step in (lambda: forward().sum().backward(), lambda: torch.autograd.grad(forward().sum(), q)):
        with pytest.raises(RuntimeError, match="captured backward pass"):
            capture(step)
        torch.cuda.synchronize()
    del eager
    graph, (got,) = capture(lambda: torch.autograd.grad(forward().sum(), q))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and q.grad is None
    graph, _ = capture(lambda: forward().sum().backward())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(q.grad, want)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["cross", "rope"])
@pytest.mark.parametrize("between", ["views", "products", "eager"])
def test_captured_backward_reaches_the_leaf_through_other_nodes(dev, op, between):
    """The same where views or products lie between the leaf and the operator, and
    where the eager graph itself is what the captured backward pass would run."""
    g = torch.Generator(device=dev).manual_seed(5)
    w = torch.randn(1, 7, 6 * 64, device=dev, dtype=torch.float16, generator=g).requires_grad_(True)

    def inputs():
        x = w * 0.5 if between == "products" else w
        return [x[..., a * 64:(a + n) * 64].view(1, 7, n, 64).transpose(1, 2) for a, n in ((0, 2), (2, 2), (4, 2))]

    def forward(qkv=None):
        q, k, v = qkv or inputs()
        return lib.cross_attention_autograd(q, k, v) if op == "cross" else lib.qk_norm_rope_autograd(q, k)[1]

    def capture(step):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        return graph, out

    want, = torch.autograd.grad(forward().sum(), w)
    held = inputs() if between == "eager" else None
    eager = None if held else forward()
    for step in (lambda: forward(held).sum().backward(), lambda: torch.autograd.grad(forward(held).sum(), w)):
        with pytest.raises(RuntimeError, match="captured backward pass"):
            capture(step)
        torch.cuda.synchronize()
    del eager, held
    graph, (got,) = capture(lambda: torch.autograd.grad(forward().sum(), w))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and w.grad is None
    graph, _ = capture(lambda: forward().sum().backward())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(w.grad, want)

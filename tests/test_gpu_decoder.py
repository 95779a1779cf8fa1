"""The operators together, as a decoder uses them: norm and rotation in front of
block-sparse and cross attention in training, and one decoding step over a
shared prefix and an encoder's states.

Tolerances: the attention gradients hold 1.5e-2 (bf16) and 3e-3 (fp16) of the
largest gradient each (their own tests); two of them and four roundings
of 16-bit tensors between the operators make 2 x that + 4 eps.  A decoding step
passes three roundings: 3 eps of the largest value, and the attentions' own
error (eps) each.
"""

import math

import pytest
import torch

from blocksparsefa_reorder_b200 import (block_sparse_attention, block_sparse_attention_autograd, cross_attention,
                                        cross_attention_autograd, qk_norm_rope, qk_norm_rope_autograd, rope_table,
                                        shared_prefix_attention)

pytestmark = pytest.mark.gpu


def _norm(x, w):
    return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w


def _turn(x, cos, sin, pos):
    c, s = cos.to(x.dtype)[pos], sin.to(x.dtype)[pos]
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat((a * c - b * s, a * s + b * c), -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_training_layer_gradients(dev, dtype):
    """Reordered tokens: positions are the permutation; self-attention over a
    block mask, then cross attention to padded encoder states."""
    torch.manual_seed(0)
    B, H, N, D, E = 2, 2, 384, 64, 200
    qkv = torch.randn(B, N, 3 * H * D, device=dev).to(dtype)
    enc_k, enc_v = (torch.randn(B, 1, E, D, device=dev).to(dtype) for _ in range(2))
    wq, wk, wc = (1 + 0.1 * torch.randn(D, device=dev) for _ in range(3))
    perm = torch.randperm(N, device=dev)
    cos, sin = rope_table(N, D, device=dev)
    mask = torch.rand(3, 3, device=dev) < 0.5
    mask |= torch.eye(3, dtype=torch.bool, device=dev)
    lens = torch.tensor([200, 77], device=dev)
    g = torch.randn(B, H, N, D, device=dev).to(dtype)

    leaves = [t.clone().requires_grad_(True) for t in (qkv, enc_k, enc_v, wq, wk, wc)]
    q, k, v = (t.view(B, N, H, D).transpose(1, 2) for t in leaves[0].split(H * D, -1))
    q, k = qk_norm_rope_autograd(q, k, leaves[3], leaves[4], positions=perm, cos=cos, sin=sin)
    o = block_sparse_attention_autograd(q, k, v.contiguous(), mask)
    c, _ = qk_norm_rope_autograd(o, None, leaves[5])
    y = cross_attention_autograd(c, leaves[1], leaves[2], k_lens=lens)
    grads = torch.autograd.grad(y, leaves, g)

    ref = [t.double().requires_grad_(True) for t in (qkv, enc_k, enc_v, wq, wk, wc)]
    q, k, v = (t.view(B, N, H, D).transpose(1, 2) for t in ref[0].split(H * D, -1))
    q, k = _turn(_norm(q, ref[3]), cos, sin, perm), _turn(_norm(k, ref[4]), cos, sin, perm)
    full = mask.repeat_interleave(128, 0).repeat_interleave(128, 1)
    o = ((q @ k.transpose(-1, -2)) / math.sqrt(D)).masked_fill(~full, -math.inf).softmax(-1) @ v
    c = _norm(o, ref[5])
    gone = (torch.arange(E, device=dev) >= lens[:, None])[:, None, None]
    yr = ((c @ ref[1].transpose(-1, -2)) / math.sqrt(D)).masked_fill(gone, -math.inf).softmax(-1) @ ref[2]
    rgrads = torch.autograd.grad(yr, ref, g.double())
    eps = torch.finfo(dtype).eps
    tol = 2 * (1.5e-2 if dtype == torch.bfloat16 else 3e-3) + 4 * eps
    assert (y.double() - yr).abs().max() <= tol * yr.abs().max()
    for name, a, r in zip(("qkv", "enc k", "enc v", "wq", "wk", "wc"), grads, rgrads):
        assert a.shape == r.shape and (a.double() - r).abs().max() <= tol * r.abs().max(), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decoding_steps_behind_a_prefix(dev, dtype):
    """Three steps of four sequences: the new token's key is normed and rotated
    into the cache, the prefix attended once for all, then the encoder; eagerly
    and as one captured graph, against plain attention over everything."""
    torch.manual_seed(1)
    B, H, Hk, P, C, E, D = 4, 8, 2, 300, 16, 150, 64
    cos, sin = rope_table(P + C, D, device=dev)
    wq, wk = (1 + 0.1 * torch.randn(D, device=dev) for _ in range(2))
    raw_p, vp = (torch.randn(1, Hk, P, D, device=dev).to(dtype) for _ in range(2))
    _, kp = qk_norm_rope(None, raw_p, None, wk, cos=cos, sin=sin)
    ek, ev = (torch.randn(B, Hk, E, D, device=dev).to(dtype) for _ in range(2))
    elens = torch.tensor([150, 1, 0, 99], device=dev)
    ck, cv = (torch.zeros(B, Hk, C, D, device=dev, dtype=dtype) for _ in range(2))
    lens = torch.zeros(B, dtype=torch.int32, device=dev)
    pos = torch.zeros(B, 1, dtype=torch.int64, device=dev)
    x, xk, xv = (torch.zeros(B, h, 1, D, device=dev, dtype=dtype) for h in (H, Hk, Hk))
    rows = torch.arange(B, device=dev)

    def step():
        lens.add_(1)
        q, k = qk_norm_rope(x, xk, wq, wk, positions=pos, cos=cos, sin=sin)
        at = lens.long() - 1
        ck[rows, :, at] = k[:, :, 0]
        cv[rows, :, at] = xv[:, :, 0]
        o = shared_prefix_attention(q, kp[0], vp[0], ck, cv, lens=lens)
        c, _ = qk_norm_rope(o, None, wq)
        return o, cross_attention(c, ek, ev, k_lens=elens)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    eps = torch.finfo(dtype).eps
    for run in ("eager", "graph"):
        lens.zero_(), ck.zero_(), cv.zero_()
        keys, values = [], []
        for t in range(3):
            for buf in (x, xk, xv):
                buf.copy_(torch.randn(buf.shape, device=dev))
            pos.fill_(P + t)
            if run == "graph":
                graph.replay()
                o, y = captured
            else:
                o, y = step()
            keys.append(_turn(_norm(xk.double(), wk), cos, sin, pos[0])), values.append(xv.double())
            q = _turn(_norm(x.double(), wq), cos, sin, pos[0])
            kk = torch.cat((kp.double().expand(B, -1, -1, -1), *keys), 2).repeat_interleave(H // Hk, 1)
            vv = torch.cat((vp.double().expand(B, -1, -1, -1), *values), 2).repeat_interleave(H // Hk, 1)
            ro = ((q @ kk.transpose(-1, -2)) / math.sqrt(D)).softmax(-1) @ vv
            assert (o.double() - ro).abs().max() <= 4 * eps * max(1.0, ro.abs().max().item()), (run, t)
            c = _norm(ro, wq)
            for b, n in enumerate(elens.tolist()):
                if n == 0:
                    assert (y[b] == 0).all()
                    continue
                kb = ek[b, :, :n].double().repeat_interleave(H // Hk, 0)
                vb = ev[b, :, :n].double().repeat_interleave(H // Hk, 0)
                ry = ((c[b] @ kb.transpose(-1, -2)) / math.sqrt(D)).softmax(-1) @ vb
                # o's error is taken up by the norm: relative to o's size, not to 1
                size = ro[b].square().mean(-1).sqrt().min().item()
                assert (y[b].double() - ry).abs().max() <= (4 * eps / size + 4 * eps) * vb.abs().max(), (run, t, b)


def test_norm_and_rotation_in_front_of_the_reordered_forward(dev):
    """Rotating the original order and reordering inside the attention equals
    rotating reordered rows by their true positions."""
    torch.manual_seed(2)
    B, H, N, D = 1, 2, 256, 64
    q, k, v = (torch.randn(B, H, N, D, device=dev, dtype=torch.float16) for _ in range(3))
    w = 1 + 0.1 * torch.randn(D, device=dev)
    perm = torch.randperm(N, device=dev)
    cos, sin = rope_table(N, D, device=dev)
    mask = torch.tensor([[True, False], [True, True]], device=dev)
    a, b = qk_norm_rope(q, k, w, w, cos=cos, sin=sin)
    o = block_sparse_attention(a, b, v, mask, q_perm=perm, kv_perm=perm)
    a, b = qk_norm_rope(q[:, :, perm], k[:, :, perm], w, w, positions=perm, cos=cos, sin=sin)
    o2 = block_sparse_attention(a, b, v[:, :, perm].contiguous(), mask)
    assert torch.equal(o[:, :, perm], o2)


def test_runner_times_the_norm_and_rotation(dev, capsys):
    from blocksparsefa_reorder_b200.runners import run_experiments_B200
    from blocksparsefa_reorder_b200.utils import Args

    args = Args(matrix_mtx=None, block_size=128, head_dim=64, num_heads=2, row_reorder=None, col_reorder=None, mode="B200")
    mask = torch.ones(1, 2, 2, 2, dtype=torch.bool, device=dev)
    perm = torch.randperm(256, device=dev)
    r = run_experiments_B200(args, mask, 256, row_perm=perm, col_perm=perm, warmup=1, reps=2, qk_norm_rope=True)
    assert r["ms_with_norm_rope"] > 0 and "Average time with norm, rotation and reordering" in capsys.readouterr().out
    r = run_experiments_B200(args, mask, 256, warmup=1, reps=2)
    assert "ms_with_norm_rope" not in r

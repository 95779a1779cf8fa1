"""The attention-side operators of language models as measured cases.

Each case is one call (or one training step) of an operator of this library:

* ``qk_norm_rope``: root-mean-square norm of every query and key head and the
  rotation of its position, in one pass, with its gradient;
* ``cross_attention``: queries of one length over an encoder's states of
  another, padded per sequence, with shared key / value heads, with its gradient;
* ``shared_prefix_attention``: a batch of sequences that continue one long
  prefix: the prefix is attended once for all of them, each sequence's own
  keys behind it.

``run`` computes them in plain torch operations in 32 bits, or, where ``own``
is set, calls this library.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
LOG2E = 1.4426950408889634


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _rope(name, B, H, Hk, N, D, R, dtype, interleaved=False, train=False, fused_qkv=False, span=65536):
    """B sequences of N tokens, H query and Hk key heads of D, the first R dimensions rotated; positions up to `span`."""
    return {"name": name, "op": "rope", "B": B, "H": H, "Hk": Hk, "N": N, "D": D, "R": R, "dtype": dtype,
            "interleaved": interleaved, "train": train, "fused_qkv": fused_qkv, "span": span}


def _cross(name, B, H, Hk, M, N, D, dtype, lo, train=False):
    """M queries a sequence over N encoder states, of which from `lo` to N are valid, evenly spread over the batch."""
    return {"name": name, "op": "cross", "B": B, "H": H, "Hk": Hk, "M": M, "N": N, "D": D, "dtype": dtype, "lo": lo,
            "train": train}


def _prefix(name, B, H, Hk, T, P, C, D, dtype, lo):
    """T new tokens of B sequences behind P shared keys; each sequence holds from `lo` to C keys of its own."""
    return {"name": name, "op": "prefix", "B": B, "H": H, "Hk": Hk, "T": T, "P": P, "C": C, "D": D, "dtype": dtype,
            "lo": lo}


def listed():
    return [
        # one decoding step of 8 sequences at far positions: latency alone
        _rope("rope_token", 8, 16, 4, 1, 128, 128, "bf16"),
        # a whole prompt at the benchmark's size (16 heads, 16384 tokens), its tokens reordered: positions permuted
        _rope("rope_prompt", 1, 16, 16, 16384, 128, 128, "bf16", span=16384),
        # a training step on views of a fused projection's output, neighbouring pairs rotated
        _rope("rope_train", 2, 16, 4, 8192, 64, 64, "fp16", interleaved=True, train=True, fused_qkv=True, span=8192),
        # a training step in 32 bits, odd sizes, half of each head rotated
        _rope("rope_train_odd", 3, 12, 3, 1531, 128, 64, "fp32", train=True, span=4096),
        # a translation or speech decoder's step: one token a sequence over a padded batch of encoder states
        _cross("cross_token", 16, 16, 16, 1, 1500, 64, "fp16", 211),
        # one token over the long-context configuration's 65536 states, key / value heads shared by four
        _cross("cross_token_long", 4, 32, 8, 1, 65536, 128, "bf16", 16000),
        # a prompt's tokens over long encoded documents, at the benchmark's heads
        _cross("cross_forward", 1, 16, 16, 4096, 16384, 128, "bf16", 16384),
        # a training step of an encoder-decoder layer with shared key / value heads
        _cross("cross_train", 2, 16, 4, 2048, 4096, 128, "bf16", 4001, train=True),
        # a training step of a padded batch, odd lengths, one sequence without any encoder state
        _cross("cross_train_odd", 3, 6, 2, 777, 1531, 64, "fp16", 0, train=True),
        # a few chats behind a short system prompt
        _prefix("prefix_small", 4, 16, 4, 1, 1000, 64, 64, "fp16", 1),
        # a serving batch behind a long document
        _prefix("prefix_serve", 64, 32, 8, 1, 32768, 512, 128, "bf16", 9),
        # drafted tokens checked at once: several queries a sequence
        _prefix("prefix_draft", 16, 16, 4, 7, 8192, 301, 128, "bf16", 7),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("rope", "cross", "cross", "prefix"))
    if op == "rope":
        Hk = rng.choice((1, 2, 3, 4, 8, 16))
        H = Hk * rng.choice((1, 2, 4))
        D = rng.choice((32, 64, 96, 128, 256))
        B = rng.randint(1, 8)
        N = _log(rng, 1, 16384)
        train = rng.random() < 0.5
        # at most the largest case's elements
        N = max(1, min(N, (60_000_000 if not train else 30_000_000) // (B * (H + Hk) * D)))
        return {k: v for k, v in _rope("", B, H, Hk, N, D, D if rng.random() < 0.6 else D // 2,
                                       rng.choice(("bf16", "fp16", "fp32")), rng.random() < 0.4, train,
                                       rng.random() < 0.5, max(N, _log(rng, 64, 131072))).items() if k != "name"}
    Hk = rng.choice((1, 2, 4, 8, 16))
    H = min(32, Hk * rng.choice((1, 2, 3, 4, 8)) if Hk < 16 else Hk * rng.choice((1, 2)))
    D, dtype = rng.choice((64, 128)), rng.choice(("bf16", "fp16"))
    if op == "cross":
        B = rng.randint(1, 16)
        M = rng.randint(1, 4) if rng.random() < 0.4 else _log(rng, 5, 4096)
        N = _log(rng, 1, 65536 if M <= 4 else 16384)
        train = M > 4 and rng.random() < 0.5
        # at most the largest case's products and stored scores
        most = (1 << 30) // (B * H * M)
        N = min(N, most // 4 if train else most, (1 << 31) // (B * Hk * 1024))
        # (a softmax over one key has no gradient but rounding: training starts at 16 states)
        N = max(16 if train else 1, N)
        lo = rng.randint(0, N)
        return {k: v for k, v in _cross("", B, H, Hk, M, N, D, dtype, lo, train).items() if k != "name"}
    B = _log(rng, 1, 96)
    T = 1 if rng.random() < 0.6 else rng.randint(2, 24)
    P = _log(rng, 1, 32768)
    C = T + _log(rng, 1, 1024)
    P = max(1, min(P, (1 << 27) // (B * H * T)))
    lo = rng.randint(T, C)
    return {k: v for k, v in _prefix("", B, H, Hk, T, P, C, D, dtype, lo).items() if k != "name"}


def _lens(case, n, count):
    """Valid keys of each sequence: `lo` .. n evenly spread (one sequence: n)."""
    if count == 1:
        return [n]
    return [case["lo"] + round((n - case["lo"]) * i / (count - 1)) for i in range(count)]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt, scale=1.0):
        x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32 if dtype == torch.float32 else dtype)
        return x if scale == 1.0 else x.mul_(scale)

    s = {"case": case}
    if case["op"] == "rope":
        B, H, Hk, N, D, R = (case[x] for x in ("B", "H", "Hk", "N", "D", "R"))
        if case["fused_qkv"]:
            # the output of one projection [B, N, (H + 2 Hk) D]: queries, keys and values side by side
            qkv = randn(B, N, (H + 2 * Hk) * D)
            s["q"] = qkv[..., :H * D].view(B, N, H, D).transpose(1, 2)
            s["k"] = qkv[..., H * D:(H + Hk) * D].view(B, N, Hk, D).transpose(1, 2)
        else:
            s["q"], s["k"] = randn(B, H, N, D), randn(B, Hk, N, D)
        s["wq"] = 1 + 0.2 * randn(D, dtype=torch.float32)
        s["wk"] = 1 + 0.2 * randn(D, dtype=torch.float32)
        # distinct positions of each sequence where the span allows it, as reordered or sampled tokens have them
        pos = torch.rand(B, case["span"], generator=g, device="cuda").argsort(1)[:, :N] if case["span"] >= N else None
        s["positions"] = pos.to(torch.int32).contiguous()
        # the rotation's table, kept by the program: angles in 64 bits
        inv = 10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
        ang = torch.arange(case["span"], device="cuda", dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        if case["train"]:
            s["dq"], s["dk"] = randn(B, H, N, D), randn(B, Hk, N, D)
        return s
    if case["op"] == "cross":
        B, H, Hk, M, N, D = (case[x] for x in ("B", "H", "Hk", "M", "N", "D"))
        # score deviation 1.5: a softmax with some dozens of keys that matter
        s["q"], s["k"], s["v"] = randn(B, H, M, D, scale=1.5), randn(B, Hk, N, D), randn(B, Hk, N, D)
        if case["train"]:
            s["do"] = randn(B, H, M, D)
        lens = _lens(case, N, B)
    else:
        B, H, Hk, T, P, C, D = (case[x] for x in ("B", "H", "Hk", "T", "P", "C", "D"))
        s["q"], s["kp"], s["vp"] = randn(B, H, T, D, scale=1.5), randn(Hk, P, D), randn(Hk, P, D)
        s["k"], s["v"] = randn(B, Hk, C, D), randn(B, Hk, C, D)
        lens = _lens(case, C, B)
    order = torch.randperm(B, generator=g, device="cuda")
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")[order].contiguous()
    return s


# ---------------------------------------------------------------------------
# Plain forms: elementary operations in 32 bits, rounded once
# ---------------------------------------------------------------------------
def _pairs(x, interleaved):
    """The two halves of the rotated pairs of x [..., R]."""
    h = x.shape[-1] // 2
    return (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :h], x[..., h:])


def _turn(x, c, s, R, interleaved):
    a, b = _pairs(x[..., :R], interleaved)
    y0, y1 = a * c - b * s, a * s + b * c
    y = torch.stack((y0, y1), -1).flatten(-2) if interleaved else torch.cat((y0, y1), -1)
    return torch.cat((y, x[..., R:]), -1)


def _plain_rope(st):
    case = st["case"]
    R, il = case["R"], case["interleaved"]
    at = st["positions"].long()
    c, s = st["cos"][at][:, None], st["sin"][at][:, None]

    def forward(x, w):
        xf = x.float()
        r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
        return _turn(xf * r * w, c, s, R, il).to(x.dtype)

    def backward(x, w, dy):
        xf = x.float()
        r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
        n = xf * r
        t = _turn(dy.float(), c, -s, R, il)  # the rotation turned back
        dw = (t * n).sum((0, 1, 2))
        t = t * w
        return ((t - n * (t * n).mean(-1, keepdim=True)) * r).to(x.dtype), dw

    q, k = forward(st["q"], st["wq"]), forward(st["k"], st["wk"])
    if not case["train"]:
        return q, k
    dq, dwq = backward(st["q"], st["wq"], st["dq"])
    dk, dwk = backward(st["k"], st["wk"], st["dk"])
    return q, k, dq, dk, dwq, dwk


def _softmax(s):
    """Weights not yet divided, their sums, and the log2 of the scores' sum of exponentials."""
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = (s - m).exp()
    l = p.sum(-1, keepdim=True)
    return p, l, (m + l.log()) * LOG2E


def _plain_cross(st):
    case = st["case"]
    B, H, Hk, M, N, D = (case[x] for x in ("B", "H", "Hk", "M", "N", "D"))
    scale = 1 / math.sqrt(D)
    q = st["q"].float().view(B, Hk, H // Hk * M, D)
    k, v = st["k"].float(), st["v"].float()
    gone = torch.arange(N, device="cuda") >= st["lens"][:, None, None, None]
    p, l, lse = _softmax((q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(gone, -math.inf))
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    of = p @ v
    o = of.to(st["q"].dtype).view(B, H, M, D)
    if not case["train"]:
        return o, lse.view(B, H, M)
    do = st["do"].float().view(q.shape)
    ds = p * (do @ v.transpose(-1, -2) - (do * of).sum(-1, keepdim=True))
    dq, dk, dv = (ds @ k) * scale, (ds.transpose(-1, -2) @ q) * scale, p.transpose(-1, -2) @ do
    return o, dq.view(B, H, M, D).to(o.dtype), dk.to(o.dtype), dv.to(o.dtype)


def _plain_prefix(st):
    case = st["case"]
    B, H, Hk, T, P, C, D = (case[x] for x in ("B", "H", "Hk", "T", "P", "C", "D"))
    G, scale = H // Hk, 1 / math.sqrt(D)
    q = st["q"].float().view(B, Hk, G * T, D)
    # the prefix once for all: the batch's queries are the rows of one product for each key head
    sp = q.transpose(0, 1).reshape(Hk, B * G * T, D) @ st["kp"].float().transpose(-1, -2)
    sp = sp.view(Hk, B, G * T, P).transpose(0, 1)
    ss = q @ st["k"].float().transpose(-1, -2)
    t = torch.arange(T, device="cuda").repeat(G)[:, None]
    seen = torch.arange(C, device="cuda") < (st["lens"][:, None, None, None] - (T - 1 - t))
    p, l, lse = _softmax(torch.cat((sp, ss.masked_fill(~seen, -math.inf)), -1) * scale)
    pp = p[..., :P].transpose(0, 1).reshape(Hk, B * G * T, P)
    o = (pp @ st["vp"].float()).view(Hk, B, G * T, D).transpose(0, 1) + p[..., P:] @ st["v"].float()
    o = o / torch.where(l > 0, l, torch.ones_like(l))
    return o.to(st["q"].dtype).reshape(B, H, T, D)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _own_rope(st):
    from blocksparsefa_reorder_b200 import qk_norm_rope, qk_norm_rope_autograd

    case = st["case"]
    kw = dict(positions=st["positions"], cos=st["cos"], sin=st["sin"], eps=EPS, interleaved=case["interleaved"])
    if not case["train"]:
        return qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], **kw)
    leaves = [st[x].detach().requires_grad_(True) for x in ("q", "k", "wq", "wk")]
    q, k = qk_norm_rope_autograd(*leaves, **kw)
    dq, dk, dwq, dwk = torch.autograd.grad((q, k), leaves, (st["dq"], st["dk"]))
    return q.detach(), k.detach(), dq, dk, dwq, dwk


def _own_cross(st):
    from blocksparsefa_reorder_b200 import cross_attention, cross_attention_autograd

    if not st["case"]["train"]:
        return cross_attention(st["q"], st["k"], st["v"], k_lens=st["lens"], return_lse=True)
    leaves = [st[x].detach().requires_grad_(True) for x in ("q", "k", "v")]
    o = cross_attention_autograd(*leaves, k_lens=st["lens"])
    return (o.detach(), *torch.autograd.grad(o, leaves, st["do"]))


def _own_prefix(st):
    from blocksparsefa_reorder_b200 import shared_prefix_attention

    return shared_prefix_attention(st["q"], st["kp"], st["vp"], st["k"], st["v"], lens=st["lens"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rope": _own_rope, "cross": _own_cross, "prefix": _own_prefix}[op](state)
    return {"rope": _plain_rope, "cross": _plain_cross, "prefix": _plain_prefix}[op](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rope":
        B, H, Hk, N, D, R = (case[x] for x in ("B", "H", "Hk", "N", "D", "R"))
        x = B * (H + Hk) * N * D
        # each position's row of the table once, at most the table
        table = min(B * N, case["span"]) * R * 4 + B * N * 4
        if not case["train"]:
            return {"bytes": 2 * x * e + table + 8 * D, "flops": 7 * x}
        # forward: x in, y out; backward: x and dy in, dx out (x is read by both, as the two are separate calls)
        return {"bytes": 5 * x * e + 2 * table + 24 * D, "flops": 22 * x}
    B, H, Hk, D = (case[x] for x in ("B", "H", "Hk", "D"))
    if case["op"] == "cross":
        M, keys = case["M"], sum(_lens(case, case["N"], B))
        q, kv, pairs = B * H * M * D * e, 2 * keys * Hk * D * e, H * M * keys
        if not case["train"]:
            return {"bytes": 2 * q + kv + 4 * B * H * M + 4 * B, "flops": 4 * pairs * D}
        # the backward's gradients of k and v are written whole, padded rows too; it reads q, k, v, o and do again
        full = 2 * B * Hk * case["N"] * D * e
        return {"bytes": 2 * q + kv + 3 * q + kv + q + full + 8 * B, "flops": 14 * pairs * D}
    T, P = case["T"], case["P"]
    keys = sum(_lens(case, case["C"], B))
    q = B * H * T * D * e
    return {"bytes": 2 * q + 2 * P * Hk * D * e + 2 * keys * Hk * D * e + 4 * B,
            "flops": 4 * H * T * D * (B * P + keys)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rope(st):
    case = st["case"]
    R, il = case["R"], case["interleaved"]
    turn = torch.complex(st["cos"].double(), st["sin"].double())[st["positions"].long()][:, None]

    def op(x, w):
        y = x / ((x ** 2).mean(-1, keepdim=True) + EPS).sqrt() * w
        z = y[..., :R]
        z = torch.view_as_complex(z.unflatten(-1, (R // 2, 2)).contiguous()) if il else \
            torch.view_as_complex(z.unflatten(-1, (2, R // 2)).transpose(-1, -2).contiguous())
        z = torch.view_as_real(z * turn)
        z = z.flatten(-2) if il else z.transpose(-1, -2).flatten(-2)
        return torch.cat((z, y[..., R:]), -1)

    x = [st[n].double().requires_grad_(True) for n in ("q", "k", "wq", "wk")]
    q, k = op(x[0], x[2]), op(x[1], x[3])
    if not case["train"]:
        return q.detach(), k.detach()
    g = torch.autograd.grad((q, k), x, (st["dq"].double(), st["dk"].double()))
    return (q.detach(), k.detach(), *g)


def _exact_cross(st):
    case = st["case"]
    B, H, Hk, M, N, D = (case[x] for x in ("B", "H", "Hk", "M", "N", "D"))
    o = torch.zeros(B, H, M, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, M), -math.inf, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(B, h, n, D, dtype=torch.float64, device="cuda") for h, n in ((H, M), (Hk, N), (Hk, N))]
    for b, n in enumerate(st["lens"].tolist()):
        for h in range(H):
            if not n:
                continue
            j = h // (H // Hk)
            q, k, v = st["q"][b, h].double(), st["k"][b, j, :n].double(), st["v"][b, j, :n].double()
            s = torch.einsum("md,nd->mn", q, k) / math.sqrt(D)
            lse[b, h] = s.logsumexp(-1) / math.log(2)
            p = s.softmax(-1)
            o[b, h] = p @ v
            if case["train"]:
                do = st["do"][b, h].double()
                dp = do @ v.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(D)
                grads[0][b, h] = ds @ k
                grads[1][b, j, :n] += ds.T @ q
                grads[2][b, j, :n] += p.T @ do
    return (o, *grads) if case["train"] else (o, lse)


def _exact_prefix(st):
    case = st["case"]
    B, H, Hk, T, D = (case[x] for x in ("B", "H", "Hk", "T", "D"))
    G = H // Hk
    o = torch.zeros(B, H, T, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["lens"].tolist()):
        for t in range(T):
            own_keys = max(0, n - (T - 1 - t))
            k = torch.cat((st["kp"], st["k"][b, :, :own_keys]), 1).double()
            v = torch.cat((st["vp"], st["v"][b, :, :own_keys]), 1).double()
            q = st["q"][b, :, t].double().view(Hk, G, D)
            o[b, :, t] = ((q @ k.transpose(1, 2) / math.sqrt(D)).softmax(-1) @ v).view(H, D)
    return o


def exact(case, seed):
    st = prepare(case, seed)
    return {"rope": _exact_rope, "cross": _exact_cross, "prefix": _exact_prefix}[case["op"]](st)

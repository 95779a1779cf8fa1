"""Norm of every query and key head and the rotation of its position, fused.

The step in front of an attention call: one pass over q and k that scales each
head's row to unit root mean square, multiplies the norm's weight in and turns
the row by its token's position, and the gradient of that pass.  The tensors
are the ``[B, H, N, D]`` views :func:`~blocksparsefa_reorder_b200.block_sparse_attention`
takes, so views of a fused projection need no copy and the outputs go straight
into it; with reordered tokens, ``positions`` are the permutation itself
(``perm[i]`` = the old, i.e. true, position of row ``i``).
The reference has no counterpart: its inputs are q and k as attention takes
them.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .api import _DTYPES, _check_err, _require_cuda, _stream

_INDEX = {torch.int32: _lib.INDEX_I32, torch.int64: _lib.INDEX_I64}


def rope_table(length: int, dim: int, base: float = 10000.0, device="cuda"):
    """``(cos, sin)``, each float32 ``[length, dim / 2]``: the angles
    ``pos * base^(-2 i / dim)`` of every position below ``length``, computed in
    64 bits (a far position's angle has lost its fraction in 32)."""
    if dim <= 0 or dim % 2:
        raise ValueError(f"dim must be even and positive, got {dim}")
    if length <= 0:
        raise ValueError(f"length must be positive, got {length}")
    inv = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    ang = torch.arange(length, dtype=torch.float64, device=device)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _check_side(x, w, name: str, like=None):
    _require_cuda(x, name)
    if x.dim() != 4:
        raise ValueError(f"{name} must be [B, H, N, D], got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {x.dtype}")
    if like is not None:
        if (x.shape[0], x.shape[2], x.shape[3]) != (like.shape[0], like.shape[2], like.shape[3]):
            raise ValueError(f"q and k must share B, N and D, got {tuple(like.shape)} and {tuple(x.shape)}")
        if x.dtype != like.dtype:
            raise TypeError(f"q and k must share a dtype, got {like.dtype} and {x.dtype}")
        if x.device != like.device:
            raise ValueError("q and k must be on one device")
    if w is not None:
        _require_cuda(w, f"{name}_weight")
        if tuple(w.shape) != (x.shape[3],) or not w.is_contiguous():
            raise ValueError(f"{name}_weight must be a contiguous [{x.shape[3]}] tensor, got {tuple(w.shape)}")
        if w.dtype not in (torch.float32, x.dtype):
            raise TypeError(f"{name}_weight must be float32 or {x.dtype}, got {w.dtype}")
        if w.device != x.device:
            raise ValueError(f"{name}_weight is on another device")


def _t4(t: torch.Tensor, name: str) -> _lib.Tensor4d:
    if t.stride(3) != 1 and t.shape[3] > 1:
        raise ValueError(f"the last (head) dimension of {name} must be contiguous")
    return _lib.Tensor4d(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _out(out, x, name: str) -> torch.Tensor:
    if out is None:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{name} has the wrong shape, dtype or device")
    return out


def _args(q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved):
    """Checks, and the C arguments but for the outputs."""
    if q is None and k is None:
        raise ValueError("pass q or k")
    if q is not None:
        _check_side(q, q_weight, "q")
    if k is not None:
        _check_side(k, k_weight, "k", q)
    x = q if q is not None else k
    a = _lib.RopeArgs()
    a.B, a.N, a.D = x.shape[0], x.shape[2], x.shape[3]
    a.H = q.shape[1] if q is not None else 0
    a.Hk = k.shape[1] if k is not None else 0
    a.dtype = _DTYPES[x.dtype]
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise TypeError("q_weight and k_weight must share a dtype")
    w = q_weight if q_weight is not None else k_weight
    a.weight_dtype = _DTYPES[w.dtype] if w is not None else a.dtype
    if q is not None:
        a.q = _t4(q, "q")
        a.q_weight = q_weight.data_ptr() if q_weight is not None else None
    if k is not None:
        a.k = _t4(k, "k")
        a.k_weight = k_weight.data_ptr() if k_weight is not None else None
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    a.eps = eps
    a.interleaved = 1 if interleaved else 0
    if (cos is None) != (sin is None):
        raise ValueError("pass both cos and sin, or neither (norm only)")
    if cos is None:
        if positions is not None:
            raise ValueError("positions need the cos and sin tables")
        return a, x
    for name, t in (("cos", cos), ("sin", sin)):
        _require_cuda(t, name)
        if t.dtype != torch.float32 or t.dim() != 2:
            raise TypeError(f"{name} must be a float32 [length, R / 2] table")
        if t.device != x.device:
            raise ValueError(f"{name} is on another device")
    if cos.shape != sin.shape or cos.stride() != sin.stride() or cos.stride(1) != 1:
        raise ValueError("cos and sin must share their shape and strides, with contiguous rows")
    a.R = 2 * cos.shape[1]
    a.cos, a.sin, a.table_len = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
    a.table_stride = max(cos.stride(0), cos.shape[1])
    if positions is not None:
        _require_cuda(positions, "positions")
        if positions.dtype not in _INDEX:
            raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.device != x.device:
            raise ValueError("positions are on another device")
        if tuple(positions.shape) not in ((a.N,), (a.B, a.N)) or (positions.stride(-1) != 1 and a.N > 1):
            raise ValueError(f"positions must be [{a.N}] or [{a.B}, {a.N}] with contiguous rows, "
                             f"got {tuple(positions.shape)}")
        a.positions, a.pos_dtype = positions.data_ptr(), _INDEX[positions.dtype]
        a.pos_stride_b = positions.stride(0) if positions.dim() == 2 else 0
    return a, x


def qk_norm_rope(q: Optional[torch.Tensor], k: Optional[torch.Tensor], q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, *, positions: Optional[torch.Tensor] = None,
                 cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False, out=None, check_errors: bool = False):
    """``R(pos) (x / sqrt(mean(x^2) + eps) * w)`` of every row of q and k.

    q: CUDA ``[B, H, N, D]``, k: ``[B, Hk, N, D]`` (any number of heads), one
    dtype of bf16 / fp16 / fp32, last dim contiguous, rows 16-byte aligned, D a
    multiple of 8 up to 256; either may be None (that output is None then).
    q_weight / k_weight: ``[D]`` in float32 or q's dtype, None = ones.
    cos, sin: float32 ``[length, R / 2]`` tables (:func:`rope_table`), R a
    multiple of 16 up to D: the first R dimensions are rotated, in pairs
    ``(i, i + R / 2)`` or, with ``interleaved``, ``(2 i, 2 i + 1)``.  None: no
    rotation.  positions: int ``[N]`` or ``[B, N]`` rows of the tables, None =
    0 .. N - 1.  A position outside the tables gives a NaN row, and an error
    with ``check_errors`` (which synchronises).
    out: optional ``(q_out, k_out)``, e.g. views of a key cache or the inputs
    themselves.  Returns ``(q_out, k_out)``; sums, norm and rotation are fp32,
    rounded once.
    """
    a, x = _args(q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved)
    oq, ok = out if out is not None else (None, None)
    oq = _out(oq, q, "q_out") if q is not None else None
    ok = _out(ok, k, "k_out") if k is not None else None
    if x.shape[0] == 0 or x.shape[2] == 0 or a.H + a.Hk == 0:
        return oq, ok
    if oq is not None:
        a.q_out = _t4(oq, "q_out")
    if ok is not None:
        a.k_out = _t4(ok, "k_out")
    err = torch.zeros(1, dtype=torch.int32, device=x.device) if check_errors else None
    a.err_flag = err.data_ptr() if err is not None else None
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().bsa_qk_norm_rope(ctypes.byref(a), _stream(x.device)), "bsa_qk_norm_rope")
    _check_err(err, "qk_norm_rope")
    return oq, ok


def qk_norm_rope_backward(dq_out: Optional[torch.Tensor], dk_out: Optional[torch.Tensor], q: Optional[torch.Tensor],
                          k: Optional[torch.Tensor], q_weight: Optional[torch.Tensor] = None,
                          k_weight: Optional[torch.Tensor] = None, *, positions: Optional[torch.Tensor] = None,
                          cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, eps: float = 1e-6,
                          interleaved: bool = False, check_errors: bool = False):
    """Gradients of :func:`qk_norm_rope` for the output gradients ``dq_out``,
    ``dk_out`` (the forward's inputs again, same keywords): returns
    ``dq, dk, dq_weight, dk_weight`` (None for what is absent).  The weights'
    gradients are summed over batch, heads and tokens in fp32 in a fixed order."""
    a, x = _args(q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved)
    outs = []
    for name, t, g, w in (("q", q, dq_out, q_weight), ("k", k, dk_out, k_weight)):
        if t is None:
            outs += [None, None]
            continue
        _require_cuda(g, f"d{name}_out")
        if g.shape != t.shape or g.dtype != t.dtype or g.device != t.device:
            raise ValueError(f"d{name}_out must have {name}'s shape, dtype and device")
        dx = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        dw = torch.empty_like(w) if w is not None else None
        outs += [dx, dw]
        setattr(a, f"{name}_out", _t4(dx, f"d{name}"))
        setattr(a, f"d{name}_out", _t4(g, f"d{name}_out"))
        setattr(a, f"d{name}_weight", dw.data_ptr() if dw is not None else None)
    dq, dqw, dk, dkw = outs
    if x.shape[0] == 0 or x.shape[2] == 0 or a.H + a.Hk == 0:
        for dw in (dqw, dkw):
            if dw is not None:
                dw.zero_()
        return dq, dk, dqw, dkw
    err = torch.zeros(1, dtype=torch.int32, device=x.device) if check_errors else None
    a.err_flag = err.data_ptr() if err is not None else None
    L = _lib.lib()
    with torch.cuda.device(x.device):
        nbytes = ctypes.c_size_t()
        _lib.check(L.bsa_qk_norm_rope_bwd_workspace_bytes(ctypes.byref(a), ctypes.byref(nbytes)),
                   "bsa_qk_norm_rope_bwd_workspace_bytes")
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=x.device) if nbytes.value else None
        _lib.check(L.bsa_qk_norm_rope_bwd(ctypes.byref(a), ws.data_ptr() if ws is not None else None, nbytes.value,
                                          _stream(x.device)), "bsa_qk_norm_rope_bwd")
    _check_err(err, "qk_norm_rope_backward")
    return dq, dk, dqw, dkw


def _rows(g: torch.Tensor) -> torch.Tensor:
    """A gradient as the kernels read it: contiguous rows of its own (autograd
    hands out expanded and transposed ones)."""
    ok = g.stride(3) == 1 and all(s * g.element_size() % 16 == 0 for s in g.stride()[:3]) and g.data_ptr() % 16 == 0
    return g if ok else g.contiguous()


class _QkNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, cos, sin)
        ctx.eps, ctx.interleaved = eps, interleaved
        ctx.set_materialize_grads(False)
        return qk_norm_rope(q, k, q_weight, k_weight, positions=positions, cos=cos, sin=sin, eps=eps,
                            interleaved=interleaved)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, qw, kw, positions, cos, sin = ctx.saved_tensors
        # a side whose output took no part has no gradient
        has_q, has_k = dq_out is not None, dk_out is not None
        if not has_q and not has_k:
            return (None,) * 9
        dq, dk, dqw, dkw = qk_norm_rope_backward(
            _rows(dq_out) if has_q else None, _rows(dk_out) if has_k else None, q if has_q else None,
            k if has_k else None, qw if has_q else None, kw if has_k else None, positions=positions, cos=cos, sin=sin,
            eps=ctx.eps, interleaved=ctx.interleaved)
        return dq, dk, dqw, dkw, None, None, None, None, None


def qk_norm_rope_autograd(q: Optional[torch.Tensor], k: Optional[torch.Tensor],
                          q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *,
                          positions: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                          sin: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False):
    """:func:`qk_norm_rope` as a differentiable op (gradients of q, k and the
    weights; the tables and positions have none)."""
    return _QkNormRopeFn.apply(q, k, q_weight, k_weight, positions, cos, sin, float(eps), bool(interleaved))

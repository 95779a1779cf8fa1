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
import math
from typing import Optional

import torch

from . import _lib
from .api import _DTYPES, _check_err, _require_cuda, on_device, raw_stream

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


def _t4(t: torch.Tensor, name: str):
    s = t.stride()
    if s[3] != 1 and t.shape[3] > 1:
        raise ValueError(f"the last (head) dimension of {name} must be contiguous")
    return t.data_ptr(), s[0], s[1], s[2]


def _check_weight(w, x, name: str) -> int:
    _require_cuda(w, name)
    if w.dim() != 1 or w.shape[0] != x.shape[3] or not w.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{x.shape[3]}] tensor, got {tuple(w.shape)}")
    if w.dtype != torch.float32 and w.dtype != x.dtype:
        raise TypeError(f"{name} must be float32 or {x.dtype}, got {w.dtype}")
    if w.device != x.device:
        raise ValueError(f"{name} is on another device")
    return w.data_ptr()


def _check_tables(x, N: int, B: int, positions, cos, sin):
    """(cos, sin, table_stride, table_len, R, positions, pos_dtype, pos_stride_b)"""
    for name, t in (("cos", cos), ("sin", sin)):
        _require_cuda(t, name)
        if t.dtype != torch.float32 or t.dim() != 2:
            raise TypeError(f"{name} must be a float32 [length, R / 2] table")
        if t.device != x.device:
            raise ValueError(f"{name} is on another device")
    length, half = cos.shape
    stride = cos.stride()
    if sin.shape != cos.shape or sin.stride() != stride or (stride[1] != 1 and half > 1):
        raise ValueError("cos and sin must share their shape and strides, with contiguous rows")
    if half == 0 or length == 0:
        raise ValueError("cos and sin must not be empty (pass None for the norm alone)")
    pos, pos_dtype, pos_stride = 0, _lib.INDEX_I32, 0
    if positions is not None:
        _require_cuda(positions, "positions")
        if positions.dtype not in _INDEX:
            raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.device != x.device:
            raise ValueError("positions are on another device")
        shape = tuple(positions.shape)
        if (shape != (N,) and shape != (B, N)) or (positions.stride(-1) != 1 and N > 1):
            raise ValueError(f"positions must be [{N}] or [{B}, {N}] with contiguous rows, got {shape}")
        pos, pos_dtype = positions.data_ptr(), _INDEX[positions.dtype]
        pos_stride = positions.stride(0) if len(shape) == 2 else 0
    return cos.data_ptr(), sin.data_ptr(), max(stride[0], half), length, 2 * half, pos, pos_dtype, pos_stride


class _Call:
    """The checked arguments of a forward or backward call."""

    __slots__ = ("x", "B", "N", "D", "H", "Hk", "head", "q", "k", "weights", "table", "tail")

    def __init__(self, q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved):
        x = q if q is not None else k
        if x is None:
            raise ValueError("pass q or k")
        for name, t in (("q", q), ("k", k)):
            if t is None:
                continue
            _require_cuda(t, name)
            if t.dim() != 4:
                raise ValueError(f"{name} must be [B, H, N, D], got {tuple(t.shape)}")
            if t.dtype not in _DTYPES:
                raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
        B, _, N, D = x.shape
        if q is not None and k is not None:
            if k.shape[0] != B or k.shape[2] != N or k.shape[3] != D:
                raise ValueError(f"q and k must share B, N and D, got {tuple(q.shape)} and {tuple(k.shape)}")
            if k.dtype != q.dtype:
                raise TypeError(f"q and k must share a dtype, got {q.dtype} and {k.dtype}")
            if k.device != q.device:
                raise ValueError("q and k must be on one device")
        dtype = wdtype = _DTYPES[x.dtype]
        wq = _check_weight(q_weight, q, "q_weight") if q is not None and q_weight is not None else 0
        wk = _check_weight(k_weight, k, "k_weight") if k is not None and k_weight is not None else 0
        if wq or wk:
            if wq and wk and q_weight.dtype != k_weight.dtype:
                raise TypeError("q_weight and k_weight must share a dtype")
            wdtype = _DTYPES[(q_weight if wq else k_weight).dtype]
        if not 0 <= eps < math.inf:
            raise ValueError("eps must be finite and not negative")
        if (cos is None) != (sin is None):
            raise ValueError("pass both cos and sin, or neither (norm only)")
        if cos is not None:
            c, s, stride, length, R, pos, pos_dtype, pos_stride = _check_tables(x, N, B, positions, cos, sin)
        elif positions is not None:
            raise ValueError("positions need the cos and sin tables")
        else:
            c, s, stride, length, R, pos, pos_dtype, pos_stride = 0, 0, 0, 0, 0, 0, _lib.INDEX_I32, 0
        self.x, self.B, self.N, self.D = x, B, N, D
        self.H = q.shape[1] if q is not None else 0
        self.Hk = k.shape[1] if k is not None else 0
        self.head = (B, self.H, self.Hk, N, D, R, dtype, wdtype)
        self.q = _t4(q, "q") if q is not None else _lib.NO_TENSOR
        self.k = _t4(k, "k") if k is not None else _lib.NO_TENSOR
        self.weights = (wq, wk)
        self.table = (c, s, stride, length, pos_dtype, pos, pos_stride)
        self.tail = (eps, 1 if interleaved else 0)

    @property
    def empty(self) -> bool:
        return self.B == 0 or self.N == 0 or self.H + self.Hk == 0

    def pack(self, q_out, k_out, dq_out, dk_out, dqw, dkw, err) -> bytes:
        return _lib.ROPE_ARGS.pack(*self.head, *self.q, *self.k, *q_out, *k_out, *dq_out, *dk_out, *self.weights,
                                   *self.table, *self.tail, dqw, dkw, err.data_ptr() if err is not None else 0)


def _contiguous_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _out(out, x, name: str) -> torch.Tensor:
    if out is None:
        return _contiguous_like(x)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{name} has the wrong shape, dtype or device")
    return out


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
    c = _Call(q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved)
    oq, ok = out if out is not None else (None, None)
    oq = _out(oq, q, "q_out") if q is not None else None
    ok = _out(ok, k, "k_out") if k is not None else None
    if c.empty:
        return oq, ok
    device = c.x.device
    err = torch.zeros(1, dtype=torch.int32, device=device) if check_errors else None
    none = _lib.NO_TENSOR
    a = c.pack(_t4(oq, "q_out") if oq is not None else none, _t4(ok, "k_out") if ok is not None else none, none, none,
               0, 0, err)
    with on_device(device):
        _lib.check(_lib.lib().bsa_qk_norm_rope(a, raw_stream(device)), "bsa_qk_norm_rope")
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
    c = _Call(q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved)
    dx, dw, outs, grads = [None, None], [None, None], [_lib.NO_TENSOR] * 2, [_lib.NO_TENSOR] * 2
    for i, (name, t, g, w) in enumerate((("q", q, dq_out, q_weight), ("k", k, dk_out, k_weight))):
        if t is None:
            continue
        _require_cuda(g, f"d{name}_out")
        if g.shape != t.shape or g.dtype != t.dtype or g.device != t.device:
            raise ValueError(f"d{name}_out must have {name}'s shape, dtype and device")
        dx[i] = _contiguous_like(t)
        outs[i], grads[i] = _t4(dx[i], f"d{name}"), _t4(g, f"d{name}_out")
        if w is not None:
            dw[i] = torch.empty_like(w)
    if c.empty:
        for t in dw:
            if t is not None:
                t.zero_()
        return (*dx, *dw)
    device = c.x.device
    err = torch.zeros(1, dtype=torch.int32, device=device) if check_errors else None
    a = c.pack(*outs, *grads, *(t.data_ptr() if t is not None else 0 for t in dw), err)
    L = _lib.lib()
    with on_device(device):
        nbytes = ctypes.c_size_t()
        _lib.check(L.bsa_qk_norm_rope_bwd_workspace_bytes(a, ctypes.byref(nbytes)),
                   "bsa_qk_norm_rope_bwd_workspace_bytes")
        n = nbytes.value
        ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
        _lib.check(L.bsa_qk_norm_rope_bwd(a, ws.data_ptr() if n else None, n, raw_stream(device)),
                   "bsa_qk_norm_rope_bwd")
    _check_err(err, "qk_norm_rope_backward")
    return (*dx, *dw)


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

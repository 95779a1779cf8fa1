"""Attention whose keys are not the queries' own tokens.

* :func:`cross_attention`: queries of one length over an encoder's states of
  another, padded per sequence, key / value heads shared by groups of query
  heads; one token or many, with its gradient
  (:func:`cross_attention_backward`, :func:`cross_attention_autograd`).
* :func:`shared_prefix_attention`: new tokens of a batch of sequences that all
  continue one long prefix, whose keys are read once for the whole batch.

Both keep :func:`~blocksparsefa_reorder_b200.block_sparse_attention`'s
conventions: ``[B, H, N, D]`` views with a contiguous last dimension, log2 LSE,
``o = 0`` and ``lse = -inf`` for a row that sees no key, the current stream, no
CPU path.  The reference has no counterpart (its queries and keys share one
length).
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from .api import _DTYPES, _check_err, _require_cuda, on_device, raw_stream

_INDEX = {torch.int32: _lib.INDEX_I32, torch.int64: _lib.INDEX_I64}
_HALF = (torch.float16, torch.bfloat16)


def _t4(t: torch.Tensor, name: str):
    """Address and batch, head and token strides; heads or tokens expanded from
    one are spread out before (:func:`_spread`)."""
    s = t.stride()
    if s[-1] != 1:
        raise ValueError(f"the last (head) dimension of {name} must be contiguous")
    return (t.data_ptr(), s[0], s[1], s[2]) if len(s) == 4 else (t.data_ptr(), 0, s[0], s[1])


def _spread(t: torch.Tensor) -> torch.Tensor:
    """Heads or tokens expanded from one (stride 0) get memory of their own: the
    TMA descriptors need real strides there.  An expanded batch is kept."""
    s = t.stride()
    if s[-3] and s[-2]:
        return t
    return t.contiguous() if (not s[-3] and t.shape[-3] > 1) or (not s[-2] and t.shape[-2] > 1) else t


def _check_tensors(q, others) -> None:
    """dtype and device of every tensor against q's."""
    if q.dtype not in _HALF:
        raise TypeError(f"q must be float16 or bfloat16, got {q.dtype}")
    for name, t in others:
        _require_cuda(t, name)
        if t.dtype != q.dtype:
            raise TypeError(f"{name} must have q's dtype {q.dtype}, got {t.dtype}")
        if t.device != q.device:
            raise ValueError(f"{name} is on another device than q")


def _check_lens(lens, B: int, q, name: str) -> None:
    _require_cuda(lens, name)
    if lens.dtype not in _INDEX:
        raise TypeError(f"{name} must be int32 or int64, got {lens.dtype}")
    if tuple(lens.shape) != (B,) or not lens.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{B}] tensor, got {tuple(lens.shape)}")
    if lens.device != q.device:
        raise ValueError(f"{name} is on another device than q")


def _scale(sm_scale, D: int) -> float:
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    if not 0 < scale < math.inf:
        raise ValueError("sm_scale must be positive and finite")
    return scale


def _outputs(q, out, return_lse: bool, lse_out):
    if out is None:
        o = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        o = out
        if o.shape != q.shape or o.dtype != q.dtype or o.device != q.device:
            raise ValueError("out has the wrong shape, dtype or device")
    lse = None
    if return_lse or lse_out is not None:
        lse = lse_out if lse_out is not None else torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
        if lse_out is not None and (lse.shape != q.shape[:3] or lse.dtype != torch.float32 or
                                    not lse.is_contiguous() or lse.device != q.device):
            raise ValueError("lse_out must be a contiguous float32 [B, H, tokens] tensor on q's device")
    return o, lse


def _flag(check_errors: bool, device):
    """(error word or None, its address)"""
    if not check_errors:
        return None, 0
    err = torch.zeros(1, dtype=torch.int32, device=device)
    return err, err.data_ptr()


def _launch(name: str, query, call, a: bytes, device, err) -> None:
    """Workspace query, workspace, launch, optional device check."""
    with on_device(device):
        nbytes = ctypes.c_size_t()
        _lib.check(query(a, ctypes.byref(nbytes)), name)
        n = nbytes.value
        ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
        _lib.check(call(a, ws.data_ptr() if n else None, n, raw_stream(device)), name)
    _check_err(err, name)


def _check_cross(q, k, v, k_lens):
    _require_cuda(q, "q")
    if q.dim() != 4:
        raise ValueError(f"q must be [B, H, M, D], got {tuple(q.shape)}")
    _check_tensors(q, (("k", k), ("v", v)))
    B, H, M, D = q.shape
    if k.dim() != 4 or v.shape != k.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"k and v must be [{B}, Hk, N, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
    Hk, N = k.shape[1], k.shape[2]
    if Hk == 0 or H % Hk:
        raise ValueError(f"the query heads ({H}) must be a multiple of the key / value heads ({Hk})")
    if k_lens is not None:
        _check_lens(k_lens, B, q, "k_lens")
    return B, H, Hk, M, N, D


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, k_lens: Optional[torch.Tensor] = None,
                    sm_scale: Optional[float] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None,
                    lse_out: Optional[torch.Tensor] = None, check_errors: bool = False):
    """Attention of M queries over N keys of another sequence.

    ``o = softmax(q k^T * sm_scale over keys j < k_lens[b]) v`` per (b, h).

    q: CUDA ``[B, H, M, D]``, k and v: ``[B, Hk, N, D]``, bf16 or fp16, D 64 or
    128, last dim contiguous, rows 16-byte aligned; H a multiple of Hk, query
    head h reads key head ``h // (H // Hk)``.  M and N are free, from one token
    on.  k and v may be one copy expanded over the batch.
    k_lens: optional int ``[B]`` on the device: valid keys of each sequence
    (0 gives ``o = 0``, ``lse = -inf``); what lies behind them is never read
    into the result, NaN included.  Lengths outside [0, N] are clamped, and an
    error with ``check_errors`` (which synchronises).
    return_lse: also return the row log-sum-exp in log2 units, ``[B, H, M]``.
    """
    B, H, Hk, M, N, D = _check_cross(q, k, v, k_lens)
    scale = _scale(sm_scale, D)
    o, lse = _outputs(q, out, return_lse, lse_out)
    if B == 0 or M == 0 or H == 0:
        return (o, lse) if return_lse else o
    q, k, v = _spread(q), _spread(k), _spread(v)
    err, flag = _flag(check_errors, q.device)
    a = _lib.CROSS_ARGS.pack(B, H, Hk, M, N, D, _DTYPES[q.dtype], _INDEX[k_lens.dtype] if k_lens is not None else 0,
                             *_t4(q, "q"), *_t4(o, "out"), *_t4(k, "k"), *_t4(v, "v"),
                             k_lens.data_ptr() if k_lens is not None else 0, lse.data_ptr() if lse is not None else 0,
                             flag, scale)
    L = _lib.lib()
    _launch("bsa_cross_fwd", L.bsa_cross_fwd_workspace_bytes, L.bsa_cross_fwd, a, q.device, err)
    return (o, lse) if return_lse else o


def cross_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                             dout: torch.Tensor, *, k_lens: Optional[torch.Tensor] = None,
                             sm_scale: Optional[float] = None, check_errors: bool = False):
    """Gradients of :func:`cross_attention`: ``dq, dk, dv`` for the output
    gradient ``dout``, from the forward's ``o`` and log2 ``lse``.

    dk and dv are summed over the query heads of each key / value head and are
    zero behind ``k_lens[b]``; every gradient row is written by one CTA (no
    atomics, deterministic).
    """
    B, H, Hk, M, N, D = _check_cross(q, k, v, k_lens)
    _check_tensors(q, (("o", o), ("dout", dout)))
    if o.shape != q.shape or dout.shape != q.shape:
        raise ValueError("o and dout must have q's shape")
    _require_cuda(lse, "lse")
    if lse.shape != q.shape[:3] or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != q.device:
        raise ValueError("lse must be the forward's contiguous float32 [B, H, M] LSE")
    scale = _scale(sm_scale, D)
    dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    if B == 0 or M == 0 or H == 0:
        return dq, dk.zero_(), dv.zero_()
    q, k, v, o, dout = _spread(q), _spread(k), _spread(v), _spread(o), _spread(dout)
    delta = torch.empty_like(lse)
    err, flag = _flag(check_errors, q.device)
    a = _lib.CROSS_BWD_ARGS.pack(B, H, Hk, M, N, D, _DTYPES[q.dtype],
                                 _INDEX[k_lens.dtype] if k_lens is not None else 0, *_t4(q, "q"), *_t4(k, "k"),
                                 *_t4(v, "v"), *_t4(o, "o"), *_t4(dout, "dout"), *_t4(dq, "dq"), *_t4(dk, "dk"),
                                 *_t4(dv, "dv"), k_lens.data_ptr() if k_lens is not None else 0, lse.data_ptr(),
                                 delta.data_ptr(), flag, scale)
    with on_device(q.device):
        _lib.check(_lib.lib().bsa_cross_bwd(a, raw_stream(q.device)), "bsa_cross_bwd")
    _check_err(err, "cross_attention_backward")
    return dq, dk, dv


def _rows(g: torch.Tensor) -> torch.Tensor:
    """A gradient as the kernels read it (autograd hands out expanded and
    transposed ones)."""
    ok = g.stride(3) == 1 and all(s * 2 % 16 == 0 for s in g.stride()[:3]) and g.data_ptr() % 16 == 0
    return g if ok else g.contiguous()


class _CrossAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, k_lens, sm_scale):
        o, lse = cross_attention(q, k, v, k_lens=k_lens, sm_scale=sm_scale, return_lse=True)
        ctx.save_for_backward(q, k, v, o, lse, k_lens)
        ctx.sm_scale = sm_scale
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, o, lse, k_lens = ctx.saved_tensors
        dq, dk, dv = cross_attention_backward(q, k, v, o, lse, _rows(dout), k_lens=k_lens, sm_scale=ctx.sm_scale)
        return dq, dk, dv, None, None


def cross_attention_autograd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                             k_lens: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None) -> torch.Tensor:
    """:func:`cross_attention` as a differentiable op (gradients of q, k, v);
    k and v expanded over the batch get the sum of its gradients."""
    return _CrossAttentionFn.apply(q, k, v, k_lens, sm_scale)


def shared_prefix_attention(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, k: torch.Tensor,
                            v: torch.Tensor, *, lens: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
                            return_lse: bool = False, out: Optional[torch.Tensor] = None,
                            lse_out: Optional[torch.Tensor] = None, check_errors: bool = False):
    """Attention of T new tokens a sequence behind a prefix all sequences share.

    q: CUDA ``[B, H, T, D]``; k_prefix, v_prefix: ``[Hk, P, D]``, seen whole by
    every token and read once for the batch; k, v: ``[B, Hk, C, D]``, each
    sequence's own keys, of which the first ``lens[b]`` are valid (None = C),
    the last T of them those of the new tokens themselves: token t sees own
    keys ``j < lens[b] - (T - 1 - t)`` (it needs them in the cache already).
    P or C may be 0.  bf16 or fp16, D 64 or 128, H a multiple of Hk, rows
    16-byte aligned.  What lies behind ``lens[b]`` is never read into the
    result; a value row that only later tokens of a sequence see has to be
    finite (earlier ones take it times 0).  Lengths outside [0, C] are clamped,
    and an error with ``check_errors`` (which synchronises).
    return_lse: also return the row log-sum-exp in log2 units, ``[B, H, T]``.
    """
    _require_cuda(q, "q")
    if q.dim() != 4:
        raise ValueError(f"q must be [B, H, T, D], got {tuple(q.shape)}")
    _check_tensors(q, (("k_prefix", k_prefix), ("v_prefix", v_prefix), ("k", k), ("v", v)))
    B, H, T, D = q.shape
    if k_prefix.dim() != 3 or v_prefix.shape != k_prefix.shape or k_prefix.shape[2] != D:
        raise ValueError(f"k_prefix and v_prefix must be [Hk, P, {D}], got {tuple(k_prefix.shape)} and "
                         f"{tuple(v_prefix.shape)}")
    Hk, P = k_prefix.shape[0], k_prefix.shape[1]
    if k.dim() != 4 or v.shape != k.shape or (k.shape[0], k.shape[1], k.shape[3]) != (B, Hk, D):
        raise ValueError(f"k and v must be [{B}, {Hk}, C, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if Hk == 0 or H % Hk:
        raise ValueError(f"the query heads ({H}) must be a multiple of the key / value heads ({Hk})")
    if lens is not None:
        _check_lens(lens, B, q, "lens")
    scale = _scale(sm_scale, D)
    o, lse = _outputs(q, out, return_lse, lse_out)
    if B == 0 or T == 0 or H == 0:
        return (o, lse) if return_lse else o
    q, k_prefix, v_prefix, k, v = (_spread(t) for t in (q, k_prefix, v_prefix, k, v))
    err, flag = _flag(check_errors, q.device)
    a = _lib.PREFIX_ARGS.pack(B, H, Hk, T, P, k.shape[2], D, _DTYPES[q.dtype],
                              _INDEX[lens.dtype] if lens is not None else 0, *_t4(q, "q"), *_t4(o, "out"),
                              *_t4(k_prefix, "k_prefix"), *_t4(v_prefix, "v_prefix"), *_t4(k, "k"), *_t4(v, "v"),
                              lens.data_ptr() if lens is not None else 0, lse.data_ptr() if lse is not None else 0,
                              flag, scale)
    L = _lib.lib()
    _launch("bsa_prefix_fwd", L.bsa_prefix_fwd_workspace_bytes, L.bsa_prefix_fwd, a, q.device, err)
    return (o, lse) if return_lse else o

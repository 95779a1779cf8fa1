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

from typing import Optional

import torch

from . import _lib
from .api import _check_err


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


def _error_word(check_errors: bool, q, k):
    x = q if q is not None else k
    return torch.zeros(1, dtype=torch.int32, device=x.device) if check_errors and x is not None else None


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
    themselves; outputs that overlap each other or another input are refused.
    Returns ``(q_out, k_out)``; sums, norm and rotation are fp32,
    rounded once.
    """
    q_out, k_out = out if out is not None else (None, None)
    err = _error_word(check_errors, q, k)
    o = _lib.native().qk_norm_rope(q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved, q_out, k_out, err)
    _check_err(err, "qk_norm_rope")
    return o


def qk_norm_rope_backward(dq_out: Optional[torch.Tensor], dk_out: Optional[torch.Tensor], q: Optional[torch.Tensor],
                          k: Optional[torch.Tensor], q_weight: Optional[torch.Tensor] = None,
                          k_weight: Optional[torch.Tensor] = None, *, positions: Optional[torch.Tensor] = None,
                          cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, eps: float = 1e-6,
                          interleaved: bool = False, check_errors: bool = False):
    """Gradients of :func:`qk_norm_rope` for the output gradients ``dq_out``,
    ``dk_out`` (the forward's inputs again, same keywords): returns
    ``dq, dk, dq_weight, dk_weight`` (None for what is absent).  The weights'
    gradients are summed over batch, heads and tokens in fp32 in a fixed order."""
    err = _error_word(check_errors, q, k)
    g = _lib.native().qk_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, positions, cos, sin, eps,
                                            interleaved, err)
    _check_err(err, "qk_norm_rope_backward")
    return g


def qk_norm_rope_autograd(q: Optional[torch.Tensor], k: Optional[torch.Tensor],
                          q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *,
                          positions: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                          sin: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False):
    """:func:`qk_norm_rope` as a differentiable op (gradients of q, k and the
    weights; the tables and positions have none, and the gradient itself is not
    differentiable)."""
    return _lib.native().qk_norm_rope_autograd(q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved)

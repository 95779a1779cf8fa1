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

from typing import Optional

import torch

from . import _lib
from .api import _check_err


def _error_word(check_errors: bool, q):
    return torch.zeros(1, dtype=torch.int32, device=q.device) if check_errors else None


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, k_lens: Optional[torch.Tensor] = None,
                    sm_scale: Optional[float] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None,
                    lse_out: Optional[torch.Tensor] = None, o_rest: Optional[torch.Tensor] = None,
                    check_errors: bool = False):
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
    o_rest: optional tensor laid out as the output that receives what rounding
    left of the result (fp32 result - o), for :func:`cross_attention_backward`.
    Outputs given (out, lse_out, o_rest) that overlap each other or an input are
    refused.
    """
    err = _error_word(check_errors, q)
    o, lse = _lib.native().cross_attention(q, k, v, k_lens, sm_scale, return_lse, out, lse_out, o_rest, err)
    _check_err(err, "cross_attention")
    return (o, lse) if return_lse else o


def cross_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                             dout: torch.Tensor, *, k_lens: Optional[torch.Tensor] = None,
                             sm_scale: Optional[float] = None, o_rest: Optional[torch.Tensor] = None,
                             check_errors: bool = False):
    """Gradients of :func:`cross_attention`: ``dq, dk, dv`` for the output
    gradient ``dout``, from the forward's ``o`` and log2 ``lse``.

    dk and dv are summed over the query heads of each key / value head and are
    zero behind ``k_lens[b]``; every gradient row is written by one CTA (no
    atomics, deterministic).  o_rest: the forward's, so that ``rowsum(dout o)``
    is formed from the unrounded output; without it o's rounding is in dq and dk
    (over few keys as much of it as their own).  P and dS are rounded to the
    inputs' type for the products, dS of fp16 inputs relative to the largest
    output gradient of its key / value head.
    """
    err = _error_word(check_errors, q)
    g = _lib.native().cross_attention_backward(q, k, v, o, lse, dout, k_lens, sm_scale, o_rest, err)
    _check_err(err, "cross_attention_backward")
    return g


def cross_attention_autograd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                             k_lens: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None) -> torch.Tensor:
    """:func:`cross_attention` as a differentiable op (gradients of q, k, v);
    k and v expanded over the batch get the sum of its gradients.  The gradient
    itself is not differentiable.

    The forward writes, beside the output, a second tensor of its size (what
    rounding left of it) and the LSE, whether a gradient is recorded or not, and
    the graph keeps them with q, k and v; the gradients of q, k and v are all
    computed, whichever are asked for.  Where none is recorded,
    :func:`cross_attention` does the same without."""
    return _lib.native().cross_attention_autograd(q, k, v, k_lens, sm_scale)


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
    Outputs given that overlap each other or an input are refused.
    """
    err = _error_word(check_errors, q)
    o, lse = _lib.native().shared_prefix_attention(q, k_prefix, v_prefix, k, v, lens, sm_scale, return_lse, out, lse_out,
                                                   err)
    _check_err(err, "shared_prefix_attention")
    return (o, lse) if return_lse else o

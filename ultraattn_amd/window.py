"""Sliding-window attention with sinks on one MI355X: forward, backward, and new tokens against a cache.

Host side of ``ua_swa_*`` in ``include/ultraattn.h``, beside the block-sparse operators of ``ops.py`` and in their manner: row tensors
``[B, S, H, D]`` with any (batch, token, head) strides (multiples of 8; from token to token of keys and values, in the backward of ``q`` and ``dout`` too,
at most 4194303 elements), ``lse`` ``[B, H, S]`` fp32 in natural logarithm, results written in place when
given (``out`` may be ``q`` itself; results overlap nothing else), everything on the current CUDA(HIP) stream, nothing synchronises.  Types are bf16 and fp16, D is 64 or 128, lengths are arbitrary, and keys
may have fewer heads than queries (each serves ``Hq / Hk`` consecutive ones).

Query i is at position ``q_start + i`` and key j at ``k_start + j``.  With ``window=(left, right)`` a query at p sees the keys at
``p - left .. p + right`` (-1: no bound on that side) and, up to ``p + right``, the first ``sinks`` positions of the sequence.
``q_start=None`` puts the last query at the last key.  A query that sees no key gets ``out = 0``, ``lse = -inf`` and no gradient, so
results over shards of the keys (``k_start``) are joined by ``merge_partials`` / ``update_out_and_lse``.
NaN or infinity in a key or value reaches the rows that see it, and may reach others of their tile of 128 rows (in a decode, of up to 32 rows of a key
head); it reaches no tile that has none that does.  So a cache may hold anything in rows that no new token sees.
"""
from typing import Optional, Tuple

import torch

from ._lib import native


def swa_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Tuple[int, int] = (-1, 0), sinks: int = 0,
            softmax_scale: Optional[float] = None, q_start: Optional[int] = None, k_start: int = 0, out: Optional[torch.Tensor] = None,
            lse: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Forward -> (out, lse).  The default window is causal attention, aligned at the last key; ``softmax_scale`` is 1 / sqrt(D)."""
    left, right = window
    return native().swa_forward(q, k, v, left, right, sinks, q_start, k_start, softmax_scale, out, lse)


def swa_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: Optional[torch.Tensor], lse: torch.Tensor,
            window: Tuple[int, int] = (-1, 0), sinks: int = 0, softmax_scale: Optional[float] = None, q_start: Optional[int] = None, k_start: int = 0,
            dq: Optional[torch.Tensor] = None, dk: Optional[torch.Tensor] = None, dv: Optional[torch.Tensor] = None,
            softmax_d: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Backward -> (dq, dk, dv), with the arguments of the forward.  ``lse`` and ``softmax_d`` (rowsum(dout * out), as ``bsa_bwd`` takes it; then
    ``out`` is ignored) are the rows' global statistics; dk and dv are summed over the query heads of a key head.  The same call gives the same bits."""
    left, right = window
    return native().swa_backward(dout, q, k, v, out, lse, dq, dk, dv, softmax_d, left, right, sinks, q_start, k_start, softmax_scale)


def swa_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor, window: int = -1, sinks: int = 0,
               softmax_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
               lse: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """T new tokens of every sequence, q ``[B, T, Hq, D]``, against the caches ``[B, room, Hk, D]`` that hold them already -> (out, lse).

    ``lens`` (int32 ``[B]`` on the device) counts the new tokens: token t of sequence b is at position ``lens[b] - T + t`` and sees the keys up to
    itself, at most ``window`` behind it (-1: all) and the first ``sinks``.  A token before position 0 sees nothing.  What lies behind ``lens[b]`` in the
    caches is not read.  Meant for few tokens (a step's one, or several proposed ones); a prompt's go through ``swa_fwd``."""
    return native().swa_decode(q, k_cache, v_cache, lens, window, sinks, softmax_scale, out, lse)

"""Rotary positions of Q and K on one MI355X: forward, backward, and the serving form that also fills a cache.

Host side of ``ua_rope`` / ``ua_rope_append`` in ``include/ultraattn.h``.  Row tensors are ``[B, S, H, D]`` in bf16, fp16 or
fp32, head_dim contiguous, any strides; results are written in place when given.  Everything runs on the current CUDA(HIP) stream; nothing
synchronises or keeps state, so every call can be captured into a HIP graph.
"""
import math
from typing import Optional, Tuple

import torch

from ._lib import native


def rope_freqs(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
               original_length: Optional[int] = None, slow: float = 1.0, fast: float = 32.0,
               device=None) -> Tuple[torch.Tensor, float]:
    """(freqs, scale): the angles per position of ``rotary_dim / 2`` pairs as float64 on ``device``, and the factor of the
    turned entries, as the other functions take them.  Made once, kept like a weight.

    Without ``scaling`` f_i = base^(-2 i / rotary_dim) and scale = 1.  For contexts ``factor`` times as long:

    * ``"linear"``: positions are interpolated, f_i / factor;
    * ``"ntk"``: the base grows so that the last pair is interpolated and the first is not, base * factor^(rotary_dim / (rotary_dim - 2));
    * ``"yarn"`` (Peng et al. 2023, "YaRN"): a pair that makes fewer than ``slow`` turns over ``original_length`` tokens is interpolated, one that
      makes more than ``fast`` keeps its frequency, those between are blended linearly in the number of turns; scale = 0.1 ln(factor) + 1."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    if not (base > 0 and factor > 0 and math.isfinite(base) and math.isfinite(factor)):
        raise ValueError("base and factor must be positive numbers")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    if scaling is None and factor != 1.0:
        raise ValueError("factor needs a scaling")
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("'ntk' needs more than one pair")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freqs = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    scale = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "yarn":
        if original_length is None or original_length <= 0 or not 0 <= slow < fast:
            raise ValueError("'yarn' needs original_length > 0 and 0 <= slow < fast")
        keep = ((original_length * freqs / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        freqs = freqs / factor * (1 - keep) + freqs * keep
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return freqs.to(device) if device is not None else freqs, scale


def rope_fwd(q: torch.Tensor, k: Optional[torch.Tensor], freqs: torch.Tensor, positions: Optional[torch.Tensor] = None, start: int = 0,
             interleaved: bool = False, scale: float = 1.0, q_out: Optional[torch.Tensor] = None,
             k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Turns q ``[B, S, Hq, D]`` and k ``[B, S, Hk, D]`` (or None) by their positions -> (q_out, k_out), one launch for both.

    Pair i is turned by ``position * freqs[i]`` and multiplied by ``scale``; pairs are ``(x[i], x[i + n])`` of the first ``2 n``
    entries, ``n = len(freqs)``, or with ``interleaved`` ``(x[2i], x[2i + 1])``; what is behind them passes through.  Token s is at
    ``start + s``, or at ``positions`` (int32 or int64, ``[S]`` or ``[B, S]``, in any order).  Angles are reduced in more than
    64 bits, so far positions (up to 2^53 in size; ``start`` is checked) are as exact as near ones.  ``q_out=q`` works in place; an output may not overlap an input otherwise."""
    return native().rope(q, k, freqs, positions, start, interleaved, False, scale, q_out, k_out)


def rope_bwd(dq: torch.Tensor, dk: Optional[torch.Tensor], freqs: torch.Tensor, positions: Optional[torch.Tensor] = None, start: int = 0,
             interleaved: bool = False, scale: float = 1.0, dq_out: Optional[torch.Tensor] = None,
             dk_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Gradients of ``rope_fwd``'s inputs from those of its outputs (the turn by the negative angles), with the same arguments."""
    return native().rope(dq, dk, freqs, positions, start, interleaved, True, scale, dq_out, dk_out)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor,
                freqs: torch.Tensor, interleaved: bool = False, scale: float = 1.0, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A serving step's T new tokens of every sequence, one launch: returns q ``[B, T, Hq, D]`` turned, and writes k, turned, and v
    ``[B, T, Hk, D]`` to their rows of the caches ``[B, room, Hk, D]``.

    ``lens`` (int32 ``[B]`` on the device) counts the new tokens: token t of sequence b is at position ``lens[b] - T + t``, which is also its
    row.  Tokens whose row is not in the cache (negative: a sequence shorter than T; or beyond ``room``) are not
    written, and no other row is touched."""
    return native().rope_append(q, k, v, k_cache, v_cache, lens, freqs, interleaved, scale, q_out)

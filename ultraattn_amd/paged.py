"""A paged key and value cache on one MI355X: new tokens' rows written with their rotary positions, attention of a chain or a tree of new tokens against it,
and the rows of a tree's accepted branch moved together.

Host side of ``ua_paged_*`` in ``include/ultraattn.h``, beside ``rope_append`` and ``swa_decode`` for contiguous caches and in their manner: row tensors
``[B, T, H, D]``, any (batch, token, head) strides, results written in place when given, everything on the current CUDA(HIP) stream; nothing synchronises or keeps
state, so every call can be captured into a HIP graph, and one captured call serves all lengths, tables and trees.

The cache is two pools ``[n_pages, page, Hk, D]`` (any page size and strides, views of one tensor too) and a ``table``, int32 ``[B, max_pages]`` on the device: row r of
sequence b is slot ``r % page`` of page ``table[b, r // page]``.  An entry outside the pool (-1, say) is a page that is not there: nothing is written to it, and its rows
are not seen, so that pages behind a window may be given back.  A contiguous cache ``[B, room, Hk, D]`` is one too, with ``table = arange(B)[:, None]``.  ``paged_decode`` reads caches of bf16 or fp16 with heads of 64 or 128;
``paged_append`` and ``paged_keep`` also take fp32 and other head sizes, for readers of the caller's own.

A step brings T tokens of every sequence, of which ``n_new`` (int32 ``[B]``; None: all) are real.  ``lens`` (int32 ``[B]``) counts the real ones: token t is row
``base + t`` of its sequence, ``base = lens - n_new``.  The tokens are a chain, or with ``parents`` (int32 ``[B, T]``, or ``[T]`` for one tree in all sequences, T up to 256)
a tree of drafts: ``parents[b, t] < t`` is the token before token t, any other value says that it follows the cache's last row.  A token's position is ``base`` plus the number of
tokens before it in its branch.

A serving step that verifies a tree::

    lens += n_new                                                                       # all of them on the device
    q = paged_append(q, k, v, k_pages, v_pages, table, lens, freqs, n_new, parents)     # in every layer
    out, lse = paged_decode(q, k_pages, v_pages, table, lens, n_new, parents)
    ...                                                                                 # logits, and which branch is accepted
    paged_keep(k_pages, v_pages, table, lens, n_new, path, n_kept)                      # [layers, n_pages, page, Hk, D]: once for all layers
    lens += n_kept - n_new
"""
from typing import Optional, Tuple, Union

import torch

from ._lib import native


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                 freqs: torch.Tensor, n_new: Optional[torch.Tensor] = None, parents: Optional[torch.Tensor] = None, interleaved: bool = False,
                 scale: float = 1.0, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Returns q ``[B, T, Hq, D]`` turned by its positions, and writes k, turned, and v ``[B, T, Hk, D]`` to their rows; one launch.

    ``freqs``, ``interleaved`` and ``scale`` as in ``rope_fwd``; bf16, fp16 or fp32, any D up to 512.  Rows that the table has no page for are not written, and no other
    row is touched.  Of tokens that are not real nothing is written, and their q is 0."""
    return native().paged_append(q, k, v, k_pages, v_pages, table, lens, freqs, n_new, parents, interleaved, scale, q_out)


def paged_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, n_new: Optional[torch.Tensor] = None,
                 parents: Optional[torch.Tensor] = None, window: int = -1, sinks: int = 0, softmax_scale: Optional[float] = None,
                 out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The new tokens, q ``[B, T, Hq, D]``, against the cache that holds them already -> (out, lse), lse ``[B, Hq, T]`` fp32 in natural logarithm.

    A token sees the rows before ``base`` and its own branch, itself included; with ``window >= 0`` of both only what is at most ``window`` positions before it, and the first
    ``sinks`` positions.  One that sees nothing, or is not real, gets ``out = 0``, ``lse = -inf``.  bf16 or fp16, D 64 or 128, Hq a multiple of Hk, strides multiples of 8
    elements.  What lies behind ``lens``, and rows that no token sees, may be anything; NaN in a drafted token's key or value may reach all drafts of its sequence, in
    another row that is seen also rows beside those that see it.  Probabilities are rounded to the type before they meet the values; sums and ``lse`` are 32 bits."""
    return native().paged_decode(q, k_pages, v_pages, table, lens, n_new, parents, window, sinks, softmax_scale, out, lse)


def paged_keep(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, n_new: Union[torch.Tensor, int], path: torch.Tensor,
               n_kept: torch.Tensor) -> None:
    """After a verification: the first ``n_kept`` (int32 ``[B]``) tokens of ``path`` (int32 ``[B, M]``) become the sequence's next rows, in place and in one launch: row
    ``base + i`` takes what row ``base + path[b, i]`` holds, K and V.

    The pools may have a leading axis of layers, ``[layers, n_pages, page, Hk, D]``; bf16, fp16 or fp32, any D.  ``lens`` and ``n_new`` are the verified step's (``n_new`` may be
    one number for all sequences).  ``path`` rises along a branch, as the tokens before a token have lower numbers; where an entry is below its place or not a real token,
    or a page is not there, the row stays as it is.  What follows the kept rows is left as it was: set ``lens`` to ``base + n_kept`` for the next step."""
    native().paged_keep(k_pages, v_pages, table, lens, n_new, path, n_kept)

"""Drafted tokens of a serving batch: their tree's masks, and which of them stay.

A step that looks at several drafted tokens of each row at once takes the row's last token and its drafts as tokens 0 to
M - 1 through the model (``paged.rope_append``, ``paged.tree_attention``), and ``verify_tokens`` then keeps those that the
model's own probabilities agree with, so that what comes out is distributed as if every token had been drawn by itself.

No counterpart in the reference, which leaves generation to the caller.  There is no CPU path for ``verify_tokens``.
"""

from __future__ import annotations

import torch

from . import _native
from .paged import _scratch, _stream

__all__ = ["tree_tables", "verify_tokens"]


def tree_tables(parents: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(depths, visible) of trees of tokens: int32 ``[..., M]`` and ``[..., M, ceil(M / 32)]``.

    ``parents[..., t]`` is the token before token t, less than t; a token whose parent is negative is a root, as is one
    whose parent is not before it.  visible has the bits of each token and its ancestors, as ``paged.tree_attention``
    takes them.
    """
    if parents.dtype not in (torch.int32, torch.int64) or parents.dim() == 0:
        raise TypeError("tree_tables takes int32 or int64 parents [..., M]")
    m = parents.shape[-1]
    words = -(-m // 32)
    depths = torch.zeros(parents.shape, dtype=torch.int32, device=parents.device)
    bits = torch.zeros(*parents.shape, 32 * words, dtype=torch.bool, device=parents.device)
    for t in range(m):
        parent = parents[..., t : t + 1].long()
        has = (parent >= 0) & (parent < t)
        parent = parent.clamp(0, max(0, t - 1))
        depths[..., t : t + 1] = torch.where(has, depths.gather(-1, parent) + 1, 0)
        before = bits.gather(-2, parent[..., None].expand(*parent.shape, 32 * words))[..., 0, :]
        bits[..., t, :] = before & has
        bits[..., t, t] = True
    place = torch.arange(32, device=parents.device)
    packed = (bits.unflatten(-1, (words, 32)).long() << place).sum(-1)
    return depths, torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def verify_tokens(logits: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor, *,
                  parents: torch.Tensor | None = None, draft_probs: torch.Tensor | None = None,
                  temperature: torch.Tensor | None = None,
                  seq_lens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted tokens of each row stay, and the token that follows them: (path, counts, next).

    Token 0 of ``tokens`` (int32 or int64 ``[rows, M]``) is the row's last token, tokens 1 to ``min(seq_lens[b], M) - 1``
    are drafts: of a line, or, with ``parents`` (int32 ``[rows, M]`` or ``[M]``), of a tree in which token n stands behind
    token ``parents[n] < n``.  ``logits`` ``[rows, M, vocab]`` (float32, bfloat16, float16, of any strides of row and
    token) are the model's for what follows each token, p their softmax at the row's ``temperature`` (fp32, 1 unless
    given; at 0 the first largest logit has all of p).  ``uniforms`` are fp32 ``[rows, M]`` random numbers in [0, 1).  From
    token 0 on:

    * without ``draft_probs``, ``uniforms[n]`` draws v from p.  The row goes on with the first draft behind n that holds
      v, or stops, and v follows;
    * with ``draft_probs`` (fp32 ``[rows, M - 1, vocab]``, a line: ``draft_probs[n]`` is the q that token n + 1 was drawn
      from) the row goes on to token n + 1 where ``uniforms[n] * q < p`` at it.  Else it stops, and the uniform of the
      row's last token draws what follows from ``max(p - q, 0)``, or from p behind the last draft.

    A draw takes the first v whose running sum passes the uniform times the sum; weights and sums are 64-bit.  A row stops
    with -1 at logits that have NaN or +inf, or nothing but -inf (a grammar that allows nothing), and at a temperature that
    is negative or not finite; a row of no token gives 0 and -1.

    path (int32 ``[rows, M]``) has the numbers of the tokens that stay, from 0 on and -1 behind them, counts (int32
    ``[rows]``) how many they are, token 0 among them, as ``paged.keep_tokens`` takes them; next is int64 ``[rows]``.
    """
    stream = _stream(logits)
    sizes = logits.shape if logits.dim() == 3 and logits.numel() < 1 << 62 else (0, 0, 0)  # the call refuses others
    return _native.tensor_calls().verify_tokens(logits, tokens, uniforms, parents, draft_probs, temperature, seq_lens,
                                                *_scratch(logits, stream, "verify", *sizes), stream)

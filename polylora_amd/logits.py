"""Logits of a serving batch before the next tokens are picked: penalties of repeated tokens, biases, grammar masks.

No counterpart in the reference, which leaves generation to the caller.  There is no CPU path.
"""

from __future__ import annotations

import torch

from . import _native
from .paged import _stream

__all__ = ["adjust_logits", "pack_allowed"]


def pack_allowed(mask: torch.Tensor) -> torch.Tensor:
    """int32 ``[..., ceil(vocab / 32)]`` words of a boolean ``[..., vocab]``: bit ``v % 32`` of word ``v // 32`` is mask[v]."""
    if mask.dtype is not torch.bool or mask.dim() == 0:
        raise TypeError("pack_allowed takes a boolean [..., vocab] tensor")
    mask = torch.nn.functional.pad(mask, (0, -mask.shape[-1] % 32)).unflatten(-1, (-1, 32))
    words = (mask.long() << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def adjust_logits(logits: torch.Tensor, *, tokens: torch.Tensor | None = None, lens: torch.Tensor | None = None,
                  prompt_lens: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                  presence: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                  bias_ids: torch.Tensor | None = None, bias_values: torch.Tensor | None = None,
                  allowed: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """The logits ``[rows, vocab]`` of each row's next token, adjusted as the row's request asks; fp32, in this order:

    1. ``v`` among the row's first ``lens`` of ``tokens`` (prompt and output): ``x / repetition`` where x > 0, else
       ``x * repetition``;
    2. ``v`` n > 0 times among those from ``prompt_lens`` on (the output): ``x - (frequency * n + presence)``;
    3. ``x +`` the row's bias for v (``bias_values`` at v's places in ``bias_ids``, summed in order; -inf bans it);
    4. ``-inf`` where v's bit of ``allowed`` is 0 (words as ``pack_allowed`` makes them).

    tokens int32 or int64 ``[rows, n]`` (n to 1048575; right-padded, what is beyond lens is not read as tokens), lens
    and prompt_lens int32 ``[rows]``, the penalties fp32 ``[rows]``, bias_ids int32 and bias_values fp32 ``[rows, m]`` (or
    ``[m]`` for all rows; m to 2047), allowed int32 ``[rows, ceil(vocab / 32)]`` (or one row for all); each is optional,
    ids outside the vocabulary match nothing; bias_ids and bias_values of several rows have one row stride.  Logits in
    float32, bfloat16 or float16, rows of any stride.  The result goes into ``out`` (fp32, or the logits' dtype; the
    logits themselves too; rows apart) or a new fp32 tensor.
    """
    return _native.tensor_calls().adjust_logits(logits, tokens, lens, prompt_lens, repetition, presence, frequency,
                                                bias_ids, bias_values, allowed, out, _stream(logits))

"""Logits of a serving batch before the next tokens are picked: penalties of repeated tokens, biases, grammar masks.

No counterpart in the reference, which leaves generation to the caller.  There is no CPU path.
"""

from __future__ import annotations

import torch

from . import _native
from .paged import _check_tensor, _gpu

__all__ = ["adjust_logits", "pack_allowed"]


def pack_allowed(mask: torch.Tensor) -> torch.Tensor:
    """int32 ``[..., ceil(vocab / 32)]`` words of a boolean ``[..., vocab]``: bit ``v % 32`` of word ``v // 32`` is mask[v]."""
    if mask.dtype is not torch.bool or mask.dim() == 0:
        raise TypeError("pack_allowed takes a boolean [..., vocab] tensor")
    mask = torch.nn.functional.pad(mask, (0, -mask.shape[-1] % 32)).unflatten(-1, (-1, 32))
    words = (mask.long() << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _rows_of(name: str, t: torch.Tensor, dtype: torch.dtype, device: int, rows: int) -> tuple[int, int]:
    """(columns, row stride) of a list per row ``[rows, n]`` or one ``[n]`` that all rows share."""
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, not on the GPU of the other arguments")
    if not 1 <= t.dim() <= 2 or (t.dim() == 2 and t.shape[0] != rows):
        raise ValueError(f"{name} must be [{rows}, n], or [n] for all rows, not {list(t.shape)}")
    if t.numel() and t.stride(-1) != 1:
        raise ValueError(f"the rows of {name} must be contiguous")
    return t.shape[-1], t.stride(0) if t.dim() == 2 else 0


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
    ids outside the vocabulary match nothing.  Logits in float32, bfloat16 or float16, rows of any stride.  The result
    goes into ``out`` (fp32, or the logits' dtype; the logits themselves too) or a new fp32 tensor.
    """
    device = _gpu(logits, "adjust_logits")
    if logits.dim() != 2:
        raise ValueError(f"logits must be [rows, vocab], not {list(logits.shape)}")
    rows, vocab = logits.shape
    code = _native.dtype_code(logits.dtype)
    if logits.numel() and logits.stride(1) != 1:
        raise ValueError("the rows of logits must be contiguous")
    if out is None:
        out = torch.empty((rows, vocab), dtype=torch.float32, device=logits.device)
        out_code = _native.PL_F32
    else:
        if out.dtype is not torch.float32 and out.dtype is not logits.dtype:
            raise TypeError(f"out must be float32 or {logits.dtype}, not {out.dtype}")
        _check_tensor("out", out, out.dtype, device, (rows, vocab), dense=False)
        if out.numel() and out.stride(1) != 1:
            raise ValueError("the rows of out must be contiguous")
        out_code = _native.dtype_code(out.dtype)
    history = token_bytes = ld_tokens = n_bias = ld_bias = ld_allowed = 0
    if tokens is None:
        if lens is not None or prompt_lens is not None:
            raise ValueError("lens and prompt_lens count tokens, which are missing")
        if repetition is not None or presence is not None or frequency is not None:
            raise ValueError("penalties need the tokens they are for")
    else:
        if tokens.dtype is not torch.int64 and tokens.dtype is not torch.int32:
            raise TypeError(f"tokens must be int64 or int32, not {tokens.dtype}")
        if lens is None:
            raise ValueError("tokens need lens, the number of them in each row")
        history, ld_tokens = _rows_of("tokens", tokens, tokens.dtype, device, rows)
        token_bytes = tokens.element_size()
        _check_tensor("lens", lens, torch.int32, device, (rows,))
        if prompt_lens is not None:
            _check_tensor("prompt_lens", prompt_lens, torch.int32, device, (rows,))
        for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
            if t is not None:
                _check_tensor(name, t, torch.float32, device, (rows,))
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("bias_ids and bias_values go together")
    if bias_ids is not None:
        n_bias, ld_bias = _rows_of("bias_ids", bias_ids, torch.int32, device, rows)
        if _rows_of("bias_values", bias_values, torch.float32, device, rows) != (n_bias, ld_bias):
            raise ValueError("bias_ids and bias_values must have one shape and row stride")
    if allowed is not None:
        words, ld_allowed = _rows_of("allowed", allowed, torch.int32, device, rows)
        if words * 32 < vocab:
            raise ValueError(f"allowed has {words} words a row for a vocabulary of {vocab}")
    rc = _native.calls().pl_adjust_logits(
        code, out_code, logits.data_ptr(), logits.stride(0), out.data_ptr(), out.stride(0), rows, vocab,
        None if tokens is None else tokens.data_ptr(), token_bytes, ld_tokens, history,
        None if lens is None else lens.data_ptr(), None if prompt_lens is None else prompt_lens.data_ptr(),
        None if repetition is None else repetition.data_ptr(), None if presence is None else presence.data_ptr(),
        None if frequency is None else frequency.data_ptr(), None if bias_ids is None else bias_ids.data_ptr(),
        None if bias_values is None else bias_values.data_ptr(), ld_bias, n_bias,
        None if allowed is None else allowed.data_ptr(), ld_allowed, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        _native.check(rc, "pl_adjust_logits")
    return out

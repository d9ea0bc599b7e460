"""Paged key-value cache of a serving batch: append with the rotation by position, attention of one new token.

Every row of a batch is a request with its own adapter and its own length; its keys and values lie in pages of one
pool, in the order of its row of a page table.  ``rope_append`` rotates the new tokens' queries and keys and writes
keys and values to their places, ``paged_attention`` reads them for the row's newest token.  Rows are right-padded as
in the rest of the package: token t of row b counts for ``t < min(seq_lens[b], M)``.

A cache is ``[pages, kv_heads, page_size, head_dim]`` (any strides with a contiguous last dimension, so a permuted
``[pages, page_size, kv_heads, head_dim]`` too) in the model's dtype, or ``torch.float8_e4m3fn`` for 16-bit models with
an fp32 scale per key head; ``page_size`` is a power of two of at least 16, ``head_dim`` a multiple of 16 up to 256.

No counterpart in the reference, which leaves attention to the wrapped model.  There is no CPU path and no backward.
"""

from __future__ import annotations

import torch

from . import _native, sgmv

__all__ = ["paged_attention", "rope_append", "rope_table"]

_FP8 = torch.float8_e4m3fn


def rope_table(positions: int, rot: int, base: float = 10000.0, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), fp32 ``[positions, rot / 2]``: the angle of pair i at position p is ``p * base ** (-2 i / rot)``."""
    if rot < 0 or rot % 2:
        raise ValueError(f"the rotated part of a head is a whole number of pairs, not {rot} elements")
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2.0 * i / max(1, rot))
    return angle.cos().float(), angle.sin().float()



def _check_tensor(name: str, t: torch.Tensor, dtype: torch.dtype, device: int, shape: tuple, dense: bool = True) -> None:
    """A tensor argument: its dtype, its GPU, its shape (None: any size) and, if `dense`, that it is contiguous."""
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, not on the GPU of the other arguments")
    got = t.shape
    if len(got) != len(shape) or any(w is not None and w != g for g, w in zip(got, shape)):
        raise ValueError(f"{name} must have shape {['any' if w is None else w for w in shape]}, not {list(got)}")
    if dense and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _gpu(t: torch.Tensor, what: str) -> int:
    device = t.get_device()
    if not t.is_cuda:
        raise RuntimeError(f"{what}: polylora_amd computes only on a ROCm GPU through its HIP library; got a CPU "
                           "tensor (there is no CPU fallback)")
    return device


def _check_cache(key: torch.Tensor, value: torch.Tensor, table: torch.Tensor, rows: int, dim: int, dtype: torch.dtype,
                 device: int, k_scale, v_scale) -> int:
    """The cache arguments of both calls; returns the cache's dtype code."""
    if key.dim() != 4 or key.shape != value.shape:
        raise ValueError("the caches must be [pages, kv_heads, page_size, head_dim], both alike, not "
                         f"{list(key.shape)} and {list(value.shape)}")
    _, kv_heads, page_size, head_dim = key.shape
    if head_dim != dim:
        raise ValueError(f"the caches hold heads of {head_dim} elements, not {dim}")
    if key.dtype is dtype:
        code = _native.dtype_code(dtype)
        if k_scale is not None or v_scale is not None:
            raise ValueError("scales belong to an 8-bit cache")
    elif key.dtype is _FP8 and dtype is not torch.float32:
        code = _native.PL_F8E4M3
        if k_scale is None or v_scale is None:
            raise ValueError("an 8-bit cache needs k_scale and v_scale")
        _check_tensor("k_scale", k_scale, torch.float32, device, (kv_heads,))
        _check_tensor("v_scale", v_scale, torch.float32, device, (kv_heads,))
    else:
        raise TypeError(f"a cache holds the model's dtype ({dtype}) or, for 16-bit models, {_FP8}, not {key.dtype}")
    if value.dtype is not key.dtype or key.get_device() != device or value.get_device() != device:
        raise TypeError("the caches must have one dtype and lie on the GPU of the other arguments")
    if key.numel() and (key.stride(3) != 1 or value.stride(3) != 1):
        raise ValueError("the last dimension of the caches must be contiguous")
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError(f"a page must hold a power of two of at least 16 tokens, not {page_size}")
    _check_tensor("page_table", table, torch.int32, device, (rows, None), dense=False)
    if table.numel() and table.stride(1) != 1:
        raise ValueError("the rows of page_table must be contiguous")
    return code


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                page_table: torch.Tensor, past_lens: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                seq_lens: torch.Tensor | None = None, interleaved: bool = False, k_scale: torch.Tensor | None = None,
                v_scale: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate the new tokens' q and k by position, append k and v to the rows' pages; returns the rotated q.

    q ``[rows, M, heads, dim]``, k and v ``[rows, M, kv_heads, dim]`` with a contiguous last dimension (views of one
    fused projection too).  Token t of row b (``t < min(seq_lens[b], M)``; all M without seq_lens) has position
    ``past_lens[b] + t``; cos and sin are fp32 ``[positions, rot / 2]`` (``rope_table``) and rotate the first ``rot``
    elements of a head: its halves against each other, or the pairs (2i, 2i + 1) with ``interleaved``.  Both in fp32,
    rounded once.  page_table, past_lens and seq_lens are int32.  An 8-bit cache takes ``x / scale``, saturated.

    The rotated q comes back as a new contiguous tensor, 0 for padding tokens; ``k_out``, a contiguous tensor like k,
    also receives the rotated k, for attention inside a prompt.  A token beyond the cos table or on a page the table
    does not hold (an id outside the pool) counts as padding.
    """
    device = _gpu(q, "rope_append")
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError("q and k must be [rows, M, heads, dim] and [rows, M, kv_heads, dim], not "
                         f"{list(q.shape)} and {list(k.shape)}")
    rows, row_len, heads, dim = q.shape
    kv_heads = k.shape[2]
    dtype = q.dtype
    code = _native.dtype_code(dtype)
    _check_tensor("k", k, dtype, device, (rows, row_len, kv_heads, dim), dense=False)
    _check_tensor("v", v, dtype, device, (rows, row_len, kv_heads, dim), dense=False)
    cache_code = _check_cache(key_cache, value_cache, page_table, rows, dim, dtype, device, k_scale, v_scale)
    if key_cache.shape[1] != kv_heads or kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} heads and {kv_heads} key heads over a cache of {key_cache.shape[1]}")
    if q.numel() and (q.stride(3) != 1 or k.stride(3) != 1 or v.stride(3) != 1):
        raise ValueError("the last dimension of q, k and v must be contiguous")
    _check_tensor("past_lens", past_lens, torch.int32, device, (rows,))
    if seq_lens is not None:
        _check_tensor("seq_lens", seq_lens, torch.int32, device, (rows,))
    _check_tensor("cos", cos, torch.float32, device, (None, None))
    _check_tensor("sin", sin, torch.float32, device, tuple(cos.shape))
    positions, half = cos.shape
    if 2 * half > dim:
        raise ValueError(f"cos and sin rotate {2 * half} elements of heads of {dim}")
    if k_out is not None:
        _check_tensor("k_out", k_out, dtype, device, (rows, row_len, kv_heads, dim))
    q_out = torch.empty((rows, row_len, heads, dim), dtype=dtype, device=q.device)
    rc = _native.calls().pl_rope_append(
        code, cache_code, q.data_ptr(), q.stride()[:3], k.data_ptr(), k.stride()[:3], v.data_ptr(), v.stride()[:3],
        q_out.data_ptr(), None if k_out is None else k_out.data_ptr(), key_cache.data_ptr(), key_cache.stride()[:3],
        value_cache.data_ptr(), value_cache.stride()[:3], key_cache.shape[0], key_cache.shape[2],
        page_table.data_ptr(), page_table.stride(0), page_table.shape[1], past_lens.data_ptr(),
        None if seq_lens is None else seq_lens.data_ptr(), rows, row_len, heads, kv_heads, dim, cos.data_ptr(),
        sin.data_ptr(), positions, 2 * half, int(interleaved), None if k_scale is None else k_scale.data_ptr(),
        None if v_scale is None else v_scale.data_ptr(), torch._C._cuda_getCurrentRawStream(device))
    if rc:
        _native.check(rc, "pl_rope_append")
    return q_out


# One set of counters for each (device, stream), kept as the decode launch's are.
_COUNTERS: dict[tuple[int, int], sgmv._HandoffCounters] = {}


def _scratch(device: int, stream: int, dim: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The stream's workspace for parts of rows and its zeroed arrival counters."""
    held = _COUNTERS.get((device, stream))
    if held is None:
        held = _COUNTERS[device, stream] = sgmv._HandoffCounters(torch.device("cuda", device))
    nbytes = _native.load().pl_paged_attention_workspace_bytes(dim)
    return (sgmv._workspace(held.device, stream, "attention").get(nbytes),
            held.get(_native.PL_ATTENTION_COUNTER_INTS))


def paged_attention(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, page_table: torch.Tensor,
                    lens: torch.Tensor, *, scale: float | None = None, window: int | None = None,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per row over the row's pages: ``softmax(scale * q . keys) . values``.

    q ``[rows, heads, dim]`` (last dimension contiguous); heads is a multiple of the cache's kv_heads, each key head
    serving as many query heads in a row.  ``lens`` (int32) counts the row's tokens, the new one included (append it
    first); with ``window`` only the last that many of them count.  ``scale`` is ``dim ** -0.5`` unless given.  Sums and
    the softmax are fp32, the output is rounded once, into ``out`` (contiguous, like q) or a new tensor.  A row without
    a token gives 0; slots of pages beyond a row's tokens are never part of a result, whatever they hold.
    """
    device = _gpu(q, "paged_attention")
    if q.dim() != 3:
        raise ValueError(f"q must be [rows, heads, dim], not {list(q.shape)}")
    rows, heads, dim = q.shape
    dtype = q.dtype
    code = _native.dtype_code(dtype)
    cache_code = _check_cache(key_cache, value_cache, page_table, rows, dim, dtype, device, k_scale, v_scale)
    kv_heads = key_cache.shape[1]
    if kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} heads over a cache of {kv_heads} key heads")
    if q.numel() and q.stride(2) != 1:
        raise ValueError("the last dimension of q must be contiguous")
    _check_tensor("lens", lens, torch.int32, device, (rows,))
    if window is not None and window < 1:
        raise ValueError(f"window must be at least one token, not {window}")
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=dtype, device=q.device)
    else:
        _check_tensor("out", out, dtype, device, (rows, heads, dim))
    stream = torch._C._cuda_getCurrentRawStream(device)
    ws, counters = _scratch(device, stream, dim)
    rc = _native.calls().pl_paged_attention(
        code, cache_code, q.data_ptr(), q.stride()[:2], key_cache.data_ptr(), key_cache.stride()[:3],
        value_cache.data_ptr(), value_cache.stride()[:3], key_cache.shape[0], key_cache.shape[2],
        page_table.data_ptr(), page_table.stride(0), page_table.shape[1], lens.data_ptr(), rows, heads, kv_heads, dim,
        dim ** -0.5 if scale is None else scale, window or 0, None if k_scale is None else k_scale.data_ptr(),
        None if v_scale is None else v_scale.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(),
        counters.data_ptr(), counters.numel(), stream)
    if rc:
        _native.check(rc, "pl_paged_attention")
    return out

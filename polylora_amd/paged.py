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

import threading

import torch

from . import _native, sgmv

__all__ = ["paged_attention", "rope_append", "rope_table"]


def rope_table(positions: int, rot: int, base: float = 10000.0, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), fp32 ``[positions, rot / 2]``: the angle of pair i at position p is ``p * base ** (-2 i / rot)``."""
    if rot < 0 or rot % 2:
        raise ValueError(f"the rotated part of a head is a whole number of pairs, not {rot} elements")
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2.0 * i / max(1, rot))
    return angle.cos().float(), angle.sin().float()


def _stream(t: torch.Tensor) -> int:
    """The current stream of the tensor's GPU; 0 for a tensor on none, which the call refuses."""
    device = t.get_device()
    return torch._C._cuda_getCurrentRawStream(device) if device >= 0 else 0


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                page_table: torch.Tensor, past_lens: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                seq_lens: torch.Tensor | None = None, interleaved: bool = False, k_scale: torch.Tensor | None = None,
                v_scale: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate the new tokens' q and k by position, append k and v to the rows' pages; returns the rotated q.

    q ``[rows, M, heads, dim]``, k and v ``[rows, M, kv_heads, dim]`` with a contiguous last dimension (views of one
    fused projection too).  Token t of row b (``t < min(seq_lens[b], M)``; all M without seq_lens) has position
    ``past_lens[b] + t``; cos and sin are fp32 ``[positions, rot / 2]`` (``rope_table``) and rotate the first ``rot``
    elements of a head: its halves against each other, or the pairs (2i, 2i + 1) with ``interleaved``.  Both in fp32,
    rounded once.  page_table ``[rows, columns]`` (rows may share one, expanded), past_lens and seq_lens ``[rows]`` are
    int32.  An 8-bit cache takes ``x / scale``, saturated.  No two elements of the caches may share a place.

    The rotated q comes back as a new contiguous tensor, 0 for padding tokens; ``k_out``, a contiguous tensor like k,
    also receives the rotated k, for attention inside a prompt.  A token beyond the cos table or on a page the table
    does not hold (an id outside the pool) counts as padding.
    """
    return _native.tensor_calls().rope_append(q, k, v, key_cache, value_cache, page_table, past_lens, cos, sin, seq_lens,
                                              interleaved, k_scale, v_scale, k_out, _stream(q))


class _Scratch:
    """What the attention's launches use that run one after the other: the workspace for parts of rows, and arrival
    counters that are zero between launches."""

    def __init__(self, device: int) -> None:
        self.workspace = sgmv._Workspace(torch.device("cuda", device))
        self.counters: torch.Tensor | None = None
        self.args: dict[int, tuple[int, int, int, int]] = {}  # by head size; replaced workspaces stay allocated

    def get(self, dim: int) -> tuple[int, int, int, int]:
        return self.args.get(dim) or self._make(dim)

    def _make(self, dim: int) -> tuple[int, int, int, int]:
        with _LOCK:
            buf = self.workspace.get(int(_native.load().pl_paged_attention_workspace_bytes(dim)))
            if self.counters is None:
                # by a fill kernel on the current stream, the launch's, which a HIP graph records like any other
                self.counters = torch.empty(_native.PL_ATTENTION_COUNTER_INTS, dtype=torch.int32, device=buf.device).zero_()
            args = buf.data_ptr(), buf.numel(), self.counters.data_ptr(), self.counters.numel()
            self.args[dim] = args
            return args


_LOCK = threading.Lock()
# One for each (device, stream), for the life of the process.
_SCRATCH: dict[tuple[int, int], _Scratch] = {}
# What the last HIP graph captured on a (device, stream) got: (capture id, its own).  Graphs captured on one stream may
# be replayed beside each other and beside the stream's own work, so they share nothing with either.  The memory is
# the graph's, from the pool that it is captured into, and lasts as long as that.
_CAPTURED: dict[tuple[int, int], tuple[int, _Scratch]] = {}


def _scratch(t: torch.Tensor, stream: int) -> tuple[int, int, int, int]:
    device = t.get_device()
    if device < 0 or t.dim() == 0:
        return 0, 0, 0, 0  # the call refuses the tensor
    key = device, stream
    capture = _native.tensor_calls().stream_capture_id(stream)
    if capture:
        held = _CAPTURED.get(key)
        if held is None or held[0] != capture or capture < 0:  # below 0: a capture of unknown id
            held = _CAPTURED[key] = capture, _Scratch(device)
        return held[1].get(t.shape[-1])
    held = _SCRATCH.get(key)
    if held is None:
        held = _SCRATCH.setdefault(key, _Scratch(device))
    return held.get(t.shape[-1])


def paged_attention(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, page_table: torch.Tensor,
                    lens: torch.Tensor, *, scale: float | None = None, window: int | None = None,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per row over the row's pages: ``softmax(scale * q . keys) . values``.

    q ``[rows, heads, dim]`` (last dimension contiguous); heads is a multiple of the cache's kv_heads, each key head
    serving as many query heads in a row.  ``lens`` (int32) counts the row's tokens, the new one included (append it
    first); with ``window`` only the last that many of them count.  ``scale`` is ``dim ** -0.5`` unless given.  Sums and
    the softmax are fp32, the output is rounded once, into ``out`` (contiguous, like q) or a new tensor.  A row without
    a token, or whose scores are all -inf, gives 0; slots of pages beyond a row's tokens are never part of a result,
    whatever they hold.

    Calls on one stream share a workspace and counters; a HIP graph has its own, so its replays may overlap other work,
    but not each other.
    """
    stream = _stream(q)
    return _native.tensor_calls().paged_attention(q, key_cache, value_cache, page_table, lens, scale, window, k_scale,
                                                  v_scale, out, *_scratch(q, stream), stream)

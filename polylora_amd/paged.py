"""Paged key-value cache of a serving batch: append with the rotation by position, attention of new and drafted tokens.

Every row of a batch is a request with its own adapter and its own length; its keys and values lie in pages of one
pool, in the order of its row of a page table.  ``rope_append`` rotates the new tokens' queries and keys and writes
keys and values to their places, ``paged_attention`` reads them for the row's newest token.  Rows are right-padded as
in the rest of the package: token t of row b counts for ``t < min(seq_lens[b], M)``.

Where several tokens of a row are drafted and looked at in one pass, ``rope_append`` appends all of them (``depths``
where they form a tree), ``tree_attention`` is their attention over the pages and over one another,
``drafts.verify_tokens`` says which of them stay, and ``keep_tokens`` moves those up behind the row's tokens.

A cache is ``[pages, kv_heads, page_size, head_dim]`` (any strides with a contiguous last dimension, so a permuted
``[pages, page_size, kv_heads, head_dim]`` too) in the model's dtype, or ``torch.float8_e4m3fn`` for 16-bit models with
an fp32 scale per key head; ``page_size`` is a power of two of at least 16, ``head_dim`` a multiple of 16 up to 256.

No counterpart in the reference, which leaves attention to the wrapped model.  There is no CPU path and no backward.
"""

from __future__ import annotations

import threading

import torch

from . import _native, sgmv

__all__ = ["keep_tokens", "paged_attention", "rope_append", "rope_table", "tree_attention"]


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
                v_scale: torch.Tensor | None = None, k_out: torch.Tensor | None = None,
                q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                depths: torch.Tensor | None = None) -> torch.Tensor:
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

    With ``q_norm`` and ``k_norm`` (``[dim]``, fp32 or q's dtype, both of one; either may be None) each head of q and k is
    first divided by ``sqrt(mean(x ** 2) + eps)`` and multiplied by the weights, in fp32 like the rest and not rounded in
    between (its squares too: elements beyond 2 ** 59 may give 0).  ``depths`` (int32 ``[rows, M]``, or ``[M]`` for all
    rows) is for tokens that form a tree: token t is rotated by position ``past_lens[b] + depths[b, t]``, its place in the
    pages stays ``past_lens[b] + t``.
    """
    return _native.tensor_calls().rope_append(q, k, v, key_cache, value_cache, page_table, past_lens, cos, sin, seq_lens,
                                              interleaved, k_scale, v_scale, k_out, q_norm, k_norm, eps, depths,
                                              _stream(q))


class _Scratch:
    """What launches use that run one after the other: a workspace for parts of the work, and arrival counters that are
    zero between launches."""

    def __init__(self, device: int) -> None:
        self.workspace = sgmv._Workspace(torch.device("cuda", device))
        self.counters: torch.Tensor | None = None
        self.retired: list[torch.Tensor] = []
        # by call and its sizes; replaced buffers stay allocated
        self.args: dict[tuple, tuple[int, int, int, int]] = {}

    def get(self, call: str, *sizes: int) -> tuple[int, int, int, int]:
        return self.args.get((call, *sizes)) or self._make(call, *sizes)

    def _make(self, call: str, *sizes: int) -> tuple[int, int, int, int]:
        lib = _native.load()
        with _LOCK:
            buf = self.workspace.get(int(getattr(lib, f"pl_{call}_workspace_bytes")(*sizes)))
            ints = int(lib.pl_verify_counter_ints(*sizes[:2])) if call == "verify" else 0
            ints = max(ints, _native.PL_ATTENTION_COUNTER_INTS)
            if self.counters is None or self.counters.numel() < ints:
                if self.counters is not None:
                    self.retired.append(self.counters)
                    ints = max(ints, 2 * self.counters.numel())
                # by a fill kernel on the current stream, the launch's, which a HIP graph records like any other
                self.counters = torch.empty(ints, dtype=torch.int32, device=buf.device).zero_()
            args = buf.data_ptr(), buf.numel(), self.counters.data_ptr(), self.counters.numel()
            if len(self.args) >= 4096:  # a batch of every size
                self.args.clear()
            self.args[(call, *sizes)] = args
            return args


_LOCK = threading.Lock()
# One for each (device, stream), for the life of the process.
_SCRATCH: dict[tuple[int, int], _Scratch] = {}
# What the last HIP graph captured on a (device, stream) got: (capture id, its own).  Graphs captured on one stream may
# be replayed beside each other and beside the stream's own work, so they share nothing with either.  The memory is
# the graph's, from the pool that it is captured into, and lasts as long as that.
_CAPTURED: dict[tuple[int, int], tuple[int, _Scratch]] = {}


def _scratch(t: torch.Tensor, stream: int, call: str, *sizes: int) -> tuple[int, int, int, int]:
    device = t.get_device()
    if device < 0:
        return 0, 0, 0, 0  # the call refuses the tensor
    key = device, stream
    capture = _native.tensor_calls().stream_capture_id(stream)
    if capture:
        held = _CAPTURED.get(key)
        if held is None or held[0] != capture or capture < 0:  # below 0: a capture of unknown id
            held = _CAPTURED[key] = capture, _Scratch(device)
        return held[1].get(call, *sizes)
    held = _SCRATCH.get(key)
    if held is None:
        held = _SCRATCH.setdefault(key, _Scratch(device))
    return held.get(call, *sizes)


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

    Calls on one stream share a workspace and counters (``tree_attention``'s too); a HIP graph has its own, so its replays
    may overlap other work, but not each other.
    """
    stream = _stream(q)
    return _native.tensor_calls().paged_attention(q, key_cache, value_cache, page_table, lens, scale, window, k_scale,
                                                  v_scale, out, *_scratch(q, stream, "paged_attention", *(q.shape[-1:] or (0,))), stream)


def tree_attention(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, page_table: torch.Tensor,
                   past_lens: torch.Tensor, *, seq_lens: torch.Tensor | None = None,
                   visible: torch.Tensor | None = None, depths: torch.Tensor | None = None,
                   scale: float | None = None, window: int | None = None, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of several new tokens of each row, drafts or a piece of a prompt, over its pages and one another.

    q ``[rows, M, heads, dim]`` (last dimension contiguous): token t of row b (``t < min(seq_lens[b], M)``) was appended
    to place ``past_lens[b] + t`` (``rope_append``).  It sees the row's ``past_lens[b]`` tokens before these and, of
    these, itself and those before it; or, with ``visible``, those whose bit is set in its mask: int32
    ``[rows, M, words]`` (or ``[M, words]`` for all rows), bit ``j % 32`` of word ``j // 32`` for token j
    (``drafts.tree_tables`` makes them from the tokens' parents).  With ``window`` a token sees the last that many, itself
    included, by position; in a tree, of at most ``window`` tokens, that is by ``depths`` and holds for the tokens before
    the tree.  scale, scales, precision, ``out`` and rows that see nothing are ``paged_attention``'s; padding tokens get 0.
    """
    stream = _stream(q)
    # columns of the products: the workspace goes by whether they are few, which those of fp32 count as
    fits = q.dim() == 4 and key_cache.dim() == 4 and q.dtype != torch.float32
    columns = q.shape[1] * q.shape[2] // max(1, key_cache.shape[1]) if fits else 0
    return _native.tensor_calls().tree_attention(q, key_cache, value_cache, page_table, past_lens, seq_lens, visible,
                                                 depths, scale, window, k_scale, v_scale, out,
                                                 *_scratch(q, stream, "tree_attention", *(q.shape[-1:] or (0,)), min(columns, 128)),
                                                 stream)


def keep_tokens(key_caches, value_caches, page_table: torch.Tensor, past_lens: torch.Tensor, path: torch.Tensor,
                counts: torch.Tensor) -> None:
    """Move the keys and values of the tokens that stay up behind the row's tokens, in every layer's caches.

    ``key_caches`` and ``value_caches`` are sequences of caches, one for each layer, alike in shape, strides and dtype and
    none over another.  Row b keeps the tokens at places ``past_lens[b] + path[b, i]``, ``i < counts[b]``: they move to
    ``past_lens[b] + i``.  path is int32 ``[rows, n]`` and ascends (``drafts.verify_tokens`` gives it; a row's path ends at
    an entry that does not); counts and past_lens are int32 ``[rows]``.  Moves from or to pages that the table does not
    hold are left out.  Rows that move tokens do not share the pages they move them in.
    """
    _native.tensor_calls().keep_tokens(key_caches, value_caches, page_table, past_lens, path, counts, _stream(path))

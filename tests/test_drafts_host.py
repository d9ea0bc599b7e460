"""The drafted tokens' operators on the host: refusals that come before any launch, trees' tables, the plain forms."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from oracle import decode as one_token
from oracle import drafts as plain
from polylora_amd import _native
from polylora_amd.drafts import tree_tables, verify_tokens
from polylora_amd.paged import keep_tokens, rope_append, rope_table, tree_attention


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 2, 32)
    key, table = torch.zeros(1, 2, 16, 32), torch.zeros(1, 1, dtype=torch.int32)
    lens = torch.zeros(1, dtype=torch.int32)
    cos, sin = rope_table(4, 32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rope_append(x, x, x, key, key, table, lens, cos, sin, q_norm=torch.ones(32))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        tree_attention(x, key, key, table, lens)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        keep_tokens([key], [key], table, lens, torch.zeros(1, 2, dtype=torch.int32), lens)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        verify_tokens(torch.zeros(1, 2, 8), torch.zeros(1, 2, dtype=torch.int64), torch.zeros(1, 2))
    with pytest.raises(TypeError, match="sequence"):
        keep_tokens(3, [key], table, lens, table, lens)
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        _native.tensor_calls().verify_tokens(*[None] * 7, 0, 0, 0, 0, 0)


def test_tree_tables_of_a_tree():
    parents = torch.tensor([-1, 0, 0, 1, 3, 2, -1], dtype=torch.int32)
    depths, visible = tree_tables(parents)
    assert depths.tolist() == [0, 1, 1, 2, 3, 2, 0] and depths.dtype == visible.dtype == torch.int32
    seen = [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {0, 1, 3, 4}, {0, 2, 5}, {6}]
    assert visible.tolist() == [[sum(1 << j for j in s)] for s in seen]
    with pytest.raises(TypeError):
        tree_tables(torch.zeros(3))


@pytest.mark.parametrize("m", [0, 1, 31, 32, 33, 70])
def test_tree_tables_of_batches(m):
    gen = torch.Generator().manual_seed(m)
    parents = torch.tensor([[-1 if t == 0 else int(torch.randint(-1 if t % 7 == 0 else 0, t, (), generator=gen))
                             for t in range(m)] for _ in range(3)], dtype=torch.int64).view(3, m)
    depths, visible = tree_tables(parents)
    assert depths.shape == (3, m) and visible.shape == (3, m, -(-m // 32))
    for b in range(3):
        for t in range(m):
            line, a = set(), t
            while a >= 0:
                line.add(a)
                a = int(parents[b, a])
            assert int(depths[b, t]) == len(line) - 1
            assert {j for j in range(m) if int(visible[b, t, j // 32]) >> (j % 32) & 1} == line


def _i64(*v):
    return ctypes.cast((ctypes.c_int64 * len(v))(*v), ctypes.c_void_p)


def _pointers(*v):
    return ctypes.cast((ctypes.c_void_p * len(v))(*v), ctypes.c_void_p)


def _refused(fn, args, **changes):
    """Status of a call whose arguments the library refuses before it launches anything."""
    got = dict(args)
    got.update(changes)
    rc = fn(*got.values())
    assert rc != 0 and _native.load().pl_last_error()
    return rc


def test_norm_append_refusals_of_the_library():
    lib = _native.load()
    s, p = _i64(64, 32, 16), 4096
    good = dict(dtype=1, cache=1, q=p, qs=s, k=2 * p, ks=s, v=3 * p, vs=s, out=1 << 20, k_out=None, key=p, keys=s, value=p,
                values=s, pages=4, page=16, table=p, ld=2, cols=2, past=p, seq=None, rows=1, m=2, heads=2, kv=2, dim=16,
                cos=p, sin=p, positions=8, rot=16, inter=0, ksc=None, vsc=None, qn=p, kn=p, norm=1, eps=1e-6, depths=p,
                depths_ld=2, stream=None)
    call = lib.pl_norm_rope_append
    assert _refused(call, good, norm=2) == _native.PL_ERR_ARG  # fp16 weights for a bf16 model
    assert _refused(call, good, eps=0.0) == _native.PL_ERR_ARG
    assert _refused(call, good, eps=-1.0) == _native.PL_ERR_ARG
    assert _refused(call, good, eps=math.inf) == _native.PL_ERR_ARG
    assert _refused(call, good, eps=math.nan) == _native.PL_ERR_ARG
    assert _refused(call, good, heads=3) == _native.PL_ERR_ARG
    assert _refused(call, good, out=p) == _native.PL_ERR_ARG  # over q
    assert _refused(call, good, dim=24) == _native.PL_ERR_LIMIT
    assert call(*{**good, "rows": 0}.values()) == 0 and call(*{**good, "m": 0}.values()) == 0  # nothing to do


def test_keep_refusals_of_the_library():
    lib = _native.load()
    p = 4096
    good = dict(dtype=1, layers=2, keys=_pointers(p, 2 * p), values=_pointers(3 * p, 4 * p), strides=_i64(512, 256, 16),
                pages=4, page=16, kv=2, dim=16, table=p, ld=2, cols=2, past=p, path=p, path_ld=4, n=4, counts=p, rows=2,
                stream=None)
    call = lib.pl_keep_tokens
    assert _refused(call, good, dtype=9) == _native.PL_ERR_ARG
    assert _refused(call, good, layers=-1) == _native.PL_ERR_ARG
    assert _refused(call, good, n=-1) == _native.PL_ERR_ARG
    assert _refused(call, good, path_ld=3) == _native.PL_ERR_ARG
    assert _refused(call, good, keys=None) == _native.PL_ERR_ARG
    assert _refused(call, good, keys=_pointers(p, None)) == _native.PL_ERR_ARG
    assert _refused(call, good, keys=_pointers(p, p + 8)) == _native.PL_ERR_ALIGN
    assert _refused(call, good, strides=_i64(512, 256, 8)) == _native.PL_ERR_ARG  # slots over one another
    assert _refused(call, good, strides=_i64(512, 256, 17)) == _native.PL_ERR_ALIGN
    assert _refused(call, good, counts=None) == _native.PL_ERR_ARG
    assert _refused(call, good, path=None) == _native.PL_ERR_ARG
    assert _refused(call, good, page=8) == _native.PL_ERR_LIMIT
    for nothing in ({"rows": 0}, {"n": 0}, {"layers": 0}, {"pages": 0}):
        assert call(*{**good, **nothing}.values()) == 0


def test_tree_attention_refusals_of_the_library():
    lib = _native.load()
    s, p = _i64(64, 32, 16), 4096
    good = dict(dtype=1, cache=1, q=p, qs=s, key=p, keys=s, value=p, values=s, pages=4, page=16, table=p, ld=2, cols=2,
                past=p, seq=None, visible=p, vrow=8, vtoken=1, words=1, depths=p, drow=4, rows=2, m=4, heads=2, kv=2,
                dim=16, scale=1.0, window=0, ksc=None, vsc=None, out=1 << 20)
    good.update(_TREE_SCRATCH)
    call = lib.pl_tree_attention
    assert _refused(call, good, window=-1) == _native.PL_ERR_ARG
    assert _refused(call, good, window=3) == _native.PL_ERR_ARG  # shorter than the tree
    assert _refused(call, good, window=8, depths=None) == _native.PL_ERR_ARG
    assert _refused(call, good, m=33) == _native.PL_ERR_ARG  # more tokens than bits
    assert _refused(call, good, past=None) == _native.PL_ERR_ARG
    assert _refused(call, good, out=p) == _native.PL_ERR_ARG  # over q
    assert _refused(call, good, value=p + 8) == _native.PL_ERR_ALIGN
    assert _refused(call, good, heads=3) == _native.PL_ERR_ARG
    assert _refused(call, good, wsb=lib.pl_tree_attention_workspace_bytes(16, 4) - 1) == _native.PL_ERR_ARG
    assert _refused(call, good, counters=None) == _native.PL_ERR_ARG
    assert _refused(call, good, ints=16) == _native.PL_ERR_ARG
    assert _refused(call, good, heads=2050, qs=_i64(1 << 20, 1 << 17, 16)) == _native.PL_ERR_LIMIT
    assert _refused(call, good, keys=_i64(64, 32, 1 << 30)) == _native.PL_ERR_LIMIT
    assert _refused(call, good, rows=1 << 20, cols=1 << 26, ld=1 << 26, out=1 << 60) == _native.PL_ERR_LIMIT
    need = lib.pl_tree_attention_workspace_bytes
    assert need(0, 4) == need(257, 4) == need(64, -1) == 0 and need(64, 96) < need(64, 97)
    assert call(*{**good, "rows": 0}.values()) == 0 and call(*{**good, "m": 0}.values()) == 0


# What a call gets beside its arguments proper.
_TREE_SCRATCH = {"ws": 4096, "wsb": 1 << 30, "counters": 4096, "ints": _native.PL_ATTENTION_COUNTER_INTS, "stream": None}
_VERIFY_SCRATCH = {"ws": 4096, "wsb": 1 << 30, "counters": 4096, "ints": 1 << 20, "stream": None}


def test_verification_refusals_of_the_library():
    lib = _native.load()
    p = 4096
    good = dict(dtype=0, logits=p, row=80, node=16, tokens=p, token_bytes=8, ld_tokens=5, uniforms=p, ld_uniforms=5,
                parents=None, ld_parents=0, probs=p, probs_row=64, probs_node=16, heat=p, seq=None, rows=2, nodes=5,
                vocab=16, path=p, counts=p, next=p)
    good.update(_VERIFY_SCRATCH)
    call = lib.pl_verify_tokens
    assert _refused(call, good, dtype=3) == _native.PL_ERR_ARG
    assert _refused(call, good, token_bytes=2) == _native.PL_ERR_ARG
    assert _refused(call, good, vocab=-1) == _native.PL_ERR_ARG
    assert _refused(call, good, vocab=1 << 30) == _native.PL_ERR_LIMIT
    assert _refused(call, good, parents=p) == _native.PL_ERR_ARG  # probabilities of a tree
    for name in ("logits", "tokens", "uniforms", "path", "counts", "next"):
        assert _refused(call, good, **{name: None}) == _native.PL_ERR_ARG
    assert _refused(call, good, nodes=1025) == _native.PL_ERR_LIMIT
    assert _refused(call, good, wsb=lib.pl_verify_workspace_bytes(2, 5, 16) - 1) == _native.PL_ERR_ARG
    assert _refused(call, good, ints=lib.pl_verify_counter_ints(2, 5) - 1) == _native.PL_ERR_ARG
    assert _refused(call, good, counters=None) == _native.PL_ERR_ARG
    assert call(*{**good, "rows": 0}.values()) == 0


def test_plain_tree_attention_of_one_token_is_the_single_tokens():
    gen = torch.Generator().manual_seed(3)
    key, value = (torch.randn(6, 2, 16, 16, generator=gen) for _ in range(2))
    table = torch.tensor([[3, 0, -1], [5, 2, 1]], dtype=torch.int32)
    lens = torch.tensor([20, 37])
    q = torch.randn(2, 1, 4, 16, generator=gen)
    for window in (None, 7):
        want = one_token.paged_attention(q[:, 0], key, value, table, lens, window=window)[0]
        got = plain.tree_attention(q, key, value, table, lens - 1, window=window)[0][:, 0]
        assert float((got - want).abs().max()) < 1e-12


def test_plain_line_is_a_tree_of_one_branch():
    gen = torch.Generator().manual_seed(4)
    key, value = (torch.randn(6, 2, 16, 16, generator=gen) for _ in range(2))
    table = torch.tensor([[3, 0, 4], [5, 2, 1]], dtype=torch.int32)
    past = torch.tensor([20, 31])
    q = torch.randn(2, 5, 4, 16, generator=gen)
    seen = torch.ones(5, 5, dtype=torch.bool).tril().expand(2, 5, 5)
    depths = torch.arange(5).expand(2, 5)
    for window in (None, 9):
        a = plain.tree_attention(q, key, value, table, past, visible=seen, depths=depths, window=window)[0]
        b = plain.tree_attention(q, key, value, table, past, window=window)[0]
        assert float((a - b).abs().max()) < 1e-12


def test_plain_verification_keeps_the_models_distribution():
    """What follows token 0 is distributed as the model has it, whatever the drafts' probabilities: summed over a grid of
    random numbers, each of which stands for as much."""
    gen = torch.Generator().manual_seed(5)
    vocab, steps = 5, 40
    logits = torch.randn(1, 2, vocab, generator=gen)
    q = torch.softmax(torch.randn(1, 1, vocab, generator=gen), -1)
    p = torch.softmax(logits[0, 0].double(), -1)
    grid = (torch.arange(steps) + 0.5) / steps
    got = torch.zeros(vocab, dtype=torch.float64)
    for d in range(vocab):
        tokens = torch.tensor([[0, d]])
        for u in grid.tolist():
            for w in grid.tolist():
                path, counts, following = plain.verify_tokens(logits, tokens, torch.tensor([[u, w]]), draft_probs=q)
                stays = int(counts[0]) == 2
                got[d if stays else int(following[0])] += float(q[0, 0, d]) / steps**2
    # each of the grid's borders is off by at most one of its steps, in acceptance and in drawing
    assert float((got - p).abs().max()) < 2.0 / steps
    assert abs(float(got.sum()) - 1) < 1e-5

"""Faults that a step over drafted tokens once had and that the host alone shows."""

from __future__ import annotations

import pytest
import torch

from polylora_amd import _native
from polylora_amd.drafts import tree_tables

from .test_drafts_host import _TREE_SCRATCH, _VERIFY_SCRATCH, _i64, _refused


@pytest.mark.parametrize("shift", [16, 64])
def test_attention_workspaces_begin_with_a_line(shift):
    """Parts of two workgroups on one line of the L2 could not be handed over."""
    lib = _native.load()
    s, p = _i64(64, 32, 16), 4096
    good = dict(dtype=1, cache=1, q=p, qs=s, key=p, keys=s, value=p, values=s, pages=4, page=16, table=p, ld=2, cols=2,
                past=p, seq=None, visible=None, vrow=0, vtoken=0, words=0, depths=None, drow=0, rows=2, m=4, heads=2, kv=2,
                dim=16, scale=1.0, window=0, ksc=None, vsc=None, out=1 << 20)
    good.update(_TREE_SCRATCH)
    assert _refused(lib.pl_tree_attention, good, ws=4096 + shift) == _native.PL_ERR_ALIGN
    good = dict(dtype=1, cache=1, q=p, qs=s, key=p, keys=s, value=p, values=s, pages=4, page=16, table=p, ld=2, cols=2,
                lens=p, rows=2, heads=2, kv=2, dim=16, scale=1.0, window=0, ksc=None, vsc=None, out=1 << 20)
    good.update(_TREE_SCRATCH)
    assert _refused(lib.pl_paged_attention, good, ws=4096 + shift) == _native.PL_ERR_ALIGN


def test_attention_workspaces_are_no_larger_than_what_is_launched_takes():
    """Two parts of 512 workers of 16 columns of heads above 128 elements, of 32 below; fp32 has no kernel for more columns."""
    lib = _native.load()
    need = lib.pl_tree_attention_workspace_bytes
    part = {64: 16 * (64 + 2) * 4, 128: 16 * (128 + 2) * 4, 256: 16 * (256 + 2) * 4}  # 16 columns, and two sums to each
    for dim, dp, sixteens in ((16, 64, 2), (64, 64, 2), (80, 128, 2), (128, 128, 2), (144, 256, 1), (256, 256, 1)):
        assert need(dim, 1) == need(dim, 32) == 2 * 512 * sixteens * part[dp]
        assert need(dim, 1) <= 17 << 20
    s, p = _i64(1 << 20, 64 * 40, 64), 4096
    good = dict(dtype=0, cache=0, q=p, qs=s, key=p, keys=_i64(2048, 1024, 64), value=p, values=_i64(2048, 1024, 64), pages=4,
                page=16, table=p, ld=2, cols=2, past=p, seq=None, visible=None, vrow=0, vtoken=0, words=0, depths=None,
                drow=0, rows=2, m=9, heads=40, kv=1, dim=64, scale=1.0, window=0, ksc=None, vsc=None, out=1 << 40)
    good.update(_TREE_SCRATCH)
    # fp32 of 360 columns takes what one column does: no later check finds fault but the workspace's place
    assert _refused(lib.pl_tree_attention, good, ws=4096 + 64, wsb=need(64, 1)) == _native.PL_ERR_ALIGN
    assert _refused(lib.pl_tree_attention, good, ws=4096 + 64, wsb=need(64, 1) - 1) == _native.PL_ERR_ARG
    assert _refused(lib.pl_tree_attention, good, ws=4096 + 64, wsb=need(64, 1), dtype=1, cache=1) == _native.PL_ERR_ARG


@pytest.mark.parametrize("name", ["pl_rope_append", "pl_norm_rope_append"])
def test_append_refusals_name_the_function_that_was_called(name):
    lib = _native.load()
    s, p = _i64(64, 32, 16), 4096
    good = dict(dtype=1, cache=1, q=p, qs=s, k=2 * p, ks=s, v=3 * p, vs=s, out=1 << 20, k_out=None, key=p, keys=s, value=2 * p,
                values=s, pages=4, page=16, table=p, ld=2, cols=2, past=p, seq=None, rows=1, m=2, heads=2, kv=2, dim=16,
                cos=p, sin=p, positions=8, rot=16, inter=0, ksc=None, vsc=None)
    if name == "pl_norm_rope_append":
        good.update(qn=p, kn=p, norm=1, eps=1e-6, depths=None, depths_ld=0)
    good["stream"] = None
    for bad in (dict(dim=24), dict(rot=3), dict(past=None), dict(out=p), dict(value=p), dict(rows=1 << 30)):
        _refused(getattr(lib, name), good, **bad)
        assert lib.pl_last_error().decode().startswith(name + ": "), (bad, lib.pl_last_error())


def test_append_without_norms_does_not_look_at_eps():
    """Refused for what comes after eps, not for it."""
    lib = _native.load()
    s, p = _i64(64, 32, 16), 4096
    good = dict(dtype=1, cache=1, q=p, qs=s, k=2 * p, ks=s, v=3 * p, vs=s, out=1 << 20, k_out=None, key=p, keys=s, value=2 * p,
                values=s, pages=4, page=16, table=p, ld=2, cols=2, past=p, seq=None, rows=1, m=2, heads=2, kv=2, dim=24,
                cos=p, sin=p, positions=8, rot=16, inter=0, ksc=None, vsc=None, qn=None, kn=None, norm=1, eps=0.0, depths=p,
                depths_ld=2, stream=None)
    for eps in (0.0, -1.0, float("nan")):
        assert _refused(lib.pl_norm_rope_append, good, eps=eps) == _native.PL_ERR_LIMIT  # the head size
        assert _refused(lib.pl_norm_rope_append, good, eps=eps, kn=p) == _native.PL_ERR_ARG


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_a_token_whose_parent_is_not_before_it_is_a_root(dtype):
    """Token 0 as its own parent too: it was one deeper than a root, and all tokens behind it."""
    parents = torch.tensor([[0, 0, 1, 1, 9], [-1, 1, 0, 4, 2], [-7, 2**30, 1, 0, 4]], dtype=dtype)
    depths, visible = tree_tables(parents)
    assert depths.tolist() == [[0, 1, 2, 2, 0], [0, 0, 1, 0, 2], [0, 0, 1, 1, 0]]
    assert visible[..., 0].tolist() == [[1, 3, 7, 11, 16], [1, 2, 5, 8, 21], [1, 2, 6, 9, 16]]
    depths, visible = tree_tables(parents[:, :0])
    assert depths.shape == (3, 0) and visible.shape == (3, 0, 0)


def test_verification_scratch_is_aligned_as_the_header_says():
    lib = _native.load()
    p = 4096
    good = dict(dtype=0, logits=p, row=80, node=16, tokens=p, token_bytes=8, ld_tokens=5, uniforms=p, ld_uniforms=5,
                parents=None, ld_parents=0, probs=p, probs_row=64, probs_node=16, heat=p, seq=None, rows=2, nodes=5,
                vocab=16, path=p, counts=p, next=p)
    good.update(_VERIFY_SCRATCH)
    for bad in (dict(ws=p + 8), dict(ws=p + 64), dict(counters=p + 4)):
        assert _refused(lib.pl_verify_tokens, good, **bad) == _native.PL_ERR_ALIGN

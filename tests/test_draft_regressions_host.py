"""Faults that a step over drafted tokens once had and that the host alone shows."""

from __future__ import annotations

import pytest

from polylora_amd import _native

from .test_drafts_host import _TREE_SCRATCH, _i64, _refused


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

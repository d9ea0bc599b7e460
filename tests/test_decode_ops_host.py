"""The decode operators' host side: refusals that come before any launch, masks, angles, the plain forms themselves."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from oracle import decode as plain
from polylora_amd import _native
from polylora_amd.logits import adjust_logits, pack_allowed
from polylora_amd.paged import paged_attention, rope_append, rope_table


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 2, 32)
    key, table = torch.zeros(1, 2, 16, 32), torch.zeros(1, 1, dtype=torch.int32)
    lens = torch.zeros(1, dtype=torch.int32)
    cos, sin = rope_table(4, 32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rope_append(x, x, x, key, key, table, lens, cos, sin)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_attention(x[:, 0], key, key, table, lens)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        adjust_logits(torch.zeros(1, 8))


def test_things_that_are_no_tensors_are_refused():
    calls = _native.tensor_calls()
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        calls.adjust_logits(*[None] * 11, 0)
    with pytest.raises(TypeError, match="taken"):
        calls.paged_attention(1, 2)


def test_pack_allowed_places_each_bit():
    gen = torch.Generator().manual_seed(0)
    for vocab in (1, 31, 32, 33, 100):
        mask = torch.rand(3, vocab, generator=gen) < 0.5
        words = pack_allowed(mask)
        assert words.shape == (3, -(-vocab // 32)) and words.dtype == torch.int32
        for b in range(3):
            for v in range(vocab):
                assert bool(int(words[b, v // 32]) >> (v % 32) & 1) == bool(mask[b, v])
    assert pack_allowed(torch.ones(32, dtype=torch.bool)).tolist() == [-1]
    with pytest.raises(TypeError):
        pack_allowed(torch.ones(4))


def test_rope_table_angles():
    cos, sin = rope_table(5, 6, base=100.0)
    assert cos.shape == sin.shape == (5, 3) and cos.dtype == torch.float32
    for p in range(5):
        for i in range(3):
            angle = p * 100.0 ** (-2 * i / 6)
            assert abs(float(cos[p, i]) - math.cos(angle)) < 1e-7 and abs(float(sin[p, i]) - math.sin(angle)) < 1e-7
    assert rope_table(4, 0)[0].shape == (4, 0)
    with pytest.raises(ValueError):
        rope_table(4, 5)


def _i64(*v):
    return ctypes.cast((ctypes.c_int64 * len(v))(*v), ctypes.c_void_p)


def _refused(fn, args, **changes):
    """Status of a call whose arguments the library refuses before it launches anything."""
    got = dict(args)
    got.update(changes)
    rc = fn(*got.values())
    assert rc != 0 and _native.load().pl_last_error()
    return rc


def test_append_refusals_of_the_library():
    lib = _native.load()
    s, p = _i64(64, 32, 16), 4096
    good = dict(dtype=1, cache=1, q=p, qs=s, k=2 * p, ks=s, v=3 * p, vs=s, out=1 << 20, k_out=None, key=p, keys=s, value=p,
                values=s, pages=4, page=16, table=p, ld=2, cols=2, past=p, seq=None, rows=1, m=2, heads=2, kv=2, dim=16,
                cos=p, sin=p, positions=8, rot=16, inter=0, ksc=None, vsc=None, stream=None)
    one = lib.pl_rope_append
    assert _refused(one, good, dtype=7) == _native.PL_ERR_ARG
    assert _refused(one, good, dtype=0, cache=3, ksc=p, vsc=p) == _native.PL_ERR_ARG  # 8 bits for fp32
    assert _refused(one, good, cache=3) == _native.PL_ERR_ARG  # no scales
    assert _refused(one, good, ksc=p) == _native.PL_ERR_ARG  # scales of a 16-bit cache
    assert _refused(one, good, heads=3) == _native.PL_ERR_ARG
    assert _refused(one, good, dim=24) == _native.PL_ERR_LIMIT
    assert _refused(one, good, dim=272) == _native.PL_ERR_LIMIT
    assert _refused(one, good, page=24) == _native.PL_ERR_LIMIT
    assert _refused(one, good, page=8) == _native.PL_ERR_LIMIT
    assert _refused(one, good, ld=1) == _native.PL_ERR_ARG
    assert _refused(one, good, cols=1 << 30, ld=1 << 30) == _native.PL_ERR_ARG  # 2^34 positions
    assert _refused(one, good, table=None) == _native.PL_ERR_ARG
    assert _refused(one, good, key=p + 2) == _native.PL_ERR_ALIGN
    assert _refused(one, good, keys=_i64(64, 32, 17)) == _native.PL_ERR_ALIGN
    assert _refused(one, good, rot=17) == _native.PL_ERR_ARG
    assert _refused(one, good, rot=18) == _native.PL_ERR_ARG
    assert _refused(one, good, past=None) == _native.PL_ERR_ARG
    assert _refused(one, good, cos=None) == _native.PL_ERR_ARG
    assert _refused(one, good, out=p) == _native.PL_ERR_ARG  # over q
    assert _refused(one, good, k_out=3 * p) == _native.PL_ERR_ARG  # over v
    assert one(*{**good, "rows": 0}.values()) == 0 and one(*{**good, "m": 0}.values()) == 0  # nothing to do


def test_attention_refusals_of_the_library():
    lib = _native.load()
    s, p = _i64(64, 32, 16), 4096
    need = lib.pl_paged_attention_workspace_bytes(64)
    assert need > 0 and lib.pl_paged_attention_workspace_bytes(0) == lib.pl_paged_attention_workspace_bytes(257) == 0
    good = dict(dtype=1, cache=1, q=p, qs=_i64(64, 16), key=p, keys=s, value=p, values=s, pages=4, page=16, table=p, ld=2,
                cols=2, lens=p, rows=1, heads=2, kv=2, dim=16, scale=1.0, window=0, ksc=None, vsc=None, out=1 << 20, ws=p,
                wsb=need, counters=p, ints=_native.PL_ATTENTION_COUNTER_INTS, stream=None)
    one = lib.pl_paged_attention
    assert _refused(one, good, window=-1) == _native.PL_ERR_ARG
    assert _refused(one, good, lens=None) == _native.PL_ERR_ARG
    assert _refused(one, good, out=p) == _native.PL_ERR_ARG  # over q
    assert _refused(one, good, wsb=need // 2) == _native.PL_ERR_ARG
    assert _refused(one, good, counters=None) == _native.PL_ERR_ARG
    assert _refused(one, good, ints=16) == _native.PL_ERR_ARG
    assert _refused(one, good, keys=_i64(64, 32, 1 << 30)) == _native.PL_ERR_LIMIT
    assert _refused(one, good, rows=1 << 30, cols=1 << 26, ld=1 << 26, out=1 << 60) == _native.PL_ERR_LIMIT
    assert _refused(one, good, value=p + 8) == _native.PL_ERR_ALIGN
    assert one(*{**good, "rows": 0}.values()) == 0


def test_logits_refusals_of_the_library():
    lib = _native.load()
    p = 4096
    good = dict(dtype=1, out_dtype=0, logits=p, ld=64, out=1 << 20, ld_out=64, rows=2, vocab=64, tokens=p, token_bytes=8,
                ld_tokens=4, history=4, lens=p, prompt=None, rep=None, pres=None, freq=None, ids=p, values=p, ld_bias=2,
                n_bias=2, allowed=None, ld_allowed=0, stream=None)
    one = lib.pl_adjust_logits
    assert _refused(one, good, out_dtype=2) == _native.PL_ERR_ARG
    assert _refused(one, good, vocab=-1) == _native.PL_ERR_ARG
    assert _refused(one, good, history=1 << 20) == _native.PL_ERR_LIMIT
    assert _refused(one, good, n_bias=2048) == _native.PL_ERR_LIMIT
    assert _refused(one, good, token_bytes=2) == _native.PL_ERR_ARG
    assert _refused(one, good, lens=None) == _native.PL_ERR_ARG
    assert _refused(one, good, values=None) == _native.PL_ERR_ARG
    assert _refused(one, good, out=p) == _native.PL_ERR_ARG  # fp32 over bf16
    assert _refused(one, good, out=p + 2, out_dtype=1) == _native.PL_ERR_ARG
    assert _refused(one, good, out=p, out_dtype=1, ld_out=65) == _native.PL_ERR_ARG
    assert one(*{**good, "rows": 0}.values()) == 0


def test_plain_attention_is_a_softmax_over_the_rows_tokens():
    """The oracle against torch's own attention on a row gathered by hand, and its empty rows."""
    gen = torch.Generator().manual_seed(1)
    key, value = (torch.randn(5, 2, 16, 8, generator=gen) for _ in range(2))
    table = torch.tensor([[3, 1], [0, -1], [4, 2]], dtype=torch.int32)
    lens = torch.tensor([20, 0, 32])
    q = torch.randn(3, 4, 8, generator=gen)
    out, _, _ = plain.paged_attention(q, key, value, table, lens)
    assert not out[1].any()
    for b in (0, 2):
        k, v = (torch.cat([c[table[b, 0]], c[table[b, 1]]], 1)[:, : lens[b]].repeat_interleave(2, 0) for c in (key, value))
        want = torch.nn.functional.scaled_dot_product_attention(q[b][:, None].double(), k.double(), v.double())[:, 0]
        torch.testing.assert_close(out[b], want, rtol=1e-12, atol=1e-12)


def test_plain_rotation_is_a_complex_product():
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(3, 8, generator=gen, dtype=torch.float64)
    angle = torch.randn(3, generator=gen, dtype=torch.float64)
    y = plain.rotate(x, angle.cos(), angle.sin(), True)
    z = torch.view_as_complex(x[:, :6].reshape(3, 3, 2).contiguous()) * torch.exp(1j * angle)
    torch.testing.assert_close(y[:, :6], torch.view_as_real(z).reshape(3, 6))
    assert torch.equal(y[:, 6:], x[:, 6:])
    half = plain.rotate(x[:, [0, 2, 4, 1, 3, 5, 6, 7]], angle.cos(), angle.sin(), False)
    torch.testing.assert_close(half[:, [0, 3, 1, 4, 2, 5, 6, 7]], y)


def test_logits_rows_of_the_output_never_overlap():
    lib = _native.load()
    p = 4096
    args = dict(dtype=1, out_dtype=0, logits=p, ld=64, out=1 << 20, ld_out=63, rows=2, vocab=64, tokens=None, token_bytes=0,
                ld_tokens=0, history=0, lens=None, prompt=None, rep=None, pres=None, freq=None, ids=None, values=None,
                ld_bias=0, n_bias=0, allowed=None, ld_allowed=0, stream=None)
    assert _refused(lib.pl_adjust_logits, args) == _native.PL_ERR_ARG
    assert _refused(lib.pl_adjust_logits, args, ld_out=0) == _native.PL_ERR_ARG  # one row expanded to all
    assert _refused(lib.pl_adjust_logits, args, ld=0, out=p, out_dtype=1, ld_out=0) == _native.PL_ERR_ARG  # in place


def test_append_never_writes_a_place_twice():
    lib = _native.load()
    s, p = _i64(64, 32, 16), 4096
    dense, other = _i64(512, 256, 16), _i64(512, 16, 32)  # pages by head and by slot
    args = dict(dtype=1, cache=1, q=p, qs=s, k=2 * p, ks=s, v=3 * p, vs=s, out=1 << 20, k_out=None, key=4 * p, keys=dense,
                value=64 * p, values=other, pages=4, page=16, table=p, ld=2, cols=2, past=p, seq=None, rows=1, m=2, heads=2,
                kv=2, dim=16, cos=p, sin=p, positions=8, rot=16, inter=0, ksc=None, vsc=None, stream=None)
    one = lib.pl_rope_append
    for bad in (_i64(0, 256, 16), _i64(512, 0, 16), _i64(512, 256, 0), _i64(504, 256, 16), _i64(512, 16, 16), _i64(512, 256, 8)):
        assert _refused(one, args, keys=bad) == _native.PL_ERR_ARG
        assert b"share their places" in lib.pl_last_error()
        assert _refused(one, args, values=bad) == _native.PL_ERR_ARG
        assert b"share their places" in lib.pl_last_error()
    assert _refused(one, args, value=4 * p) == _native.PL_ERR_ARG
    assert b"share their places" in lib.pl_last_error()


def test_a_shared_page_table_is_no_reason_to_refuse():
    """table_ld 0 passes the table's check and meets the next one; a row that runs into the next is refused as before."""
    lib = _native.load()
    s, p = _i64(64, 32, 16), 4096
    args = dict(dtype=1, cache=1, q=p, qs=_i64(64, 16), key=p, keys=s, value=p, values=s, pages=4, page=16, table=p, ld=0,
                cols=2, lens=None, rows=2, heads=2, kv=2, dim=16, scale=1.0, window=0, ksc=None, vsc=None, out=1 << 20,
                ws=p, wsb=1 << 30, counters=p, ints=_native.PL_ATTENTION_COUNTER_INTS, stream=None)
    _refused(lib.pl_paged_attention, args)
    assert b"null pointer" in lib.pl_last_error()
    for ld in (1, -2):
        _refused(lib.pl_paged_attention, args, ld=ld)
        assert b"page table" in lib.pl_last_error()


def test_attention_counts_stay_within_32_bits():
    """Table columns whose last token's tile, and batches whose last run, would pass them."""
    lib = _native.load()
    s, p = _i64(64, 32, 16), 4096
    args = dict(dtype=1, cache=1, q=p, qs=_i64(64, 16), key=p, keys=s, value=p, values=s, pages=4, page=16, table=p,
                ld=1 << 27, cols=2, lens=p, rows=1, heads=2, kv=2, dim=16, scale=1.0, window=0, ksc=None, vsc=None, out=1 << 60,
                ws=p, wsb=1 << 30, counters=p, ints=_native.PL_ATTENTION_COUNTER_INTS, stream=None)
    one = lib.pl_paged_attention
    assert _refused(one, args, cols=(1 << 27) - 1) == _native.PL_ERR_LIMIT
    assert _refused(one, args, cols=(1 << 27) - 1, window=5) == _native.PL_ERR_LIMIT
    assert _refused(one, args, rows=(1 << 30) - 1) == _native.PL_ERR_LIMIT


def test_logits_places_stay_within_32_bits():
    lib = _native.load()
    p = 4096
    args = dict(dtype=1, out_dtype=0, logits=p, ld=1 << 31, out=1 << 60, ld_out=1 << 31, rows=1, vocab=(1 << 31) - 1, tokens=None,
                token_bytes=0, ld_tokens=0, history=0, lens=None, prompt=None, rep=None, pres=None, freq=None, ids=None,
                values=None, ld_bias=0, n_bias=0, allowed=None, ld_allowed=0, stream=None)
    assert _refused(lib.pl_adjust_logits, args) == _native.PL_ERR_LIMIT
    assert _refused(lib.pl_adjust_logits, args, vocab=(1 << 31) - (1 << 14)) == _native.PL_ERR_LIMIT

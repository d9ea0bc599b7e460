"""A step over drafted tokens against 64-bit plain forms: head norms and depths, tree attention, verification, moves."""

from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from oracle import drafts as plain
from polylora_amd.drafts import tree_tables, verify_tokens
from polylora_amd.paged import keep_tokens, paged_attention, rope_append, rope_table, tree_attention

from .test_gpu_paged import DTYPES, FP8, STEP, UNIT, attention_tolerance, back, pool, put

pytestmark = pytest.mark.gpu


def on(gpu, **tensors):
    return {name: None if t is None else t.to(gpu) for name, t in tensors.items()}


def random_parents(gen, rows, m, roots=False):
    return torch.tensor([[-1 if t == 0 else int(torch.randint(-1 if roots else 0, t, (), generator=gen))
                          for t in range(m)] for _ in range(rows)], dtype=torch.int32).view(rows, m)


def seen_of(visible, m):
    """Boolean [rows, M, M] of packed masks."""
    return ((visible[..., None] >> torch.arange(32, dtype=torch.int32) & 1) > 0).flatten(-2)[..., :m]


# ----------------------------------------------------------------------------- append


def check_norm_append(got, want, unit_of, sizes):
    """One rounding to the type, and before it 32 units of fp32 on the sum of magnitudes: half of 23 for a sum of at most
    256 squares by lanes (16 to a lane, six steps, the squares themselves), 6 for mean, root, reciprocal and two
    products, 3 for the turn."""
    got = back(got).double()
    assert torch.equal(got.isnan(), want.isnan())
    got, want, sizes = got.nan_to_num(0.0), want.nan_to_num(0.0), sizes.nan_to_num(0.0)
    tol = UNIT[unit_of] * want.abs() + STEP[unit_of] / 2 + 2.0**-19 * sizes
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() - tol).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,m,heads,kv_heads,dim,page,rot,interleaved,fp8,tree,wide,norms", [
    (1, 1, 4, 1, 16, 16, 16, False, False, False, False, "qk"),
    (3, 6, 32, 8, 128, 16, 128, False, False, True, False, "qk"),
    (5, 7, 6, 2, 80, 32, 80, False, False, True, True, "qk"),
    (4, 37, 4, 4, 96, 16, 48, True, False, False, False, "qk"),
    (2, 5, 3, 1, 256, 64, 10, False, False, True, True, "q"),
    (2, 9, 5, 5, 48, 16, 30, True, False, True, False, "k"),
    (3, 4, 2, 2, 64, 16, 0, False, False, False, False, "qk"),
    (3, 11, 8, 2, 128, 16, 128, False, True, True, False, "qk"),
    (2, 18, 4, 2, 80, 32, 40, False, True, False, True, "qk"),
    (2, 3, 4, 2, 256, 16, 254, True, True, True, False, "qk"),
    (2, 3, 4, 2, 256, 16, 2, False, False, True, False, ""),
    (300, 8, 4, 2, 64, 16, 64, False, False, True, False, "qk"),
])
def test_norm_append_matches_the_plain_form(gpu, dtype, rows, m, heads, kv_heads, dim, page, rot, interleaved, fp8, tree,
                                            wide, norms):
    if fp8 and dtype == torch.float32:
        pytest.skip("an 8-bit cache serves 16-bit models")
    if rows > 100 and dtype != torch.bfloat16:
        pytest.skip("one type at that size")
    gen = torch.Generator().manual_seed(rows * 100 + m + dim)
    past = torch.randint(0, 3 * page, (rows,), generator=gen)
    seq = torch.randint(0, m + 3, (rows,), generator=gen)  # rows of no new token, and lengths above m
    seq[0] = m
    key, value, table, ks, vs = pool(gen, rows, [int(p) + m for p in past], kv_heads, dim, page, dtype, fp8)
    if rows > 2:
        table[-1, int(past[-1]) // page] = -1  # a page that the table does not hold
    qkv = (torch.randn(rows, m, heads + 2 * kv_heads, dim, generator=gen) * 3).to(dtype)
    q, k, v = qkv.split((heads, kv_heads, kv_heads), 2)
    cos, sin = rope_table(int(past.max()) + m, rot, 10000.0)
    weights = [(torch.randn(dim, generator=gen) * 0.3 + 1).to(torch.float32 if wide else dtype) if n in norms else None
               for n in "qk"]
    depths = tree_tables(random_parents(gen, rows, m))[0] if tree else None
    eps = 1e-5
    want = plain.norm_rope_append(q, k, v, key, value, table, past, cos, sin, seq, interleaved, ks, vs, *weights, eps,
                                  depths)
    qkv = qkv.to(gpu)
    gq, gk, gv = qkv.split((heads, kv_heads, kv_heads), 2)
    gkey, gvalue = put(key, gpu), put(value, gpu)
    k_out = torch.full((rows, m, kv_heads, dim), 7.0, dtype=dtype, device=gpu)
    up = on(gpu, k_scale=ks, v_scale=vs, q_norm=weights[0], k_norm=weights[1], depths=depths)
    q_out = rope_append(gq, gk, gv, gkey, gvalue, table.to(gpu), past.int().to(gpu), cos.to(gpu), sin.to(gpu),
                        seq_lens=seq.int().to(gpu), interleaved=interleaved, k_out=k_out, eps=eps, **up)
    check_norm_append(q_out, want[0], dtype, want[4])
    check_norm_append(k_out, want[1], dtype, want[5])
    # the keys' sizes, in their places; 0 where nothing was written, which has to be the same bits
    live = torch.zeros(key.shape, dtype=torch.float64)
    for b in range(rows):
        for t in range(min(m, int(seq[b]))):
            at = plain.place(table, b, int(past[b]) + t, key.shape[0], page)
            if at is not None:
                live[at[0], :, at[1]] = want[5][b, t] if ks is None else want[5][b, t] / ks.double()[:, None]
    cache_type = FP8 if fp8 else dtype
    check_norm_append(gkey, want[2], cache_type, live)
    check_norm_append(gvalue, want[3], cache_type, live * 0)


def test_norms_without_weights_of_one_turn_nothing_else(gpu):
    """Depths 0 .. M - 1 and no norms: the append of tokens in a line, bit for bit."""
    gen = torch.Generator().manual_seed(2)
    rows, m, heads, kv, dim = 3, 6, 8, 2, 64
    key, value, table, _, _ = pool(gen, rows, [20, 30, 9], kv, dim, 16, torch.bfloat16)
    q, k, v = (torch.randn(rows, m, n, dim, generator=gen).bfloat16().to(gpu) for n in (heads, kv, kv))
    past = torch.tensor([14, 24, 3], dtype=torch.int32, device=gpu)
    cos, sin = rope_table(40, dim, device=gpu)
    out = []
    for depths in (None, torch.arange(m, dtype=torch.int32, device=gpu)):
        caches = key.to(gpu), value.to(gpu)
        out.append((rope_append(q, k, v, *caches, table.to(gpu), past, cos, sin, depths=depths), *caches))
    for a, b in zip(*out):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_norm_append_odd_strides_and_weights(gpu):
    """Heads that start at any element, and weights that do."""
    gen = torch.Generator().manual_seed(8)
    rows, m, heads, kv, dim = 2, 3, 4, 2, 64
    past = torch.tensor([3, 17])
    for shift in (1, 2, 4):
        key, value, table, _, _ = pool(gen, rows, [int(p) + m for p in past], kv, dim, 16, torch.bfloat16)
        store = torch.randn(rows, m, heads + 2 * kv, dim + shift, generator=gen).bfloat16()
        weights = torch.randn(2, dim + shift, generator=gen).bfloat16()
        cos, sin = rope_table(32, dim)
        parts = store[..., shift:].split((heads, kv, kv), 2)
        want = plain.norm_rope_append(*parts, key, value, table, past, cos, sin, q_norm=weights[0, shift:],
                                      k_norm=weights[1, shift:])
        gkey, gvalue, w = key.to(gpu), value.to(gpu), weights.to(gpu)
        q_out = rope_append(*store.to(gpu)[..., shift:].split((heads, kv, kv), 2), gkey, gvalue, table.to(gpu),
                            past.int().to(gpu), cos.to(gpu), sin.to(gpu), q_norm=w[0, shift:], k_norm=w[1, shift:])
        check_norm_append(q_out, want[0], torch.bfloat16, want[4])


def test_append_refuses(gpu):
    x = torch.zeros(1, 2, 2, 32, device=gpu, dtype=torch.bfloat16)
    key, value = (torch.zeros(2, 2, 16, 32, device=gpu, dtype=torch.bfloat16) for _ in range(2))
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
    cos, sin = rope_table(16, 32, device=gpu)
    w = torch.ones(32, device=gpu)

    def call(**more):
        return rope_append(x, x, x, key, value, table, lens, cos, sin, **more)

    call(q_norm=w, k_norm=w)
    with pytest.raises(TypeError):
        call(q_norm=w.half())
    with pytest.raises(TypeError):
        call(q_norm=w, k_norm=w.bfloat16())
    with pytest.raises(ValueError):
        call(q_norm=w[:16])
    with pytest.raises(ValueError):
        call(k_norm=torch.ones(64, device=gpu)[::2])
    with pytest.raises(ValueError):
        call(q_norm=w.cpu())
    with pytest.raises(RuntimeError, match="eps"):
        call(q_norm=w, eps=0.0)
    with pytest.raises(TypeError):
        call(depths=torch.zeros(1, 2, device=gpu))
    with pytest.raises(ValueError):
        call(depths=torch.zeros(1, 3, dtype=torch.int32, device=gpu))
    with pytest.raises(RuntimeError, match="gradient"):
        call(q_norm=w.clone().requires_grad_())


# ----------------------------------------------------------------------------- tree attention


def check_tree(gpu, dtype, past, seq, m, heads, kv_heads, dim, page, tree=True, fp8=False, order="head", window=None,
               scale=None, seed=0, holes=False, shared=False, extra=0, q_gain=1.5, columns=0):
    gen = torch.Generator().manual_seed(seed + dim + heads + m)
    rows = len(past)
    new = [min(m, n) for n in (seq or [m] * rows)]
    held = [min(max(0, p) + max(0, n), (columns or 10**9) * page) for p, n in zip(past, new)]
    key, value, table, ks, vs = pool(gen, rows, held, kv_heads, dim, page, dtype, fp8)
    if holes:
        table[::2, 0] = -1
        table[1::2, 0] = key.shape[0]
    q = (torch.randn(rows, m + 1, heads + 1, dim, generator=gen) * q_gain).to(dtype)[:, 1:, 1:]
    visible = depths = seen = None
    if tree:
        parents = random_parents(gen, 1 if shared else rows, m, roots=extra == 1)
        depths, visible = tree_tables(parents)
        if extra == 2:  # any bits at all, rows of none among them
            visible = torch.randint(-2**31, 2**31, visible.shape, generator=gen).int()
            visible[:, ::5] = 0
        seen = seen_of(visible, m).expand(rows, m, m)
        depths = depths.expand(rows, m)
        if shared:
            visible = visible[0]
    lens, n = torch.tensor(past, dtype=torch.int32), None if seq is None else torch.tensor(seq, dtype=torch.int32)
    want, spread, reach = plain.tree_attention(q, key, value, table, lens, n, seen, depths, scale, window, ks, vs)
    up = on(gpu, k_scale=ks, v_scale=vs, seq_lens=n, visible=visible, depths=depths)
    args = (q.to(gpu), put(key, gpu, order), put(value, gpu, order), table.to(gpu), lens.to(gpu))
    got = tree_attention(*args, scale=scale, window=window, **up)
    tol = attention_tolerance(want, spread, reach, dtype, dim, max(1, *(p + m for p in past)))
    err = (got.cpu().double() - want).abs()
    assert not got.isnan().any()
    assert bool((err <= tol).all()), (float((err / tol).max()), float(err.max()))
    again = torch.full_like(got, 7.0)
    assert tree_attention(*args, scale=scale, window=window, out=again, **up) is again
    assert torch.equal(again, got)  # the same bits each time
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 1, 16, 16), (8, 2, 64, 16), (12, 4, 80, 32), (9, 3, 96, 16),
                                                     (8, 2, 128, 16), (5, 5, 112, 64), (4, 2, 256, 16), (20, 1, 144, 16),
                                                     (40, 2, 64, 128)])
@pytest.mark.parametrize("tree", [False, True])
def test_tree_attention_matches_the_plain_form(gpu, dtype, heads, kv_heads, dim, page, tree):
    check_tree(gpu, dtype, [0, 1, 15, 33, 140], [7, 5, 0, 9, 7], 7, heads, kv_heads, dim, page, tree)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 32, 33, 64, 65, 100])
@pytest.mark.parametrize("group", [1, 4, 5])
def test_tree_attention_of_any_number_of_tokens(gpu, m, group):
    check_tree(gpu, torch.bfloat16, [0, 50, 131], None, m, 2 * group, 2, 64, 16, tree=True)
    check_tree(gpu, torch.float16, [17, 0, 300], [m, m // 2, max(1, m - 1)], m, 2 * group, 2, 128, 32, tree=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [32, 64, 80, 128, 256])
@pytest.mark.parametrize("m,group", [(3, 4), (9, 4), (40, 2), (5, 20)])
def test_tree_attention_over_8_bits(gpu, dtype, dim, m, group):
    check_tree(gpu, dtype, [0, 77, 500], [m, m, m // 2], m, 2 * group, 2, dim, 16, fp8=True, q_gain=0.2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extra", [1, 2])
def test_tree_attention_of_several_roots_and_of_any_bits(gpu, dtype, extra):
    check_tree(gpu, dtype, [0, 0, 40], [34, 20, 34], 34, 4, 2, 64, 16, extra=extra)
    check_tree(gpu, dtype, [0, 9], [11, 1], 11, 8, 2, 128, 16, extra=extra, shared=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 16, 33, 100, 1000])
@pytest.mark.parametrize("tree", [False, True])
def test_tree_attention_of_a_window(gpu, dtype, window, tree):
    m = min(window, 12) if tree else 12
    check_tree(gpu, dtype, [0, 5, 64, 300, 411], [m, m, 1, m, m // 2], m, 8, 2, 64, 16, tree, window=window)


def test_tree_attention_layouts_holes_and_scales(gpu):
    for order in ("head", "slot"):
        check_tree(gpu, torch.bfloat16, [200, 63, 0, 16], None, 6, 8, 2, 128, 64, order=order, scale=0.3)
    check_tree(gpu, torch.bfloat16, [200, 63, 0, 16], None, 6, 8, 2, 128, 16, holes=True)
    check_tree(gpu, torch.float32, [200, 63, 0, 16], None, 20, 8, 2, 64, 16, holes=True, tree=False)
    check_tree(gpu, torch.float16, [200, 63, 0, -3], [6, 0, -1, 4], 6, 8, 2, 128, 16, tree=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,m,heads,kv_heads,dim,lens", [
    (1, 5, 32, 8, 128, 5000), (1, 64, 32, 8, 128, 1700), (3, 16, 8, 1, 64, 3000), (70, 2, 8, 2, 64, 400),
    (300, 3, 4, 2, 64, 90), (2, 33, 28, 4, 128, 900), (1, 1, 8, 1, 128, 9000), (9, 64, 32, 1, 128, 300),
])
def test_tree_attention_of_long_and_of_many_rows(gpu, dtype, rows, m, heads, kv_heads, dim, lens):
    gen = torch.Generator().manual_seed(rows + m)
    past = torch.randint(0, lens + 1, (rows,), generator=gen).tolist()
    past[-1] = lens
    check_tree(gpu, dtype, past, None, m, heads, kv_heads, dim, 16, tree=m > 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,group,tree,window", [(300, 8, False, None), (300, 8, False, 40), (130, 20, True, None),
                                                 (130, 20, True, 150), (600, 2, False, 7)])
def test_tree_attention_of_more_columns_than_one_launch_takes(gpu, dtype, m, group, tree, window):
    check_tree(gpu, dtype, [0, 37, 300], [m, m // 3, m - 1], m, group, 1, 32, 16, tree, window=window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [48, 64, 80, 128, 144, 256])
@pytest.mark.parametrize("m,group", [(16, 6), (33, 1), (8, 4), (97, 1), (16, 8), (15, 9), (52, 5)])
def test_tree_attention_where_many_columns_begin(gpu, dtype, dim, m, group):
    check_tree(gpu, dtype, [0, 1, 77, 400], [m, 0, m // 2, m], m, 2 * group, 2, dim, 16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [12, 33, 100, 1000])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("heads", [12, 40])
def test_tree_attention_of_a_window_and_many_columns(gpu, dtype, window, tree, heads):
    check_tree(gpu, dtype, [0, 5, 64, 300, 411], [12, 12, 1, 12, 6], 12, heads, 2, 64, 16, tree, window=window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [12, 40])
def test_tree_attention_of_many_columns_where_the_table_ends_before_the_row(gpu, dtype, heads):
    check_tree(gpu, dtype, [60, 64, 200, 0], None, 12, heads, 2, 64, 16, columns=4)
    check_tree(gpu, dtype, [0, 0, 40], [12, 0, 12], 12, heads, 2, 128, 16, extra=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [5, 30])
def test_tree_attention_where_the_table_ends_before_the_row(gpu, dtype, m):
    """Tokens behind the table's last column are left out, of the drafts and of what lies before them."""
    check_tree(gpu, dtype, [60, 64, 200, 0], None, m, 8, 2, 64, 16, columns=4)
    check_tree(gpu, dtype, [60, 64, 200, 0], None, m, 8, 2, 64, 16, tree=False, columns=4, window=33)


def test_tree_attention_of_lengths_near_32_bits(gpu):
    q = torch.ones(2, 3, 4, 64, device=gpu, dtype=torch.bfloat16)
    key = torch.ones(2, 2, 16, 64, device=gpu, dtype=torch.bfloat16)
    table = torch.tensor([[0, 1]] * 2, dtype=torch.int32, device=gpu)
    past = torch.tensor([2**31 - 1, 2**31 - 3], dtype=torch.int32, device=gpu)
    for heads in (4, 2):
        for window in (None, 5, 2**31 - 1):
            got = tree_attention(q[:, :, :heads], key, key, table, past, window=window)
            assert torch.equal(got, torch.zeros_like(got) if window == 5 else torch.ones_like(got))


def test_one_drafted_token_is_the_single_tokens_attention(gpu):
    gen = torch.Generator().manual_seed(3)
    lens = [40, 300, 1]
    key, value, table, _, _ = pool(gen, 3, lens, 2, 64, 16, torch.float32)
    q = torch.randn(3, 1, 8, 64, generator=gen).to(gpu)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    args = key.to(gpu), value.to(gpu), table.to(gpu)
    a, b = tree_attention(q, *args, n - 1)[:, 0], paged_attention(q[:, 0], *args, n)
    assert float((a - b).abs().max()) < 1e-5


def test_tree_attention_takes_empty_batches(gpu):
    key = torch.zeros(2, 1, 16, 16, device=gpu)
    for rows, m in ((0, 3), (2, 0)):
        q = torch.zeros(rows, m, 1, 16, device=gpu)
        table, past = torch.zeros(rows, 1, dtype=torch.int32, device=gpu), torch.zeros(rows, dtype=torch.int32, device=gpu)
        assert tree_attention(q, key, key, table, past).shape == (rows, m, 1, 16)
    q, past = torch.ones(2, 3, 1, 16, device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    for pages, columns in ((0, 2), (2, 0)):
        key, table = torch.zeros(pages, 1, 16, 16, device=gpu), torch.zeros(2, columns, dtype=torch.int32, device=gpu)
        assert not tree_attention(q, key, key, table, past).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [4, 40])
def test_tree_attention_reads_nothing_that_no_token_sees(gpu, dtype, heads):
    """NaN in places beyond the row's tokens, before every window and at drafts that a token does not see."""
    gen = torch.Generator().manual_seed(6)
    page, m, past = 16, 6, 70
    key, value, table, _, _ = pool(gen, 1, [past + m], 2, 64, page, dtype)
    q = torch.randn(1, m, heads, 64, generator=gen).to(dtype)
    parents = torch.tensor([[-1, 0, 0, 1, 2, 4]], dtype=torch.int32)
    depths, visible = tree_tables(parents)
    lens = torch.tensor([past], dtype=torch.int32)
    for t in range(m):
        k2, v2 = key.clone(), value.clone()
        hidden = [past + j for j in range(m) if not int(visible[0, t, 0]) >> j & 1] + list(range(past - 20))
        for p in hidden:
            at = plain.place(table, 0, p, key.shape[0], page)
            k2[at[0], :, at[1]] = v2[at[0], :, at[1]] = float("nan")
        args = on(gpu, visible=visible, depths=depths)
        clean = tree_attention(q.to(gpu), key.to(gpu), value.to(gpu), table.to(gpu), lens.to(gpu), window=20, **args)
        got = tree_attention(q.to(gpu), k2.to(gpu), v2.to(gpu), table.to(gpu), lens.to(gpu), window=20, **args)
        assert torch.equal(got[:, t], clean[:, t]), t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [2, 24])
def test_tree_attention_infinities_and_nan_stay_where_they_are(gpu, dtype, heads):
    gen = torch.Generator().manual_seed(7)
    key, value, table, _, _ = pool(gen, 1, [90], 1, 64, 16, dtype)
    q = torch.randn(1, 5, heads, 64, generator=gen).to(dtype)
    q[0, 2, 1, 5] = float("nan")
    at = plain.place(table, 0, 30, key.shape[0], 16)
    value[at[0], :, at[1], 7] = float("inf")
    lens = torch.tensor([85], dtype=torch.int32)
    got = tree_attention(q.to(gpu), key.to(gpu), value.to(gpu), table.to(gpu), lens.to(gpu)).cpu()
    nan = torch.zeros(5, heads, 64, dtype=torch.bool)
    nan[2, 1] = True
    assert torch.equal(got[0].isnan(), nan)
    assert bool((got[0, :, :, 7] == float("inf")).logical_or(nan[:, :, 7]).all())
    assert int(got.isinf().sum()) == 5 * heads - 1


def test_tree_attention_refuses(gpu):
    q = torch.zeros(2, 4, 4, 64, device=gpu, dtype=torch.bfloat16)
    key, value = (torch.zeros(4, 2, 16, 64, device=gpu, dtype=torch.bfloat16) for _ in range(2))
    table = torch.zeros(2, 2, dtype=torch.int32, device=gpu)
    past = torch.zeros(2, dtype=torch.int32, device=gpu)
    masks, depths = torch.ones(2, 4, 1, dtype=torch.int32, device=gpu), torch.zeros(2, 4, dtype=torch.int32, device=gpu)

    def call(q=q, key=key, value=value, table=table, past=past, **more):
        return tree_attention(q, key, value, table, past, **more)

    call(visible=masks, depths=depths, window=4)
    for bad in (dict(q=q[0]), dict(key=key[:, :1]), dict(table=table[:1]), dict(past=past[:1]), dict(window=0),
                dict(visible=masks[:, :3]), dict(visible=masks[:1]), dict(visible=masks[..., :0]),
                dict(visible=masks, window=4), dict(visible=masks, depths=depths, window=3),
                dict(visible=masks, depths=depths[:, :3]), dict(out=q[:1]), dict(out=q.transpose(1, 2)),
                dict(q=q[..., ::2]), dict(seq_lens=past[:1]), dict(past=past.cpu()),
                dict(k_scale=torch.ones(2, device=gpu), v_scale=torch.ones(2, device=gpu))):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(past=past.long()), dict(visible=masks.long()), dict(visible=masks, depths=depths.float()),
                dict(key=key.half(), value=value.half()), dict(q=q.double())):
        with pytest.raises(TypeError):
            call(**bad)
    with pytest.raises(RuntimeError, match="overlaps"):
        call(out=q)
    with pytest.raises(RuntimeError, match="gradient"):
        call(q=q.clone().requires_grad_())


def test_tree_attention_in_graphs_and_on_streams(gpu):
    """Replays with other lengths, two graphs and eager calls on two streams beside each other."""
    gen = torch.Generator().manual_seed(9)
    rows, m, page = 3, 9, 16
    key, value, table, _, _ = pool(gen, rows, [700, 500, 900], 2, 64, page, torch.bfloat16)
    key, value = key.nan_to_num(0.0).to(gpu), value.nan_to_num(0.0).to(gpu)
    table = table.to(gpu)
    visible = tree_tables(random_parents(gen, rows, m))[1].to(gpu)
    qs = [torch.randn(rows, m, 8, 64, generator=gen).bfloat16().to(gpu) for _ in range(2)]
    past = torch.zeros(rows, dtype=torch.int32, device=gpu)
    lengths = [[0, 3, 50], [690, 400, 891], [100, 491, 7]]
    want = {}
    for i, lens in enumerate(lengths):
        past.copy_(torch.tensor(lens))
        for j, q in enumerate(qs):
            want[i, j] = tree_attention(q, key, value, table, past, visible=visible)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for q in qs:
        with torch.cuda.stream(side):
            tree_attention(q, key, value, table, past, visible=visible)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(tree_attention(q, key, value, table, past, visible=visible))
        graphs.append(graph)
    others = [torch.cuda.Stream() for _ in range(2)]
    for i, lens in enumerate(lengths * 2):
        past.copy_(torch.tensor(lens))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, others):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [tree_attention(q, key, value, table, past, visible=visible) for q in qs]
        torch.cuda.synchronize()
        for j in range(2):
            assert torch.equal(outs[j], want[i % 3, j]) and torch.equal(eager[j], want[i % 3, j])


def test_tree_attention_from_threads(gpu):
    gen = torch.Generator().manual_seed(10)
    key, value, table, _, _ = pool(gen, 2, [500, 800], 2, 64, 16, torch.bfloat16)
    key, value, table = key.to(gpu), value.to(gpu), table.to(gpu)
    past = torch.tensor([490, 790], dtype=torch.int32, device=gpu)
    qs = [torch.randn(2, 10, 8, 64, generator=gen).bfloat16().to(gpu) for _ in range(4)]
    want = [tree_attention(q, key, value, table, past) for q in qs]
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [tree_attention(qs[i], key, value, table, past) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
        return all(torch.equal(g, want[i]) for g in got)

    with ThreadPoolExecutor(4) as pool_of_threads:
        assert all(pool_of_threads.map(work, range(4)))


# ----------------------------------------------------------------------------- verification


def check_verify(gpu, logits, tokens, uniforms, **more):
    want = plain.verify_tokens(logits, tokens, uniforms, **more)
    got = verify_tokens(logits.to(gpu), tokens.to(gpu), uniforms.to(gpu), **on(gpu, **more))
    assert [t.dtype for t in got] == [torch.int32, torch.int32, torch.int64]
    for name, a, b in zip(("path", "counts", "next"), got, want):
        assert torch.equal(a.cpu(), b), (name, a.tolist(), b.tolist())
    return got


def drafted(gen, rows, m, vocab, dtype, kind, peak=2.5):
    """Arguments of a step: logits, tokens that often agree with them, uniforms, and what `kind` adds."""
    logits = (torch.randn(rows, m, vocab, generator=gen) * peak).to(dtype)
    uniforms = torch.rand(rows, m, generator=gen)
    more = {"temperature": torch.tensor([(0.0, 0.7, 1.0, 1.3)[b % 4] for b in range(rows)]),
            "seq_lens": torch.randint(0, m + 2, (rows,), generator=gen).int()}
    more["seq_lens"][0] = m
    if kind == "line":
        q = torch.softmax(logits[:, : m - 1].float() + torch.randn(rows, max(0, m - 1), vocab, generator=gen), -1)
        drawn = torch.multinomial(q.flatten(0, 1), 1, generator=gen) if m > 1 else q.new_zeros(0)
        tokens = torch.cat((torch.zeros(rows, 1), drawn.view(rows, m - 1)), 1).long()
        more["draft_probs"] = q
    else:
        more["parents"] = random_parents(gen, rows, m) if kind == "tree" else None
        best = logits.float().topk(min(3, vocab), -1).indices
        tokens = torch.zeros(rows, m, dtype=torch.int64)
        for b in range(rows):
            for t in range(1, m):
                parent = int(more["parents"][b, t]) if kind == "tree" else t - 1
                tokens[b, t] = best[b, parent, int(torch.randint(0, best.shape[-1], (), generator=gen))]
    return logits, tokens, uniforms, more


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["line", "tree", "sure"])
@pytest.mark.parametrize("rows,m,vocab", [(1, 1, 1), (2, 3, 2), (9, 6, 7), (40, 5, 64), (7, 9, 1000), (3, 4, 4096),
                                          (3, 5, 4097), (2, 33, 515), (4, 6, 12289), (1, 4, 32003)])
def test_verification_matches_the_plain_form(gpu, dtype, kind, rows, m, vocab):
    gen = torch.Generator().manual_seed(rows + m + vocab)
    logits, tokens, uniforms, more = drafted(gen, rows, m, vocab, dtype, kind)
    check_verify(gpu, logits, tokens, uniforms, **more)
    check_verify(gpu, logits, tokens.int(), uniforms, **{**more, "seq_lens": None, "temperature": None})


@pytest.mark.parametrize("kind", ["line", "tree"])
def test_verification_of_a_large_vocabulary(gpu, kind):
    gen = torch.Generator().manual_seed(1)
    logits, tokens, uniforms, more = drafted(gen, 3, 4, 128256, torch.float32, kind, peak=4)
    check_verify(gpu, logits, tokens, uniforms, **more)


@pytest.mark.parametrize("kind", ["line", "tree"])
def test_verification_of_many_rows(gpu, kind):
    gen = torch.Generator().manual_seed(2)
    logits, tokens, uniforms, more = drafted(gen, 700, 4, 331, torch.bfloat16, kind)
    check_verify(gpu, logits, tokens, uniforms, **more)


@pytest.mark.parametrize("kind", ["line", "tree", "sure"])
@pytest.mark.parametrize("rows,m,vocab", [(64, 4, 66000), (256, 2, 70001), (2, 2, 1100000)])
def test_verification_of_many_large_rows(gpu, kind, rows, m, vocab):
    gen = torch.Generator().manual_seed(8)
    logits, tokens, uniforms, more = drafted(gen, rows, m, vocab, torch.bfloat16, kind, peak=4)
    check_verify(gpu, logits, tokens, uniforms, **more)


@pytest.mark.parametrize("kind", ["line", "tree", "sure"])
@pytest.mark.parametrize("rows,m,vocab,dtype", [(1500, 3, 300, torch.float32), (130, 33, 515, torch.float16),
                                                (684, 3, 65600, torch.bfloat16)])
def test_verification_of_thousands_of_tokens(gpu, kind, rows, m, vocab, dtype):
    gen = torch.Generator().manual_seed(10)
    logits, tokens, uniforms, more = drafted(gen, rows, m, vocab, dtype, kind, peak=4)
    check_verify(gpu, logits, tokens, uniforms, **more)


def test_verification_where_a_row_stops_without_a_distribution_before_others_would_draw(gpu):
    """Many workgroups to a row, the first token's logits unusable, those behind it fine: again and again."""
    gen = torch.Generator().manual_seed(9)
    logits, tokens, uniforms, more = drafted(gen, 8, 5, 40000, torch.float32, "line")
    more["seq_lens"], more["temperature"] = None, None
    logits[::2, 0, 7] = float("nan")
    want = plain.verify_tokens(logits, tokens, uniforms, **more)
    args, more = (logits.to(gpu), tokens.to(gpu), uniforms.to(gpu)), on(gpu, **more)
    for _ in range(50):
        got = verify_tokens(*args, **more)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind", ["line", "tree", "sure"])
def test_verification_without_a_distribution(gpu, kind):
    """NaN, +inf, nothing allowed, a whole slice banned, bad temperatures: the row stops there, with -1."""
    gen = torch.Generator().manual_seed(3)
    rows, m, vocab = 14, 4, 9000
    logits, tokens, uniforms, more = drafted(gen, rows, m, vocab, torch.float32, kind)
    more["seq_lens"] = None
    more["temperature"] = torch.tensor([0.0, 1.0] * 7)
    more["temperature"][8:14] = torch.tensor([-1.0, float("inf"), float("nan"), 1e-30, 1e30, 1.0])
    logits[0, 0, 5000] = logits[1, 0, 5000] = float("nan")
    logits[2, 0, 17] = logits[3, 1, 17] = float("inf")
    logits[4, 0] = logits[5, 1] = float("-inf")
    logits[6, :, :8192] = logits[7, :, 100:] = float("-inf")
    check_verify(gpu, logits, tokens, uniforms, **more)


@pytest.mark.parametrize("kind", ["line", "tree", "sure"])
def test_verification_ties_and_border_numbers(gpu, kind):
    gen = torch.Generator().manual_seed(4)
    rows, m, vocab = 12, 4, 5000
    logits, tokens, uniforms, more = drafted(gen, rows, m, vocab, torch.bfloat16, kind, peak=0.5)
    logits = logits.round()  # ties everywhere
    uniforms[::3] = 0.0
    uniforms[1::3] = 1 - 2.0**-24
    more["seq_lens"] = None
    check_verify(gpu, logits, tokens, uniforms, **more)
    more["temperature"] = torch.zeros(rows)
    check_verify(gpu, logits, tokens, uniforms, **more)


def test_verification_of_equal_and_of_disjoint_probabilities(gpu):
    vocab, m = 4500, 3
    logits = torch.full((6, m, vocab), float("-inf"))
    logits[:, :, 4200:4204] = 0.0  # a quarter each, exactly
    q = torch.zeros(6, m - 1, vocab)
    q[0, :, 4200:4204] = 0.25  # the model's own
    q[1, :, :4] = 0.25  # none of it
    q[2, :, 4200:4202] = 0.5  # a part of it
    q[3, :, 4200:4204] = 0.5  # more than it: nothing rests, so p itself is drawn from
    q[4, :, 3] = 1.0
    tokens = torch.tensor([[0, 4201, 4203], [0, 1, 2], [0, 4201, 4200], [0, 4200, 4201], [0, 4500, -1], [0, 4202, 9]])
    uniforms = torch.tensor([[0.99, 0.99, 0.6], [0.0, 0.5, 0.3], [0.4, 0.7, 0.9], [0.9, 0.9, 0.55], [0.0, 0.0, 0.99],
                             [0.0, 0.0, 0.1]])
    path, counts, following = check_verify(gpu, logits, tokens, uniforms, draft_probs=q)
    assert counts.tolist() == [3, 1, 2, 1, 1, 2] and following.tolist()[:4] == [4202, 4201, 4203, 4202]


def test_verification_takes_any_strides_and_shared_trees(gpu):
    gen = torch.Generator().manual_seed(5)
    rows, m, vocab = 5, 6, 777
    logits, tokens, uniforms, more = drafted(gen, rows, m, vocab, torch.float16, "tree")
    parents = random_parents(gen, 1, m)[0]
    want = plain.verify_tokens(logits, tokens, uniforms, parents=parents, seq_lens=more["seq_lens"])
    store = torch.zeros(m, rows, vocab + 3, dtype=torch.float16, device=gpu)
    store[..., 1 : vocab + 1] = logits.transpose(0, 1).to(gpu)
    wide_tokens, wide_u = (torch.zeros(rows, m + 2, dtype=t.dtype, device=gpu) for t in (tokens, uniforms))
    wide_tokens[:, 1:-1], wide_u[:, 1:-1] = tokens.to(gpu), uniforms.to(gpu)
    got = verify_tokens(store.transpose(0, 1)[..., 1 : vocab + 1], wide_tokens[:, 1:-1], wide_u[:, 1:-1],
                        **on(gpu, parents=parents, seq_lens=more["seq_lens"]))
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    # one row's logits for all of them
    logits, tokens, uniforms, more = drafted(gen, 1, m, vocab, torch.float32, "line")
    tokens, uniforms, q = tokens.expand(4, m), torch.rand(4, m, generator=gen), more["draft_probs"].expand(4, m - 1, vocab)
    want = plain.verify_tokens(logits.expand(4, m, vocab), tokens, uniforms, draft_probs=q)
    got = verify_tokens(logits.to(gpu).expand(4, m, vocab), tokens.to(gpu), uniforms.to(gpu),
                        draft_probs=more["draft_probs"].to(gpu).expand(4, m - 1, vocab))
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


def test_verification_of_nothing(gpu):
    for rows, m, vocab in ((0, 3, 5), (2, 0, 5), (2, 3, 0)):
        path, counts, following = verify_tokens(torch.zeros(rows, m, vocab, device=gpu),
                                                torch.zeros(rows, m, dtype=torch.int64, device=gpu),
                                                torch.zeros(rows, m, device=gpu))
        assert path.shape == (rows, m) and following.tolist() == [-1] * rows
        assert counts.tolist() == [min(m, 1)] * rows


def test_verification_refuses(gpu):
    logits, tokens = torch.zeros(2, 3, 8, device=gpu), torch.zeros(2, 3, dtype=torch.int64, device=gpu)
    u, q = torch.zeros(2, 3, device=gpu), torch.zeros(2, 2, 8, device=gpu)
    tree = torch.zeros(2, 3, dtype=torch.int32, device=gpu)

    def call(logits=logits, tokens=tokens, u=u, **more):
        return verify_tokens(logits, tokens, u, **more)

    call(draft_probs=q)
    for bad in (dict(logits=logits[0]), dict(logits=logits[..., ::2]), dict(tokens=tokens[:1]), dict(u=u[:, :2]),
                dict(parents=tree, draft_probs=q), dict(parents=tree[:, :2]), dict(draft_probs=q[:, :1]),
                dict(draft_probs=q[..., :4]), dict(temperature=u[:, 0]), dict(temperature=torch.ones(2)),
                dict(seq_lens=tree[:, 0].contiguous()[:1]), dict(u=u.cpu())):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(logits=logits.double()), dict(tokens=tokens.float()), dict(u=u.double()), dict(draft_probs=q.half()),
                dict(parents=tree.long()), dict(temperature=torch.ones(2, device=gpu).double())):
        with pytest.raises(TypeError):
            call(**bad)
    with pytest.raises(RuntimeError, match="gradient"):
        call(logits=logits.clone().requires_grad_())


def test_verification_in_graphs_and_on_streams(gpu):
    gen = torch.Generator().manual_seed(6)
    cases = [drafted(gen, 6, 5, 9001, torch.float32, kind) for kind in ("line", "tree", "line", "tree")]
    want = [plain.verify_tokens(logits, tokens, u, **more) for logits, tokens, u, more in cases]
    held = [(logits.to(gpu), tokens.to(gpu), u.to(gpu), on(gpu, **more)) for logits, tokens, u, more in cases]
    side = torch.cuda.Stream()
    graphs = []
    for kind in range(2):
        args = tuple(t.clone() for t in held[kind][:3])
        more = {name: None if t is None else t.clone() for name, t in held[kind][3].items()}
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            verify_tokens(*args, **more)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = verify_tokens(*args, **more)
        graphs.append((graph, args, more, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(4):
        for kind, (graph, args, more, _) in enumerate(graphs):
            source = held[kind + 2 * (turn % 2)]
            for a, b in zip(args, source):
                a.copy_(b)
            for name, t in more.items():
                if t is not None:
                    t.copy_(source[3][name])
        torch.cuda.synchronize()
        for (graph, *_), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [verify_tokens(*h[:3], **h[3]) for h in held]
        torch.cuda.synchronize()
        for got, w in zip(eager, want):
            assert all(torch.equal(a.cpu(), b) for a, b in zip(got, w))
        for kind, (*_, out) in enumerate(graphs):
            assert all(torch.equal(a.cpu(), b) for a, b in zip(out, want[kind + 2 * (turn % 2)]))


# ----------------------------------------------------------------------------- moves


def bits_of(x):
    return back(x).view(torch.uint8 if x.dtype == FP8 else torch.int16 if x.element_size() == 2 else torch.int32)


@pytest.mark.parametrize("dtype", DTYPES + [FP8])
@pytest.mark.parametrize("layers,rows,m,kv_heads,dim,page,order", [
    (1, 1, 2, 1, 16, 16, "head"), (3, 4, 9, 2, 80, 16, "slot"), (2, 6, 40, 2, 128, 32, "head"),
    (70, 2, 6, 3, 32, 16, "head"), (1, 3, 600, 1, 16, 64, "slot"),
])
def test_moves_match_the_plain_form(gpu, dtype, layers, rows, m, kv_heads, dim, page, order):
    gen = torch.Generator().manual_seed(layers + rows + m)
    past = torch.randint(0, 3 * page, (rows,), generator=gen).int()
    past[0] = 0
    counts = torch.randint(0, m + 2, (rows,), generator=gen).int()
    path = torch.full((rows, m), -1, dtype=torch.int32)
    for b in range(rows):
        k = min(m, int(counts[b]))
        path[b, :k] = torch.randperm(m, generator=gen)[:k].sort().values
    if rows > 2:
        path[-1, : min(4, m)] = torch.tensor([0, 2, 2, 3])[: min(4, m)]  # ends at the second 2
        counts[-1] = m
        path[-2, 0] = -1  # nothing moves
    model = torch.bfloat16 if dtype == FP8 else dtype
    keys, values = [], []
    state = gen.get_state()
    for _ in range(layers):
        gen.set_state(state)  # the same pages in every layer
        key, value, table, _, _ = pool(gen, rows, [int(p) + m for p in past], kv_heads, dim, page, model, dtype == FP8)
        shift = torch.randn(1, generator=gen) if dtype != FP8 else 0
        keys.append(key if dtype == FP8 else (key + len(keys)).to(dtype))
        values.append(value if dtype == FP8 else (value + shift).to(dtype))
    if rows > 2:
        table[1, -1] = -1
    up = [[put(x, gpu, order) for x in xs] for xs in (keys, values)]
    assert keep_tokens(*up, *(t.to(gpu) for t in (table, past, path, counts))) is None
    for before, after in zip(keys + values, up[0] + up[1]):
        assert torch.equal(bits_of(after), bits_of(plain.keep_tokens(before, table, past, path, counts)))


def test_moves_of_stacked_layers_and_of_nothing(gpu):
    gen = torch.Generator().manual_seed(1)
    stack = torch.randn(2, 3, 5, 2, 16, 32, generator=gen)  # keys and values of three layers in one tensor
    table = torch.tensor([[4, 1]], dtype=torch.int32, device=gpu)
    past, counts = torch.tensor([14], dtype=torch.int32, device=gpu), torch.tensor([3], dtype=torch.int32, device=gpu)
    path = torch.tensor([[0, 3, 4]], dtype=torch.int32, device=gpu)
    up = stack.to(gpu)
    keep_tokens(up[0], up[1], table, past, path, counts)
    for i in range(2):
        for layer in range(3):
            want = plain.keep_tokens(stack[i, layer], *(t.cpu() for t in (table, past, path, counts)))
            assert torch.equal(up[i, layer].cpu(), want)
    before = up.clone()
    keep_tokens([], [], table, past, path, counts)
    keep_tokens(up[0], up[1], table, past, path, counts * 0)
    keep_tokens(up[0], up[1], table[:0], past[:0], path[:0], counts[:0])
    keep_tokens(up[0], up[1], table, past, path[:, :0], counts)
    keep_tokens(up[0], up[1], table, past, torch.arange(3, dtype=torch.int32, device=gpu)[None], counts)
    assert torch.equal(up, before)


def test_moves_refuse(gpu):
    key, value = (torch.zeros(4, 2, 16, 32, device=gpu) for _ in range(2))
    table, path = torch.zeros(2, 2, dtype=torch.int32, device=gpu), torch.zeros(2, 3, dtype=torch.int32, device=gpu)
    n = torch.zeros(2, dtype=torch.int32, device=gpu)

    def call(keys=(key,), values=(value,), table=table, past=n, path=path, counts=n):
        return keep_tokens(keys, values, table, past, path, counts)

    call()
    for bad in (dict(keys=(key, key)), dict(keys=(key,), values=(key,)), dict(values=(value[:3],)),
                dict(values=(value.bfloat16(),)), dict(values=(torch.zeros(4, 16, 2, 32, device=gpu).transpose(1, 2),)),
                dict(keys=(key[0],), values=(value[0],)), dict(table=table[:1]), dict(past=n[:1]), dict(path=path[0]),
                dict(counts=n[:1]), dict(keys=(key.cpu(),), values=(value.cpu(),)),
                dict(keys=(torch.zeros(4, 2, 8, 32, device=gpu),), values=(torch.zeros(4, 2, 8, 32, device=gpu),))):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(path=path.long()), dict(counts=n.long()), dict(keys=(key.double(),), values=(value.double(),)),
                dict(keys=3), dict(keys=(3,))):
        with pytest.raises(TypeError):
            call(**bad)
    wide = torch.zeros(4, 1, 16, 32, device=gpu).expand(4, 2, 16, 32)
    with pytest.raises(RuntimeError, match="share"):
        call(keys=(wide,), values=(torch.zeros(4, 1, 16, 32, device=gpu).expand(4, 2, 16, 32),))

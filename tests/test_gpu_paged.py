"""The paged cache's operators against their 64-bit plain forms: sizes, types, layouts, masks, streams, refusals."""

from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from oracle import decode as plain
from polylora_amd.paged import paged_attention, rope_append, rope_table

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
# half a unit in the last place of each type, relative
UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, FP8: 2.0**-4}
# and the smallest step of its subnormals
STEP = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24, FP8: 2.0**-9}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def pool(gen, rows, lens, kv_heads, dim, page, dtype, fp8=False, columns=0):
    """CPU (key, value, table, k_scale, v_scale): random pages in random places, NaN in slots without a token."""
    counts = [-(-n // page) for n in lens]
    total = sum(counts) + 3
    ids = torch.randperm(total, generator=gen).tolist()
    width = max(1, columns, *counts)
    table = torch.full((rows, width), -1, dtype=torch.int32)
    held = torch.zeros(total, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(counts):
        for i in range(n):
            table[b, i] = ids[at]
            held[ids[at], : min(page, lens[b] - i * page)] = True
            at += 1
    caches, scales = [], []
    for _ in range(2):
        x = torch.randn(total, kv_heads, page, dim, generator=gen)
        scale = torch.rand(kv_heads, generator=gen) * 0.05 + 0.01
        x = (x / scale[:, None, None]).clamp(-448, 448) if fp8 else x
        x = x.masked_fill(~held[:, None, :, None], float("nan")).to(FP8 if fp8 else dtype)
        caches.append(x)
        scales.append(scale if fp8 else None)
    return caches[0], caches[1], table, scales[0], scales[1]


def put(x, gpu, order="head"):
    """A cache on the GPU with its pages laid out by head or by slot."""
    if x is None:
        return None
    if order == "head":
        return x.to(gpu)
    bits = x.view(torch.uint8) if x.dtype == FP8 else x
    return bits.transpose(1, 2).contiguous().to(gpu).view(x.dtype).transpose(1, 2)


def back(x):
    return x.cpu().contiguous()


# ----------------------------------------------------------------------------- append


def check_append(got, want, unit_of, sizes):
    """One rounding to the type, and fp32 products and sums before it (three roundings each)."""
    got, want = back(got).double(), want
    assert torch.equal(got.isnan(), want.isnan())
    got, want, sizes = got.nan_to_num(0.0), want.nan_to_num(0.0), sizes.nan_to_num(0.0)
    tol = UNIT[unit_of] * want.abs() + STEP[unit_of] / 2 + 2.0**-21 * sizes
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() - tol).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,m,heads,kv_heads,dim,page,rot,interleaved,fp8,order", [
    (1, 1, 4, 1, 16, 16, 16, False, False, "head"),
    (3, 1, 32, 8, 128, 16, 128, False, False, "head"),
    (5, 7, 6, 2, 80, 32, 80, False, False, "slot"),
    (4, 37, 4, 4, 96, 16, 48, True, False, "head"),
    (2, 5, 3, 1, 256, 64, 10, False, False, "slot"),
    (2, 9, 5, 5, 48, 16, 30, True, False, "head"),
    (3, 4, 2, 2, 64, 16, 0, False, False, "head"),
    (3, 11, 8, 2, 128, 16, 128, False, True, "head"),
    (2, 18, 4, 2, 80, 32, 40, False, True, "slot"),
    (2, 3, 4, 2, 32, 16, 32, True, True, "head"),
])
def test_append_matches_the_plain_form(gpu, dtype, rows, m, heads, kv_heads, dim, page, rot, interleaved, fp8, order):
    if fp8 and dtype == torch.float32:
        pytest.skip("an 8-bit cache serves 16-bit models")
    gen = torch.Generator().manual_seed(rows * 100 + m + dim)
    past = torch.randint(0, 3 * page, (rows,), generator=gen)
    seq = torch.randint(0, m + 3, (rows,), generator=gen)  # rows of no new token, and lengths above m
    seq[0] = m
    key, value, table, ks, vs = pool(gen, rows, [int(p) + m for p in past], kv_heads, dim, page, dtype, fp8)
    if rows > 2:
        table[-1, int(past[-1]) // page] = -1  # a page that the table does not hold
    qkv = torch.randn(rows, m, heads + 2 * kv_heads, dim, generator=gen).to(dtype)
    q, k, v = qkv.split((heads, kv_heads, kv_heads), 2)
    cos, sin = rope_table(int(past.max()) + m, rot, 10000.0)
    if fp8:
        v[0, 0] *= 1000  # saturates
    want = plain.rope_append(q, k, v, key, value, table, past, cos, sin, seq, interleaved, ks, vs)
    # |x c| + |z s|, which the rounding errors are proportional to: the first of a pair with one sign, its second with the other
    sizes = [plain.rope_append(q.abs(), k.abs(), v.abs(), key.double().abs(), value.double().abs(), table, past,
                               cos.abs(), sign * sin.abs(), seq, interleaved, ks, vs) for sign in (-1, 1)]
    qkv = qkv.to(gpu)
    gq, gk, gv = qkv.split((heads, kv_heads, kv_heads), 2)
    gkey, gvalue = put(key, gpu, order), put(value, gpu, order)
    k_out = torch.full((rows, m, kv_heads, dim), 7.0, dtype=dtype, device=gpu)
    up = {"k_scale": None if ks is None else ks.to(gpu), "v_scale": None if vs is None else vs.to(gpu)}
    q_out = rope_append(gq, gk, gv, gkey, gvalue, table.to(gpu), past.int().to(gpu), cos.to(gpu), sin.to(gpu),
                        seq_lens=seq.int().to(gpu), interleaved=interleaved, k_out=k_out, **up)
    both = [torch.maximum(a, b) for a, b in zip(*sizes)]
    check_append(q_out, want[0], dtype, both[0])
    check_append(k_out, want[1], dtype, both[1])
    cache_type = FP8 if fp8 else dtype
    check_append(gkey, want[2], cache_type, both[2])
    check_append(gvalue, want[3], cache_type, both[3])


def test_append_keeps_every_other_byte_and_rounds_once(gpu):
    """Values are copied bit for bit; bytes of other slots, pages and table columns stay."""
    gen = torch.Generator().manual_seed(5)
    dtype, page = torch.bfloat16, 16
    past = [0, 15, 16, 31]
    key, value, table, _, _ = pool(gen, 4, [p + 2 for p in past], 2, 64, page, dtype)
    q = torch.randn(4, 2, 4, 64, generator=gen).to(dtype)
    k, v = (torch.randn(4, 2, 2, 64, generator=gen).to(dtype) for _ in range(2))
    cos, sin = torch.ones(64, 32), torch.zeros(64, 32)  # no turn: keys are copied too
    gkey, gvalue = key.to(gpu), value.to(gpu)
    q_out = rope_append(q.to(gpu), k.to(gpu), v.to(gpu), gkey, gvalue, table.to(gpu),
                        torch.tensor(past, dtype=torch.int32, device=gpu), cos.to(gpu), sin.to(gpu))
    for b, p in enumerate(past):
        for t in range(2):
            at = plain.place(table, b, p + t, key.shape[0], page)
            key[at[0], :, at[1]], value[at[0], :, at[1]] = k[b, t], v[b, t]
    assert torch.equal(back(gkey).view(torch.int16), key.view(torch.int16))
    assert torch.equal(back(gvalue).view(torch.int16), value.view(torch.int16))
    assert torch.equal(q_out.cpu(), q)


def test_append_takes_empty_batches(gpu):
    key = torch.zeros(2, 1, 16, 16, device=gpu)
    cos, sin = rope_table(4, 16, device=gpu)
    for rows, m in ((0, 3), (2, 0)):
        x = torch.zeros(rows, m, 1, 16, device=gpu)
        table = torch.zeros(rows, 1, dtype=torch.int32, device=gpu)
        past = torch.zeros(rows, dtype=torch.int32, device=gpu)
        assert rope_append(x, x, x, key, key.clone(), table, past, cos, sin).shape == (rows, m, 1, 16)


def test_append_skips_positions_outside_the_table_and_the_angles(gpu):
    key = torch.zeros(2, 1, 16, 16, device=gpu)
    value = torch.zeros(2, 1, 16, 16, device=gpu)
    x = torch.ones(5, 1, 1, 16, device=gpu)
    table = torch.tensor([[0], [0], [2], [-5], [1]], dtype=torch.int32, device=gpu)
    past = torch.tensor([16, -1, 3, 3, 9], dtype=torch.int32, device=gpu)  # past the columns, below 0, no such page (2x), past cos
    cos, sin = rope_table(9, 16, device=gpu)
    q = rope_append(x, x, x, key, value, table, past, cos, sin)
    assert not q.any() and not key.any() and not value.any()


# ----------------------------------------------------------------------------- attention


def attention_tolerance(want, spread, reach, dtype, dim, tokens):
    """One rounding of the output; scores off by (dim + 8) fp32 roundings of |q| . |k| and exponents and factors by a
    few more, which move each weight by that share; weights of 16-bit values kept to 2 ** -15; sums of at most one
    addition for every 32 tokens and 64 more."""
    weights = 2.0**-24 * (4 * (dim + 8) * reach + 16) + 2.0**-24 * (tokens / 32 + 64)
    if dtype != torch.float32:
        weights = weights + 2.0**-15
    return UNIT[dtype] * want.abs() + STEP[dtype] + weights * spread


def check_attention(gpu, dtype, lens, heads, kv_heads, dim, page, fp8=False, order="head", window=None, scale=None,
                    seed=0, q_gain=1.5, holes=False, columns=0):
    gen = torch.Generator().manual_seed(seed + dim + heads)
    rows = len(lens)
    held = [min(n, (columns or 10**9) * page) for n in lens]
    key, value, table, ks, vs = pool(gen, rows, held, kv_heads, dim, page, dtype, fp8, columns=columns)
    if holes:
        table[::2, 0] = -1
        table[1::2, 0] = key.shape[0]
    q = (torch.randn(rows, heads + 1, dim, generator=gen) * q_gain).to(dtype)
    n = torch.tensor(lens, dtype=torch.int32)
    want, spread, reach = plain.paged_attention(q[:, 1:], key, value, table, n, scale, window, ks, vs)
    up = {"k_scale": None if ks is None else ks.to(gpu), "v_scale": None if vs is None else vs.to(gpu)}
    args = (q.to(gpu)[:, 1:], put(key, gpu, order), put(value, gpu, order), table.to(gpu), n.to(gpu))
    got = paged_attention(*args, scale=scale, window=window, **up)
    tol = attention_tolerance(want, spread, reach, dtype, dim, max(1, *lens))
    err = (got.cpu().double() - want).abs()
    assert not got.isnan().any()
    assert bool((err <= tol).all()), (float((err / tol).max()), float(err.max()))
    again = torch.full_like(got, 7.0)
    assert paged_attention(*args, scale=scale, window=window, out=again, **up) is again
    assert torch.equal(again, got)  # the same bits each time
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (1, 1, 16, 16), (4, 1, 32, 16), (32, 8, 128, 16), (12, 12, 80, 32), (28, 4, 96, 64), (9, 3, 256, 16),
    (16, 1, 64, 128), (17, 1, 64, 16), (40, 2, 48, 16), (6, 2, 192, 32), (3, 1, 112, 16), (5, 5, 144, 16),
    (48, 1, 64, 16), (71, 1, 64, 16), (66, 2, 128, 16), (130, 1, 256, 16), (64, 2, 80, 32),
])
def test_attention_matches_the_plain_form(gpu, dtype, heads, kv_heads, dim, page):
    check_attention(gpu, dtype, [1, 0, 2, 15, 16, 17, 33, 100, 257], heads, kv_heads, dim, page)


@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("heads,kv_heads,dim,page,order", [
    (4, 1, 16, 16, "head"), (32, 8, 128, 16, "slot"), (12, 4, 96, 32, "head"), (8, 8, 80, 16, "head"),
    (20, 1, 64, 64, "slot"), (4, 2, 256, 16, "head"),
])
def test_attention_over_an_8_bit_cache(gpu, dtype, heads, kv_heads, dim, page, order):
    check_attention(gpu, dtype, [3, 0, 31, 64, 65, 300], heads, kv_heads, dim, page, fp8=True, order=order)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 16, 31, 63, 64, 1000])
def test_attention_windows(gpu, dtype, window):
    check_attention(gpu, dtype, [0, 1, 16, 40, 63, 64, 65, 200], 8, 2, 64, 16, window=window, order="slot")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,heads,kv_heads", [([5000], 8, 2), ([3000, 1, 2999], 4, 4), ([2049] * 4 + [0] * 9, 16, 1),
                                                 ([4000, 700], 40, 2), ([3000], 71, 1)])
def test_attention_over_long_rows(gpu, dtype, lens, heads, kv_heads):
    check_attention(gpu, dtype, lens, heads, kv_heads, 128, 16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_many_rows(gpu, dtype):
    gen = torch.Generator().manual_seed(3)
    check_attention(gpu, dtype, torch.randint(0, 70, (700,), generator=gen).tolist(), 4, 2, 64, 16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_leaves_out_pages_the_table_does_not_hold(gpu, dtype):
    check_attention(gpu, dtype, [10, 16, 17, 40, 300], 8, 2, 64, 16, holes=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_clamps_lengths_to_the_table(gpu, dtype):
    check_attention(gpu, dtype, [10_000, 64, 65, 0], 8, 2, 64, 16, columns=4)


def test_attention_of_negative_lengths_is_empty(gpu):
    key = torch.ones(2, 1, 16, 64, dtype=torch.bfloat16, device=gpu)
    table = torch.zeros(2, 1, dtype=torch.int32, device=gpu)
    q = torch.ones(2, 1, 64, dtype=torch.bfloat16, device=gpu)
    assert not paged_attention(q, key, key, table, torch.tensor([-1, -100], dtype=torch.int32, device=gpu)).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale,gain", [(1.0, 20.0), (0.0, 1.0), (-0.3, 1.0), (0.125, 40.0)])
def test_attention_scales_and_peaks(gpu, dtype, scale, gain):
    """One token that takes all of the weight, all tokens alike, and a negative scale."""
    check_attention(gpu, dtype, [1, 30, 64, 129, 1000], 4, 2, 64, 16, scale=scale, q_gain=gain)


def test_attention_takes_no_rows_and_no_pages(gpu):
    key = torch.zeros(0, 2, 16, 64, dtype=torch.bfloat16, device=gpu)
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=gpu)
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    assert paged_attention(q, key, key, none.view(0, 0), none).shape == (0, 4, 64)
    q = torch.ones(3, 4, 64, dtype=torch.bfloat16, device=gpu)
    table = torch.full((3, 2), -1, dtype=torch.int32, device=gpu)
    assert not paged_attention(q, key, key, table, torch.full((3,), 20, dtype=torch.int32, device=gpu)).any()
    assert not paged_attention(q, key, key, table[:, :0], torch.full((3,), 20, dtype=torch.int32, device=gpu)).any()


# ----------------------------------------------------------------------------- values that are easily lost


# rows that a wave has to itself, rows that a workgroup takes whole, a row that is split over workgroups
DEALS = {"alone": [300] * 300, "whole": [600] * 128, "split": [8192]}


@pytest.mark.parametrize("deal", DEALS)
@pytest.mark.parametrize("dtype,fp8", [(d, False) for d in DTYPES] + [(d, True) for d in DTYPES[:2]])
def test_attention_keeps_tokens_far_below_the_highest_score(gpu, deal, dtype, fp8):
    """A first token of value 0 that stands 2 to 22 above all others: the output is the others' alone."""
    lens, kv_heads, dim, page = DEALS[deal], 2, 64, 64
    above = torch.tensor([2.0, 12.0, 14.0, 16.0, 18.0, 20.0, 22.0])
    gen = torch.Generator().manual_seed(21)
    key, value, table, ks, vs = pool(gen, len(lens), lens, kv_heads, dim, page, dtype, fp8)
    key = torch.where(key.float().isnan(), float("nan"), 0.0)
    value = value.float().abs()
    first = table[:, 0].long()
    key[first, :, 0, 0], value[first, :, 0] = 1.0, 0.0
    key, value, ks = key.to(FP8 if fp8 else dtype), value.to(FP8 if fp8 else dtype), torch.ones(kv_heads) if fp8 else None
    q = torch.zeros(len(lens), kv_heads * len(above), dim, dtype=dtype)
    q[:, :, 0] = above.repeat(kv_heads)
    n = torch.tensor(lens, dtype=torch.int32)
    want, spread, reach = plain.paged_attention(q, key, value, table, n, 1.0, None, ks, vs)
    up = {"k_scale": ks.to(gpu), "v_scale": vs.to(gpu)} if fp8 else {}
    got = paged_attention(q.to(gpu), key.to(gpu), value.to(gpu), table.to(gpu), n.to(gpu), scale=1.0, **up)
    # the first token's value of 0 adds nothing to `spread`: what is allowed is relative to the output
    tol = attention_tolerance(want, spread, reach, dtype, dim, max(lens))
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def _finite_batch(gpu, dtype, deal, fp8=False):
    """Arguments on the GPU, two query heads to each of two key heads, and the page and slot of a token in the middle
    of the last row."""
    lens, page = DEALS[deal], 16
    gen = torch.Generator().manual_seed(22)
    key, value, table, ks, vs = pool(gen, len(lens), lens, 2, 64, page, dtype, fp8)
    q = torch.randn(len(lens), 4, 64, generator=gen).to(dtype)
    at = plain.place(table, len(lens) - 1, lens[-1] // 2, key.shape[0], page)
    args = [x.to(gpu) for x in (q, key, value, table, torch.tensor(lens, dtype=torch.int32))]
    return args, {"k_scale": ks.to(gpu), "v_scale": vs.to(gpu)} if fp8 else {}, at


@pytest.mark.parametrize("deal", DEALS)
@pytest.mark.parametrize("dtype,fp8", [(d, False) for d in DTYPES] + [(torch.bfloat16, True)])
def test_attention_hands_on_nan_that_counts(gpu, deal, dtype, fp8):
    """NaN in a query, in a key and in a value: NaN comes out where it goes in, and nowhere else."""
    (q, key, value, table, lens), scales, (page, slot) = _finite_batch(gpu, dtype, deal, fp8)
    clean = paged_attention(q, key, value, table, lens, **scales)
    assert not clean.isnan().any()

    def check(where, *args):
        got = paged_attention(*args, table, lens, **scales)
        assert torch.equal(got.isnan(), where)
        assert torch.equal(got[~where], clean[~where])

    where = torch.zeros(clean.shape, dtype=torch.bool, device=gpu)
    bad = q.clone()
    bad[-1, 1, 5] = float("nan")
    where[-1, 1] = True
    check(where, bad, key, value)
    bits = torch.tensor(float("nan")).to(key.dtype).view(torch.uint8 if fp8 else key.dtype).to(gpu)
    bad = key.clone()
    (bad.view(torch.uint8) if fp8 else bad)[page, 1, slot, 7] = bits
    where.zero_()[-1, 2:] = True
    check(where, q, bad, value)
    bad = value.clone()
    (bad.view(torch.uint8) if fp8 else bad)[page, 1, slot, 7] = bits
    where.zero_()[-1, 2:, 7] = True
    check(where, q, key, bad)


@pytest.mark.parametrize("deal", DEALS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_hands_on_infinite_values(gpu, deal, dtype):
    """An infinite value has a weight above 0, so its sum is infinite; the largest score's, whose weight is 1, among them."""
    (q, key, value, table, lens), _, (page, slot) = _finite_batch(gpu, dtype, deal)
    key[page, 1, slot] = q[-1, 2] * 2  # the highest score of one query head, an ordinary one of the other
    clean = paged_attention(q, key, value, table, lens)
    value[page, 1, slot, 7], value[page, 1, slot, 60] = float("inf"), float("-inf")
    got = paged_attention(q, key, value, table, lens)
    assert bool((got[-1, 2:, 7] == float("inf")).all()) and bool((got[-1, 2:, 60] == float("-inf")).all())
    same = torch.ones(clean.shape, dtype=torch.bool, device=gpu)
    same[-1, 2:, 7] = same[-1, 2:, 60] = False
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("dtype", DTYPES[:2])
def test_append_stores_quotients_in_8_bits(gpu, dtype):
    """Values half way between two e4m3 numbers, over scales whose reciprocals are rounded: the even one, as x / scale is."""
    heads = torch.arange(3, 8 if dtype == torch.bfloat16 else 64, 2)
    scale = heads / 256.0
    x = (torch.arange(16, 32) / 16.0)[None] * scale[:, None]
    k = x.to(dtype)[None, None]
    assert torch.equal(k.float()[0, 0], x)
    want = (k.float()[0, 0] / scale[:, None]).to(FP8).float()
    key = torch.zeros(1, len(heads), 16, 16, device=gpu).to(FP8)
    value, k, up = key.clone(), k.to(gpu), scale.to(gpu)
    cos, sin = rope_table(4, 0, device=gpu)
    zero = torch.zeros(1, dtype=torch.int32, device=gpu)
    rope_append(k, k, k, key, value, zero[None], zero, cos, sin, k_scale=up, v_scale=up)
    assert torch.equal(key[0, :, 0].float().cpu(), want)
    assert torch.equal(value[0, :, 0].float().cpu(), want)


# ----------------------------------------------------------------------------- what large batches alone reach


def _ragged(gen, rows, low, high):
    return torch.randint(low, high + 1, (rows,), generator=gen).tolist()


@pytest.mark.parametrize("dtype,fp8", [(d, False) for d in DTYPES] + [(torch.float16, True)])
@pytest.mark.parametrize("kv_heads,heads,dim", [(16, 16, 64), (16, 32, 128)])
def test_attention_of_more_pairs_than_waves(gpu, dtype, fp8, kv_heads, heads, dim):
    """4800 pairs: every wave takes a run of whole pairs, which begin and end inside rows, some of them empty."""
    gen = torch.Generator().manual_seed(41)
    check_attention(gpu, dtype, _ragged(gen, 300, 0, 200), heads, kv_heads, dim, 16, fp8=fp8)


@pytest.mark.parametrize("dtype,fp8", [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("rows,low,high", [(70, 400, 520), (6, 6000, 8192), (40, 1, 4000)])
def test_attention_of_many_tokens(gpu, dtype, fp8, rows, low, high):
    """2048 atoms and more: one workgroup on a CU, pairs alone and split."""
    gen = torch.Generator().manual_seed(42)
    check_attention(gpu, dtype, _ragged(gen, rows, low, high), 8, 8, 128, 64, fp8=fp8)


@pytest.mark.parametrize("dtype,fp8", [(d, False) for d in DTYPES] + [(d, True) for d in DTYPES[:2]])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens", [[100] * 40 + [0, 1, 33], [3000, 17]])
def test_attention_over_a_pool_larger_than_the_last_cache(gpu, dtype, fp8, dim, lens):
    """Pages marked as read once, out of more than 256 MiB of them: the bits that a small pool gives."""
    gen = torch.Generator().manual_seed(43)
    kv_heads, page = 4, 64
    key, value, table, ks, vs = pool(gen, len(lens), lens, kv_heads, dim, page, dtype, fp8)
    n = key.shape[0]
    large = (257 << 20) // (2 * kv_heads * page * dim * key.element_size()) + 1
    ids = torch.randperm(large, generator=gen)[:n]
    up = {"k_scale": ks.to(gpu), "v_scale": vs.to(gpu)} if fp8 else {}
    q = torch.randn(len(lens), 8, dim, generator=gen).to(dtype).to(gpu)
    lens = torch.tensor(lens, dtype=torch.int32, device=gpu)
    want = paged_attention(q, key.to(gpu), value.to(gpu), table.to(gpu), lens, **up)
    assert not want.isnan().any()
    wide = []
    for c in (key, value):
        bits = c.view(torch.uint8) if fp8 else c
        x = torch.full((large, *c.shape[1:]), 127 if fp8 else float("nan"), dtype=bits.dtype, device=gpu)
        x[ids.to(gpu)] = bits.to(gpu)
        wide.append(x.view(c.dtype))
    moved = torch.where((table >= 0) & (table < n), ids[table.clamp(0, n - 1).long()], -1).int()
    assert torch.equal(paged_attention(q, *wide, moved.to(gpu), lens, **up), want)


def _append_by_rows(q, k, v, key, value, table, past, cos, sin, seq, interleaved, ks, vs):
    """oracle.decode.rope_append, a row's tokens at once."""
    m, page = q.shape[1], key.shape[2]
    out = [torch.zeros(x.shape, dtype=torch.float64) for x in (q, k)]
    caches = [key.double().clone(), value.double().clone()]
    for b in range(q.shape[0]):
        n = min(m, int(seq[b]))
        pos = int(past[b]) + torch.arange(n)
        c, s = (t[pos].double()[:, None] for t in (cos, sin))
        h = c.shape[-1]
        for x, y in zip((q, k), out):
            x = x[b, :n].double()
            i = torch.arange(h) * 2 if interleaved else torch.arange(h)
            j = i + 1 if interleaved else i + h
            y[b, :n] = x
            y[b, :n, :, i], y[b, :n, :, j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
        for cache, x, scale in zip(caches, (out[1][b, :n], v[b, :n].double()), (ks, vs)):
            x = x if scale is None else (x / scale.double()[:, None]).clamp(-448, 448)
            cache[table[b].long()[pos // page], :, pos % page] = x
    return *out, *caches


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_plain_append_by_rows_is_the_plain_append(interleaved):
    gen = torch.Generator().manual_seed(44)
    key, value, table, ks, vs = pool(gen, 3, [40, 20, 33], 2, 32, 16, torch.bfloat16, True)
    q, k, v = (torch.randn(3, 7, h, 32, generator=gen) for h in (4, 2, 2))
    past, seq = torch.tensor([33, 5, 0]), torch.tensor([7, 0, 4])
    cos, sin = rope_table(40, 20)
    args = (q, k, v, key, value, table, past, cos, sin, seq, interleaved, ks, vs)
    for a, b in zip(_append_by_rows(*args), plain.rope_append(*args)):
        assert torch.equal(a.isnan(), b.isnan())
        torch.testing.assert_close(a.nan_to_num(0.0), b.nan_to_num(0.0), rtol=1e-14, atol=1e-14)


@pytest.mark.parametrize("dtype,fp8", [(d, False) for d in DTYPES] + [(d, True) for d in DTYPES[:2]])
@pytest.mark.parametrize("rows,m,heads,kv_heads,dim,rot,interleaved", [
    (1, 4099, 8, 2, 64, 64, False),  # two tokens to a workgroup, an odd number of them
    (3, 2735, 4, 2, 64, 64, True),  # four
    (3, 5461, 3, 1, 80, 40, False),
    (2, 4100, 4, 1, 256, 256, False),  # as many as its places leave threads for
    (5, 1700, 6, 2, 48, 30, True),  # single elements
])
def test_append_of_many_tokens(gpu, dtype, fp8, rows, m, heads, kv_heads, dim, rot, interleaved):
    """Outputs past the caches and several tokens to a workgroup, the last one part full, rows part full."""
    gen = torch.Generator().manual_seed(45)
    past, page = torch.randint(0, 50, (rows,), generator=gen), 64
    seq = torch.randint(m // 2, m + 1, (rows,), generator=gen)
    seq[0] = m
    key, value, table, ks, vs = pool(gen, rows, [int(p + n) for p, n in zip(past, seq)], kv_heads, dim, page, dtype, fp8)
    q, k, v = torch.randn(rows, m, heads + 2 * kv_heads, dim, generator=gen).to(dtype).split((heads, kv_heads, kv_heads), 2)
    cos, sin = rope_table(m + 50, rot)
    args = (q, k, v, key, value, table, past, cos, sin, seq, interleaved, ks, vs)
    want = _append_by_rows(*args)
    sizes = [_append_by_rows(q.abs(), k.abs(), v.abs(), key.float().abs(), value.float().abs(), table, past, cos.abs(),
                             sign * sin.abs(), seq, interleaved, ks, vs) for sign in (-1, 1)]
    sizes = [torch.maximum(a, b) for a, b in zip(*sizes)]
    gkey, gvalue, k_out = key.to(gpu), value.to(gpu), torch.full((rows, m, kv_heads, dim), 7.0, dtype=dtype, device=gpu)
    up = {"k_scale": ks.to(gpu), "v_scale": vs.to(gpu)} if fp8 else {}
    q_out = rope_append(q.to(gpu), k.to(gpu), v.to(gpu), gkey, gvalue, table.to(gpu), past.int().to(gpu), cos.to(gpu),
                        sin.to(gpu), seq_lens=seq.int().to(gpu), interleaved=interleaved, k_out=k_out, **up)
    for got, one, size, kind in zip((q_out, k_out, gkey, gvalue), want, sizes, (dtype, dtype, FP8 if fp8 else dtype,
                                                                             FP8 if fp8 else dtype)):
        check_append(got, one, kind, size)


# ----------------------------------------------------------------------------- streams and graphs


def _step(gpu, gen, rows=6, dtype=torch.bfloat16, longest=900):
    past = torch.randint(0, longest, (rows,), generator=gen)
    key, value, table, _, _ = pool(gen, rows, [int(p) + 1 for p in past], 2, 64, 16, dtype)
    q, k, v = (torch.randn(rows, 1, h, 64, generator=gen).to(dtype).to(gpu) for h in (8, 2, 2))
    cos, sin = rope_table(longest + 1, 64, device=gpu)
    key, value, table, past = key.to(gpu), value.to(gpu), table.to(gpu), past.int().to(gpu)

    def run():
        turned = rope_append(q, k, v, key, value, table, past, cos, sin)
        return paged_attention(turned[:, 0], key, value, table, past + 1)

    return run, q


def test_append_then_attend_on_two_streams(gpu):
    gen = torch.Generator().manual_seed(11)
    steps = [_step(gpu, gen)[0] for _ in range(2)]
    want = [s() for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(3):
        got = []
        for s, step in zip(streams, steps):
            with torch.cuda.stream(s):
                got.append(step())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("warm", [True, False])
def test_append_then_attend_in_a_graph(gpu, warm):
    """Replays with new inputs between them, and eager calls of other sizes on the same stream."""
    gen = torch.Generator().manual_seed(12)
    run, q = _step(gpu, gen)
    other, _ = _step(gpu, gen, rows=3, longest=5000)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        if warm:
            run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = run()
    other_want = other()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=gen).to(q.dtype))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        with torch.cuda.stream(stream):
            assert torch.equal(other(), other_want)
            assert torch.equal(run(), got)
        torch.cuda.synchronize()


def _capture(fn, stream=None):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = fn()
    return graph, out


@pytest.mark.parametrize("warm", [True, False])
def test_graphs_of_one_capture_stream_replayed_beside_each_other(gpu, warm):
    """Two graphs captured on the same stream, with rows that are split, on two other streams at once, and eager calls
    on the capture stream beside them."""
    gen = torch.Generator().manual_seed(13)
    steps = [_step(gpu, gen, rows=2, longest=9000)[0] for _ in range(3)]
    want = [s() for s in steps]
    capture = torch.cuda.Stream()
    capture.wait_stream(torch.cuda.current_stream())
    if warm:
        with torch.cuda.stream(capture):
            steps[2]()
    torch.cuda.synchronize()
    graphs = [_capture(s, capture) for s in steps[:2]]
    streams = [torch.cuda.Stream() for _ in graphs]
    got = [[], [], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, (graph, out), kept in zip(streams, graphs, got):
            with torch.cuda.stream(stream):
                graph.replay()
                kept.append(out.clone())
        with torch.cuda.stream(capture):
            got[2].append(steps[2]())
    torch.cuda.synchronize()
    for kept, one in zip(got, want):
        assert all(torch.equal(x, one) for x in kept)


def test_a_graph_keeps_its_scratch_when_others_are_captured(gpu):
    """Head sizes that need larger workspaces, graphs captured and dropped, and eager allocations between replays."""
    gen = torch.Generator().manual_seed(14)
    run, _ = _step(gpu, gen, rows=2, longest=9000)
    want = run()
    torch.cuda.synchronize()
    graph, out = _capture(run)
    for i in range(4):
        other, _ = _step(gpu, gen, rows=2, longest=3000 + i)
        torch.cuda.synchronize()
        dropped, _ = _capture(other)
        dropped.replay()
        torch.cuda.synchronize()
        del dropped
        noise = [torch.full((1 << 20,), -1, dtype=torch.int32, device=gpu) for _ in range(8)]
        torch.cuda.synchronize()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(bool((x == -1).all()) for x in noise)


def test_threads_that_share_a_stream(gpu):
    gen = torch.Generator().manual_seed(15)
    steps = [_step(gpu, gen, rows=2, longest=5000)[0] for _ in range(2)]
    want = [s() for s in steps]
    stream = torch.cuda.Stream()  # no scratch yet
    torch.cuda.synchronize()

    def work(step):
        with torch.cuda.stream(stream):
            return [step() for _ in range(30)]

    with ThreadPoolExecutor(2) as pool:
        got = list(pool.map(work, steps))
    torch.cuda.synchronize()
    for kept, one in zip(got, want):
        assert all(torch.equal(x, one) for x in kept)


# ----------------------------------------------------------------------------- refusals


def _good(gpu, dtype=torch.bfloat16):
    key = torch.zeros(3, 2, 16, 32, dtype=dtype, device=gpu)
    i32 = dict(dtype=torch.int32, device=gpu)
    a = {"q": torch.zeros(2, 4, 32, dtype=dtype, device=gpu), "key_cache": key, "value_cache": key.clone(),
         "page_table": torch.zeros(2, 1, **i32), "lens": torch.ones(2, **i32)}
    cos, sin = rope_table(4, 32, device=gpu)
    x = torch.zeros(2, 1, 2, 32, dtype=dtype, device=gpu)
    b = {"q": torch.zeros(2, 1, 4, 32, dtype=dtype, device=gpu), "k": x, "v": x.clone(), "key_cache": key,
         "value_cache": key.clone(), "page_table": a["page_table"], "past_lens": torch.zeros(2, **i32), "cos": cos, "sin": sin}
    return a, b


def test_refusals_of_both(gpu):
    attend, append = _good(gpu)
    paged_attention(**attend)
    rope_append(**append)
    key = attend["key_cache"]
    fp8 = torch.zeros(3, 2, 16, 32, dtype=FP8, device=gpu)
    ones = torch.ones(2, device=gpu)
    bad = [
        ({"key_cache": key[:, :, :, :16]}, ValueError),  # another head size
        ({"key_cache": key[:2]}, ValueError),  # caches of two sizes
        ({"key_cache": key.float(), "value_cache": key.float()}, TypeError),
        ({"value_cache": key.half()}, TypeError),
        ({"key_cache": fp8, "value_cache": fp8}, ValueError),  # no scales
        ({"key_cache": fp8, "value_cache": fp8, "k_scale": ones, "v_scale": ones[:1]}, ValueError),
        ({"key_cache": fp8, "value_cache": fp8, "k_scale": ones, "v_scale": ones.double()}, TypeError),
        ({"k_scale": ones, "v_scale": ones}, ValueError),  # scales without an 8-bit cache
        ({"key_cache": key[:, :, :8], "value_cache": key[:, :, :8]}, ValueError),  # pages of 8 tokens
        ({"key_cache": key.new_zeros(3, 2, 48, 32), "value_cache": key.new_zeros(3, 2, 48, 32)}, ValueError),
        ({"key_cache": key.transpose(2, 3).contiguous().transpose(2, 3)}, ValueError),
        ({"key_cache": key.cpu()}, (TypeError, ValueError)),
        ({"page_table": attend["page_table"].long()}, TypeError),
        ({"page_table": attend["page_table"][:1]}, ValueError),
        ({"page_table": attend["page_table"][:, 0]}, ValueError),
        ({"page_table": attend["page_table"].cpu()}, ValueError),
        # strides that are no whole 16-byte pieces
        ({"key_cache": key.new_zeros(3, 2, 16, 33)[..., :32]}, RuntimeError),
    ]
    for change, error in bad:
        for fn, good in ((paged_attention, attend), (rope_append, append)):
            with pytest.raises(error):
                fn(**{**good, **change})


def test_refusals_of_the_attention(gpu):
    good, _ = _good(gpu)
    q, key = good["q"], good["key_cache"]
    odd = key.new_zeros(3, 2, 16, 24)
    bad = [
        ({"q": q.cpu()}, RuntimeError),
        ({"q": q[:, :3]}, ValueError),  # three heads over two
        ({"q": q[0]}, ValueError),
        ({"q": q.double()}, TypeError),
        ({"q": q.transpose(1, 2).contiguous().transpose(1, 2)}, ValueError),
        ({"lens": good["lens"].long()}, TypeError),
        ({"lens": good["lens"][:1]}, ValueError),
        ({"window": 0}, ValueError),
        ({"window": -4}, ValueError),
        ({"out": torch.empty(2, 4, 32, device=gpu)}, TypeError),
        ({"out": torch.empty(2, 4, 16, dtype=q.dtype, device=gpu)}, ValueError),
        ({"out": q}, RuntimeError),  # over the queries
        ({"q": q.new_zeros(2, 4, 24), "key_cache": odd, "value_cache": odd}, RuntimeError),  # heads of 24
        ({"q": q.new_zeros(2, 4, 272), "key_cache": key.new_zeros(3, 2, 16, 272),
          "value_cache": key.new_zeros(3, 2, 16, 272)}, RuntimeError),
    ]
    for change, error in bad:
        with pytest.raises(error):
            paged_attention(**{**good, **change})


def test_refusals_of_the_append(gpu):
    _, good = _good(gpu)
    k, cos = good["k"], good["cos"]
    bad = [
        ({"q": good["q"].cpu()}, RuntimeError),
        ({"q": good["q"][:, 0]}, ValueError),
        ({"k": k[:1]}, ValueError),
        ({"v": k[:, :, :1]}, ValueError),
        ({"v": k.float()}, TypeError),
        ({"k": k[:, :, :1], "v": k[:, :, :1]}, ValueError),  # fewer heads than the cache
        ({"past_lens": good["past_lens"].long()}, TypeError),
        ({"past_lens": good["past_lens"][:1]}, ValueError),
        ({"seq_lens": good["past_lens"].long()}, TypeError),
        ({"cos": cos.half()}, TypeError),
        ({"sin": cos[:1]}, ValueError),
        ({"cos": cos[:, :4].t(), "sin": cos[:, :4].t()}, ValueError),
        ({"cos": torch.ones(4, 17, device=gpu), "sin": torch.ones(4, 17, device=gpu)}, ValueError),
        ({"k_out": k[:, :, :1]}, ValueError),
        ({"k_out": k}, RuntimeError),  # over the keys
    ]
    for change, error in bad:
        with pytest.raises(error):
            rope_append(**{**good, **change})


def test_tensors_that_want_derivatives_are_refused(gpu):
    """Any floating-point argument, not only the queries; under no_grad they are taken."""
    dtype = torch.bfloat16
    attend, append = _good(gpu, dtype)
    fp8 = torch.zeros(3, 2, 16, 32, device=gpu).to(FP8)
    ones = torch.ones(2, device=gpu)
    scaled = {"key_cache": fp8, "value_cache": fp8.clone(), "k_scale": ones, "v_scale": ones.clone()}
    attend["out"] = torch.empty_like(attend["q"])
    append["k_out"] = torch.empty_like(append["k"])
    for fn, good in ((paged_attention, attend), (rope_append, append), (paged_attention, {**attend, **scaled}),
                     (rope_append, {**append, **scaled})):
        for name, t in good.items():
            if t.dtype not in (torch.float32, dtype):
                continue
            held = t.detach().clone().requires_grad_()
            with pytest.raises(RuntimeError, match="no backward"):
                fn(**{**good, name: held})
            with torch.no_grad():
                fn(**{**good, name: held})
            with torch.autograd.forward_ad.dual_level():
                dual = torch.autograd.forward_ad.make_dual(t.detach().clone(), torch.ones_like(t))
                with pytest.raises(RuntimeError, match="no forward derivative"):
                    fn(**{**good, name: dual})


def test_append_into_caches_of_any_layout_that_is_apart(gpu):
    """Slices of wider buffers, keys beside values, one page or one key head of any stride."""
    gen = torch.Generator().manual_seed(31)
    cos, sin = rope_table(20, 32, device=gpu)
    past = torch.tensor([3], dtype=torch.int32, device=gpu)
    one = torch.zeros(1, 1, dtype=torch.int32, device=gpu)
    for kv, pages in ((2, 3), (1, 3), (2, 1), (1, 1)):
        x = torch.randn(1, 2, kv, 32, generator=gen).to(gpu)
        wide = torch.zeros(pages, 2, kv, 16, 48, device=gpu)
        by_slot = torch.zeros(pages, 16, kv, 2, 32, device=gpu).permute(3, 0, 2, 1, 4)
        want = None
        for key, value in ((wide[:, 0, :, :, :32], wide[:, 1, :, :, 16:]), (by_slot[0], by_slot[1]),
                           (torch.zeros(pages, kv, 16, 32, device=gpu), torch.zeros(kv, 16, pages, 32, device=gpu).permute(2, 0, 1, 3))):
            rope_append(x, x, x, key, value, one, past, cos, sin)
            got = torch.stack((key, value))
            want = got if want is None else want
            assert torch.equal(got, want) and bool((got[:, 0, :, 3:5] != 0).any())


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")
def test_tensors_of_a_gpu_that_is_not_the_current_one(gpu):
    other = torch.device("cuda", 1)
    with torch.cuda.device(other):
        attend, append = _good(other)
        attend["lens"].fill_(9)
        attend["value_cache"].fill_(2.0)
        want, turned = paged_attention(**attend), rope_append(**append)
    with torch.cuda.device(gpu):
        assert torch.equal(paged_attention(**attend), want) and torch.equal(rope_append(**append), turned)
        assert torch.cuda.current_device() == gpu.index


def test_rows_that_share_one_page_table(gpu):
    """A table expanded over the rows: several continuations of one prompt, of lengths of their own."""
    gen = torch.Generator().manual_seed(32)
    key, value, table, _, _ = pool(gen, 1, [400], 2, 64, 16, torch.bfloat16)
    key, value, table = key.to(gpu), value.to(gpu), table.to(gpu)
    q = torch.randn(5, 4, 64, generator=gen).to(torch.bfloat16).to(gpu)
    lens = torch.tensor([400, 1, 0, 17, 399], dtype=torch.int32, device=gpu)
    want = paged_attention(q, key, value, table.repeat(5, 1), lens)
    assert torch.equal(paged_attention(q, key, value, table.expand(5, -1), lens), want)
    x = torch.randn(5, 1, 2, 64, generator=gen).to(torch.bfloat16).to(gpu)
    past = torch.tensor([0, 31, 16, 350, 128], dtype=torch.int32, device=gpu)
    cos, sin = rope_table(400, 64, device=gpu)
    caches = [[c.clone() for c in (key, value)] for _ in range(2)]
    for (k, v), t in zip(caches, (table.repeat(5, 1), table.expand(5, -1))):
        rope_append(x, x, x, k, v, t, past, cos, sin)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(*caches))


def test_dimensions_of_one_may_have_any_stride(gpu):
    """One key head, one page or one column of a table, out of buffers whose other strides are odd."""
    gen = torch.Generator().manual_seed(33)
    key, value = (torch.randn(1, 1, 16, 32, generator=gen).to(gpu) for _ in range(2))
    x = torch.randn(3, 1, 2, 32, generator=gen).to(gpu)
    lens = torch.tensor([16, 3, 9], dtype=torch.int32, device=gpu)
    table = torch.zeros(3, 1, dtype=torch.int32, device=gpu)
    odd_key, odd_value = (torch.as_strided(c.clone(), (1, 1, 16, 32), (515, 513, 32, 1)) for c in (key, value))
    odd_table = torch.zeros(1, 3, dtype=torch.int32, device=gpu).t()
    assert odd_table.stride(1) == 3
    want = paged_attention(x[:, 0], key, value, table, lens)
    assert torch.equal(paged_attention(x[:, 0], odd_key, odd_value, odd_table, lens), want)
    cos, sin = rope_table(16, 32, device=gpu)
    past = torch.tensor([4, 5, 6], dtype=torch.int32, device=gpu)
    rope_append(x, x[:, :, :1], x[:, :, 1:], key, value, table, past, cos, sin)
    rope_append(x, x[:, :, :1], x[:, :, 1:], odd_key, odd_value, odd_table, past, cos, sin)
    assert torch.equal(odd_key, key) and torch.equal(odd_value, value)


def test_append_into_a_lazy_clone_leaves_the_original(gpu):
    _, good = _good(gpu)
    key, value = good["key_cache"], good["value_cache"]
    good["k"], good["v"] = torch.ones_like(good["k"]), torch.ones_like(good["v"])
    good["page_table"] = torch.tensor([[0], [1]], dtype=torch.int32, device=gpu)
    copies = torch._lazy_clone(key), torch._lazy_clone(value)
    rope_append(**{**good, "key_cache": copies[0], "value_cache": copies[1]})
    assert not key.any() and not value.any()
    assert bool(copies[0].any()) and bool(copies[1].any())

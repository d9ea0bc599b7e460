"""Adjusted logits against their 64-bit plain form: histories, biases, masks, layouts, refusals."""

from __future__ import annotations

import pytest
import torch

from oracle import decode as plain
from polylora_amd.logits import adjust_logits, pack_allowed

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def build(gen, rows, vocab, dtype, history=0, bias=0, grammar=False, token_dtype=torch.int64, pad=0):
    """CPU arguments of a call; the logits are the first columns of rows of vocab + pad."""
    a = {"logits": (torch.randn(rows, vocab + pad, generator=gen) * 4).to(dtype)[:, :vocab]}
    if history:
        ids = (torch.rand(rows, history, generator=gen) ** 2 * (vocab + 2)).long() - 1  # -1 and vocab among them
        lens = torch.randint(0, history + 1, (rows,), generator=gen)
        lens[0] = history
        prompt = (lens * torch.rand(rows, generator=gen)).long()
        a.update(tokens=ids.to(token_dtype), lens=lens.int(), prompt_lens=prompt.int())
        a.update({name: torch.rand(rows, generator=gen) + 0.5 for name in ("repetition", "presence", "frequency")})
    if bias:
        ids = torch.randint(-2, vocab + 2, (rows, bias), generator=gen)
        ids[:, bias // 2] = ids[:, 0]  # an id twice
        values = torch.randn(rows, bias, generator=gen)
        values[:, -1] = float("-inf")
        a.update(bias_ids=ids.int(), bias_values=values)
    if grammar:
        allowed = torch.rand(rows, vocab, generator=gen) < 0.4
        allowed[0] = False  # a row that nothing is allowed in
        a["allowed"] = pack_allowed(allowed)
    return a


def check(gpu, a, out_dtype=None, in_place=False):
    want, size = plain.adjust_logits(**a)
    up = {name: t.to(gpu) for name, t in a.items()}
    wide = a["logits"]._base if a["logits"]._base is not None else a["logits"]
    held = wide.to(gpu)
    up["logits"] = held[:, : a["logits"].shape[1]]
    dtype = torch.float32
    if in_place:
        dtype, up["out"] = a["logits"].dtype, up["logits"]
    elif out_dtype is not None:
        dtype, up["out"] = out_dtype, torch.full(a["logits"].shape, 7.0, dtype=out_dtype, device=gpu)
    got = adjust_logits(**up)
    assert got.dtype is dtype and got.shape == want.shape
    assert torch.equal(held[:, a["logits"].shape[1] :].cpu(), wide[:, a["logits"].shape[1] :])
    got = got.cpu().double()
    fine = want.isfinite()
    assert torch.equal(got[~fine], want[~fine]) and bool(got[fine].isfinite().all())
    # at most eight fp32 operations (and one for each bias) on magnitudes that add up to `size`, and the output's rounding
    count = 8 + (a["bias_ids"].shape[-1] if "bias_ids" in a else 0)
    tol = UNIT[dtype] * want.abs() + count * 2.0**-24 * size + 1e-30
    err = (got - want).abs()
    assert bool((err[fine] <= tol[fine]).all()), float((err - tol)[fine].max())
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,history,bias,grammar,pad", [
    (1, 1, 3, 2, True, 0), (2, 31, 40, 0, True, 0), (3, 1000, 0, 0, False, 8), (3, 1003, 77, 5, True, 0),
    (2, 4096, 300, 0, False, 0), (2, 4097, 300, 9, True, 3), (5, 9001, 1000, 40, True, 1), (1, 20000, 5, 300, False, 0),
    (2, 33000, 0, 1, True, 0), (17, 257, 700, 3, False, 0),
])
def test_matches_the_plain_form(gpu, dtype, rows, vocab, history, bias, grammar, pad):
    gen = torch.Generator().manual_seed(vocab + rows)
    a = build(gen, rows, vocab, dtype, history, bias, grammar, pad=pad)
    wide = check(gpu, a)
    if dtype != torch.float32:
        check(gpu, a, out_dtype=dtype)
    assert torch.equal(check(gpu, a), wide)


def test_the_longest_lists(gpu):
    """A history beyond one look of a workgroup and a bias list at its limit, most of it in one slice."""
    gen = torch.Generator().manual_seed(6)
    a = build(gen, 2, 20000, torch.bfloat16, 9000, 2047, True)
    a["bias_ids"][1] = a["bias_ids"][1] % 600
    check(gpu, a)


@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place_rows_of_any_stride(gpu, dtype):
    gen = torch.Generator().manual_seed(1)
    check(gpu, build(gen, 3, 5001, dtype, 90, 4, True, pad=7), in_place=True)


@pytest.mark.parametrize("missing", ["prompt_lens", "repetition", "presence", "frequency"])
def test_each_penalty_may_be_missing(gpu, missing):
    a = build(torch.Generator().manual_seed(2), 3, 700, torch.float32, 200)
    del a[missing]
    check(gpu, a)


def test_histories_of_32_bits_and_lists_shared_by_rows(gpu):
    gen = torch.Generator().manual_seed(3)
    a = build(gen, 4, 900, torch.bfloat16, 50, 6, True, token_dtype=torch.int32)
    check(gpu, a)
    for name in ("tokens", "bias_ids", "bias_values", "allowed"):
        a[name] = a[name][1].contiguous()
    check(gpu, a)


def test_a_token_repeated_past_16_bits(gpu):
    """Counts are exact: 70000 times the same token."""
    a = {"logits": torch.zeros(1, 40), "tokens": torch.full((1, 70000), 5), "lens": torch.tensor([70000], dtype=torch.int32),
         "frequency": torch.tensor([1.0])}
    assert float(check(gpu, a)[0, 5]) == -70000.0


def test_lengths_beyond_the_history_and_below_zero(gpu):
    a = {"logits": torch.ones(2, 64), "tokens": torch.arange(10).expand(2, 10).contiguous(),
         "lens": torch.tensor([99, -4], dtype=torch.int32), "presence": torch.ones(2)}
    got = check(gpu, a)
    assert float(got[0, :10].sum()) == 0 and float(got[1].sum()) == 64


def test_infinities_and_nan(gpu):
    """Banned and overflowed logits keep their meaning; what the mask forbids is -inf whatever was there."""
    x = torch.tensor([[float("-inf"), float("inf"), float("nan"), torch.finfo(torch.float32).min, 1.0, float("nan")]])
    a = dict(tokens=torch.tensor([[0, 1, 3, 4]], device=gpu), lens=torch.tensor([4], dtype=torch.int32, device=gpu),
             repetition=torch.tensor([2.0], device=gpu), presence=torch.tensor([1.0], device=gpu),
             allowed=pack_allowed(torch.tensor([[True, True, True, True, True, False]])).to(gpu))
    got = adjust_logits(x.to(gpu), **a).cpu()[0]
    assert got[0] == float("-inf") and got[1] == float("inf") and got[2].isnan()
    assert got[3] == float("-inf")  # the lowest value times 2 is past it
    assert got[4] == -0.5 and got[5] == float("-inf")


def test_no_rows_and_no_history(gpu):
    assert adjust_logits(torch.zeros(0, 50, device=gpu)).shape == (0, 50)
    x = torch.randn(2, 50, device=gpu)
    none = torch.zeros(2, 0, dtype=torch.int64, device=gpu)
    assert torch.equal(adjust_logits(x, tokens=none, lens=torch.ones(2, dtype=torch.int32, device=gpu)), x)


def test_on_another_stream_and_in_a_graph(gpu):
    gen = torch.Generator().manual_seed(4)
    a = {name: t.to(gpu) for name, t in build(gen, 3, 6000, torch.bfloat16, 100, 5, True).items()}
    want = adjust_logits(**a)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert torch.equal(adjust_logits(**a), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = adjust_logits(**a)
    for i in range(3):
        a["logits"].copy_(torch.randn(3, 6000, generator=gen).to(torch.bfloat16))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, adjust_logits(**a))


def test_refusals(gpu):
    i32 = dict(dtype=torch.int32, device=gpu)
    good = {"logits": torch.zeros(2, 64, device=gpu), "tokens": torch.zeros(2, 3, dtype=torch.int64, device=gpu),
            "lens": torch.ones(2, **i32), "repetition": torch.ones(2, device=gpu), "bias_ids": torch.zeros(2, 2, **i32),
            "bias_values": torch.zeros(2, 2, device=gpu), "allowed": torch.zeros(2, 2, **i32)}
    adjust_logits(**good)
    x = good["logits"]
    bad = [
        ({"logits": x.cpu()}, RuntimeError),
        ({"logits": x[0]}, ValueError),
        ({"logits": x.double()}, TypeError),
        ({"logits": torch.zeros(64, 2, device=gpu).t()}, ValueError),
        ({"tokens": None}, ValueError),
        ({"tokens": None, "lens": None}, ValueError),
        ({"lens": None}, ValueError),
        ({"tokens": good["tokens"].float()}, TypeError),
        ({"tokens": good["tokens"][:1]}, ValueError),
        ({"tokens": good["tokens"].cpu()}, ValueError),
        ({"tokens": torch.zeros(2, 1 << 20, dtype=torch.int64, device=gpu)}, RuntimeError),
        ({"lens": good["lens"].long()}, TypeError),
        ({"prompt_lens": good["lens"][:1]}, ValueError),
        ({"repetition": torch.ones(1, device=gpu)}, ValueError),
        ({"presence": torch.ones(2, dtype=torch.float64, device=gpu)}, TypeError),
        ({"bias_ids": None}, ValueError),
        ({"bias_values": good["bias_values"][:, :1]}, ValueError),
        ({"bias_ids": good["bias_ids"].long()}, TypeError),
        ({"bias_ids": torch.zeros(2, 2048, **i32), "bias_values": torch.zeros(2, 2048, device=gpu)}, RuntimeError),
        ({"allowed": good["allowed"][:, :1]}, ValueError),
        ({"allowed": good["allowed"].long()}, TypeError),
        ({"out": torch.zeros(2, 64, dtype=torch.float16, device=gpu)}, TypeError),
        ({"out": torch.zeros(2, 63, device=gpu)}, ValueError),
        ({"out": torch.zeros(64, 2, device=gpu).t()}, ValueError),
    ]
    for change, error in bad:
        with pytest.raises(error):
            adjust_logits(**{**good, **change})
    wide = torch.zeros(2, 65, device=gpu)
    with pytest.raises(RuntimeError):  # over the logits, one element on
        adjust_logits(wide[:, :64], out=wide[:, 1:])


def test_tensors_that_want_derivatives_are_refused(gpu):
    """Any floating-point argument, not only the logits; under no_grad they are taken."""
    good = {name: t.to(gpu) for name, t in build(torch.Generator().manual_seed(8), 2, 40, torch.float32, 5, 3).items()}
    good["out"] = torch.empty_like(good["logits"])
    for name, t in good.items():
        if t.dtype != torch.float32:
            continue
        held = t.detach().clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no backward"):
            adjust_logits(**{**good, name: held})
        with torch.no_grad():
            adjust_logits(**{**good, name: held})
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(t.detach().clone(), torch.ones_like(t))
            with pytest.raises(RuntimeError, match="no forward derivative"):
                adjust_logits(**{**good, name: dual})


def test_lists_of_one_row_of_any_stride(gpu):
    """A single row's ids as a slice of a wider buffer beside dense values."""
    a = {name: t.to(gpu) for name, t in build(torch.Generator().manual_seed(9), 1, 300, torch.bfloat16, 20, 6, True).items()}
    want = adjust_logits(**a)
    for name in ("bias_ids", "tokens", "allowed"):
        wide = torch.zeros(1, a[name].shape[1] + 5, dtype=a[name].dtype, device=gpu)
        wide[:, : a[name].shape[1]] = a[name]
        assert torch.equal(adjust_logits(**{**a, name: wide[:, : a[name].shape[1]]}), want)
    assert torch.equal(adjust_logits(**{**a, "bias_values": a["bias_values"][0]}), want)  # one list, a row or not


def test_dimensions_of_one_may_have_any_stride(gpu):
    """A vocabulary of one, a history of one token, a list of one bias."""
    x = torch.tensor([[2.0, 3.0]], device=gpu).t()
    one = torch.zeros(1, 2, dtype=torch.int32, device=gpu).t()
    lens = torch.ones(2, dtype=torch.int32, device=gpu)
    assert x.stride(1) == one.stride(1) == 2
    got = adjust_logits(x, tokens=one, lens=lens, presence=torch.ones(2, device=gpu), bias_ids=one,
                        bias_values=torch.full((1, 2), 0.5, device=gpu).t())
    assert got.tolist() == [[1.5], [2.5]]

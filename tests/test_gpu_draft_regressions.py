"""Faults that a step over drafted tokens once had, each with the call that showed it or would have."""

from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from oracle import drafts as plain
from polylora_amd.drafts import tree_tables, verify_tokens
from polylora_amd.paged import keep_tokens, paged_attention, rope_append, rope_table, tree_attention

from .test_gpu_drafts import random_parents, seen_of
from .test_gpu_draft_steps import VOCAB, Server, Weights, plain_logits
from .test_gpu_paged import pool

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- verification


def drafted_on(gpu, seed, rows, m, vocab, dtype, tree):
    """A step's arguments, made on the GPU, other ones for each seed: (logits, tokens, uniforms, what else)."""
    gen = torch.Generator(device=gpu).manual_seed(seed)
    logits = (torch.randn(rows, m, vocab, generator=gen, device=gpu) * 4.5).to(dtype)
    tokens = torch.zeros(rows, m, dtype=torch.int64, device=gpu)
    heat = torch.tensor([(0.7, 1.0, 0.9, 0.0)[(b + seed) % 4] for b in range(rows)], device=gpu)
    more = {"temperature": heat, "seq_lens": torch.randint((m + 1) // 2, m + 1, (rows,), generator=gen, device=gpu).int()}
    if tree:
        parents = random_parents(torch.Generator().manual_seed(seed), rows, m)
        best = logits.float().topk(3, -1).indices
        nth = torch.randint(0, 3, (rows, m), generator=gen, device=gpu)
        up = parents.to(gpu).clamp(min=0).long()
        tokens = best.gather(1, up[..., None].expand(-1, -1, 3)).gather(2, nth[..., None])[..., 0]
        more["parents"] = parents.to(gpu)
    else:
        near = logits[:, :-1].float() + 0.5 * torch.randn(rows, m - 1, vocab, generator=gen, device=gpu)
        q = torch.softmax(near / torch.where(heat == 0, 1.0, heat)[:, None, None], -1)
        tokens[:, 1:] = (q / torch.empty_like(q).exponential_(generator=gen)).argmax(-1)
        more["draft_probs"] = q
    return logits, tokens, torch.rand(rows, m, generator=gen, device=gpu), more


@pytest.mark.parametrize("rows,m,vocab,dtype,tree", [
    (256, 6, 128256, torch.float32, False), (64, 6, 128256, torch.float32, False), (32, 32, 32003, torch.bfloat16, True),
    (100, 32, 32003, torch.bfloat16, True),
])
def test_verification_of_other_inputs_in_each_call(gpu, rows, m, vocab, dtype, tree):
    """What one call leaves in the workspace is not the next one's: sums of the call before, seen in place of this one's,
    are right where inputs repeat and move `next` where they do not."""
    for seed in range(4):
        *args, more = drafted_on(gpu, seed, rows, m, vocab, dtype, tree)
        got = verify_tokens(*args, **more)
        want = plain.verify_tokens(*args, **more)
        for name, a, b in zip(("path", "counts", "next"), got, want):
            assert torch.equal(a.cpu(), b), (seed, name, (a.cpu() != b).nonzero().tolist())


# ----------------------------------------------------------------------------- threads


def on_one_stream(calls, repeats=30):
    """What each call gives where each is a thread's and all threads launch on one stream, which has no scratch yet."""
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()

    def work(call):
        with torch.cuda.stream(stream):
            return [call() for _ in range(repeats)]

    with ThreadPoolExecutor(len(calls)) as threads:
        got = list(threads.map(work, calls))
    torch.cuda.synchronize()
    return got


def test_verification_from_threads_that_share_a_stream(gpu):
    """A call is several launches: those of another on the stream do not come between them."""
    calls, want = [], []
    for seed, (rows, m, vocab, tree) in enumerate([(3, 6, 40000, False), (7, 4, 9001, False), (5, 6, 20000, True)]):
        *args, more = drafted_on(gpu, seed, rows, m, vocab, torch.float32, tree)
        calls.append(lambda args=args, more=more: verify_tokens(*args, **more))
        want.append(plain.verify_tokens(*args, **more))
    for kept, w in zip(on_one_stream(calls), want):
        for got in kept:
            assert all(torch.equal(a.cpu(), b) for a, b in zip(got, w))


def test_attention_from_threads_that_share_a_stream(gpu):
    """Many columns and few rows are two launches; one thread has single tokens over the same pages."""
    gen = torch.Generator().manual_seed(1)
    key, value, table, _, _ = pool(gen, 2, [3000, 2500], 2, 64, 16, torch.bfloat16)
    key, value, table = key.nan_to_num(0.0).to(gpu), value.nan_to_num(0.0).to(gpu), table.to(gpu)
    past = torch.tensor([2900, 2400], dtype=torch.int32, device=gpu)
    calls = []
    for m in (40, 64, 9):  # 160 and 256 columns, and 36
        q = torch.randn(2, m, 8, 64, generator=gen).bfloat16().to(gpu)
        calls.append(lambda q=q: tree_attention(q, key, value, table, past))
    one = torch.randn(2, 8, 64, generator=gen).bfloat16().to(gpu)
    calls.append(lambda: paged_attention(one, key, value, table, past))
    want = [call() for call in calls]
    for kept, w in zip(on_one_stream(calls), want):
        assert all(torch.equal(got, w) for got in kept)


# ----------------------------------------------------------------------------- weights of a drafted token's attention


@pytest.mark.parametrize("dtype,fp8", [(torch.float32, False), (torch.bfloat16, False), (torch.float16, False),
                                       (torch.bfloat16, True), (torch.float16, True)])
@pytest.mark.parametrize("heads", [4, 40])  # 20 and 200 columns: both kernels
@pytest.mark.parametrize("dim", [64, 144])
def test_weights_are_held_in_32_bits(gpu, dtype, fp8, heads, dim):
    """Two values, 1 and -1, with weights 1 and exp(-d), d down to 2^-13: out is tanh(d / 2), a small difference.

    Weights are off by 2^-22 at most (of exp2's argument and result a unit each of fp32, half of one in their sum); two
    fp16 parts keep 2^-21 of one.  Half of that, over the sum of weights, which is nearly 2, and the output's own rounding."""
    d = torch.tensor([2.0**-e * f for e in (7, 9, 11, 12, 13) for f in (1.0, 1.25, 1.75)], dtype=torch.float64)
    rows, m = len(d), 5
    key = torch.zeros(rows, 1, 16, dim, dtype=dtype)
    value = torch.zeros(rows, 1, 16, dim, dtype=dtype)
    value[:, :, 0], value[:, :, 1] = 1.0, -1.0
    key[:, 0, 1, 3] = -1.0 if fp8 else -d.to(dtype)
    more = {}
    if fp8:
        key, value = (x.to(torch.float8_e4m3fn) for x in (key, value))
        more = {"k_scale": torch.ones(1, device=gpu), "v_scale": torch.ones(1, device=gpu)}
    q = torch.zeros(rows, m, heads, dim, dtype=dtype)
    q[..., 3] = d.to(dtype)[:, None, None] if fp8 else 1.0
    table = torch.arange(rows, dtype=torch.int32)[:, None]
    got = tree_attention(q.to(gpu), key.to(gpu), value.to(gpu), table.to(gpu),
                         torch.full((rows,), 2, dtype=torch.int32, device=gpu),
                         visible=torch.zeros(m, 1, dtype=torch.int32, device=gpu), scale=1.0, **more)
    want = torch.tanh(d / 2)[:, None, None, None].expand(got.shape)
    weight = 2.0**-22 + (2.0**-21 if dtype == torch.float16 else 0.0)
    tol = torch.finfo(dtype).eps / 2 * want + weight / 2
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


# ----------------------------------------------------------------------------- infinities and NaN that some tokens see


@pytest.mark.parametrize("dtype,fp8", [(torch.float32, False), (torch.bfloat16, False), (torch.float16, False),
                                       (torch.bfloat16, True), (torch.float16, True)])
@pytest.mark.parametrize("dim", [64, 80, 256])
@pytest.mark.parametrize("heads", [2, 40])  # 16 and 320 columns
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("window", [None, 40])
def test_infinities_and_nan_reach_the_tokens_that_see_them_and_no_others(gpu, dtype, fp8, dim, heads, tree, window):
    """Among the drafts, in the tile where they begin and where windows begin: each comes out, whatever its weight, at its
    element of the tokens that see its place; all else is what finite values in its place give, bit for bit."""
    gen = torch.Generator().manual_seed(dim + heads)
    rows, m, page = 2, 8, 16
    past = [133, 77]
    key, value, table, ks, vs = pool(gen, rows, [p + m for p in past], 1, dim, page, dtype, fp8)
    q = (torch.randn(rows, m, heads, dim, generator=gen) * (0.2 if fp8 else 1.0)).to(dtype)
    depths = seen = None
    more = {"k_scale": ks, "v_scale": vs, "visible": None, "depths": None}
    if tree:
        parents = random_parents(gen, rows, m)
        depths, visible = tree_tables(parents)
        seen = seen_of(visible, m)
        more.update(visible=visible, depths=depths)
    bits = value.view(torch.uint8) if fp8 else value
    inf = float("inf")
    kinds = [0x7F, 0xFF] if fp8 else [inf, -inf, float("nan")]
    hit = torch.zeros(rows, m, dim, 3, dtype=torch.bool)  # +inf, -inf and NaN that a token sees at an element
    clean = bits.clone()
    for b in range(rows):
        places = [past[b] + j for j in range(m)] + [past[b] - 1, past[b] - 6]
        if window:  # places where some windows begin and others do not reach
            places += [past[b] - window + j for j in range(m + 1)]
        for i, p in enumerate(places):
            at = plain.place(table, b, p, key.shape[0], page)
            # elements at both ends and in the middle, the same one for several places
            for d in (i % 3, dim // 2 + i, dim - 1 - i % 2):
                kind = (i + d) % len(kinds)
                bits[at[0], 0, at[1], d] = kinds[kind]
                clean[at[0], 0, at[1], d] = 0
                for t in range(m):
                    if p in plain.seen_places(past[b], m, t, m, None if seen is None else seen[b, t].tolist(),
                                              None if depths is None else int(depths[b, t]), window):
                        hit[b, t, d, 2 if fp8 else kind] = True
    some = hit.any(-1).sum(1)
    assert bool((some == m).any()) and bool(((some > 0) & (some < m)).any())  # seen by all, and by a part of the tokens
    args = (table.to(gpu), torch.tensor(past, dtype=torch.int32, device=gpu))
    more = {name: None if t is None else t.to(gpu) for name, t in more.items()}
    got = tree_attention(q.to(gpu), key.to(gpu), value.to(gpu), *args, window=window, **more).cpu()
    want = tree_attention(q.to(gpu), key.to(gpu), clean.view(value.dtype).to(gpu), *args, window=window, **more).cpu()
    assert not want.isnan().any() and not want.isinf().any()
    nan = hit[..., 2] | (hit[..., 0] & hit[..., 1])
    for name, where, x in (("nan", nan, float("nan")), ("+inf", hit[..., 0] & ~nan, inf), ("-inf", hit[..., 1] & ~nan, -inf)):
        want = torch.where(where[:, :, None], x, want)
    same = (got == want) | (got.isnan() & want.isnan())
    assert bool(same.all()), [(i, float(got[tuple(i)]), float(want[tuple(i)])) for i in (~same).nonzero().tolist()[:5]]


# ----------------------------------------------------------------------------- sizes


def test_verification_of_more_rows_than_their_pieces_would_fit_a_grid(gpu):
    """Tokens that are taken whole are as many workgroups, not as many as they have pieces."""
    gen = torch.Generator().manual_seed(2)
    rows, m, vocab = 4096, 33, 128256
    logits = (torch.randn(1, m, vocab, generator=gen) * 4.5).to(gpu).expand(rows, m, vocab)
    uniforms = torch.rand(rows, m, generator=gen)
    tokens = logits[0].argmax(-1).cpu().roll(1).expand(rows, m).clone()
    got = verify_tokens(logits, tokens.to(gpu), uniforms.to(gpu))
    some = torch.randperm(rows, generator=gen)[:24]
    want = plain.verify_tokens(logits[:24], tokens[some], uniforms[some])
    assert int(want[1].max()) > 1
    for a, b in zip(got, want):
        assert torch.equal(a.cpu()[some], b)


# ----------------------------------------------------------------------------- append


def test_append_by_depths_without_norms_takes_any_eps(gpu):
    gen = torch.Generator().manual_seed(3)
    key, value, table, _, _ = pool(gen, 2, [9, 20], 1, 32, 16, torch.float32)
    x = torch.randn(2, 4, 1, 32, generator=gen).to(gpu)
    past = torch.tensor([3, 14], dtype=torch.int32, device=gpu)
    depths = torch.tensor([0, 1, 1, 2], dtype=torch.int32, device=gpu)
    args = (x, x, x, key.to(gpu), value.to(gpu), table.to(gpu), past, *rope_table(32, 32, device=gpu))
    want = rope_append(*args, depths=depths)
    assert torch.equal(rope_append(*args, depths=depths, eps=0.0), want)
    with pytest.raises(RuntimeError, match="eps"):
        rope_append(*args, depths=depths, eps=0.0, k_norm=torch.ones(32, device=gpu))


# ----------------------------------------------------------------------------- whole steps of lines with probabilities


def test_steps_over_lines_with_probabilities(gpu):
    """Each pass's logits are those of the row's tokens alone, and what stays and follows is what the definition has."""
    gen = torch.Generator().manual_seed(4)
    w = Weights(gpu, torch.float32)
    rows = [torch.randint(0, VOCAB, (n,), generator=gen).tolist() for n in (3, 20, 35)]
    server = Server(gpu, w, rows, 128)
    heat = torch.tensor([0.0, 0.8, 1.1])
    kept = refused = 0
    for _ in range(10):
        m = int(torch.randint(2, 7, (), generator=gen))
        n = torch.randint(1, m + 1, (len(rows),), generator=gen).int()
        drafts, q = torch.zeros(len(rows), m - 1, dtype=torch.int64), torch.zeros(len(rows), m - 1, VOCAB)
        want = [[] for _ in rows]
        for b, tokens in enumerate(rows):
            for t in range(m):
                behind = plain_logits(w, tokens + drafts[b, :t].tolist()).cpu()
                want[b].append(behind)
                if t < m - 1:
                    near = behind.float() + 1.5 * torch.randn(VOCAB, generator=gen)
                    q[b, t] = torch.softmax(near / float(heat[b] or 1), -1)
                    drafts[b, t] = int(torch.multinomial(q[b, t], 1, generator=gen)) if heat[b] else int(near.argmax())
        ids = torch.cat((torch.tensor([r[-1:] for r in rows]), drafts), 1)
        uniforms = torch.rand(len(rows), m, generator=gen)
        logits = server.forward(ids.to(gpu), n.to(gpu))
        for b in range(len(rows)):
            for t in range(int(n[b])):
                # fp32 sums of other orders, over logits of size 10 (the greedy steps' bound)
                assert float((logits[b, t].cpu().double() - want[b][t]).abs().max()) < 1e-4
        more = dict(draft_probs=q, temperature=heat, seq_lens=n)
        path, counts, following = verify_tokens(logits, ids.to(gpu), uniforms.to(gpu),
                                                **{k: v.to(gpu) for k, v in more.items()})
        for a, b in zip((path, counts, following), plain.verify_tokens(logits.cpu(), ids, uniforms, **more)):
            assert torch.equal(a.cpu(), b)
        keep_tokens(server.keys, server.values, server.table, server.lens, path, counts)
        server.lens += counts
        for b, c in enumerate(counts.tolist()):
            rows[b] += ids[b, 1:c].tolist() + [int(following[b])]
            kept, refused = kept + c - 1, refused + int(n[b]) - c
    assert kept > 5 and refused > 5


# ----------------------------------------------------------------------------- shared scratch


SHAPES = [(700, 4, 331, torch.bfloat16, True), (3, 5, 9001, torch.float32, False), (1100, 2, 66000, torch.bfloat16, False),
          (1, 1024, 50, torch.float32, True), (600, 4, 1500, torch.float16, False), (1, 1024, 50, torch.float32, False),
          (40, 30, 66000, torch.bfloat16, True), (5, 1, 4097, torch.float32, False)]


def test_verification_of_one_shape_after_another(gpu):
    """A stream's counters are as the next call wants them, whatever its sizes and the kernels that they choose, and an
    attention's in between."""
    key = torch.randn(40, 1, 16, 64, generator=torch.Generator().manual_seed(1)).to(gpu)
    table = torch.arange(40, dtype=torch.int32, device=gpu)[None]
    past = torch.tensor([600], dtype=torch.int32, device=gpu)
    q = torch.randn(1, 5, 8, 64, generator=torch.Generator().manual_seed(2)).to(gpu)
    with torch.cuda.stream(torch.cuda.Stream()):
        attended = tree_attention(q, key, key, table, past)
        for turn in range(2):
            for i, shape in enumerate(SHAPES[::-1] if turn else SHAPES):
                *args, more = drafted_on(gpu, 10 * turn + i, *shape)
                got = verify_tokens(*args, **more)
                want = plain.verify_tokens(*args, **more)
                for a, b in zip(got, want):
                    assert torch.equal(a.cpu(), b), (turn, shape)
                assert torch.equal(tree_attention(q, key, key, table, past), attended)


def test_verification_of_many_tokens_in_a_graph(gpu):
    """Replays with other inputs, eager calls of other sizes between them."""
    for shape in (SHAPES[0], SHAPES[2], SHAPES[4], SHAPES[6]):
        *args, more = drafted_on(gpu, 0, *shape)
        verify_tokens(*args, **more)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = verify_tokens(*args, **more)
        for seed in (1, 2, 3):
            *others, also = drafted_on(gpu, seed, *shape)
            for a, b in zip([*args, *more.values()], [*others, *also.values()]):
                a.copy_(b)
            graph.replay()
            *small, rest = drafted_on(gpu, seed, 3, 5, 9001, torch.float32, False)
            for got, want in ((out, plain.verify_tokens(*others, **also)),
                              (verify_tokens(*small, **rest), plain.verify_tokens(*small, **rest))):
                for a, b in zip(got, want):
                    assert torch.equal(a.cpu(), b), (seed, shape)

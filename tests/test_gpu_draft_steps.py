"""Whole steps over drafted tokens, all operators together, against a decode that keeps no cache and drafts nothing."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from oracle.drafts import head_norm
from polylora_amd.drafts import tree_tables, verify_tokens
from polylora_amd.logits import adjust_logits
from polylora_amd.paged import keep_tokens, rope_append, rope_table, tree_attention

pytestmark = pytest.mark.gpu

VOCAB, HIDDEN, HEADS, KV, DIM, LAYERS, PAGE = 211, 96, 6, 2, 32, 3, 16


class Weights:
    def __init__(self, gpu, dtype):
        gen = torch.Generator().manual_seed(11)

        def w(*shape, scale=1.0):
            return (torch.randn(*shape, generator=gen) * scale).to(gpu, dtype)

        self.embed, self.head = w(VOCAB, HIDDEN), w(HIDDEN, VOCAB, scale=0.5)
        self.layers = [dict(q=w(HIDDEN, HEADS * DIM, scale=0.1), k=w(HIDDEN, KV * DIM, scale=0.1),
                            v=w(HIDDEN, KV * DIM, scale=0.1), o=w(HEADS * DIM, HIDDEN, scale=0.07),
                            q_norm=w(DIM, scale=0.2) + 1, k_norm=w(DIM, scale=0.2) + 1,
                            up=w(HIDDEN, 2 * HIDDEN, scale=0.1), down=w(2 * HIDDEN, HIDDEN, scale=0.1))
                       for _ in range(LAYERS)]


def rms(x):
    return x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt()


def plain_logits(w, tokens):
    """Logits behind the last of a row's tokens, in 64 bits, every token by itself."""
    n = len(tokens)
    h = w.embed[torch.tensor(tokens, device=w.embed.device)].double()
    i = torch.arange(DIM // 2, dtype=torch.float64, device=h.device)
    angle = torch.arange(n, device=h.device, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * i / DIM)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turn(x):
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    for p in w.layers:
        x = rms(h)
        q, k, v = ((x @ p[m].double()).unflatten(-1, (-1, DIM)) for m in "qkv")
        q, k = turn(head_norm(q, p["q_norm"], 1e-6)), turn(head_norm(k, p["k_norm"], 1e-6))
        k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, v))
        s = (q.transpose(0, 1) @ k.permute(1, 2, 0).contiguous()) * DIM**-0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=h.device).triu(1), float("-inf"))
        out = (s.softmax(-1) @ v.transpose(0, 1).contiguous()).transpose(0, 1).flatten(1)
        h = h + out @ p["o"].double()
        h = h + F.silu(rms(h) @ p["up"].double()) @ p["down"].double()
    return rms(h[-1]) @ w.head.double()


class Server:
    """Rows of requests over paged caches; the pages of a row lie anywhere."""

    def __init__(self, gpu, w, prompts, room):
        self.w, self.gpu, rows = w, gpu, len(prompts)
        width = -(-room // PAGE)
        order = torch.randperm(rows * width + 3, generator=torch.Generator().manual_seed(5))
        self.table = order[: rows * width].view(rows, width).int().to(gpu)
        dtype = w.embed.dtype
        shape = (rows * width + 3, KV, PAGE, DIM)
        self.keys = [torch.full(shape, float("nan"), dtype=dtype, device=gpu) for _ in range(LAYERS)]
        self.values = [torch.full(shape, float("nan"), dtype=dtype, device=gpu) for _ in range(LAYERS)]
        self.lens = torch.zeros(rows, dtype=torch.int32, device=gpu)
        self.cos, self.sin = rope_table(room, DIM, device=gpu)
        self.last = torch.tensor([p[-1] for p in prompts], device=gpu)
        # the prompts up to their last token, right-padded, in one pass
        m = max(len(p) - 1 for p in prompts)
        ids = torch.tensor([p[:-1] + [0] * (m - len(p) + 1) for p in prompts], device=gpu)
        n = torch.tensor([len(p) - 1 for p in prompts], dtype=torch.int32, device=gpu)
        self.forward(ids, n)
        self.lens += n

    def forward(self, ids, n, parents=None):
        depths, visible = (None, None) if parents is None else tree_tables(parents)
        h = self.w.embed[ids]
        for i, p in enumerate(self.w.layers):
            x = rms(h)
            q, k, v = ((x @ p[m]).unflatten(-1, (-1, DIM)) for m in "qkv")
            q = rope_append(q, k, v, self.keys[i], self.values[i], self.table, self.lens, self.cos, self.sin, seq_lens=n,
                            q_norm=p["q_norm"], k_norm=p["k_norm"], depths=depths)
            out = tree_attention(q, self.keys[i], self.values[i], self.table, self.lens, seq_lens=n, visible=visible)
            h = h + out.flatten(2) @ p["o"]
            h = h + F.silu(rms(h) @ p["up"]) @ p["down"]
        return rms(h) @ self.w.head

    def step(self, drafts, parents, n, temperature, uniforms):
        """One pass over the last tokens and their drafts; the tokens that each row gains."""
        ids = torch.cat((self.last[:, None], drafts), 1)
        logits = self.forward(ids, n, parents)
        logits = adjust_logits(logits.flatten(0, 1)).view_as(logits)  # no rules: the same numbers
        path, counts, following = verify_tokens(logits, ids, uniforms, parents=parents, temperature=temperature,
                                                seq_lens=n)
        keep_tokens(self.keys, self.values, self.table, self.lens, path, counts)
        self.lens += counts
        self.last = following
        kept = ids.gather(1, path.clamp(min=0).long())
        return [kept[b, 1 : int(counts[b])].tolist() + [int(following[b])] for b in range(len(n))]


def drafts_of(gen, truth, m):
    """A tree behind a row's last token that holds some of what comes (truth) among what does not."""
    parents, tokens, on_way, depth = [-1], [0], [True], [0]
    for _ in range(m - 1):
        p = int(torch.randint(max(0, len(parents) - 3), len(parents), (), generator=gen))
        right = on_way[p] and depth[p] < len(truth) and not any(
            q == p and ok for q, ok in zip(parents[1:], on_way[1:])) and float(torch.rand((), generator=gen)) < 0.7
        parents.append(p)
        tokens.append(truth[depth[p]] if right else (truth[depth[p]] + 1 + int(torch.randint(
            0, VOCAB - 1, (), generator=gen))) % VOCAB if depth[p] < len(truth) else 0)
        on_way.append(right)
        depth.append(depth[p] + 1)
    return parents, tokens[1:]


def test_greedy_steps_give_what_single_tokens_give(gpu):
    gen = torch.Generator().manual_seed(1)
    w = Weights(gpu, torch.float32)
    prompts = [torch.randint(0, VOCAB, (n,), generator=gen).tolist() for n in (2, 40, 17, 90)]
    steps = 24
    truth = []
    for p in prompts:
        tokens = list(p)
        for _ in range(steps + 8):
            best = plain_logits(w, tokens).topk(2)
            # fp32 sums of other orders move logits of size 10 by less than this
            assert float(best.values[0] - best.values[1]) > 1e-4
            tokens.append(int(best.indices[0]))
        truth.append(tokens[len(p) :])
    server = Server(gpu, w, prompts, 160)
    got = [[] for _ in prompts]
    most = 0
    while min(len(g) for g in got) < steps:
        m = int(torch.randint(1, 13, (), generator=gen))
        rows = [drafts_of(gen, truth[b][len(got[b]) :], m) for b in range(len(prompts))]
        n = torch.randint(1, m + 1, (len(prompts),), generator=gen).int()
        done = [len(g) >= steps for g in got]
        n[torch.tensor(done)] = 0  # rows that have what they wanted rest
        last = server.last.clone()
        gained = server.step(torch.tensor([r[1] for r in rows], device=gpu).view(len(rows), m - 1),
                             torch.tensor([r[0] for r in rows], dtype=torch.int32, device=gpu), n.to(gpu),
                             torch.zeros(len(prompts), device=gpu), torch.zeros(len(prompts), m, device=gpu))
        for b, tokens in enumerate(gained):
            if done[b]:
                assert tokens == [-1]
                server.last[b] = last[b]
            else:
                got[b] += tokens
                most = max(most, len(tokens))
        assert all(g == t[: len(g)] for g, t in zip(got, truth)), (got, truth)
    assert most > 2  # drafts were kept and moved


def test_drawn_steps_do_not_depend_on_the_drafts(gpu):
    """A sure draft stays exactly where the row's own draw gives it: the same random numbers, the same tokens."""
    gen = torch.Generator().manual_seed(2)
    w = Weights(gpu, torch.float32)
    prompts = [torch.randint(0, VOCAB, (n,), generator=gen).tolist() for n in (5, 33)]
    heat = torch.tensor([0.8, 1.0], device=gpu)
    u = torch.rand(2, 12, generator=gen)
    server = Server(gpu, w, prompts, 64)
    want = [[], []]
    none = torch.zeros(2, 0, dtype=torch.int64, device=gpu)
    for i in range(12):
        root = torch.full((2, 1), -1, dtype=torch.int32, device=gpu)
        one = server.step(none, root, torch.ones(2, dtype=torch.int32, device=gpu), heat, u[:, i : i + 1].to(gpu))
        for b in range(2):
            want[b] += one[b]
    server, got = Server(gpu, w, prompts, 64), [[], []]
    while min(len(g) for g in got) < 12:
        at = [len(g) for g in got]
        m = 4
        # a line of what comes, its third draft wrong; the random numbers go by the tokens' places
        tokens = [[want[b][min(at[b] + j, 11)] if j != 2 else (want[b][min(at[b] + j, 11)] + 1) % VOCAB for j in range(3)]
                  for b in range(2)]
        n = torch.tensor([min(m, 12 - at[b]) for b in range(2)], dtype=torch.int32)
        us = torch.stack([F.pad(u[b, at[b] : at[b] + m], (0, m))[:m] for b in range(2)])
        line = torch.tensor([[-1, 0, 1, 2]] * 2, dtype=torch.int32, device=gpu)
        last = server.last.clone()
        gained = server.step(torch.tensor(tokens, device=gpu), line, n.to(gpu), heat, us.to(gpu))
        for b in range(2):
            if at[b] < 12:
                got[b] += gained[b]
            else:
                server.last[b] = last[b]
    assert got == want

"""A step of speculative decoding beside the Linears, as cases to time and compare.

A small model (or a table of n-grams) drafts a few tokens behind each row's newest one, the large model takes them all
in one pass, and the row keeps those that its probabilities agree with.  Four operators carry that pass over a paged
cache, for a batch in which every row is a request of its own:

* ``append``  paged.rope_append with the norms of queries and keys of each head in the same pass, and with the depth of
              a token in a tree of drafts in place of its number
* ``tree``    paged.tree_attention: the drafted tokens of each row over its pages and over their own ancestors
* ``verify``  drafts.verify_tokens: which drafts stay, and the token behind them, from given random numbers
* ``keep``    paged.keep_tokens: keys and values of the drafts that stay move up behind the row's tokens, in every layer

A case is a dict of plain values.  Lengths, trees, page orders and values all come from the seed: rows hold between an
eighth of ``context`` tokens and all of them (one row all of them, the first ``empty`` rows none), the pages of a row
lie anywhere in the pool, and the slots of a row's last page that hold no token hold NaN.
"""

from __future__ import annotations

import functools
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_FP8 = torch.float8_e4m3fn


def _append(name, dtype, rows, new, heads, kv_heads, dim, page, context, tree=False, rot=None, interleaved=False,
            fp8=False):
    return {"name": name, "op": "append", "dtype": dtype, "rows": rows, "new": new, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "context": context, "tree": tree,
            "rot": dim if rot is None else rot, "interleaved": interleaved, "fp8": fp8}


def _tree(name, dtype, rows, new, context, heads, kv_heads, dim, page, tree=True, window=0, empty=0, fp8=False):
    return {"name": name, "op": "tree", "dtype": dtype, "rows": rows, "new": new, "context": context, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "tree": tree, "window": window, "empty": empty, "fp8": fp8}


def _verify(name, dtype, rows, new, vocab, tree=False):
    return {"name": name, "op": "verify", "dtype": dtype, "rows": rows, "new": new, "vocab": vocab, "tree": tree}


def _keep(name, dtype, rows, new, layers, kv_heads, dim, page, context, fp8=False):
    return {"name": name, "op": "keep", "dtype": dtype, "rows": rows, "new": new, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "page": page, "context": context, "fp8": fp8}


def listed():
    return [
        # one request, its newest token and a tree of five drafts: latency alone
        _append("append_norm_1x6", "bf16", 1, 6, 32, 8, 128, 16, 700, tree=True),
        # the prompts of a full batch
        _append("append_norm_prompts_32x1024", "bf16", 32, 1024, 32, 8, 128, 64, 0),
        # one request early in its answer, five drafts in a line: latency alone
        _tree("tree_1x6_700", "bf16", 1, 6, 700, 32, 8, 128, 16, tree=False),
        # one layer of a serving step, seven drafts in a line for each of 64 requests
        _tree("tree_64x8_4096", "bf16", 64, 8, 4096, 32, 8, 128, 16, tree=False),
        # few requests, large trees of drafts: many queries to a key
        _tree("tree_16x64_8192", "bf16", 16, 64, 8192, 32, 8, 128, 16),
        # one request over a long document, 8-bit cache
        _tree("tree_1x16_131072_fp8", "bf16", 1, 16, 131072, 32, 8, 128, 64, fp8=True),
        # a small fp32 model with a key head for each query head and a window, some rows without a draft
        _tree("tree_fp32_9x13_1500", "fp32", 9, 13, 1500, 12, 12, 80, 32, window=500, empty=2),
        # one request, five drafts drawn from the drafting model's probabilities
        _verify("verify_1x6", "fp32", 1, 6, 128256),
        # a serving step of 256 requests
        _verify("verify_256x6", "fp32", 256, 6, 128256),
        # trees of a drafting model's likeliest tokens
        _verify("verify_tree_32x32", "bf16", 32, 32, 32003, tree=True),
        # every layer's cache of one request after that: latency alone
        _keep("keep_1x8", "bf16", 1, 8, 32, 8, 128, 16, 700),
        # and of a batch of trees
        _keep("keep_128x32", "bf16", 128, 32, 32, 8, 128, 16, 128),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case: lines and trees of drafts, caches of 8 to 32 bits, odd lengths and vocabularies."""
    kind = rng.choice(("append", "tree", "tree", "verify", "keep"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    heads, kv_heads = rng.choice(((32, 8), (16, 16), (12, 4), (64, 8), (28, 4), (8, 1), (40, 2), (9, 3)))
    dim = rng.choice((64, 80, 96, 128, 128, 256))
    page = rng.choice((16, 32, 64, 128))
    fp8 = dtype != "fp32" and rng.random() < 0.35
    es = 4 if dtype == "fp32" else 2
    tree = rng.random() < 0.5
    if kind == "append":
        rows = _spread(rng, 1, 256)
        new = rng.choice((1, _spread(rng, 2, 64), _spread(rng, 2, 1024)))
        most = 32768 * 48 * 128 * 2  # what the largest listed case reads
        if fp8:
            most //= 64  # an 8-bit cache comes back as the values that it stands for, a small one
        new = max(1, min(new, most // (rows * (heads + 2 * kv_heads) * dim * es)))
        c = _append("", dtype, rows, new, heads, kv_heads, dim, page, rng.choice((0, _spread(rng, 1, 2000))),
                    tree=tree and new <= 64, rot=rng.choice((dim, dim, dim // 2)), interleaved=rng.random() < 0.4,
                    fp8=fp8)
        c["context"] = min(c["context"], (3_000_000 if fp8 else 200_000_000) // (rows * kv_heads * dim))
    elif kind == "tree":
        rows, new = _spread(rng, 1, 64), _spread(rng, 1, 64)
        cs = 1 if fp8 else es
        # bytes of the caches and products, up to half of the largest listed cases', a quarter of the products in fp32
        most = min(260_000_000 // (rows * kv_heads * dim * 2 * cs),
                   (4 if dtype == "fp32" else 16) * 10**9 // (rows * new * heads * dim))
        context = min(_spread(rng, 16, 131072), max(16, most))
        window = rng.choice((0, 0, _spread(rng, 64, 4096)))
        c = _tree("", dtype, rows, new, context, heads, kv_heads, dim, page, tree=tree, window=window,
                  empty=0 if rows < 4 else rng.choice((0, 1, rows // 4)), fp8=fp8)
    elif kind == "verify":
        new = _spread(rng, 1, 32)
        vocab = _spread(rng, 1000, 128256)
        rows = max(1, min(_spread(rng, 1, 256), 190_000_000 // (vocab * new)))
        c = _verify("", dtype, rows, new, vocab, tree=tree)
    else:
        rows, new, layers = _spread(rng, 1, 128), _spread(rng, 2, 64), _spread(rng, 1, 48)
        c = _keep("", dtype, rows, new, layers, kv_heads, dim, page, rng.choice((0, _spread(rng, 1, 2000))), fp8=fp8)
        # at most what the largest listed case moves, of caches no larger than its
        c["layers"] = layers = max(1, min(layers, 32 * 8 * 128 * 2 * 128 // (rows * kv_heads * dim * es)))
        room = (100_000_000 if fp8 else 600_000_000 * 2 // es) // (layers * kv_heads * dim * 2)
        c["rows"] = max(1, min(rows, room // (c["context"] + new + page)))
        c["context"] = min(c["context"], max(0, room // c["rows"] - new - page))
    del c["name"]
    return c


# ----------------------------------------------------------------------------- inputs


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((seed * 1009 + salt) % (1 << 62))


def _lengths(case, seed):
    """(tokens that each row's cache holds before the call, new tokens of each row)."""
    rng = random.Random("%d:%d:%d" % (seed, case["rows"], case["context"]))
    top = case["context"]
    held = [rng.randint(top // 8, top) for _ in range(case["rows"])]
    held[-1] = top
    m = case["new"]
    new = [m if case["rows"] == 1 else rng.randint((m + 1) // 2, m) for _ in range(case["rows"])]
    for i in range(case.get("empty", 0)):
        held[i] = new[i] = 0
    return held, new


def _parents(case, seed):
    """Per row the parent of each token: a line, or a tree of up to four drafts to a token, a parent before its drafts."""
    rng = random.Random("%d:%d:tree" % (seed, case["rows"]))
    rows = []
    for _ in range(case["rows"]):
        if not case["tree"]:
            rows.append(list(range(-1, case["new"] - 1)))
            continue
        parents, children = [-1], [0]
        for _ in range(case["new"] - 1):
            # drafts mostly of the likeliest branch so far, so that trees are deep as well as wide
            p = max(rng.randrange(len(parents)) for _ in range(2))
            while children[p] >= 4:
                p = (p + 1) % len(parents)
            parents.append(p)
            children[p] += 1
            children.append(0)
        order = sorted(range(len(parents)), key=lambda i: (_depth(parents, i), i))
        rank = {old: i for i, old in enumerate(order)}
        rows.append([-1 if parents[i] < 0 else rank[parents[i]] for i in order])
    return rows


def _depth(parents, i):
    d = 0
    while parents[i] >= 0:
        i = parents[i]
        d += 1
    return d


def _depths(parents):
    out = []
    for row in parents:
        d = []
        for p in row:
            d.append(0 if p < 0 else d[p] + 1)
        out.append(d)
    return out


def _words(parents):
    """Per row and token the words of its mask: bit j % 32 of word j // 32 is set for itself and its ancestors j."""
    out = []
    for row in parents:
        masks = []
        for i, p in enumerate(row):
            masks.append((0 if p < 0 else masks[p]) | 1 << i)
        n = -(-len(row) // 32)
        words = [[m >> 32 * w & 0xFFFFFFFF for w in range(n)] for m in masks]
        out.append([[w - (1 << 32) if w >> 31 else w for w in line] for line in words])
    return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _scales(case, gen):
    """A scale for each key head of an 8-bit cache."""
    return torch.rand(case["kv_heads"], generator=gen, device="cuda") * 0.02 + 0.01


def _pool(case, seed, lens, dtype, layers=1):
    """([key and value cache of each layer], page table) that hold `lens` tokens of each row, NaN in the slots beyond."""
    page, gen = case["page"], _gen(seed, 2)
    counts = [-(-n // page) for n in lens]
    total = case["rows"] * -(-(case["context"] + case["new"]) // page) + 2  # room for every row at its longest
    order = list(range(total))
    random.Random(seed).shuffle(order)
    width, at, rows = max(1, max(counts)), 0, []
    for n in counts:
        rows.append(order[at : at + n] + [-1] * (width - n))
        at += n
    table = _i32(rows)
    last = [(r[n - 1], length - (n - 1) * page) for r, n, length in zip(rows, counts, lens) if n]
    caches = []
    for _ in range(2 * layers):
        x = torch.randn(total, case["kv_heads"], page, case["dim"], generator=gen, device="cuda")
        x = (x * 50).to(_FP8) if case["fp8"] else x.to(dtype)
        if last:
            ids, used = _i32([i for i, _ in last]).long(), _i32([n for _, n in last])
            stale = (torch.arange(page, device="cuda") >= used[:, None])[:, None, :, None]
            bits = x.view(torch.uint8) if case["fp8"] else x
            bits[ids] = bits[ids].masked_fill(stale, 127 if case["fp8"] else float("nan"))
        caches.append(x)
    return caches, table


def _prepare_append(case, seed):
    dtype, gen = _DTYPES[case["dtype"]], _gen(seed, 1)
    past, new = _lengths(case, seed)
    # caches as they are before the call: room for the new tokens, in pages that the rows own already
    (key, value), table = _pool(case, seed, [p + n for p, n in zip(past, new)], dtype)
    rows, m, dim = case["rows"], case["new"], case["dim"]
    # queries, keys and values as one projection gives them, side by side
    heads, kv = case["heads"], case["kv_heads"]
    qkv = (torch.randn(rows, m, heads + 2 * kv, dim, generator=gen, device="cuda") * 3).to(dtype)
    angle = torch.arange(case["context"] + m, device="cuda", dtype=torch.float64)[:, None]
    angle = angle * 500000.0 ** (-torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64) * 2 / case["rot"])
    s = {"op": "append", "q": qkv[:, :, :heads], "k": qkv[:, :, heads : heads + kv], "v": qkv[:, :, heads + kv :],
         "key": key, "value": value, "table": table, "past": _i32(past), "new": _i32(new),
         "cos": angle.cos().float(), "sin": angle.sin().float(), "interleaved": case["interleaved"], "eps": 1e-6}
    for name in ("q_norm", "k_norm"):
        s[name] = (torch.randn(dim, generator=gen, device="cuda") * 0.3 + 1).to(dtype)
    s["depths"] = _i32(_depths(_parents(case, seed))) if case["tree"] else None
    s["k_scale"], s["v_scale"] = (_scales(case, gen), _scales(case, gen)) if case["fp8"] else (None, None)
    return s


def _prepare_tree(case, seed):
    dtype, gen = _DTYPES[case["dtype"]], _gen(seed, 1)
    past, new = _lengths(case, seed)
    (key, value), table = _pool(case, seed, [p + n for p, n in zip(past, new)], dtype)
    q = torch.randn(case["rows"], case["new"], case["heads"], case["dim"], generator=gen, device="cuda") * 1.5
    s = {"op": "tree", "q": q.to(dtype), "key": key, "value": value, "table": table, "past": _i32(past),
         "new": _i32(new), "scale": case["dim"] ** -0.5, "window": case["window"], "visible": None, "depths": None}
    if case["tree"]:
        parents = _parents(case, seed)
        s["visible"], s["depths"] = _i32(_words(parents)), _i32(_depths(parents))
    s["k_scale"], s["v_scale"] = (_scales(case, gen), _scales(case, gen)) if case["fp8"] else (None, None)
    return s


def _prepare_verify(case, seed):
    dtype, gen = _DTYPES[case["dtype"]], _gen(seed, 1)
    rows, m, vocab = case["rows"], case["new"], case["vocab"]
    rng = random.Random(seed)
    new = [m if rows == 1 else rng.randint((m + 1) // 2, m) for _ in range(rows)]
    # greedy rows among them
    heat = [0.8 if rows == 1 else rng.choice((0.0, 0.7, 0.9, 1.0)) for _ in range(rows)]
    s = {"op": "verify", "new": _i32(new), "temperature": torch.tensor(heat, device="cuda"), "parents": None,
         "draft_probs": None}
    logits = torch.empty(rows, m, vocab, dtype=dtype, device="cuda")
    tokens = torch.zeros(rows, m, dtype=torch.int64, device="cuda")
    parents = _parents(case, seed) if case["tree"] else None
    if parents is not None:
        s["parents"] = _i32(parents)
    else:
        s["draft_probs"] = torch.empty(rows, m - 1, vocab, device="cuda")
    for b in range(rows):
        # a drafting model that thinks nearly as the large one does
        x = torch.randn(m, vocab, generator=gen, device="cuda") * (6 if case["tree"] else 4.5)
        logits[b] = (x + torch.randn(m, vocab, generator=gen, device="cuda") * 0.5).to(dtype)
        if case["tree"]:
            # the drafts of a token are its likeliest successors
            best = x.topk(4, -1).indices
            row = parents[b]
            nth, seen = [], {}
            for p in row:
                nth.append(seen.get(p, 0))
                seen[p] = nth[-1] + 1
            if m > 1:
                tokens[b, 1:] = best[_i32(row[1:]).long(), _i32(nth[1:]).long()]
        elif m > 1:
            p = torch.softmax(x[: m - 1] / (heat[b] or 1.0), -1)
            s["draft_probs"][b] = p
            noise = torch.empty_like(p).exponential_(generator=gen)
            tokens[b, 1:] = (p / noise).argmax(-1)
    s["logits"], s["tokens"] = logits, tokens
    s["uniforms"] = torch.rand(rows, m, generator=gen, device="cuda")
    return s


def _kept(case, seed, new):
    """(node numbers of the tokens that stay, ascending from the first one; how many) of each row.

    A node stays where it is or comes from beyond the places that are written, so that a pass may be run again."""
    rng = random.Random("%d:kept" % seed)
    paths, counts = [], []
    for n in new:
        k = min(n, rng.randint(1, 6))
        beyond = sorted(rng.sample(range(k, n), min(k - 1, n - k)))
        paths.append(list(range(k - len(beyond))) + beyond)
        counts.append(k)
    return [p + [-1] * (case["new"] - len(p)) for p in paths], counts


def _prepare_keep(case, seed):
    past, new = _lengths(case, seed)
    caches, table = _pool(case, seed, [p + n for p, n in zip(past, new)], _DTYPES[case["dtype"]], case["layers"])
    path, counts = _kept(case, seed, new)
    return {"op": "keep", "keys": caches[0::2], "values": caches[1::2], "table": table, "past": _i32(past),
            "path": _i32(path), "counts": _i32(counts), "fp8": case["fp8"]}


def prepare(case, seed):
    return {"append": _prepare_append, "tree": _prepare_tree, "verify": _prepare_verify,
            "keep": _prepare_keep}[case["op"]](case, seed)


# ----------------------------------------------------------------------------- plain forms


def _norm(x, weight, eps):
    return x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.float()


def _turn(x, cos, sin, interleaved):
    """x [..., heads, dim] rotated by cos, sin [..., 1, rot / 2]."""
    h = cos.shape[-1]
    a, b = (x[..., 0 : 2 * h : 2], x[..., 1 : 2 * h : 2]) if interleaved else (x[..., :h], x[..., h : 2 * h])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., 2 * h :]), -1)


def _store(cache, x, scale):
    """x [tokens, kv_heads, dim] in the cache's type, as bits that can be put in place."""
    if scale is None:
        return cache, x.to(cache.dtype)
    return cache.view(torch.uint8), (x / scale[:, None]).clamp(-448, 448).to(_FP8).view(torch.uint8)


def _append_plain(s):
    page, m = s["key"].shape[2], s["q"].shape[1]
    t = torch.arange(m, device="cuda")
    live = t < s["new"][:, None]
    slot = torch.where(live, s["past"][:, None] + t, 0)
    pos = slot if s["depths"] is None else torch.where(live, s["past"][:, None] + s["depths"], 0)
    cos, sin = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
    q = _turn(_norm(s["q"].float(), s["q_norm"], s["eps"]), cos, sin, s["interleaved"])
    q = torch.where(live[:, :, None, None], q, 0.0).to(s["q"].dtype)
    k = _turn(_norm(s["k"].float(), s["k_norm"], s["eps"]), cos, sin, s["interleaved"])
    at = (s["table"].long().gather(1, slot // page)[live], slice(None), (slot % page)[live])
    for cache, x, scale in ((s["key"], k, s["k_scale"]), (s["value"], s["v"].float(), s["v_scale"])):
        bits, x = _store(cache, x[live], scale)
        bits[at] = x
    return {"q": q, "key": s["key"], "value": s["value"]}


def _gathered(cache, table, scale):
    """[rows, kv_heads, positions, dim] of the rows' pages."""
    x = cache[table] if scale is None else cache.view(torch.uint8)[table].view(_FP8)
    x = x.float().transpose(1, 2).flatten(2, 3)
    return x if scale is None else x * scale[:, None, None]


def _tree_plain(s):
    q, table = s["q"], s["table"].clamp(min=0)
    rows, m, heads, dim = q.shape
    kv_heads, page = s["key"].shape[1:3]
    past = s["past"][:, None, None]
    t = torch.arange(m, device="cuda")
    i = t[:, None]  # the drafted token that looks
    j = torch.arange(table.shape[1] * page, device="cuda")  # the place that it looks at
    draft = j - past
    if s["visible"] is None:
        seen = draft <= i
    else:
        words = s["visible"].long().gather(2, (draft.clamp(0, m - 1) // 32).expand(rows, m, -1))
        seen = (draft < 0) | (words >> draft.clamp(0, m - 1) % 32 & 1 > 0)
    seen = seen & (draft < s["new"][:, None, None])
    if s["window"]:
        depth = i if s["depths"] is None else s["depths"][:, :, None]
        seen = seen & ((draft >= 0) & (s["visible"] is not None) | (j > past + depth - s["window"]))
    live = (seen & (i < s["new"][:, None, None])).transpose(1, 2)[:, None, :, None]  # [rows, 1, positions, 1, m]
    k = _gathered(s["key"], table, s["k_scale"])
    q = q.float().view(rows, m, kv_heads, -1, dim).permute(0, 2, 4, 3, 1).flatten(3).contiguous()
    w = (k @ q * s["scale"]).unflatten(3, (-1, m))  # [rows, kv_heads, positions, group, m]
    del k
    w = w.masked_fill_(~live, float("-inf"))
    w = w.sub_(w.amax(2, keepdim=True).clamp(min=-1e30)).exp_()
    w = w.div_(w.sum(2, keepdim=True).clamp(min=1e-30)).flatten(3)
    j = torch.arange(table.shape[1] * page, device="cuda")
    held = (j < (s["past"] + s["new"])[:, None])[:, None, :, None]
    v = _gathered(s["value"], table, s["v_scale"]).masked_fill_(~held, 0.0)
    out = w.transpose(2, 3).contiguous() @ v  # [rows, kv_heads, group * m, dim]
    return out.unflatten(2, (-1, m)).permute(0, 3, 1, 2, 4).reshape(rows, m, heads, dim).to(s["q"].dtype)


def _first_above(w, u):
    """The first place of each row of w whose running sum is above u times the sum."""
    upto = w.cumsum(-1)
    return (upto <= u[:, None] * upto[:, -1:]).sum(-1).clamp(max=w.shape[-1] - 1)


def _verify_plain(s):
    """In 64 bits: a random number next to a border decides a token."""
    logits, tokens, new = s["logits"], s["tokens"], s["new"].long()
    rows, m, vocab = logits.shape
    b = torch.arange(rows, device="cuda")
    at, done = torch.zeros_like(new), new == 0
    path = torch.full((rows, m), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = torch.where(done, -1, 0)
    counts = (~done).int()
    following = torch.full_like(new, -1)
    greedy = s["temperature"] == 0
    heat = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    for step in range(1, m + 1):
        x = logits[b, at].double()
        p = torch.softmax((x - x.amax(-1, keepdim=True)) / heat, -1)
        best = torch.where(x == x.amax(-1, keepdim=True), torch.arange(vocab, device="cuda"), vocab).amin(-1)
        if s["parents"] is not None:
            drawn = torch.where(greedy, best, _first_above(p, s["uniforms"][b, at].double()))
            n = torch.arange(m, device="cuda")
            fits = (s["parents"] == at[:, None]) & (tokens == drawn[:, None]) & (n < new[:, None]) & (n > 0)
            go, child = fits.any(-1), torch.where(fits, n, m - 1).amin(-1)
        else:
            child = at + 1
            last = child >= new
            token = tokens[b, child.clamp(max=m - 1)]
            q = p.new_zeros(rows, vocab)
            if m > 1:
                q = torch.where(last[:, None], 0.0, s["draft_probs"][b, at.clamp(max=m - 2)].double())
            u = s["uniforms"][b, at].double()
            go = u * q[b, token] < p[b, token]
            go = torch.where(greedy, token == best, go) & ~last
            left = (p - q).clamp(min=0)
            left = torch.where(left.sum(-1, keepdim=True) > 0, left, p)
            u = s["uniforms"][b, (new - 1).clamp(min=0)].double()
            drawn = torch.where(greedy, best, _first_above(left, u))
        following = torch.where(done | go, following, drawn)
        done = done | ~go
        at = torch.where(done, at, child)
        counts = counts + (~done).int()
        if step < m:
            path[:, step] = torch.where(done, -1, at)
    return {"path": path, "counts": counts, "next": following}


def _keep_plain(s):
    page, m = s["keys"][0].shape[2], s["path"].shape[1]
    t = torch.arange(m, device="cuda")
    live = (t < s["counts"][:, None]) & (s["path"] != t)
    source = (s["past"][:, None] + s["path"])[live].long()
    target = (s["past"][:, None] + t)[live].long()
    row = torch.arange(len(live), device="cuda")[:, None].expand_as(live)[live]
    table = s["table"].long()
    for x in s["keys"] + s["values"]:
        bits = x.view(torch.uint8) if s["fp8"] else x
        moved = bits[table[row, source // page], :, source % page]
        bits[table[row, target // page], :, target % page] = moved
    return s["keys"] + s["values"]


@functools.cache
def _entry_points():
    from polylora_amd.drafts import verify_tokens
    from polylora_amd.paged import keep_tokens, rope_append, tree_attention

    return rope_append, tree_attention, verify_tokens, keep_tokens


def run(s):
    if not own:
        return {"append": _append_plain, "tree": _tree_plain, "verify": _verify_plain, "keep": _keep_plain}[s["op"]](s)
    rope_append, tree_attention, verify_tokens, keep_tokens = _entry_points()
    if s["op"] == "append":
        q = rope_append(s["q"], s["k"], s["v"], s["key"], s["value"], s["table"], s["past"], s["cos"], s["sin"],
                        seq_lens=s["new"], interleaved=s["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                        q_norm=s["q_norm"], k_norm=s["k_norm"], eps=s["eps"], depths=s["depths"])
        return {"q": q, "key": s["key"], "value": s["value"]}
    if s["op"] == "tree":
        return tree_attention(s["q"], s["key"], s["value"], s["table"], s["past"], seq_lens=s["new"],
                              visible=s["visible"], depths=s["depths"], scale=s["scale"], window=s["window"] or None,
                              k_scale=s["k_scale"], v_scale=s["v_scale"])
    if s["op"] == "verify":
        path, counts, following = verify_tokens(s["logits"], s["tokens"], s["uniforms"], parents=s["parents"],
                                                draft_probs=s["draft_probs"], temperature=s["temperature"],
                                                seq_lens=s["new"])
        return {"path": path, "counts": counts, "next": following}
    keep_tokens(s["keys"], s["values"], s["table"], s["past"], s["path"], s["counts"])
    return s["keys"] + s["values"]


# ----------------------------------------------------------------------------- what a pass needs, and its answer


# The share of drafted steps that come out as accepted with the inputs above.
_AGREED_LINE, _AGREED_TREE = 0.745, 0.6


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    rows, m = case["rows"], case["new"]
    if case["op"] == "verify":
        # the logits of the tokens that are reached, and where a draft fell through the probabilities that it came from
        vocab, agreed = case["vocab"], _AGREED_TREE if case["tree"] else _AGREED_LINE
        lengths = (m,) if rows == 1 else range((m + 1) // 2, m + 1)
        reached = sum(agreed**i for n in lengths for i in range(n)) / len(lengths)
        fell = 0 if case["tree"] else sum(1 - agreed ** (n - 1) for n in lengths) / len(lengths)
        nbytes = rows * vocab * (reached * es + fell * 4)
        return {"bytes": rows * m * 16 + nbytes, "flops": 4 * rows * vocab * reached}
    past, new = _lengths(case, 0)
    kv, dim, cs = case["kv_heads"], case["dim"], 1 if case["fp8"] else es
    if case["op"] == "keep":
        path, counts = _kept(case, 0, new)
        moved = sum(p != i for row, n in zip(path, counts) for i, p in enumerate(row[:n]))
        return {"bytes": 4 * moved * kv * dim * cs * case["layers"] + rows * m * 4, "flops": 0}
    heads = case["heads"]
    if case["op"] == "append":
        # live tokens read and written, dead ones' queries written, the table rows of the positions that occur
        t, all_t = sum(new), rows * m
        nbytes = t * dim * ((heads + 2 * kv) * es + 2 * kv * cs) + all_t * heads * dim * es
        nbytes += min(t, case["context"] + m) * case["rot"] * 4
        return {"bytes": nbytes, "flops": t * (heads + kv) * (3 * case["rot"] + 4 * dim)}
    w = case["window"]
    keys = [min(p, w) + n if w else p + n for p, n in zip(past, new)]
    nbytes = sum(keys) * kv * dim * 2 * cs + 2 * rows * m * heads * dim * es + 4 * (sum(keys) // case["page"])
    # a line's token sees those before it, a tree's about as many as its depth
    pairs = sum((k - n) * n + (n * 5 if case["tree"] else n * (n + 1) // 2) for k, n in zip(keys, new))
    return {"bytes": nbytes, "flops": 4 * pairs * heads * dim}


def _spun(x, cos, sin, interleaved):
    """The rotation as a product of complex numbers: x [heads, tokens, dim], cos and sin [tokens, rot / 2]."""
    h = cos.shape[1]
    re, im = (x[..., 0 : 2 * h : 2], x[..., 1 : 2 * h : 2]) if interleaved else (x[..., :h], x[..., h : 2 * h])
    z = torch.complex(re.contiguous(), im.contiguous()) * torch.complex(cos, sin)
    z = torch.stack((z.real, z.imag), -1).flatten(2) if interleaved else torch.cat((z.real, z.imag), 2)
    return torch.cat((z, x[..., 2 * h :]), 2)


def _append_exact(case, seed):
    s = _prepare_append(case, seed)
    page, cos, sin = case["page"], s["cos"].double(), s["sin"].double()
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    key, value = s["key"].double(), s["value"].double()
    past, new = _lengths(case, seed)
    for b, (p, n) in enumerate(zip(past, new)):
        if not n:
            continue
        length = math.sqrt(case["dim"])
        both = []
        for x, w in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
            x = x[b, :n].double()
            x = x / torch.hypot(torch.linalg.vector_norm(x, dim=-1, keepdim=True) / length,
                                torch.tensor(math.sqrt(s["eps"]), dtype=torch.float64, device="cuda"))
            both.append(x * w.double())
        both = torch.cat(both, 1).transpose(0, 1)  # [heads + kv_heads, n, dim]
        where = torch.arange(n, device="cuda") if s["depths"] is None else s["depths"][b, :n].long()
        turned = _spun(both, cos[p + where], sin[p + where], case["interleaved"]).transpose(0, 1)
        q[b, :n] = turned[:, : case["heads"]]
        k, v = turned[:, case["heads"] :], s["v"][b, :n].double()
        if case["fp8"]:
            k, v = (x / y.double()[:, None] for x, y in ((k, s["k_scale"]), (v, s["v_scale"])))
            k, v = k.clamp(-448, 448), v.clamp(-448, 448)
        pos = torch.arange(p, p + n, device="cuda")
        ids = s["table"][b].long()[pos // page]
        key[ids, :, pos % page], value[ids, :, pos % page] = k, v
    return {"q": q, "key": key, "value": value}


def _tree_exact(case, seed):
    s = _prepare_tree(case, seed)
    past, new = _lengths(case, seed)
    if sum((p + n) * n for p, n in zip(past, new)) * case["heads"] * case["dim"] > 2e11:
        return None
    parents, window = _parents(case, seed), case["window"]
    depths = _depths(parents)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (p, n) in enumerate(zip(past, new)):
        if not n:
            continue
        ids = s["table"][b, : -(-(p + n) // case["page"])].long()
        k, v = (c.view(torch.uint8)[ids].view(_FP8).double() if case["fp8"] else c[ids].double()
                for c in (s["key"], s["value"]))
        k, v = (x.transpose(0, 1).flatten(1, 2)[:, : p + n].contiguous() for x in (k, v))  # [kv_heads, places, dim]
        if case["fp8"]:
            k, v = k * s["k_scale"].double()[:, None, None], v * s["v_scale"].double()[:, None, None]
        for i in range(n):
            a, line = i, []
            while a >= 0:
                line.append(p + a)
                a = parents[b][a]
            first = max(0, p + depths[b][i] - window + 1) if window else 0
            rest = [j for j in line if case["tree"] or j >= first]
            picked = torch.tensor(rest[::-1], device="cuda")
            q = s["q"][b, i].double().view(case["kv_heads"], -1, case["dim"])
            low = torch.matmul(q, k[:, min(first, p) : p].transpose(1, 2).contiguous())
            own_part = torch.matmul(q, k[:, picked].transpose(1, 2).contiguous())
            w = torch.softmax(torch.cat((low, own_part), -1) * s["scale"], -1)
            split = low.shape[-1]
            o = torch.matmul(w[..., :split].contiguous(), v[:, min(first, p) : p].contiguous())
            out[b, i] = (o + torch.matmul(w[..., split:].contiguous(), v[:, picked])).flatten(0, 1)
    return out


def _verify_exact(case, seed):
    s = _prepare_verify(case, seed)
    rows, m, vocab = case["rows"], case["new"], case["vocab"]
    tokens, new, u = s["tokens"].tolist(), s["new"].tolist(), s["uniforms"].double().tolist()
    heat = s["temperature"].double().tolist()
    parents = s["parents"].tolist() if case["tree"] else None
    paths, following = [], []

    def draw_from(w, number):
        upto = torch.cumsum(w, 0)
        return min(int(torch.searchsorted(upto, upto[-1] * number, right=True)), vocab - 1)

    for b in range(rows):
        node, path, token = 0, [0] if new[b] else [], -1
        while new[b]:
            x = s["logits"][b, node].double()
            best = int((x == x.max()).nonzero()[0])
            e = torch.exp((x - x.max()) / (heat[b] or 1.0))
            p = e / e.sum()
            if case["tree"]:
                token = best if heat[b] == 0 else draw_from(p, u[b][node])
                follow = [c for c in range(1, new[b]) if parents[b][c] == node and tokens[b][c] == token]
            elif node + 1 == new[b]:
                token, follow = best if heat[b] == 0 else draw_from(p, u[b][new[b] - 1]), []
            else:
                q, t = s["draft_probs"][b, node].double(), tokens[b][node + 1]
                if heat[b] == 0:
                    follow, token = [node + 1] if t == best else [], best
                elif u[b][node] * float(q[t]) < float(p[t]):
                    follow = [node + 1]
                else:
                    follow, token = [], draw_from(torch.relu(p - q), u[b][new[b] - 1])
            if not follow:
                break
            node = follow[0]
            path.append(node)
        paths.append(path + [-1] * (m - len(path)))
        following.append(token)
    return {"path": _i32(paths), "counts": _i32([sum(n >= 0 for n in p) for p in paths]),
            "next": torch.tensor(following, device="cuda")}


def _keep_exact(case, seed):
    s = _prepare_keep(case, seed)
    page = case["page"]
    past, path, counts, table = (s[k].tolist() for k in ("past", "path", "counts", "table"))
    moves = []
    for p, line, n, pages in zip(past, path, counts, table):
        for t, node in enumerate(line[:n]):
            a, b = p + node, p + t
            if a != b:
                moves.append((pages[b // page], b % page, pages[a // page], a % page))
    to_page, to_slot, from_page, from_slot = (torch.tensor(x, dtype=torch.int64, device="cuda")
                                              for x in (zip(*moves) if moves else [[]] * 4))
    out = []
    for x in s["keys"] + s["values"]:
        y = x.clone()
        bits = (x.view(torch.uint8), y.view(torch.uint8)) if case["fp8"] else (x, y)
        bits[1][to_page, :, to_slot] = bits[0][from_page, :, from_slot]
        out.append(y)
    return out


def exact(case, seed):
    return {"append": _append_exact, "tree": _tree_exact, "verify": _verify_exact,
            "keep": _keep_exact}[case["op"]](case, seed)

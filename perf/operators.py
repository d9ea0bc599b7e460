"""A decode step's work beside the Linears, as cases to time and compare.

Three operators serve a batch in which every row is a request of its own:

* ``append``  paged.rope_append: rotates the new tokens' queries and keys by position and appends keys and values to
              the rows' pages of a paged cache
* ``attend``  paged.paged_attention: the new token of each row over the row's pages
* ``logits``  logits.adjust_logits: penalties of repeated tokens, biases and grammar masks on each row's logits

A case is a dict of plain values.  Lengths, page orders, histories and values all come from the seed: rows hold
between an eighth of ``context`` tokens and all of them (one row all of them, the first ``empty`` rows none), the pages
of a row lie anywhere in the pool, and the slots of a row's last page that hold no token hold NaN.
"""

from __future__ import annotations

import functools
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_FP8 = torch.float8_e4m3fn


def _append(name, dtype, rows, new, heads, kv_heads, dim, page, context, rot=None, interleaved=False, fp8=False):
    return {"name": name, "op": "append", "dtype": dtype, "rows": rows, "new": new, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "context": context, "rot": dim if rot is None else rot,
            "interleaved": interleaved, "fp8": fp8}


def _attend(name, dtype, rows, context, heads, kv_heads, dim, page, window=0, empty=0, fp8=False):
    return {"name": name, "op": "attend", "dtype": dtype, "rows": rows, "context": context, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "empty": empty, "fp8": fp8}


def _logits(name, dtype, rows, vocab, history, grammar, bias):
    return {"name": name, "op": "logits", "dtype": dtype, "rows": rows, "vocab": vocab, "history": history,
            "grammar": grammar, "bias": bias}


def listed():
    return [
        # one request being decoded: latency alone
        _append("append_1_row", "bf16", 1, 1, 32, 8, 128, 16, 700),
        # one layer of a serving step of 256 requests
        _append("append_256_rows", "bf16", 256, 1, 32, 8, 128, 16, 1024),
        # the prompts of a full batch
        _append("append_prompts_32x1024", "bf16", 32, 1024, 32, 8, 128, 64, 0),
        # pieces of prompts into an 8-bit cache, part of each head rotated, in pairs
        _append("append_fp8_24x77", "fp16", 24, 77, 12, 4, 96, 32, 500, rot=64, interleaved=True, fp8=True),
        # one request early in its answer: latency alone
        _attend("attend_1_row_300", "bf16", 1, 300, 32, 8, 128, 16),
        # one layer of a serving step of 256 requests
        _attend("attend_256_rows_1024", "bf16", 256, 1024, 32, 8, 128, 16),
        # one request over a long document: all of the work is along one axis
        _attend("attend_1_row_131072", "bf16", 1, 131072, 32, 8, 128, 16),
        # long conversations over an 8-bit cache
        _attend("attend_64_rows_8192_fp8", "bf16", 64, 8192, 32, 8, 128, 64, fp8=True),
        # a small fp32 model with a key head for each query head and a window, some rows without a token
        _attend("attend_fp32_37_rows", "fp32", 37, 1500, 12, 12, 80, 32, window=500, empty=3),
        # one request, its penalties and a few banned tokens
        _logits("logits_1_row", "bf16", 1, 128256, 1500, False, 16),
        # a serving step of 256 requests, half of them held to a grammar
        _logits("logits_256_rows", "bf16", 256, 128256, 2000, True, 16),
        # a vocabulary that is no whole number of anything, long bias lists
        _logits("logits_fp32_40x32003", "fp32", 40, 32003, 600, False, 300),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case: single tokens and prompts, caches of 8 to 32 bits, odd lengths and vocabularies."""
    kind = rng.choice(("append", "attend", "attend", "logits"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    heads, kv_heads = rng.choice(((32, 8), (16, 16), (12, 4), (64, 8), (28, 4), (8, 1), (40, 2), (9, 3)))
    dim = rng.choice((64, 80, 96, 128, 128, 256))
    page = rng.choice((16, 32, 64, 128))
    fp8 = dtype != "fp32" and rng.random() < 0.35
    es = 4 if dtype == "fp32" else 2
    if kind == "append":
        rows = _spread(rng, 1, 256)
        new = rng.choice((1, _spread(rng, 2, 1024)))
        most = 32768 * 48 * 128 * 2  # what the largest listed case reads
        if fp8:
            most //= 64  # an 8-bit cache comes back as the values that it stands for, a small one
        new = max(1, min(new, most // (rows * (heads + 2 * kv_heads) * dim * es)))
        c = _append("", dtype, rows, new, heads, kv_heads, dim, page, rng.choice((0, _spread(rng, 1, 2000))),
                    rot=rng.choice((dim, dim, dim // 2)), interleaved=rng.random() < 0.4, fp8=fp8)
        c["context"] = min(c["context"], (3_000_000 if fp8 else 200_000_000) // (rows * kv_heads * dim))
    elif kind == "attend":
        rows = _spread(rng, 1, 256)
        most = 590_000_000 // (rows * kv_heads * dim * 2 * (1 if fp8 else es))
        context = min(_spread(rng, 16, 131072), max(16, most))
        window = rng.choice((0, 0, _spread(rng, 1, 4096)))
        c = _attend("", dtype, rows, context, heads, kv_heads, dim, page, window=window,
                    empty=0 if rows < 4 else rng.choice((0, 1, rows // 4)), fp8=fp8)
    else:
        rows = _spread(rng, 1, 256)
        vocab = _spread(rng, 1000, 90000 if dtype == "fp32" else 128256)
        c = _logits("", dtype, rows, vocab, rng.choice((0, _spread(rng, 1, 4000), _spread(rng, 1, 4000))),
                    rng.random() < 0.5, rng.choice((0, 5, _spread(rng, 1, 300))))
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
    for i in range(case.get("empty", 0)):
        held[i] = 0
    m = case.get("new", 0)
    return held, [m if case["rows"] == 1 else rng.randint((m + 1) // 2, m) for _ in range(case["rows"])]


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _scales(case, gen):
    """A scale for each key head of an 8-bit cache."""
    return torch.rand(case["kv_heads"], generator=gen, device="cuda") * 0.02 + 0.01


def _pool(case, seed, lens, dtype):
    """(key cache, value cache, page table) that hold `lens` tokens of each row, NaN in the slots beyond them."""
    page, gen = case["page"], _gen(seed, 2)
    counts = [-(-n // page) for n in lens]
    total = case["rows"] * -(-(case["context"] + case.get("new", 0)) // page) + 2  # room for every row at its longest
    order = list(range(total))
    random.Random(seed).shuffle(order)
    width, at, rows = max(1, max(counts)), 0, []
    for n in counts:
        rows.append(order[at : at + n] + [-1] * (width - n))
        at += n
    table = _i32(rows)
    caches = []
    for salt in (0.02, 0.03):
        x = torch.randn(total, case["kv_heads"], page, case["dim"], generator=gen, device="cuda")
        x = (x * 50).to(_FP8) if case["fp8"] else x.to(dtype)
        caches.append(x)
    last = [(r[n - 1], length - (n - 1) * page) for r, n, length in zip(rows, counts, lens) if n]
    if last:
        ids, used = _i32([i for i, _ in last]).long(), _i32([n for _, n in last])
        stale = (torch.arange(page, device="cuda") >= used[:, None])[:, None, :, None]
        for x in caches:
            bits = x.view(torch.uint8) if case["fp8"] else x
            bits[ids] = bits[ids].masked_fill(stale, 127 if case["fp8"] else float("nan"))
    return caches[0], caches[1], table


def _prepare_append(case, seed):
    dtype, gen = _DTYPES[case["dtype"]], _gen(seed, 1)
    past, new = _lengths(case, seed)
    # caches as they are before the call: room for the new tokens, in pages that the rows own already
    key, value, table = _pool(case, seed, [p + n for p, n in zip(past, new)], dtype)
    rows, m, dim = case["rows"], case["new"], case["dim"]
    # queries, keys and values as one projection gives them, side by side
    heads, kv = case["heads"], case["kv_heads"]
    qkv = torch.randn(rows, m, heads + 2 * kv, dim, generator=gen, device="cuda").to(dtype)
    angle = torch.arange(case["context"] + m, device="cuda", dtype=torch.float64)[:, None]
    angle = angle * 500000.0 ** (-torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64) * 2 / case["rot"])
    s = {"op": "append", "q": qkv[:, :, :heads], "k": qkv[:, :, heads : heads + kv], "v": qkv[:, :, heads + kv :],
         "key": key, "value": value, "table": table, "past": _i32(past), "new": _i32(new),
         "cos": angle.cos().float(), "sin": angle.sin().float(), "interleaved": case["interleaved"]}
    s["k_scale"], s["v_scale"] = (_scales(case, gen), _scales(case, gen)) if case["fp8"] else (None, None)
    return s


def _prepare_attend(case, seed):
    dtype, gen = _DTYPES[case["dtype"]], _gen(seed, 1)
    lens, _ = _lengths(case, seed)
    key, value, table = _pool(case, seed, lens, dtype)
    q = torch.randn(case["rows"], case["heads"], case["dim"], generator=gen, device="cuda") * 1.5
    s = {"op": "attend", "q": q.to(dtype), "key": key, "value": value, "table": table, "lens": _i32(lens),
         "scale": case["dim"] ** -0.5, "window": case["window"]}
    s["k_scale"], s["v_scale"] = (_scales(case, gen), _scales(case, gen)) if case["fp8"] else (None, None)
    return s


def _prepare_logits(case, seed):
    dtype, gen = _DTYPES[case["dtype"]], _gen(seed, 1)
    rows, vocab, history = case["rows"], case["vocab"], case["history"]
    rng = random.Random(seed)
    s = {"op": "logits", "logits": (torch.randn(rows, vocab, generator=gen, device="cuda") * 3).to(dtype)}
    s.update(dict.fromkeys(("bias_ids", "bias_values", "allowed")))
    # frequent tokens repeat; rows are right-padded with whatever was there
    u = torch.rand(rows, history, generator=gen, device="cuda", dtype=torch.float64)
    s["tokens"] = (u**3 * vocab).long().clamp(max=vocab - 1)
    lens = [history if rows == 1 else rng.randint(0, history) for _ in range(rows)]
    s["lens"], s["prompt_lens"] = _i32(lens), _i32([rng.randint(0, n) for n in lens])
    s["repetition"] = torch.rand(rows, generator=gen, device="cuda") * 0.5 + 0.9
    s["presence"] = torch.rand(rows, generator=gen, device="cuda")
    s["frequency"] = torch.rand(rows, generator=gen, device="cuda") * 0.5
    if case["bias"]:
        n = case["bias"]
        start = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
        ids = (start + torch.arange(n, device="cuda") * (vocab // n)) % vocab
        s["bias_ids"] = ids.int()
        values = torch.randn(rows, n, generator=gen, device="cuda") * 2
        s["bias_values"] = values.masked_fill(values > 3.5, float("-inf"))
    if case["grammar"]:
        # a row is free, or held to one token of fifty, or to a token set that is empty
        share = torch.tensor([rng.choice((1.0, 1.0, 0.02, 0.02)) for _ in range(rows)], device="cuda")
        share[0] = 0.0 if rows > 4 else 0.02
        bits = torch.rand(rows, -(-vocab // 32) * 32, generator=gen, device="cuda") < share[:, None]
        place = torch.arange(32, device="cuda", dtype=torch.int64)
        words = (bits.view(rows, -1, 32).long() << place).sum(-1)
        s["allowed"] = torch.where(words >= 1 << 31, words - (1 << 32), words).int()
    return s


def prepare(case, seed):
    return {"append": _prepare_append, "attend": _prepare_attend, "logits": _prepare_logits}[case["op"]](case, seed)


# ----------------------------------------------------------------------------- plain forms


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
    pos = torch.where(live, s["past"][:, None] + t, 0)
    cos, sin = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
    q = _turn(s["q"].float(), cos, sin, s["interleaved"])
    q = torch.where(live[:, :, None, None], q, 0.0).to(s["q"].dtype)
    k = _turn(s["k"].float(), cos, sin, s["interleaved"])
    at = (s["table"].long().gather(1, pos // page)[live], slice(None), (pos % page)[live])
    for cache, x, scale in ((s["key"], k, s["k_scale"]), (s["value"], s["v"].float(), s["v_scale"])):
        bits, x = _store(cache, x[live], scale)
        bits[at] = x
    return {"q": q, "key": s["key"], "value": s["value"]}


def _gathered(cache, table, scale):
    """[rows, kv_heads, positions, dim] of the rows' pages."""
    x = cache[table] if scale is None else cache.view(torch.uint8)[table].view(_FP8)
    x = x.float().transpose(1, 2).flatten(2, 3)
    return x if scale is None else x * scale[:, None, None]


def _attend_plain(s):
    q, table = s["q"], s["table"].clamp(min=0)
    rows, heads, dim = q.shape
    kv_heads, page = s["key"].shape[1:3]
    j = torch.arange(table.shape[1] * page, device="cuda")
    live = j < s["lens"][:, None]
    if s["window"]:
        live &= j >= s["lens"][:, None] - s["window"]
    live = live[:, None, :, None]
    k = _gathered(s["key"], table, s["k_scale"])
    q = q.float().view(rows, kv_heads, -1, dim).transpose(2, 3).contiguous()
    w = (k @ q * s["scale"]).masked_fill(~live, float("-inf"))  # [rows, kv_heads, positions, group]
    del k
    w = (w - w.amax(2, keepdim=True).clamp(min=-1e30)).exp()
    w = w / w.sum(2, keepdim=True).clamp(min=1e-30)
    v = _gathered(s["value"], table, s["v_scale"]).masked_fill_(~live, 0.0)
    return (w.transpose(2, 3).contiguous() @ v).reshape(rows, heads, dim).to(s["q"].dtype)


def _logits_plain(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    i = torch.arange(s["tokens"].shape[1], device="cuda")
    live, prompt = i < s["lens"][:, None], i < s["prompt_lens"][:, None]
    zeros = torch.zeros(rows, vocab + 1, dtype=torch.int32, device="cuda")  # the last column takes what is not there
    one = torch.ones_like(s["tokens"], dtype=torch.int32)
    seen = zeros.scatter_add(1, torch.where(live, s["tokens"], vocab), one)[:, :vocab] > 0
    count = zeros.scatter_add(1, torch.where(live & ~prompt, s["tokens"], vocab), one)[:, :vocab]
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - (s["frequency"][:, None] * count + s["presence"][:, None] * (count > 0))
    if s["bias_ids"] is not None:
        x = x + torch.zeros_like(x).scatter_add(1, s["bias_ids"].long(), s["bias_values"])
    if s["allowed"] is not None:
        bits = s["allowed"][:, :, None] >> torch.arange(32, dtype=torch.int32, device="cuda") & 1
        x = x.masked_fill(bits.flatten(1)[:, :vocab] == 0, float("-inf"))
    return x


@functools.cache
def _entry_points():
    from polylora_amd.logits import adjust_logits
    from polylora_amd.paged import paged_attention, rope_append

    return rope_append, paged_attention, adjust_logits


def run(s):
    if not own:
        return {"append": _append_plain, "attend": _attend_plain, "logits": _logits_plain}[s["op"]](s)
    rope_append, paged_attention, adjust_logits = _entry_points()
    if s["op"] == "append":
        q = rope_append(s["q"], s["k"], s["v"], s["key"], s["value"], s["table"], s["past"], s["cos"], s["sin"],
                        seq_lens=s["new"], interleaved=s["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"q": q, "key": s["key"], "value": s["value"]}
    if s["op"] == "attend":
        return paged_attention(s["q"], s["key"], s["value"], s["table"], s["lens"], scale=s["scale"],
                               window=s["window"] or None, k_scale=s["k_scale"], v_scale=s["v_scale"])
    return adjust_logits(s["logits"], tokens=s["tokens"], lens=s["lens"], prompt_lens=s["prompt_lens"],
                         repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                         bias_ids=s["bias_ids"], bias_values=s["bias_values"], allowed=s["allowed"])


# ----------------------------------------------------------------------------- what a pass needs, and its answer


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "logits":
        # logits in and fp32 logits out; a bit for each where there are masks; ids of 8 bytes, of which rows hold half
        rows, vocab, history = case["rows"], case["vocab"], case["history"]
        held = rows * history * (1.0 if rows == 1 else 0.5)
        nbytes = rows * vocab * (es + 4) + held * 8 + rows * case["bias"] * 8 + rows * (vocab // 8) * case["grammar"]
        return {"bytes": nbytes, "flops": 2 * rows * vocab}
    past, new = _lengths(case, 0)
    heads, kv, dim, cs = case["heads"], case["kv_heads"], case["dim"], 1 if case["fp8"] else es
    if case["op"] == "append":
        # live tokens read and written, dead ones' queries written, the table rows of the positions that occur
        t, all_t = sum(new), case["rows"] * case["new"]
        nbytes = t * dim * ((heads + 2 * kv) * es + 2 * kv * cs) + all_t * heads * dim * es
        nbytes += min(t, case["context"] + case["new"]) * case["rot"] * 4
        return {"bytes": nbytes, "flops": 3 * t * (heads + kv) * case["rot"]}
    t = sum(min(n, case["window"] or n) for n in past)
    nbytes = t * kv * dim * 2 * cs + 2 * case["rows"] * heads * dim * es + 4 * (t // case["page"])
    return {"bytes": nbytes, "flops": 4 * t * heads * dim}


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
        both = torch.cat((s["q"][b, :n], s["k"][b, :n]), 1).double().transpose(0, 1)  # [heads + kv_heads, n, dim]
        turned = _spun(both, cos[p : p + n], sin[p : p + n], case["interleaved"]).transpose(0, 1)
        q[b, :n] = turned[:, : case["heads"]]
        k, v = turned[:, case["heads"] :], s["v"][b, :n].double()
        if case["fp8"]:
            k, v = (x / y.double()[:, None] for x, y in ((k, s["k_scale"]), (v, s["v_scale"])))
            k, v = k.clamp(-448, 448), v.clamp(-448, 448)
        pos = torch.arange(p, p + n, device="cuda")
        ids = s["table"][b].long()[pos // page]
        key[ids, :, pos % page], value[ids, :, pos % page] = k, v
    return {"q": q, "key": key, "value": value}


def _attend_exact(case, seed):
    s = _prepare_attend(case, seed)
    lens, _ = _lengths(case, seed)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if not n:
            continue
        first = max(0, n - case["window"]) if case["window"] else 0
        ids = s["table"][b, : -(-n // case["page"])].long()
        k, v = (c.view(torch.uint8)[ids].view(_FP8).double() if case["fp8"] else c[ids].double()
                for c in (s["key"], s["value"]))
        k, v = (x.transpose(0, 1).flatten(1, 2)[:, first:n] for x in (k, v))  # [kv_heads, positions, dim]
        if case["fp8"]:
            k, v = k * s["k_scale"].double()[:, None, None], v * s["v_scale"].double()[:, None, None]
        q = s["q"][b].double().view(case["kv_heads"], -1, case["dim"])
        p = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"], -1)
        out[b] = torch.matmul(p, v.contiguous()).flatten(0, 1)
    return out


def _logits_exact(case, seed):
    s = _prepare_logits(case, seed)
    x = s["logits"].double()
    vocab = case["vocab"]
    for b in range(case["rows"]):
        ids, n, p = s["tokens"][b], int(s["lens"][b]), int(s["prompt_lens"][b])
        r, f, w = (float(s[key][b]) for key in ("repetition", "frequency", "presence"))
        used = ids[:n].unique()
        y = x[b, used]
        x[b, used] = torch.where(y > 0, y / r, y * r)
        made, times = ids[p:n].unique(return_counts=True)
        x[b, made] -= f * times.double() + w
        if s["bias_ids"] is not None:
            x[b, s["bias_ids"][b].long()] += s["bias_values"][b].double()
        if s["allowed"] is not None:
            v = torch.arange(vocab, device="cuda")
            words = s["allowed"][b].long() & 0xFFFFFFFF
            x[b, (words[v // 32] >> v % 32) % 2 == 0] = float("-inf")
    return x


def exact(case, seed):
    return {"append": _append_exact, "attend": _attend_exact, "logits": _logits_exact}[case["op"]](case, seed)

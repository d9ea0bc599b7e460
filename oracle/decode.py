"""Plain 64-bit forms of a decode step's operators: append to a paged cache, attention over it, adjusted logits.

Test infrastructure, written from the operators' definitions; every loop is over rows, tokens or list entries.
"""

from __future__ import annotations

import torch

E4M3_MAX = 448.0


def place(table, row: int, position: int, num_pages: int, page_size: int):
    """(page, slot) of a row's token, or None where the table holds no page of the pool for it."""
    column = position // page_size
    if position < 0 or column >= table.shape[1]:
        return None
    page = int(table[row, column])
    return (page, position % page_size) if 0 <= page < num_pages else None


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x [heads, dim] (float64) turned by cos, sin [half] of its position."""
    half = cos.shape[0]
    y = x.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        y[:, a] = x[:, a] * cos[i] - x[:, b] * sin[i]
        y[:, b] = x[:, b] * cos[i] + x[:, a] * sin[i]
    return y


def rope_append(q, k, v, key, value, table, past, cos, sin, seq_lens=None, interleaved=False, k_scale=None,
                v_scale=None):
    """(q_out, k_out, key, value) in float64; the caches hold stored values (over the scale, saturated, unrounded) and
    keep what the call does not write."""
    rows, m, heads, dim = q.shape
    num_pages, _, page_size, _ = key.shape
    q_out = torch.zeros(q.shape, dtype=torch.float64)
    k_out = torch.zeros(k.shape, dtype=torch.float64)
    key, value = key.double().clone(), value.double().clone()
    cos, sin = cos.double(), sin.double()
    for b in range(rows):
        n = m if seq_lens is None else min(m, int(seq_lens[b]))
        for t in range(n):
            pos = int(past[b]) + t
            at = place(table, b, pos, num_pages, page_size)
            if at is None or pos >= cos.shape[0]:
                continue
            q_out[b, t] = rotate(q[b, t].double(), cos[pos], sin[pos], interleaved)
            k_out[b, t] = rotate(k[b, t].double(), cos[pos], sin[pos], interleaved)
            for cache, x, scale in ((key, k_out[b, t], k_scale), (value, v[b, t].double(), v_scale)):
                if scale is not None:
                    x = (x / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
                cache[at[0], :, at[1]] = x
    return q_out, k_out, key, value


def gather(key, value, table, lens, row: int, window=None, k_scale=None, v_scale=None):
    """(keys, values) [tokens, kv_heads, dim] in float64 that a row's new token attends to."""
    num_pages, kv_heads, page_size, dim = key.shape
    n = min(max(int(lens[row]), 0), table.shape[1] * page_size)
    places = [place(table, row, p, num_pages, page_size) for p in range(max(0, n - window) if window else 0, n)]
    places = [p for p in places if p is not None]
    if not places:
        empty = torch.zeros(0, kv_heads, dim, dtype=torch.float64)
        return empty, empty
    pages, slots = (torch.tensor(x) for x in zip(*places))
    out = []
    for cache, scale in ((key, k_scale), (value, v_scale)):
        bits = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache  # 8-bit floats take no lists
        x = bits[pages, :, slots].view(cache.dtype).double()
        out.append(x if scale is None else x * scale.double()[:, None])
    return out[0], out[1]


def paged_attention(q, key, value, table, lens, scale=None, window=None, k_scale=None, v_scale=None):
    """(out, spread, reach) in float64: the output, the same sum over |values| and the largest |q| . |k| * scale, the
    sizes that rounding errors are proportional to."""
    rows, heads, dim = q.shape
    group = heads // key.shape[1]
    scale = dim**-0.5 if scale is None else scale
    out, spread = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    reach = torch.zeros(rows, heads, 1, dtype=torch.float64)
    for b in range(rows):
        k, v = gather(key, value, table, lens, b, window, k_scale, v_scale)
        if not k.shape[0]:
            continue
        k, v = (x.repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))  # [heads, tokens, dim]
        x = q[b].double()[:, :, None]
        p = torch.softmax((k @ x)[:, :, 0] * scale, -1)[:, None]
        out[b], spread[b] = (p @ v)[:, 0], (p @ v.abs())[:, 0]
        reach[b] = (k.abs() @ x.abs()).amax(1) * abs(scale)
    return out, spread, reach


def adjust_logits(logits, tokens=None, lens=None, prompt_lens=None, repetition=None, presence=None, frequency=None,
                  bias_ids=None, bias_values=None, allowed=None):
    """(logits, size) in float64: the adjusted logits and the sum of the magnitudes that went into each."""
    x = logits.double().clone()
    size = x.abs()
    rows, vocab = x.shape

    def of(t, b, off):
        return off if t is None else float(t[b])

    for b in range(rows):
        seen, made = {}, {}
        if tokens is not None:
            for i in range(min(max(int(lens[b]), 0), tokens.shape[-1])):
                v = int(tokens[b, i] if tokens.dim() == 2 else tokens[i])
                if 0 <= v < vocab:
                    seen[v] = True
                    if prompt_lens is None or i >= int(prompt_lens[b]):
                        made[v] = made.get(v, 0) + 1
        r, f, p = of(repetition, b, 1.0), of(frequency, b, 0.0), of(presence, b, 0.0)
        for v in seen:
            x[b, v] = x[b, v] / r if x[b, v] > 0 else x[b, v] * r
            size[b, v] = x[b, v].abs()
        for v, n in made.items():
            x[b, v] -= f * n + p
            size[b, v] += abs(f) * n + abs(p)
        if bias_ids is not None:
            ids, values = (t[b] if t.dim() == 2 else t for t in (bias_ids, bias_values))
            for v, w in zip(ids.tolist(), values.tolist()):
                if 0 <= v < vocab:
                    x[b, v] += w
                    size[b, v] += abs(w)
        if allowed is not None:
            words = allowed[b] if allowed.dim() == 2 else allowed
            for v in range(vocab):
                if not (int(words[v // 32]) >> (v % 32)) & 1:
                    x[b, v], size[b, v] = float("-inf"), 0.0
    return x, size

"""Plain 64-bit forms of what a step over drafted tokens does: head norms, attention of a tree, verification, moves.

Test infrastructure, written from the operators' definitions; every loop is over rows, tokens or list entries.
"""

from __future__ import annotations

import math

import torch

from .decode import E4M3_MAX, place, rotate


def head_norm(x, weight, eps):
    """x [heads, dim] (float64) over its root mean square, times the weights; weight None leaves it."""
    if weight is None:
        return x
    return x / ((x * x).sum(-1, keepdim=True) / x.shape[-1] + eps).sqrt() * weight.double()


def norm_rope_append(q, k, v, key, value, table, past, cos, sin, seq_lens=None, interleaved=False, k_scale=None,
                     v_scale=None, q_norm=None, k_norm=None, eps=1e-6, depths=None):
    """(q_out, k_out, key, value, q_size, k_size) in float64: the results, unrounded (8-bit caches over the scale and
    saturated), and the sums of magnitudes that went into each element of q_out and k_out."""
    rows, m, heads, dim = q.shape
    num_pages, _, page_size, _ = key.shape
    q_out, q_size = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    k_out, k_size = (torch.zeros(k.shape, dtype=torch.float64) for _ in range(2))
    key, value = key.double().clone(), value.double().clone()
    cos, sin = cos.double(), sin.double()
    for b in range(rows):
        n = m if seq_lens is None else min(m, int(seq_lens[b]))
        for t in range(n):
            at = place(table, b, int(past[b]) + t, num_pages, page_size)
            depth = t if depths is None else int(depths[b, t] if depths.dim() == 2 else depths[t])
            pos = int(past[b]) + depth
            if at is None or not 0 <= pos < cos.shape[0]:
                continue
            for x, w, out, size in ((q, q_norm, q_out, q_size), (k, k_norm, k_out, k_size)):
                y = head_norm(x[b, t].double(), w, eps)
                out[b, t] = rotate(y, cos[pos], sin[pos], interleaved)
                # the first of a pair with one sign, its second with the other
                size[b, t] = torch.maximum(*(rotate(y.abs(), cos[pos].abs(), sign * sin[pos].abs(), interleaved)
                                             for sign in (-1, 1)))
            for cache, x, scale in ((key, k_out[b, t], k_scale), (value, v[b, t].double(), v_scale)):
                if scale is not None:
                    x = (x / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
                cache[at[0], :, at[1]] = x
    return q_out, k_out, key, value, q_size, k_size


def seen_places(past, n, t, m, bits=None, depth=None, window=None):
    """The places of a row that its drafted token t < n sees: bits[j] says whether it sees drafted token j."""
    if bits is None:
        first = max(0, past + t - window + 1) if window else 0
        return list(range(first, past + t + 1))
    first = max(0, past + depth - window + 1) if window else 0
    return list(range(first, past)) + [past + j for j in range(n) if bits[j]]


def tree_attention(q, key, value, table, past, seq_lens=None, visible=None, depths=None, scale=None, window=None,
                   k_scale=None, v_scale=None):
    """(out, spread, reach) in float64: the output, the same sum over |values| and the largest |q| . |k| * scale, the
    sizes that rounding errors are proportional to.  visible is boolean [rows, M, M]."""
    rows, m, heads, dim = q.shape
    num_pages, kv_heads, page_size, _ = key.shape
    group = heads // kv_heads
    scale = dim**-0.5 if scale is None else scale
    out, spread = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    reach = torch.zeros(rows, m, heads, 1, dtype=torch.float64)
    fp8 = key.dtype == torch.float8_e4m3fn
    caches = [c.view(torch.uint8) if fp8 else c for c in (key, value)]  # 8-bit floats take no lists
    for b in range(rows):
        n = m if seq_lens is None else min(m, int(seq_lens[b]))
        if int(past[b]) < 0:
            continue
        for t in range(n):
            places = seen_places(int(past[b]), n, t, m, None if visible is None else visible[b, t].tolist(),
                                 None if depths is None else max(0, int(depths[b, t])), window)
            places = [place(table, b, p, num_pages, page_size) for p in places]
            places = [p for p in places if p is not None]
            if not places:
                continue
            pages, slots = (torch.tensor(x) for x in zip(*places))
            k, v = (c[pages, :, slots].view(key.dtype).double() for c in caches)
            if k_scale is not None:
                k, v = k * k_scale.double()[:, None], v * v_scale.double()[:, None]
            k, v = (x.repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))  # [heads, places, dim]
            x = q[b, t].double()[:, :, None]
            p = torch.softmax((k @ x)[:, :, 0] * scale, -1)[:, None]
            out[b, t], spread[b, t] = (p @ v)[:, 0], (p @ v.abs())[:, 0]
            reach[b, t] = (k.abs() @ x.abs()).amax(1) * abs(scale)
    return out, spread, reach


def keep_tokens(cache, table, past, path, counts):
    """The cache after the moves: every place is read before any is written."""
    num_pages, _, page_size, _ = cache.shape
    out = cache.clone()
    for b in range(table.shape[0]):
        before = -1
        for i in range(min(int(counts[b]), path.shape[1])):
            node = int(path[b, i])
            if node <= before:
                break
            before = node
            source = place(table, b, int(past[b]) + node, num_pages, page_size)
            target = place(table, b, int(past[b]) + i, num_pages, page_size)
            if source is not None and target is not None:
                out[target[0], :, target[1]] = cache[source[0], :, source[1]]
    return out


def first_above(weights, number: float) -> int:
    """The first place whose running sum is above number times the sum; the last of any weight where none is."""
    upto = weights.cumsum(0)
    above = ((upto > number * upto[-1]) & (weights > 0)).nonzero()
    if len(above):
        return int(above[0])
    some = (weights > 0).nonzero()
    return int(some[-1]) if len(some) else -1


def verify_tokens(logits, tokens, uniforms, parents=None, draft_probs=None, temperature=None, seq_lens=None):
    """(path, counts, next) of the definition, a token at a time."""
    rows, m, vocab = logits.shape
    path = torch.full((rows, m), -1, dtype=torch.int32)
    counts = torch.zeros(rows, dtype=torch.int32)
    following = torch.full((rows,), -1, dtype=torch.int64)
    for b in range(rows):
        n = m if seq_lens is None else min(m, int(seq_lens[b]))
        heat = 1.0 if temperature is None else float(temperature[b])
        if n <= 0:
            continue
        nodes, token = [0], -1
        while True:
            node = nodes[-1]
            x = logits[b, node].double()
            if not vocab or not bool((x < math.inf).all()) or float(x.max()) == -math.inf or not 0 <= heat < math.inf:
                token = -1
                break
            best = int((x == x.max()).nonzero()[0])
            e = torch.exp((x - x.max()) / (heat or 1.0))
            u = float(uniforms[b, node])
            if draft_probs is not None:
                q = None
                if node + 1 < n:
                    q = draft_probs[b, node].double()
                    d, z = int(tokens[b, node + 1]), float(e.sum())
                    if d == best if heat == 0 else 0 <= d < vocab and u * float(q[d]) * z < float(e[d]):
                        nodes.append(node + 1)
                        continue
                if heat == 0:
                    token = best
                else:
                    last = float(uniforms[b, n - 1])
                    rest = torch.zeros_like(e) if q is None else (e - q * z).clamp(min=0)
                    token = first_above(rest if float(rest.sum()) > 0 else e, last)
                break
            token = best if heat == 0 else first_above(e, u)
            after = [c for c in range(node + 1, n)
                     if (c - 1 if parents is None else int(parents[b, c] if parents.dim() == 2 else parents[c])) == node
                     and int(tokens[b, c]) == token]
            if not after:
                break
            nodes.append(after[0])
        path[b, : len(nodes)] = torch.tensor(nodes, dtype=torch.int32)
        counts[b] = len(nodes)
        following[b] = token
    return path, counts, following

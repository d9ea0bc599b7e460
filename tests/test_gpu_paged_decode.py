"""The paged decode example against a decode that keeps no cache: dense attention over the whole row, every step."""

from __future__ import annotations

import importlib.util
import sys
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

from oracle import decode as plain

pytestmark = pytest.mark.gpu

_SPEC = importlib.util.spec_from_file_location(
    "paged_decode", Path(__file__).resolve().parents[1] / "examples" / "paged_decode.py")
example = importlib.util.module_from_spec(_SPEC)
sys.modules["paged_decode"] = example
_SPEC.loader.exec_module(example)


def dense_logits(pm, r, row_lens):
    """Logits of each row's newest token from its whole history, through the wrapped Linears and plain attention."""
    base, device = pm.base_model, r.tokens.device
    m = int(row_lens.max())
    context = pm.prepare_lora_context(r.adapter_ids, (torch.arange(m, device=device) < row_lens[:, None]).long(),
                                      r.tokens.shape[0], m, device)
    dim = base.blocks[0].dim
    i = torch.arange(dim // 2, dtype=torch.float64, device=device)
    angle = torch.arange(m, dtype=torch.float64, device=device)[:, None] * 10000.0 ** (-2 * i / dim)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x):
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    h = base.embed(r.tokens[:, :m])
    blocked = torch.ones(m, m, dtype=torch.bool, device=device).triu(1)
    with example.use_lora_context(context):
        for b in base.blocks:
            x = F.rms_norm(h, h.shape[-1:], b.norm1, 1e-5)
            q, k, v = (p(x).unflatten(-1, (-1, dim)) for p in (b.q_proj, b.k_proj, b.v_proj))
            q, k, v = (t.transpose(1, 2) for t in (turn(q), turn(k), v))
            k, v = (t.repeat_interleave(q.shape[1] // k.shape[1], 1) for t in (k, v))
            s = (q.contiguous() @ k.transpose(2, 3).contiguous()) * dim**-0.5
            out = s.masked_fill(blocked, float("-inf")).softmax(-1) @ v.contiguous()
            h = h + b.o_proj(out.transpose(1, 2).flatten(2))
            x = F.rms_norm(h, h.shape[-1:], b.norm2, 1e-5)
            h = h + b.down_proj(F.silu(b.gate_proj(x)) * b.up_proj(x))
    last = h[torch.arange(h.shape[0], device=device), (row_lens - 1).long()]
    return base.head(F.rms_norm(last, last.shape[-1:], base.norm, 1e-5))


@pytest.mark.parametrize("graph", [True, False])
def test_every_step_matches_a_decode_without_a_cache(gpu, graph):
    s = example.Sizes(vocab=331, hidden=128, inner=192, layers=2, heads=4, kv_heads=2, head_dim=32)
    rows, adapters, prompt, steps = 5, 3, 37, 12
    pm = example.build_model(s, adapters, 8, torch.float32, gpu)
    r = example.build_requests(s, rows, adapters, prompt, steps, gpu)
    cache = example.PagedCache(s, rows, prompt + steps, 16, torch.float32, gpu, False)
    got = example.generate(pm, cache, r, steps, graph=graph)
    assert torch.equal(cache.lens, r.lens - 1) and torch.equal(r.lens, r.prompt_lens + steps)
    with torch.no_grad():
        for t in range(steps):
            lens = r.prompt_lens + t
            rules = {n: x.cpu() for n, x in r.rules().items()} | {"lens": lens.cpu()}
            want, _ = plain.adjust_logits(dense_logits(pm, r, lens).cpu(), **rules)
            best = want.max(-1)
            # the picked token is the best, or as near to it as fp32 sums of other orders leave logits of size about 1
            picked = want.gather(1, got[:, t : t + 1].cpu())[:, 0]
            assert bool((best.values - picked <= 1e-3).all()), (t, best, got[:, t])


def test_an_8_bit_cache_decodes_alike(gpu):
    """The first tokens after a prompt: an e4m3 cache moves logits by its rounding, not their order here and there."""
    s = example.Sizes(vocab=331, hidden=128, inner=192, layers=2, heads=4, kv_heads=2, head_dim=32)
    rows, adapters, prompt, steps = 6, 3, 50, 6
    pm = example.build_model(s, adapters, 8, torch.bfloat16, gpu)
    out = []
    for fp8 in (False, True):
        r = example.build_requests(s, rows, adapters, prompt, steps, gpu)
        cache = example.PagedCache(s, rows, prompt + steps, 16, torch.bfloat16, gpu, fp8)
        out.append(example.generate(pm, cache, r, steps))
    assert torch.equal(out[0][:, 0], out[1][:, 0])  # the prompt's own attention reads no cache
    assert float((out[0] == out[1]).float().mean()) > 0.5

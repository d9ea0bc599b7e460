"""Faults that a step over drafted tokens once had, each with the call that showed it or would have."""

from __future__ import annotations

import pytest
import torch

from oracle import drafts as plain
from polylora_amd.drafts import verify_tokens

from .test_gpu_drafts import random_parents

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

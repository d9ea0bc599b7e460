"""Serving a batch of requests, each with its own adapter, history and sampling rules, over a paged key-value cache.

A small decoder with random weights stands for the model: its Linears are wrapped by PolyLoraModel, its attention
appends to and reads a paged cache (polylora_amd.paged), and the logits of each step pass through
polylora_amd.logits before the next tokens are picked.  Every row is a request: it has its adapter, its own prompt
length, its own pages, penalties, banned tokens and grammar.

    python examples/paged_decode.py [--steps 32] [--rows 8] [--cache fp8]

Decode steps run under a HIP graph: everything a step changes (tokens, lengths, pages) is a device tensor.
"""

from __future__ import annotations

import argparse
import sys
import time
from dataclasses import dataclass
from pathlib import Path

import torch
import torch.nn.functional as F
from torch import nn

if __name__ == "__main__":  # run from a checkout
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from polylora_amd import CpuAdapterStore, PolyLoraConfig, PolyLoraModel
from polylora_amd.context import use_lora_context
from polylora_amd.logits import adjust_logits, pack_allowed
from polylora_amd.paged import paged_attention, rope_append, rope_table
from polylora_amd.store import CpuLayerWeights

TARGETS = ["q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"]


@dataclass
class Sizes:
    vocab: int = 1024
    hidden: int = 512
    inner: int = 1024
    layers: int = 2
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64


class PagedCache:
    """Keys and values of every layer in pages of `page` tokens; row b owns pages b * width .. (b + 1) * width - 1.

    A server hands pages out as rows grow and writes their ids into `table`; here every row gets its share at once.
    """

    def __init__(self, sizes: Sizes, rows: int, longest: int, page: int, dtype: torch.dtype, device, fp8: bool) -> None:
        width = -(-longest // page)
        shape = (rows * width, sizes.kv_heads, page, sizes.head_dim)
        cache_dtype = torch.float8_e4m3fn if fp8 else dtype
        self.key = [torch.empty(shape, dtype=cache_dtype, device=device) for _ in range(sizes.layers)]
        self.value = [torch.empty(shape, dtype=cache_dtype, device=device) for _ in range(sizes.layers)]
        self.table = torch.arange(rows * width, dtype=torch.int32, device=device).view(rows, width)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=device)  # tokens of each row in the pages
        self.cos, self.sin = rope_table(longest, sizes.head_dim, device=device)
        # e4m3 holds values to 448: keys and values of unit size keep four binary digits with this
        self.scale = torch.full((sizes.kv_heads,), 1 / 16, device=device) if fp8 else None


class Block(nn.Module):
    def __init__(self, s: Sizes) -> None:
        super().__init__()
        self.dim = s.head_dim
        self.norm1 = nn.Parameter(torch.ones(s.hidden))
        self.norm2 = nn.Parameter(torch.ones(s.hidden))
        q, kv = s.heads * s.head_dim, s.kv_heads * s.head_dim
        for name, fin, fout in (("q_proj", s.hidden, q), ("k_proj", s.hidden, kv), ("v_proj", s.hidden, kv),
                                ("o_proj", q, s.hidden), ("gate_proj", s.hidden, s.inner),
                                ("up_proj", s.hidden, s.inner), ("down_proj", s.inner, s.hidden)):
            setattr(self, name, nn.Linear(fin, fout, bias=False))

    def attend(self, x: torch.Tensor, cache: PagedCache, layer: int, new: torch.Tensor) -> torch.Tensor:
        q, k, v = (p(x).unflatten(-1, (-1, self.dim)) for p in (self.q_proj, self.k_proj, self.v_proj))
        key, value, scale = cache.key[layer], cache.value[layer], cache.scale
        turned = torch.empty_like(k) if x.shape[1] > 1 else None
        q = rope_append(q, k, v, key, value, cache.table, cache.lens, cache.cos, cache.sin, seq_lens=new,
                        k_scale=scale, v_scale=scale, k_out=turned)
        if turned is None:
            out = paged_attention(q[:, 0], key, value, cache.table, cache.lens + new, k_scale=scale, v_scale=scale)
            return self.o_proj(out.flatten(1)[:, None])
        # a prompt attends to itself: right-padded, so no token sees padding
        q, k, v = (t.transpose(1, 2) for t in (q, turned, v))
        group = q.shape[1] // k.shape[1]
        k, v = (t.repeat_interleave(group, 1) for t in (k, v))
        return self.o_proj(F.scaled_dot_product_attention(q, k, v, is_causal=True).transpose(1, 2).flatten(2))

    def forward(self, h: torch.Tensor, cache: PagedCache, layer: int, new: torch.Tensor) -> torch.Tensor:
        h = h + self.attend(F.rms_norm(h, h.shape[-1:], self.norm1, 1e-5), cache, layer, new)
        x = F.rms_norm(h, h.shape[-1:], self.norm2, 1e-5)
        return h + self.down_proj(F.silu(self.gate_proj(x)) * self.up_proj(x))


class Decoder(nn.Module):
    def __init__(self, s: Sizes) -> None:
        super().__init__()
        self.embed = nn.Embedding(s.vocab, s.hidden)
        self.blocks = nn.ModuleList(Block(s) for _ in range(s.layers))
        self.norm = nn.Parameter(torch.ones(s.hidden))
        self.head = nn.Linear(s.hidden, s.vocab, bias=False)

    def forward(self, input_ids: torch.Tensor, attention_mask=None, *, cache: PagedCache, new: torch.Tensor):
        """Logits [rows, vocab] of each row's newest token; `new` counts the tokens of input_ids that are the row's."""
        h = self.embed(input_ids)
        for layer, block in enumerate(self.blocks):
            h = block(h, cache, layer, new)
        last = h[torch.arange(h.shape[0], device=h.device), (new - 1).clamp(min=0).long()]
        cache.lens += new
        return self.head(F.rms_norm(last, last.shape[-1:], self.norm, 1e-5))


@dataclass
class Requests:
    """The rows of a batch: token lists (prompt, then output) and what each request asks of its logits."""

    tokens: torch.Tensor  # int64 [rows, longest]
    lens: torch.Tensor  # int32 [rows]
    prompt_lens: torch.Tensor
    adapter_ids: list
    repetition: torch.Tensor
    presence: torch.Tensor
    frequency: torch.Tensor
    bias_ids: torch.Tensor
    bias_values: torch.Tensor
    allowed: torch.Tensor

    def rules(self) -> dict:
        return {name: getattr(self, name) for name in ("tokens", "lens", "prompt_lens", "repetition", "presence",
                                                        "frequency", "bias_ids", "bias_values", "allowed")}


def build_model(s: Sizes, adapters: int, rank: int, dtype: torch.dtype, device, seed: int = 0) -> PolyLoraModel:
    torch.manual_seed(seed)
    base = Decoder(s).to(device=device, dtype=dtype).eval().requires_grad_(False)
    store = CpuAdapterStore()
    modules = {n: m for n, m in base.named_modules() if n.split(".")[-1] in TARGETS}
    for i in range(adapters):
        store.add_adapter(f"a{i}", {
            n: CpuLayerWeights(A=torch.randn(m.in_features, rank) * 0.05, B=torch.randn(rank, m.out_features) * 0.05,
                               rank=rank, scale=2.0) for n, m in modules.items()})
    config = PolyLoraConfig(target_modules=TARGETS, max_gpu_adapters=adapters, max_rank=rank)
    return PolyLoraModel(base, config, adapter_store=store).eval()


def build_requests(s: Sizes, rows: int, adapters: int, longest_prompt: int, steps: int, device, seed: int = 1) -> Requests:
    g = torch.Generator().manual_seed(seed)
    prompt = torch.randint(1, longest_prompt + 1, (rows,), generator=g, dtype=torch.int32)
    prompt[0] = longest_prompt
    tokens = torch.randint(0, s.vocab, (rows, longest_prompt + steps), generator=g)
    allowed = torch.ones(rows, s.vocab, dtype=torch.bool)
    allowed[1::2] = torch.rand(rows // 2, s.vocab, generator=g) < 0.2  # every other request is held to a token set
    r = Requests(tokens, prompt.clone(), prompt.clone(), [f"a{i % (adapters + 1)}" for i in range(rows)],
                 torch.rand(rows, generator=g) * 0.3 + 1, torch.rand(rows, generator=g), torch.rand(rows, generator=g) * 0.3,
                 torch.randint(0, s.vocab, (rows, 4), generator=g, dtype=torch.int32),
                 torch.tensor([[2.0, -2.0, float("-inf"), 0.5]]).repeat(rows, 1), pack_allowed(allowed))
    r.adapter_ids = ["__base__" if a == f"a{adapters}" else a for a in r.adapter_ids]
    for name, value in vars(r).items():
        if torch.is_tensor(value):
            setattr(r, name, value.to(device))
    return r


def pick(logits: torch.Tensor, r: Requests) -> torch.Tensor:
    """The next token of each row, greedily, written behind its history."""
    token = adjust_logits(logits, **r.rules()).argmax(-1, keepdim=True)
    r.tokens.scatter_(1, r.lens.long()[:, None], token)
    r.lens += 1
    return token


@torch.no_grad()
def generate(pm: PolyLoraModel, cache: PagedCache, r: Requests, steps: int, graph: bool = True) -> torch.Tensor:
    """Runs the prompts, then steps - 1 single tokens per row; returns the tokens [rows, steps] that were picked."""
    rows, m = r.tokens.shape[0], int(r.lens.max())
    device = r.tokens.device
    mask = torch.arange(m, device=device) < r.lens[:, None]
    logits = pm(input_ids=r.tokens[:, :m], attention_mask=mask.long(), adapter_ids=r.adapter_ids, cache=cache, new=r.lens)
    token = pick(logits, r)

    # the adapters stay resident, so one context serves every step
    context = pm.prepare_lora_context(r.adapter_ids, None, rows, 1, device)
    one = torch.ones(rows, dtype=torch.int32, device=device)

    def step() -> None:
        with use_lora_context(context):
            token.copy_(pick(pm.base_model(token, cache=cache, new=one), r))

    done = 1
    if graph and steps > 3:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # warm: workspaces, plans, the library's choices
            for _ in range(2):
                step()
                done += 1
        torch.cuda.current_stream().wait_stream(side)
        recorded = torch.cuda.CUDAGraph()
        with torch.cuda.graph(recorded, stream=side):
            step()
        while done < steps:
            recorded.replay()
            done += 1
    while done < steps:
        step()
        done += 1
    first = r.prompt_lens.long()[:, None] + torch.arange(steps, device=device)
    return r.tokens.gather(1, first)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rows", type=int, default=8)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=200)
    ap.add_argument("--adapters", type=int, default=5)
    ap.add_argument("--cache", choices=("bf16", "fp8"), default="bf16")
    args = ap.parse_args()
    device, s = torch.device("cuda", 0), Sizes()
    pm = build_model(s, args.adapters, 16, torch.bfloat16, device)
    for attempt in ("first", "second"):
        r = build_requests(s, args.rows, args.adapters, args.prompt, args.steps, device)
        cache = PagedCache(s, args.rows, args.prompt + args.steps, 16, torch.bfloat16, device, args.cache == "fp8")
        torch.cuda.synchronize()
        t = time.perf_counter()
        out = generate(pm, cache, r, args.steps)
        torch.cuda.synchronize()
        print(f"{attempt} run: {args.rows} rows x {args.steps} tokens in {(time.perf_counter() - t) * 1e3:.1f} ms", flush=True)
    for row, ids in enumerate(out[: min(4, args.rows), :12].tolist()):
        print(f"row {row} ({r.adapter_ids[row]}): {ids}")


if __name__ == "__main__":
    main()

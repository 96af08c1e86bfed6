"""From prompts to the text condition of the denoising step, on random weights: a small decoder-only
text model built from the quantised linears and the text-side operators, then the token refiner.

    python examples/encode_prompt.py [--cache bf16|int8|e4m3] [--layers N] [--new N]

1. Two prompts of different lengths go through the model packed into one batch: a step's pages, slots and
   positions are planned on the device, head norms + rope + cache write are one launch, and the rows attend
   to one another, causal, with grouped heads.
2. Both are continued token by token (greedy), all sequences in one call: the same, with
   attention over the paged cache. A prompt may also arrive in pieces (``chunks``): the same call
   with several tokens a sequence.
3. Prompts that begin with the same text stand behind one cached copy of it, which is walked once for
   all of them.
4. The hidden states of a sequence, one row per token, are what ``H3TextRefiner`` takes.
"""
from __future__ import annotations

import argparse
from dataclasses import dataclass
from pathlib import Path
import sys
from typing import Optional

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
from wuxianhuabu_b200 import h3, text  # noqa: E402


@dataclass
class TextConfig:
    hidden: int = 512
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    ffn: int = 1024
    layers: int = 2
    vocab: int = 1000
    eps: float = 1e-6


class TextModel:
    """Pre-norm decoder layers: x += out(attention(rope(qkv(norm1 x)))), x += fc2(swiglu(fc1(norm2 x)))."""

    def __init__(self, cfg: TextConfig, positions: int, seed: int = 1):
        self.cfg = cfg
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def linear(n: int, k: int) -> h3.MfLinear:
            return h3.MfLinear.quantize(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)

        ones = torch.ones(cfg.hidden, dtype=torch.bfloat16, device="cuda")
        self.embed = torch.randn(cfg.vocab, cfg.hidden, generator=g, device="cuda").to(torch.bfloat16)
        inner, kv = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim
        self.layers = [dict(qkv=linear(inner + 2 * kv, cfg.hidden), out=linear(cfg.hidden, inner),
                            fc1=linear(2 * cfg.ffn, cfg.hidden), fc2=linear(cfg.hidden, cfg.ffn))
                       for _ in range(cfg.layers)]
        self.norm = ones
        self.head_norm = torch.ones(cfg.head_dim, dtype=torch.bfloat16, device="cuda")  # (of q's and of k's heads)
        self.rope = text.RopeTable(cfg.head_dim, positions, base=10000.0)

    def forward(self, ids, positions, slots, caches, attend):
        """ids [tokens] -> hidden states [tokens, hidden]; ``attend(layer, q, k, v)`` is the
        attention of the rows over what they may see."""
        c = self.cfg
        x = self.embed[ids]
        n, inner, kv = x.shape[0], c.heads * c.head_dim, c.kv_heads * c.head_dim
        gate = torch.ones((1, c.hidden), dtype=torch.bfloat16, device="cuda")
        row0 = torch.zeros(n, dtype=torch.int32, device="cuda")
        for i, w in enumerate(self.layers):
            qkv = w["qkv"](h3.rms_norm(x, self.norm, c.eps))
            q = qkv[:, :inner].unflatten(1, (c.heads, c.head_dim))  # slices: no copies are made
            k = qkv[:, inner:inner + kv].unflatten(1, (c.kv_heads, c.head_dim))
            v = qkv[:, inner + kv:].unflatten(1, (c.kv_heads, c.head_dim))
            q = caches[i].append_roped(q, k, v, slots, self.rope, positions, q_norm=self.head_norm,
                                       k_norm=self.head_norm, eps=c.eps)
            o = attend(i, q, k, v)
            x = w["out"](o.flatten(1), h3.EPI_GATE_RESID, gate=gate, resid=x, rowmap=row0)
            y = w["fc1"](h3.rms_norm(x, self.norm, c.eps), h3.EPI_SWIGLU)
            x = w["fc2"](y, h3.EPI_GATE_RESID, gate=gate, resid=x, rowmap=row0)
        return h3.rms_norm(x, self.norm, c.eps)


class Sequences:
    """The cached state of a batch: pages of every layer, dealt out as the sequences grow. ``common``: tokens
    that every sequence begins with, cached once, before them."""

    def __init__(self, model: TextModel, batch: int, max_tokens: int, page: int = 16, fmt: str = "bf16",
                 common: Optional[list[int]] = None):
        c = model.cfg
        self.model, self.common = model, len(common or ())
        front, blocks = -(-self.common // page), -(-max_tokens // page)
        pages = front + batch * blocks
        self.caches = [text.PagedKVCache(pages, page, c.kv_heads, c.head_dim, fmt) for _ in range(c.layers)]
        self.pool = text.PagePool(pages, page, batch, blocks)
        if common:  # a sequence of its own, whose pages stay taken
            first = Sequences.__new__(Sequences)
            first.model, first.common, first.caches = model, 0, self.caches
            first.pool = text.PagePool.from_tensors(page, self.pool.free, self.pool.taken, self.pool.lens.new_zeros(1),
                                                    self.pool.table.new_zeros(1, front))
            first.extend([common])
            self.front = first.pool.table[0]

    def _step(self, ids: list[list[int]]):
        new = torch.tensor([len(seq) for seq in ids], dtype=torch.int32, device="cuda")
        flat = torch.tensor([i for seq in ids for i in seq], device="cuda")
        return flat, self.pool.plan(new, flat.numel(), first_position=self.common), max(len(seq) for seq in ids)

    def prompts(self, ids: list[list[int]]) -> torch.Tensor:
        """Whole prompts, packed, into empty caches."""
        tok, plan, longest = self._step(ids)
        norm, eps = self.model.head_norm, self.model.cfg.eps

        def attend(i, q, k, v):
            # (the prompt attends to its own bf16 rows; only later tokens read the cache)
            k = self.model.rope.apply(k, plan.positions, norm=norm, eps=eps)
            return text.prompt_attention(q, k, v, plan.cu_seqlens, longest)

        return self.model.forward(tok, plan.positions, plan.slots, self.caches, attend)

    def extend(self, ids: list[list[int]]) -> torch.Tensor:
        """Some more tokens of every sequence, attending to all that is cached."""
        tok, plan, longest = self._step(ids)

        def attend(i, q, k, v):
            if self.common:
                return text.prefix_attention(q, self.caches[i], self.front, self.common, plan.cu_seqlens, plan.kv_lens,
                                             self.pool.table, longest)
            return text.paged_attention(q, self.caches[i], plan.cu_seqlens, plan.kv_lens, self.pool.table, longest)

        return self.model.forward(tok, plan.positions, plan.slots, self.caches, attend)


def refiner(cfg: TextConfig, seed: int = 2) -> h3.H3TextRefiner:
    dit = h3.H3DiTConfig(hidden=256, heads=2, head_dim=128, ffn=512, layers=1)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def linear(n: int, k: int) -> h3.MfLinear:
        return h3.MfLinear.quantize(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)

    def ones(n: int) -> torch.Tensor:
        return torch.ones(n, dtype=torch.bfloat16, device="cuda")

    inner = dit.heads * dit.head_dim
    block = h3.H3BlockWeights(linear(3 * inner, dit.hidden), linear(dit.hidden, inner), linear(dit.ffn, dit.hidden),
                              linear(dit.hidden, dit.ffn), ones(128), ones(128), ones(dit.hidden), ones(dit.hidden))
    return h3.H3TextRefiner(dit, linear(dit.hidden, cfg.hidden), [block], ones(dit.hidden))


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--cache", choices=("bf16", "int8", "e4m3"), default="bf16")
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--new", type=int, default=12, help="tokens generated after each prompt")
    a = ap.parse_args(argv)
    cfg = TextConfig(layers=a.layers)
    g = torch.Generator()
    g.manual_seed(3)
    prompts = [torch.randint(cfg.vocab, (n,), generator=g).tolist() for n in (77, 21)]
    model = TextModel(cfg, positions=256)

    seqs = Sequences(model, len(prompts), 128, fmt=a.cache)
    states = seqs.prompts(prompts)
    rows = [[states[:77]], [states[77:]]]
    ids = [list(p) for p in prompts]
    last = torch.stack([states[76], states[-1]])
    for _ in range(a.new):
        step = torch.argmax(last.float() @ model.embed.float().t(), dim=1).tolist()
        last = seqs.extend([[t] for t in step])
        for b, t in enumerate(step):
            ids[b].append(t)
            rows[b].append(last[b:b + 1])
    grown = [torch.cat(r) for r in rows]

    # the same tokens in one pass, and in chunks over the cache: the same states up to rounding
    whole = Sequences(model, len(prompts), 128, fmt=a.cache).prompts(ids).split([len(i) for i in ids])
    again = Sequences(model, len(prompts), 128, fmt=a.cache)
    parts = [again.extend([i[at:at + 32] for i in ids]).split([len(i[at:at + 32]) for i in ids])
             for at in range(0, max(map(len, ids)), 32)]
    chunks = [torch.cat([p[b] for p in parts]) for b in range(len(ids))]

    # the first 40 tokens of one prompt as the common beginning of three
    common = prompts[0][:40]
    ends = [prompts[0][40:], prompts[1], prompts[1][:5]]
    behind = Sequences(model, 3, 128, fmt=a.cache, common=common)
    shared = list(behind.extend(ends).split([len(e) for e in ends]))
    apart = Sequences(model, 3, 128, fmt=a.cache).prompts([common + e for e in ends]).split([40 + len(e) for e in ends])

    def differ(x, y) -> float:
        return max(float((p.float() - q.float()).norm() / q.float().norm()) for p, q in zip(x, y))

    refine = refiner(cfg)
    conditions = [refine(s) for s in grown]
    h3.context().check_device()
    result = dict(tokens=[len(i) for i in ids], stepwise=differ(grown, whole), chunked=differ(chunks, whole),
                  shared=differ(shared, [x[40:] for x in apart]),
                  conditions=[tuple(c.shape) for c in conditions],
                  finite=all(bool(torch.isfinite(c.float()).all()) for c in conditions))
    print(f"cache {a.cache}: sequences of {result['tokens']} tokens; states token by token against one pass: "
          f"{result['stepwise']:.4f}, in chunks: {result['chunked']:.4f}, behind a common beginning: "
          f"{result['shared']:.4f}; conditions {result['conditions']}")
    return result


if __name__ == "__main__":
    main()

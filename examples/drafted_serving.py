#!/usr/bin/env python3
"""Serving from a cache of 8-bit floats with drafted tokens, through one attention layer with norms of queries and keys.

    python examples/drafted_serving.py [--prompts 37 150 8] [--drafts 4] [--tokens 24] [--temperature 0.3]

The toy model of ``paged_serving.py`` with a norm of each head's queries and keys.  Prompts are read whole.  Then every
step gives each sequence its last token and up to ``--drafts`` tokens that followed the same token earlier in its text,
in one ragged batch:

* ``paged.norm_rotate_append`` writes keys and values of all of them, quantised, to the cache;
* ``paged.quantised_attention`` attends over it;
* ``paged.verify`` keeps or rejects the drafts by the target's probabilities (the drafts were certain: no probabilities
  of their own) and draws the token after those kept.  What rejected drafts left in the cache is written over.

At the end every sequence is recomputed as a whole, without a cache, in 64 bits and with keys and values rounded as the
cache rounds them, and the largest difference of a logit that a token was drawn from is printed.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))

from paged_serving import DIM, HEADS, KV_HEADS, PAGE, VOCABULARY, Model  # noqa: E402

from emmy_b200 import paged  # noqa: E402

EPS = 1e-6


class NormedModel(Model):
    def __init__(self, seed=0):
        super().__init__(seed)
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        self.weights = [(torch.rand(DIM, generator=g, device="cuda") + 0.5).bfloat16() for _ in range(2)]
        self.norm = paged.Norm(*self.weights, eps=EPS)
        # keys have a root mean square of about 1 and values of about that: 2^e of 448 covers them
        self.exponents = torch.tensor([[-5] * KV_HEADS, [-4] * KV_HEADS], dtype=torch.int32, device="cuda")

    def logits_without_cache(self, tokens):
        x = self.embedding[tokens]
        q, k, v = (x @ self.project).view(len(tokens), -1, DIM).double().split([HEADS, KV_HEADS, KV_HEADS], 1)
        angle = torch.arange(len(tokens), device="cuda").double()[:, None] * self.frequencies.double()
        c, s = angle.cos()[:, None], angle.sin()[:, None]

        def turned(y, weight):
            y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
            a, b = y.chunk(2, -1)
            return torch.cat([a * c - b * s, b * c + a * s], -1)

        def held(y, exponents):
            by = torch.exp2(exponents.double())[:, None]
            return ((y / by).clamp(-448, 448).float().to(paged.E4M3).double() * by).repeat_interleave(HEADS // KV_HEADS, 1)

        q, k, v = turned(q, self.weights[0]).bfloat16().double(), held(turned(k, self.weights[1]), self.exponents[0]), held(v, self.exponents[1])
        score = torch.einsum("qhd,khd->hqk", q, k) * DIM ** -0.5
        later = torch.ones(len(tokens), len(tokens), dtype=torch.bool, device="cuda").triu(1)
        mixed = torch.einsum("hqk,khd->qhd", score.masked_fill(later, -torch.inf).softmax(-1), v)
        return (x.double() + mixed.flatten(1) @ self.merge.double()) @ self.head.double()


class Server:
    def __init__(self, model, pages=256):
        self.model = model
        self.k_cache, self.v_cache = (torch.empty(pages, PAGE, KV_HEADS, DIM, device="cuda").to(paged.E4M3) for _ in range(2))
        self.free = list(range(pages))
        self.pages = {}                         # sequence -> its pages, in order

    def step(self, batch, starts):
        """``batch``: {sequence: tokens}, at positions from ``starts[sequence]`` on.  The logits after every token."""
        model, slots, positions = self.model, [], []
        for s, tokens in batch.items():
            mine = self.pages.setdefault(s, [])
            for at in range(starts[s], starts[s] + len(tokens)):
                if at // PAGE == len(mine):
                    mine.append(self.free.pop())
                slots.append(mine[at // PAGE] * PAGE + at % PAGE)
                positions.append(at)
        width = max(len(self.pages[s]) for s in batch)
        table = torch.tensor([self.pages[s] + [0] * (width - len(self.pages[s])) for s in batch], dtype=torch.int32, device="cuda")
        slots, positions = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (slots, positions))
        x = model.embedding[torch.tensor([t for tokens in batch.values() for t in tokens], device="cuda")]
        plan = paged.QuantisedPlan([len(t) for t in batch.values()], [starts[s] + len(t) for s, t in batch.items()], HEADS, KV_HEADS, DIM)
        q, k, v = (x @ model.project).view(len(x), -1, DIM).split([HEADS, KV_HEADS, KV_HEADS], 1)
        q = paged.norm_rotate_append(model.rotation, model.norm, q, k, v, positions, slots, self.k_cache, self.v_cache, exponents=model.exponents)
        mixed, _ = paged.quantised_attention(plan, q, self.k_cache, self.v_cache, model.exponents, table)
        y = x.float() + mixed.flatten(1).float() @ model.merge.float()
        plan.check()
        return y @ model.head.float()


def looked_up(text, most):
    """What followed the last token where it stood before."""
    for at in range(len(text) - 2, -1, -1):
        if text[at] == text[-1]:
            return text[at + 1:at + 1 + most]
    return []


def serve(prompts, drafts, tokens, temperature=0.3, seed=0):
    """Serves random prompts of the given lengths up to ``tokens`` more each; (tokens of each sequence, drafts tried and
    kept, largest difference of a logit from the computation without a cache, over the largest logit)."""
    model = NormedModel(seed)
    server, g = Server(model), torch.Generator().manual_seed(seed)
    texts = [torch.randint(0, VOCABULARY, (n,), generator=g).tolist() for n in prompts]
    seen, tried, kept = [[] for _ in texts], 0, 0
    cached = [0] * len(texts)
    while any(len(t) < n + tokens for t, n in zip(texts, prompts)):
        live = [s for s, (t, n) in enumerate(zip(texts, prompts)) if len(t) < n + tokens]
        guess = {s: looked_up(texts[s], drafts) if cached[s] else [] for s in live}
        batch = {s: texts[s][cached[s]:] + guess[s] for s in live}
        logits, at = server.step(batch, cached), 0
        rows, first, drafted = [], [0], []
        for s in live:
            end = at + len(batch[s])
            rows += range(end - len(guess[s]) - 1, end)        # the last token's row and the drafts'
            drafted += guess[s]
            first.append(len(rows))
            at = end
        target = (logits[rows] / temperature).softmax(-1)
        accepted, out = paged.verify(target, None, torch.tensor(drafted, dtype=torch.int32, device="cuda"), torch.rand(len(drafted), generator=g).cuda(),
                                     torch.rand(len(live), generator=g).cuda(), torch.tensor(first, dtype=torch.int32, device="cuda"))
        accepted, out = accepted.tolist(), out.tolist()
        for i, s in enumerate(live):
            seen[s].append(logits[rows[first[i]:first[i] + accepted[i] + 1]])
            cached[s] = len(texts[s]) + accepted[i]
            texts[s] += out[first[i]:first[i] + accepted[i] + 1]
            tried, kept = tried + len(guess[s]), kept + accepted[i]
    worst = 0.0
    for text, n, got in zip(texts, prompts, seen):
        want = model.logits_without_cache(torch.tensor(text[:-1], device="cuda"))[n - 1:]
        worst = max(worst, float((torch.cat(got).double() - want).abs().max() / want.abs().max()))
    return texts, (tried, kept), worst


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompts", type=int, nargs="+", default=[37, 150, 8])
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=24)
    ap.add_argument("--temperature", type=float, default=0.3)
    a = ap.parse_args(argv)
    texts, (tried, kept), worst = serve(a.prompts, a.drafts, a.tokens, a.temperature)
    for n, text in zip(a.prompts, texts):
        print(f"prompt of {n}: continued with {text[n:]}")
    print(f"{kept} of {tried} drafted tokens kept; largest difference from the computation without a cache: {worst:.2e} of the largest logit")
    return 0 if worst < 1e-2 else 1


if __name__ == "__main__":
    sys.exit(main())

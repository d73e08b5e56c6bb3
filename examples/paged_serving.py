#!/usr/bin/env python3
"""Serving with a paged cache: prompts prefilled in chunks, then decoded, through one attention layer.

    python examples/paged_serving.py [--prompts 37 150 8] [--chunk 64] [--steps 6]

A toy model of random weights (embedding, one layer of grouped-head attention, a
head), served as a scheduler would serve it: every step takes a
chunk of at most ``--chunk`` tokens of each prompt that is still being read and
one token of each sequence that decodes, in one ragged batch.  ``Server`` keeps
the cache, hands out its pages and calls, for every step,

* ``paged.AttentionPlan`` once (a model of many layers shares it),
* ``paged.rotate_append`` and ``paged.attention`` for the layer.

At the end every sequence is recomputed as a whole, without a cache, in 64 bits,
and the largest difference of a logit is printed.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "emmy-hackathon-2026_b200"))

from emmy_b200 import paged  # noqa: E402

VOCABULARY, WIDTH, HEADS, KV_HEADS, DIM, PAGE = 512, 256, 8, 2, 64, 16


class Model:
    def __init__(self, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(*shape):
            return (torch.randn(shape, generator=g, device="cuda") * shape[0] ** -0.5).bfloat16()

        self.embedding = weight(WIDTH, VOCABULARY).t().contiguous() * WIDTH ** 0.5
        self.project = weight(WIDTH, (HEADS + 2 * KV_HEADS) * DIM)
        self.merge = weight(HEADS * DIM, WIDTH)
        self.head = weight(WIDTH, VOCABULARY)
        self.frequencies = (10000.0 ** (-torch.arange(DIM // 2, device="cuda") / (DIM // 2))).float()
        self.rotation = paged.Rotation(self.frequencies)

    def logits_without_cache(self, tokens):
        """Logits of every position of one sequence, in 64 bits; keys, values and
        rotated queries rounded to the cache's type as the served path rounds them."""
        x = self.embedding[tokens]
        q, k, v = (x @ self.project).view(len(tokens), -1, DIM).double().split([HEADS, KV_HEADS, KV_HEADS], 1)
        angle = torch.arange(len(tokens), device="cuda").double()[:, None] * self.frequencies.double()
        c, s = angle.cos()[:, None], angle.sin()[:, None]

        def turned(y):
            a, b = y.chunk(2, -1)
            return torch.cat([a * c - b * s, b * c + a * s], -1).bfloat16().double()

        k, v = (y.repeat_interleave(HEADS // KV_HEADS, 1) for y in (turned(k), v))
        score = torch.einsum("qhd,khd->hqk", turned(q), k) * DIM ** -0.5
        later = torch.ones(len(tokens), len(tokens), dtype=torch.bool, device="cuda").triu(1)
        mixed = torch.einsum("hqk,khd->qhd", score.masked_fill(later, -torch.inf).softmax(-1), v)
        y = x.double() + mixed.flatten(1) @ self.merge.double()
        return y @ self.head.double()


class Server:
    def __init__(self, model, pages=256):
        self.model = model
        shape = (pages, PAGE, KV_HEADS, DIM)
        self.k_cache, self.v_cache = (torch.empty(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.free = list(range(pages))
        self.pages = {}                         # sequence -> its pages, in order
        self.length = {}

    def step(self, batch):
        """``batch``: {sequence: its next tokens}.  The logits after each sequence's last token."""
        model, slots, positions, ends = self.model, [], [], []
        for s, tokens in batch.items():
            mine, start = self.pages.setdefault(s, []), self.length.get(s, 0)
            for at in range(start, start + len(tokens)):
                if at // PAGE == len(mine):
                    mine.append(self.free.pop())
                slots.append(mine[at // PAGE] * PAGE + at % PAGE)
                positions.append(at)
            self.length[s] = start + len(tokens)
            ends.append(len(slots) - 1)
        width = max(len(self.pages[s]) for s in batch)
        table = torch.tensor([self.pages[s] + [0] * (width - len(self.pages[s])) for s in batch], dtype=torch.int32, device="cuda")
        slots, positions = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (slots, positions))
        x = model.embedding[torch.tensor([t for tokens in batch.values() for t in tokens], device="cuda")]

        plan = paged.AttentionPlan([len(t) for t in batch.values()], [self.length[s] for s in batch], HEADS, KV_HEADS, DIM)
        q, k, v = (x @ model.project).view(len(x), -1, DIM).split([HEADS, KV_HEADS, KV_HEADS], 1)
        q = paged.rotate_append(model.rotation, q, k, v, positions, slots, self.k_cache, self.v_cache)
        mixed, _ = paged.attention(plan, q, self.k_cache, self.v_cache, table)
        y = x.float() + mixed.flatten(1).float() @ model.merge.float()
        plan.check()
        return (y @ model.head.float())[ends]

    def finish(self, s):
        self.free += self.pages.pop(s)
        del self.length[s]


def serve(prompts, chunk, steps, seed=0):
    """Serves random prompts of the given lengths; (tokens of each sequence, largest
    difference of a logit from the computation without a cache, over the largest logit)."""
    model = Model(seed)
    g = torch.Generator().manual_seed(seed)
    texts = [torch.randint(0, VOCABULARY, (n,), generator=g).tolist() for n in prompts]
    server, read, seen, left = Server(model), [0] * len(texts), [[] for _ in texts], [steps] * len(texts)
    while any(left):
        batch = {}
        for s, text in enumerate(texts):
            if left[s]:
                batch[s] = text[read[s]:read[s] + chunk]
                read[s] += len(batch[s])
        for s, logits in zip(batch, server.step(batch)):
            if read[s] == len(texts[s]):                    # the text is read: decode
                seen[s].append(logits)
                texts[s].append(int(logits.argmax()))
                left[s] -= 1
                if not left[s]:
                    server.finish(s)
    worst = 0.0
    for s, text in enumerate(texts):
        want = model.logits_without_cache(torch.tensor(text[:-1], device="cuda"))[-steps:]
        got = torch.stack(seen[s]).double()
        worst = max(worst, float((got - want).abs().max() / want.abs().max()))
    return texts, worst


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompts", type=int, nargs="+", default=[37, 150, 8])
    ap.add_argument("--chunk", type=int, default=64)
    ap.add_argument("--steps", type=int, default=6)
    a = ap.parse_args(argv)
    texts, worst = serve(a.prompts, a.chunk, a.steps)
    for n, text in zip(a.prompts, texts):
        print(f"prompt of {n}: continued with {text[n:]}")
    print(f"largest difference from the computation without a cache: {worst:.2e} of the largest logit")
    return 0 if worst < 1e-2 else 1


if __name__ == "__main__":
    sys.exit(main())

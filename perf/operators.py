"""What the paged-cache operators are timed and compared on.

Two operators of a serving step: ``rotate_append`` (rotary positions of one or several axes applied to the new
tokens' queries and keys, keys and values written into a paged cache) and ``attention`` (a ragged chunk of new
tokens, one token upwards a sequence, over that cache).  With ``own`` false ``run`` computes them in elementary
torch operations in 32 bits; with ``own`` true it calls ``emmy_b200.paged``.
"""
import math
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
ROTATED, ATTENDED = "rotate_append", "attention"


def rotated(name, tokens, heads, kv_heads, dim, page, dtype, axes=1, interleaved=False, rotary=None, layout="token",
            reach=32768):
    """A case of rotate_append: `tokens` new tokens at positions below `reach` of each axis; `rotary` leading
    components of a head turn; the cache stores a page's tokens together ("token") or its heads ("head")."""
    return {"name": name, "op": ROTATED, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "dtype": dtype, "axes": axes, "interleaved": interleaved, "rotary": rotary or dim, "layout": layout, "reach": reach}


def attended(name, seqs, q, kv, heads, kv_heads, dim, page, dtype, window=0, layout="token", mix=1):
    """A case of attention: `seqs` sequences with q[0]..q[1] new tokens each over kv[0]..kv[1] cached ones (the new
    ones among them; lengths spread over the range by `mix`), a token seeing the last `window` positions, 0: all."""
    return {"name": name, "op": ATTENDED, "seqs": seqs, "q_low": q[0], "q_high": q[1], "kv_low": kv[0], "kv_high": kv[1],
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "window": window,
            "layout": layout, "mix": mix}


def listed():
    return [
        # one sequence being decoded: the smallest call there is
        rotated("append_one", 1, 32, 8, 128, 16, "bf16"),
        # a decoding batch, one token a sequence
        rotated("append_batch", 127, 32, 8, 64, 16, "f16", interleaved=True, layout="head"),
        # the chunks of a prefill, a quarter of each head turned
        rotated("append_chunk", 4095, 32, 32, 128, 128, "bf16", rotary=32),
        # video tokens: time, height and width turn components of their own
        rotated("append_video", 16384, 32, 8, 128, 64, "bf16", axes=3, reach=4096),
        # the first tokens of one conversation
        attended("decode_one", 1, (1, 1), (301, 301), 32, 8, 128, 16, "bf16"),
        # a decoding batch at ragged lengths
        attended("decode_batch", 64, (1, 1), (517, 8191), 32, 8, 128, 16, "bf16"),
        # one very long context
        attended("decode_long", 1, (1, 1), (131071, 131071), 32, 8, 128, 64, "bf16", layout="head"),
        # drafted tokens being verified, a head of keys for each head of queries
        attended("verify", 24, (2, 9), (65, 2047), 32, 32, 64, 32, "f16"),
        # chunks of prefills among sequences that decode
        attended("mixed", 8, (1, 511), (1025, 12288), 32, 4, 64, 32, "bf16"),
        # chunks that see the last 1,024 positions only
        attended("window", 4, (1501, 2048), (4097, 8192), 32, 8, 128, 16, "f16", window=1024, layout="head"),
        # whole prompts at once
        attended("prefill", 8, (4096, 4096), (4096, 4096), 32, 8, 128, 64, "bf16"),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    dtype, layout, dim = rng.choice(("bf16", "f16")), rng.choice(("token", "head")), rng.choice((64, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 8))
    page = rng.choice((8, 16, 32, 64, 128))
    if rng.random() < 0.4:
        case = rotated("", spread(1, 16384), heads, kv_heads, dim, page, dtype, rng.choice((1, 1, 2, 3)),
                       rng.random() < 0.5, rng.choice((dim // 4, dim // 2, dim)), layout, rng.choice((2048, 32768)))
    else:
        kind = rng.choice(("decode", "verify", "mixed", "prefill"))
        if kind == "decode":
            seqs, q, kv = spread(1, 64), (1, 1), spread(1, 65536)
            seqs = max(1, min(seqs, 500_000 // kv))
        elif kind == "verify":
            seqs, kv = spread(1, 64), spread(16, 8192)
            q = (1, rng.randint(2, 16))
        elif kind == "mixed":
            seqs, kv = rng.randint(2, 8), spread(256, 12288)
            q = (1, spread(16, 512))
        else:
            seqs, kv = rng.randint(1, 4), spread(64, 4096)
            q = (max(1, kv // 2), kv)
        window = rng.choice((0, 0, 0, spread(16, 4096)))
        case = attended("", seqs, (q[0], min(q[1], kv)), (max(q[0], kv // 3), kv), heads, kv_heads, dim, page, dtype, window, layout,
                        rng.randint(1, 1 << 20))
    del case["name"]
    return case


def lengths(case):
    """New tokens and cached tokens of every sequence; the longest of each range is among them."""
    r = random.Random(case["mix"])
    kv = [r.randint(case["kv_low"], case["kv_high"]) for _ in range(case["seqs"])]
    q = [r.randint(case["q_low"], case["q_high"]) for _ in range(case["seqs"])]
    kv[-1], q[-1] = case["kv_high"], case["q_high"]
    return [min(a, b) for a, b in zip(q, kv)], kv


def cache(case, pages, gen):
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    if case["layout"] == "head":
        shape = (shape[0], shape[2], shape[1], shape[3])
    made = torch.randn(shape, generator=gen, device="cuda", dtype=DTYPES[case["dtype"]])
    return made.transpose(1, 2) if case["layout"] == "head" else made


def frequencies(case):
    half = case["rotary"] // 2
    return torch.tensor([10000.0 ** (-i / half) for i in range(half)], dtype=torch.float32, device="cuda")


def axis_of_pair(case):
    """The pairs go to the axes in runs of equal length, the last axis taking what is left."""
    half, axes = case["rotary"] // 2, case["axes"]
    return [min(i // max(1, half // axes), axes - 1) for i in range(half)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=DTYPES[case["dtype"]])

    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    state = {"case": case}
    if case["op"] == ROTATED:
        tokens = case["tokens"]
        pages = tokens // page + 8
        # one projection's output, of which queries, keys and values are views
        joined = normal(tokens, heads + 2 * kv_heads, dim)
        state["q"], state["k"], state["v"] = joined.split([heads, kv_heads, kv_heads], dim=1)
        state["k_cache"], state["v_cache"] = cache(case, pages, gen), cache(case, pages, gen)
        state["positions"] = torch.randint(0, case["reach"], (case["axes"], tokens), generator=gen, device="cuda", dtype=torch.int32)
        # whole pages follow one another within a chunk, pages themselves lie anywhere
        order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
        at = torch.arange(tokens, device="cuda", dtype=torch.int32)
        state["slots"] = order[(at // page).long()] * page + at % page
        state["frequencies"] = frequencies(case)
        state["axis"] = torch.tensor(axis_of_pair(case), device="cuda")
    else:
        q_lens, kv_lens = lengths(case)
        need = [-(-n // page) for n in kv_lens]
        pages = sum(need) + 1
        order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
        first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
        spot = torch.arange(max(need), device="cuda")
        table = order[(first[:, None] + spot).clamp(max=pages - 1)]
        state["table"] = torch.where(spot < torch.tensor(need, device="cuda")[:, None], table, 0).to(torch.int32)
        state["q"] = normal(sum(q_lens), heads, dim)
        state["k_cache"], state["v_cache"] = cache(case, pages, gen), cache(case, pages, gen)
        state["q_lens"], state["kv_lens"] = q_lens, kv_lens
        state["q_count"], state["kv_count"] = torch.tensor(q_lens, device="cuda"), torch.tensor(kv_lens, device="cuda")
    if own:
        if "emmy-hackathon-2026_b200" not in sys.path:
            sys.path.insert(0, "emmy-hackathon-2026_b200")
        from emmy_b200 import paged
        if case["op"] == ROTATED:
            state["rotation"] = paged.Rotation(state["frequencies"], axes=axis_of_pair(case), interleaved=case["interleaved"])
        else:
            state["plan"] = paged.AttentionPlan(q_lens, kv_lens, heads, kv_heads, dim, window=case["window"] or None)
        state["paged"] = paged
    return state


def plain_rotate_append(s):
    case = s["case"]
    half, rotary, page = case["rotary"] // 2, case["rotary"], case["page"]
    angle = s["positions"].float()[s["axis"]].t() * s["frequencies"]        # tokens x pairs, each by its axis
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turned(x):
        x32 = x.float()
        if case["interleaved"]:
            a, b = x32[..., 0:rotary:2], x32[..., 1:rotary:2]
            both = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
        else:
            a, b = x32[..., :half], x32[..., half:rotary]
            both = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        return torch.cat([both, x32[..., rotary:]], dim=-1).to(x.dtype)

    at, within = s["slots"].long() // page, s["slots"].long() % page
    s["k_cache"][at, within] = turned(s["k"])
    s["v_cache"][at, within] = s["v"]
    return turned(s["q"]), s["k_cache"], s["v_cache"]


def plain_attention(s):
    case, q = s["case"], s["q"]
    tokens, heads, dim = q.shape
    kv_heads, n, most = case["kv_heads"], case["seqs"], max(s["q_lens"])
    group = heads // kv_heads
    first = s["q_count"].cumsum(0) - s["q_count"]
    i = torch.arange(most, device=q.device)
    rows = (first[:, None] + i).clamp(max=tokens - 1)
    queries = q[rows].float().view(n, most, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(n, kv_heads, most * group, dim)
    table = s["table"].long()
    keys = s["k_cache"][table].float().flatten(1, 2).permute(0, 2, 3, 1)
    scores = torch.matmul(queries, keys).mul_(dim ** -0.5)
    del keys, queries
    j = torch.arange(scores.shape[-1], device=q.device)
    place = (s["kv_count"] - s["q_count"])[:, None] + i
    seen = (j <= place[..., None]) & (j < s["kv_count"][:, None, None])
    if case["window"]:
        seen &= j > place[..., None] - case["window"]
    scores = scores.view(n, kv_heads, most, group, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    values = s["v_cache"][table].float().flatten(1, 2).permute(0, 2, 1, 3)
    out = torch.matmul(weights.view(n, kv_heads, most * group, -1), values).view(n, kv_heads, most, group, dim)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + total.log())[..., 0]
    row = torch.arange(tokens, device=q.device)
    seq = torch.searchsorted(first + s["q_count"], row, right=True)
    at = row - first[seq]
    return out[seq, :, at].reshape(tokens, heads, dim).to(q.dtype), lse[seq, :, at].reshape(tokens, heads)


def run(state):
    if own:
        paged = state["paged"]
        if state["case"]["op"] == ROTATED:
            q = paged.rotate_append(state["rotation"], state["q"], state["k"], state["v"], state["positions"], state["slots"],
                                    state["k_cache"], state["v_cache"])
            return q, state["k_cache"], state["v_cache"]
        return paged.attention(state["plan"], state["q"], state["k_cache"], state["v_cache"], state["table"])
    return plain_rotate_append(state) if state["case"]["op"] == ROTATED else plain_attention(state)


def work(case):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == ROTATED:
        tokens, rotary = case["tokens"], case["rotary"]
        moved = tokens * ((2 * heads + 4 * kv_heads) * dim * 2 + 4 * case["axes"] + 4) + rotary * 2
        return {"bytes": moved, "flops": 3 * tokens * (heads + kv_heads) * rotary}
    read = pairs = 0
    for q, kv in zip(*lengths(case)):
        window = case["window"] or kv
        read += min(kv, window + q - 1)
        # token t of the chunk sees its own position and those before it, within the window
        pairs += sum(min(kv - q + t + 1, window) for t in range(q))
    tokens = sum(lengths(case)[0])
    moved = 4 * read * kv_heads * dim + tokens * heads * (4 * dim + 4) + 4 * (read // case["page"] + case["seqs"])
    return {"bytes": moved, "flops": 4 * pairs * heads * dim}


def exact(case, seed):
    """The same outputs by the definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == ROTATED:
        rotary, pairs = case["rotary"], case["rotary"] // 2
        one = [2 * p for p in range(pairs)] if case["interleaved"] else list(range(pairs))
        two = [p + 1 for p in one] if case["interleaved"] else [p + pairs for p in one]
        angle = torch.empty(case["tokens"], pairs, dtype=torch.float64, device="cuda")
        for p, axis in enumerate(axis_of_pair(case)):
            angle[:, p] = s["positions"][axis].double() * s["frequencies"][p].double()
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]

        def turned(x):
            y = x.double()
            z = torch.complex(y[..., one], y[..., two]) * turn
            y[..., one], y[..., two] = z.real, z.imag
            return y

        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        page, within = torch.div(s["slots"], case["page"], rounding_mode="floor").long(), (s["slots"] % case["page"]).long()
        k_cache[page, within], v_cache[page, within] = turned(s["k"]), s["v"].double()
        return turned(s["q"]), k_cache, v_cache
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(sum(s["q_lens"]), heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    start = 0
    for b, (n, length) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        own_pages = s["table"][b, : -(-length // page)].long()
        for h in range(kv_heads):
            group = slice(h * (heads // kv_heads), (h + 1) * (heads // kv_heads))
            keys = s["k_cache"][own_pages, :, h].double().reshape(-1, dim)[:length]
            values = s["v_cache"][own_pages, :, h].double().reshape(-1, dim)[:length]
            score = torch.einsum("tgd,kd->gtk", s["q"][start:start + n, group].double(), keys) / math.sqrt(dim)
            ahead = torch.arange(length, device="cuda") - torch.arange(length - n, length, device="cuda")[:, None]
            hidden = (ahead > 0) | (ahead <= -case["window"]) if case["window"] else ahead > 0
            score[:, hidden] = -math.inf
            lse[start:start + n, group] = torch.logsumexp(score, -1).t()
            chance = torch.softmax(score, -1)
            out[start:start + n, group] = torch.einsum("gtk,kd->tgd", chance, values)
        start += n
    return out, lse

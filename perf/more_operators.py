"""What the operators of a serving step with an 8-bit cache and drafted tokens are timed and compared on.

``norm_rotate_append`` (norms of queries and keys for each head, rotary positions, keys and values into a paged cache
of 8-bit floats or of the inputs' type), ``quantised_attention`` (a ragged chunk of new tokens over the 8-bit cache)
and ``verify`` (drafted tokens against the target's probabilities, from given random numbers).  With ``own`` false
``run`` computes them in elementary torch operations; with ``own`` true it calls ``emmy_b200.paged``.
"""
import math
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
APPENDED, ATTENDED, VERIFIED = "norm_rotate_append", "quantised_attention", "verify"


def appended(name, tokens, heads, kv_heads, dim, page, dtype, bits8=True, norm=True, interleaved=False, rotary=None, layout="token"):
    """`tokens` new tokens; the cache holds 8-bit floats, or the inputs' type; `rotary` leading components turn; the
    cache stores a page's tokens together ("token") or its heads ("head")."""
    return {"name": name, "op": APPENDED, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "dtype": dtype, "bits8": bits8, "norm": norm, "interleaved": interleaved, "rotary": rotary or dim, "layout": layout}


def attended(name, seqs, q, kv, heads, kv_heads, dim, page, dtype, window=0, layout="token", mix=1):
    """`seqs` sequences with q[0]..q[1] new tokens each over kv[0]..kv[1] cached ones (the new ones among them; lengths
    spread over the range by `mix`), a token seeing the last `window` positions, 0: all."""
    return {"name": name, "op": ATTENDED, "seqs": seqs, "q_low": q[0], "q_high": q[1], "kv_low": kv[0], "kv_high": kv[1],
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "window": window,
            "layout": layout, "mix": mix}


def verified(name, seqs, drafts, vocabulary, proposed=True, mix=1):
    """`seqs` sequences with drafts[0]..drafts[1] drafted tokens each; `proposed`: the draft's probabilities are given,
    otherwise the drafted tokens were certain."""
    return {"name": name, "op": VERIFIED, "seqs": seqs, "drafts_low": drafts[0], "drafts_high": drafts[1],
            "vocabulary": vocabulary, "proposed": proposed, "mix": mix}


def listed():
    return [
        # one sequence being decoded: the smallest call there is
        appended("append_one", 1, 32, 8, 128, 16, "bf16"),
        # a decoding batch, a token a sequence, into a cache of the inputs' type
        appended("append_batch", 127, 32, 8, 64, 16, "f16", bits8=False, interleaved=True, layout="head"),
        # the chunks of a prefill
        appended("append_chunk", 8191, 32, 8, 128, 64, "bf16"),
        # the first tokens of one conversation
        attended("decode_one", 1, (1, 1), (301, 301), 32, 8, 128, 16, "bf16"),
        # a decoding batch at ragged lengths
        attended("decode_batch", 64, (1, 1), (517, 8191), 32, 8, 128, 16, "bf16"),
        # one very long context
        attended("decode_long", 1, (1, 1), (131071, 131071), 32, 8, 128, 64, "bf16", layout="head"),
        # drafted tokens being verified, a head of keys for each head of queries
        attended("drafts", 24, (2, 9), (65, 4095), 32, 32, 64, 32, "f16"),
        # chunks of prefills among sequences that decode, the last 4,096 positions seen
        attended("mixed", 8, (1, 511), (1025, 12288), 32, 4, 64, 32, "bf16", window=4096),
        # whole prompts at once
        attended("prefill", 4, (4096, 4096), (4096, 4096), 32, 8, 128, 64, "bf16"),
        # one sequence's drafts
        verified("verify_one", 1, (4, 4), 32000),
        # a batch's drafts
        verified("verify_batch", 64, (1, 8), 131071),
        # drafts looked up in the text, without probabilities
        verified("verify_certain", 200, (0, 5), 65536, proposed=False),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    dtype, layout, dim = rng.choice(("bf16", "f16")), rng.choice(("token", "head")), rng.choice((64, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 8))
    page = rng.choice((8, 16, 32, 64, 128))
    which = rng.random()
    if which < 0.3:
        bits8, norm = rng.choice(((True, True), (True, True), (True, False), (False, True)))
        case = appended("", spread(1, 8191), heads, kv_heads, rng.choice((dim, dim, 96, 256)), page, rng.choice((dtype, dtype, "f32")), bits8,
                        norm, rng.random() < 0.4, None, layout)
        case["rotary"] = rng.choice((case["dim"] // 4, case["dim"] // 2, case["dim"], case["dim"]))
    elif which < 0.7:
        kind = rng.choice(("decode", "drafts", "mixed", "prefill"))
        if kind == "decode":
            seqs, q, kv = spread(1, 64), (1, 1), spread(1, 65536)
            seqs = max(1, min(seqs, 500_000 // kv))
        elif kind == "drafts":
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
    else:
        seqs, vocabulary = spread(1, 256), spread(500, 131072)
        seqs = min(seqs, 64 * 131071 // vocabulary)
        high = rng.randint(1, 8)
        case = verified("", seqs, (rng.randint(0, high), high), vocabulary, rng.random() < 0.6, rng.randint(1, 1 << 20))
    del case["name"]
    return case


def lengths(case):
    """New tokens and cached tokens of every sequence; the longest of each range is among them."""
    r = random.Random(case["mix"])
    kv = [r.randint(case["kv_low"], case["kv_high"]) for _ in range(case["seqs"])]
    q = [r.randint(case["q_low"], case["q_high"]) for _ in range(case["seqs"])]
    kv[-1], q[-1] = case["kv_high"], case["q_high"]
    return [min(a, b) for a, b in zip(q, kv)], kv


def drafts(case):
    """Drafted tokens of every sequence; the most is among them."""
    r = random.Random(case["mix"])
    n = [r.randint(case["drafts_low"], case["drafts_high"]) for _ in range(case["seqs"])]
    n[-1] = case["drafts_high"]
    return n


def frequencies(case):
    half = case["rotary"] // 2
    return torch.tensor([10000.0 ** (-i / half) for i in range(half)], dtype=torch.float32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    def cache(pages, kind):
        shape = (pages, case["page"], case["kv_heads"], case["dim"])
        if case["layout"] == "head":
            shape = (shape[0], shape[2], shape[1], shape[3])
        # (a cache of 8-bit floats: values of standard deviation 24, times 2^-4 or so)
        made = normal(*shape, dtype=torch.bfloat16).mul_(24).to(E4M3) if kind is E4M3 else normal(*shape, dtype=kind)
        return made.transpose(1, 2) if case["layout"] == "head" else made

    state = {"case": case}
    if case["op"] == VERIFIED:
        n, vocabulary = drafts(case), case["vocabulary"]
        rows, seqs = sum(n) + case["seqs"], case["seqs"]
        first = torch.tensor([sum(n[:s]) + s for s in range(seqs + 1)], dtype=torch.int32)
        state["first"] = first.cuda()
        # the target row that judges each draft
        judged = torch.tensor([i for s, m in enumerate(n) for i in range(int(first[s]), int(first[s]) + m)], dtype=torch.int64, device="cuda")
        logits = normal(rows, vocabulary).mul_(2.5)
        state["target"] = torch.softmax(logits, -1)
        # the draft model's logits are near the target's
        proposal = logits[judged].add_(normal(len(judged), vocabulary), alpha=0.7).softmax(-1)
        del logits
        state["drafted"] = torch.multinomial(proposal, 1, generator=gen)[:, 0].int() if len(judged) else judged.int()
        state["proposal"] = proposal if case["proposed"] else None
        state["uniforms"] = torch.rand(len(judged), generator=gen, device="cuda")
        state["finals"] = torch.rand(seqs, generator=gen, device="cuda")
        state["most"] = case["drafts_high"]
    elif case["op"] == APPENDED:
        heads, kv_heads, dim, page, tokens = case["heads"], case["kv_heads"], case["dim"], case["page"], case["tokens"]
        dtype = DTYPES[case["dtype"]]
        pages = tokens // page + 8
        # one projection's output, of which queries, keys and values are views
        state["q"], state["k"], state["v"] = normal(tokens, heads + 2 * kv_heads, dim, dtype=dtype).split([heads, kv_heads, kv_heads], dim=1)
        kind = E4M3 if case["bits8"] else dtype
        state["k_cache"], state["v_cache"] = cache(pages, kind), cache(pages, kind)
        state["positions"] = torch.randint(0, 32768, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
        # whole pages follow one another within a chunk, pages themselves lie anywhere
        order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
        at = torch.arange(tokens, device="cuda", dtype=torch.int32)
        state["slots"] = order[(at // page).long()] * page + at % page
        state["frequencies"] = frequencies(case)
        state["q_weight"], state["k_weight"] = (normal(dim).mul_(0.2).add_(1).to(dtype) for _ in range(2))
        state["exponents"] = torch.randint(-7, -3, (2, kv_heads), generator=gen, device="cuda", dtype=torch.int32)
    else:
        heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
        q_lens, kv_lens = lengths(case)
        need = [-(-n // page) for n in kv_lens]
        pages = sum(need) + 1
        order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
        start = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
        spot = torch.arange(max(need), device="cuda")
        table = order[(start[:, None] + spot).clamp(max=pages - 1)]
        state["table"] = torch.where(spot < torch.tensor(need, device="cuda")[:, None], table, 0).to(torch.int32)
        state["q"] = normal(sum(q_lens), heads, dim, dtype=DTYPES[case["dtype"]])
        state["k_cache"], state["v_cache"] = cache(pages, E4M3), cache(pages, E4M3)
        state["exponents"] = torch.randint(-6, -3, (2, kv_heads), generator=gen, device="cuda", dtype=torch.int32)
        state["q_lens"], state["kv_lens"] = q_lens, kv_lens
        state["q_count"], state["kv_count"] = torch.tensor(q_lens, device="cuda"), torch.tensor(kv_lens, device="cuda")
    if own:
        if "emmy-hackathon-2026_b200" not in sys.path:
            sys.path.insert(0, "emmy-hackathon-2026_b200")
        from emmy_b200 import paged
        state["paged"] = paged
        if case["op"] == APPENDED:
            state["rotation"] = paged.Rotation(state["frequencies"], interleaved=case["interleaved"])
            state["norm"] = paged.Norm(state["q_weight"], state["k_weight"], eps=1e-6) if case["norm"] else None
        elif case["op"] == ATTENDED:
            state["plan"] = paged.QuantisedPlan(q_lens, kv_lens, heads, kv_heads, dim, window=case["window"] or None)
    return state


def plain_append(s):
    case = s["case"]
    half, rotary, page = case["rotary"] // 2, case["rotary"], case["page"]
    angle = s["positions"].double()[:, None] * s["frequencies"].double()
    cos, sin = angle.cos()[:, None].float(), angle.sin()[:, None].float()

    def turned(x, weight):
        y = x.float()
        if case["norm"]:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
        if case["interleaved"]:
            a, b = y[..., 0:rotary:2], y[..., 1:rotary:2]
            both = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
        else:
            a, b = y[..., :half], y[..., half:rotary]
            both = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        return torch.cat([both, y[..., rotary:]], dim=-1)

    def stored(y, which):
        if not case["bits8"]:
            return y.to(s["q"].dtype)
        return (y * torch.exp2(-s["exponents"][which].float())[:, None]).clamp(-448, 448).to(E4M3)

    at, within = s["slots"].long() // page, s["slots"].long() % page
    for cache, y in ((s["k_cache"], stored(turned(s["k"], s["k_weight"]), 0)), (s["v_cache"], stored(s["v"].float(), 1))):
        if case["bits8"]:
            cache.view(torch.uint8)[at, within] = y.view(torch.uint8)       # (8-bit floats are not put everywhere)
        else:
            cache[at, within] = y
    return turned(s["q"], s["q_weight"]).to(s["q"].dtype), s["k_cache"], s["v_cache"]


def plain_attention(s):
    case, q = s["case"], s["q"]
    tokens, heads, dim = q.shape
    kv_heads, n, most = case["kv_heads"], case["seqs"], max(s["q_lens"])
    group = heads // kv_heads
    first = s["q_count"].cumsum(0) - s["q_count"]
    i = torch.arange(most, device=q.device)
    rows = (first[:, None] + i).clamp(max=tokens - 1)
    queries = q[rows].float().view(n, most, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(n, kv_heads, most * group, dim)
    table, scale = s["table"].long(), torch.exp2(s["exponents"].float())[..., None, None]

    def cached(cache, which):
        # (read as bytes: gathers of 8-bit floats are not everywhere)
        return cache.view(torch.uint8)[table].view(E4M3).float().flatten(1, 2).permute(0, 2, 1, 3).mul_(scale[which])

    scores = torch.matmul(queries, cached(s["k_cache"], 0).transpose(-1, -2)).mul_(dim ** -0.5)
    del queries
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
    out = torch.matmul(weights.view(n, kv_heads, most * group, -1), cached(s["v_cache"], 1)).view(n, kv_heads, most, group, dim)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + total.log())[..., 0]
    row = torch.arange(tokens, device=q.device)
    seq = torch.searchsorted(first + s["q_count"], row, right=True)
    at = row - first[seq]
    return out[seq, :, at].reshape(tokens, heads, dim).to(q.dtype), lse[seq, :, at].reshape(tokens, heads)


def plain_verify(s):
    """A drafted token x is kept while uniform * proposal[x] < target[x]; the token after those kept is the first whose
    running sum of max(target - proposal, 0), or of target after the last draft, exceeds final * the whole sum."""
    target, proposal, drafted, most = s["target"], s["proposal"], s["drafted"].long(), s["most"]
    vocabulary = target.shape[1]
    first = s["first"].long()
    seqs = len(first) - 1
    count = first[1:] - first[:-1] - 1
    i = torch.arange(most + 1, device=target.device)
    row = first[:-1, None] + i                              # of the target
    draft = row - torch.arange(seqs, device=target.device)[:, None]
    tried = i < count[:, None]
    kept = torch.zeros_like(tried)
    if len(drafted):
        draft = draft.clamp(max=len(drafted) - 1)
        x = drafted[draft]
        p = target[row.clamp(max=len(target) - 1), x].double()
        q = proposal[draft, x].double() if proposal is not None else torch.ones_like(p)
        kept = tried & (s["uniforms"][draft].double() * q < p)
    accepted = kept.int().cumprod(1).sum(1)
    last = first[:-1] + accepted
    mass = target[last].double()
    whole = mass
    if len(drafted):
        at = draft[torch.arange(seqs, device=target.device), accepted]
        if proposal is not None:
            rest = (mass - proposal[at].double()).clamp_(min=0)
        else:
            rest = mass.scatter(1, drafted[at][:, None], 0.0)
        rest = torch.where((accepted < count)[:, None], rest, mass)
        whole = torch.where(rest.sum(1, keepdim=True) > 0, rest, mass)
    sums = whole.cumsum(1)
    final = torch.searchsorted(sums, s["finals"].double()[:, None] * sums[:, -1:], right=True).clamp_(max=vocabulary - 1)
    seq = torch.searchsorted(first[1:], torch.arange(len(target), device=target.device), right=True)
    place = torch.arange(len(target), device=target.device) - first[seq]
    tokens = torch.full((len(target),), -1, dtype=torch.int64, device=target.device)
    if len(drafted):
        tokens = torch.where(place < accepted[seq], drafted[draft[seq, place]], tokens)
    tokens = torch.where(place == accepted[seq], final[seq, 0], tokens)
    return accepted.int(), tokens.int()


def run(state):
    op = state["case"]["op"]
    if own:
        paged = state["paged"]
        if op == APPENDED:
            q = paged.norm_rotate_append(state["rotation"], state["norm"], state["q"], state["k"], state["v"], state["positions"],
                                         state["slots"], state["k_cache"], state["v_cache"],
                                         exponents=state["exponents"] if state["case"]["bits8"] else None)
            return q, state["k_cache"], state["v_cache"]
        if op == ATTENDED:
            return paged.quantised_attention(state["plan"], state["q"], state["k_cache"], state["v_cache"], state["exponents"], state["table"])
        return paged.verify(state["target"], state["proposal"], state["drafted"], state["uniforms"], state["finals"], state["first"])
    return {APPENDED: plain_append, ATTENDED: plain_attention, VERIFIED: plain_verify}[op](state)


def work(case):
    if case["op"] == VERIFIED:
        # one row of the target and, but where all drafts are kept (about 0.6 of them one by one), one of the proposal
        n = drafts(case)
        rows = sum(2 - 0.6 ** m if case["proposed"] else 1 for m in n)
        return {"bytes": 4 * rows * case["vocabulary"] + sum(24 * m + 16 for m in n), "flops": 2 * rows * case["vocabulary"]}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == APPENDED:
        tokens, rotary = case["tokens"], case["rotary"]
        size = 4 if case["dtype"] == "f32" else 2
        moved = tokens * ((2 * heads + 2 * kv_heads) * dim * size + 2 * kv_heads * dim * (1 if case["bits8"] else size) + 8)
        flops = tokens * (heads + kv_heads) * (3 * rotary + (4 * dim if case["norm"] else 0))
        return {"bytes": moved + rotary * 2 + 2 * dim * size, "flops": flops}
    read = pairs = 0
    for q, kv in zip(*lengths(case)):
        window = case["window"] or kv
        read += min(kv, window + q - 1)
        # token t of the chunk sees its own position and those before it, within the window
        pairs += sum(min(kv - q + t + 1, window) for t in range(q))
    tokens = sum(lengths(case)[0])
    moved = 2 * read * kv_heads * dim + tokens * heads * (4 * dim + 4) + 4 * (read // case["page"] + case["seqs"])
    return {"bytes": moved, "flops": 4 * pairs * heads * dim}


def exact(case, seed):
    """The same outputs by the definitions, in 64 bits; what the cache holds as the 8-bit floats' values."""
    s = prepare(case, seed)
    if case["op"] == VERIFIED:
        accepted, tokens, starts = [], [], s["first"].tolist()
        for b, (begin, end) in enumerate(zip(starts, starts[1:])):
            drafted = s["drafted"][begin - b:end - b - 1].tolist()
            u = s["uniforms"][begin - b:end - b - 1].tolist()
            said = []
            for i, x in enumerate(drafted):
                q = float(s["proposal"][begin - b + i, x]) if case["proposed"] else 1.0
                if u[i] * q >= float(s["target"][begin + i, x]):
                    break
                said.append(x)
            mass = s["target"][begin + len(said)].double().cpu()
            if len(said) < len(drafted):
                rest = mass.clone()
                if case["proposed"]:
                    rest = (mass - s["proposal"][begin - b + len(said)].double().cpu()).clamp(min=0)
                else:
                    rest[drafted[len(said)]] = 0
                mass = rest if bool((rest > 0).any()) else mass
            sums = torch.cumsum(mass, 0)
            past = (sums > float(s["finals"][b]) * float(sums[-1])).nonzero()
            accepted.append(len(said))
            tokens += said + [int(past[0])] + [-1] * (len(drafted) - len(said))
        return torch.tensor(accepted, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32)
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    power = torch.pow(2.0, s["exponents"].double())
    if case["op"] == APPENDED:
        rotary, pairs = case["rotary"], case["rotary"] // 2
        one = [2 * p for p in range(pairs)] if case["interleaved"] else list(range(pairs))
        two = [p + 1 for p in one] if case["interleaved"] else [p + pairs for p in one]
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(s["positions"].double(), s["frequencies"].double()))[:, None]

        def turned(x, weight):
            y = x.double()
            if case["norm"]:
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / dim + 1e-6) * weight.double()
            z = torch.complex(y[..., one], y[..., two]) * turn
            y[..., one], y[..., two] = z.real, z.imag
            return y

        def stored(y, which):
            return (y / power[which][:, None]).clamp(-448, 448).to(E4M3).double() if case["bits8"] else y

        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        where, within = torch.div(s["slots"], page, rounding_mode="floor").long(), (s["slots"] % page).long()
        k_cache[where, within], v_cache[where, within] = stored(turned(s["k"], s["k_weight"]), 0), stored(s["v"].double(), 1)
        return turned(s["q"], s["q_weight"]), k_cache, v_cache
    out = torch.zeros(sum(s["q_lens"]), heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    start = 0
    for b, (n, length) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        own_pages = s["table"][b, : -(-length // page)].long()
        for h in range(kv_heads):
            group = slice(h * (heads // kv_heads), (h + 1) * (heads // kv_heads))
            keys, values = (s[c].view(torch.uint8)[own_pages, :, h].view(E4M3).double().reshape(-1, dim)[:length] * power[i, h]
                            for i, c in enumerate(("k_cache", "v_cache")))
            score = torch.einsum("tgd,kd->gtk", s["q"][start:start + n, group].double(), keys) / math.sqrt(dim)
            ahead = torch.arange(length, device="cuda") - torch.arange(length - n, length, device="cuda")[:, None]
            hidden = (ahead > 0) | (ahead <= -case["window"]) if case["window"] else ahead > 0
            score[:, hidden] = -math.inf
            lse[start:start + n, group] = torch.logsumexp(score, -1).t()
            chance = torch.softmax(score, -1)
            out[start:start + n, group] = torch.einsum("gtk,kd->tgd", chance, values)
        start += n
    return out, lse

"""The operators of an 8-bit cache and of drafted tokens on the GPU against their definitions in 64 bits.

Tolerances.  An 8-bit float (e4m3) is off by 2^-4 of the value at most, or by 2^-10 below
its normal range.  A norm's sum of squares, its root and the products are off by (head_dim +
16) roundings of 32 bits of the head's components at most, the rotation by 2^-21 of the pair's
length.  Attention: as for a 16-bit cache -- a weight rounded to 16 bits moves an output by
at most u sum(p|v|)/l, the last rounding by u|o|, 32-bit scores, exponentials and sums by
less than 1e-4 of sum(p|v|)/l and, in the logarithm, 1e-4 -- as reading the cache is exact."""
import math
import random

import pytest
import torch

from emmy_b200 import native, paged
from test_gpu_paged import UNIT, close, definition

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# half a step below a type's normal range (float16: steps of 2^-24)
SMALL = {BF16: 0.0, F16: 2.0 ** -25, F32: 0.0}


def within(got, want, off):
    bad = ~((got.double() - want).abs() <= off)
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} are off, the first at {at}: {float(got[at])}, not {float(want[at])} +- {float(off[at])}")


def generator(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------ norm_rotate_append
def appended(tokens, heads, kv_heads, dim, rotary, page, dtype=BF16, bits8=True, norm=True, layout="token", interleaved=False, offset=0,
             cache_offset=0, in_place=False, axes=1, size=1.0, exponents=True, eps=1e-6, seed=0):
    g = generator(seed)
    flat = (torch.randn(tokens * (heads + 2 * kv_heads) * dim + offset, generator=g, device="cuda") * size).to(dtype)
    x = flat[offset:].view(tokens, heads + 2 * kv_heads, dim)
    q, k, v = x.split([heads, kv_heads, kv_heads], 1)
    pairs = rotary // 2
    frequencies = (10000.0 ** -(torch.arange(pairs, device="cuda", dtype=torch.float64) / max(1, pairs))).float()
    pair_axes = [i * axes // max(1, pairs) for i in range(pairs)]
    positions = torch.randint(-5, 1 << 20, (max(pair_axes, default=0) + 1, tokens), generator=g, device="cuda", dtype=torch.int32)
    pages = tokens // page + 3
    kind = E4M3 if bits8 else dtype
    caches = []
    for _ in range(2):
        shape = (pages, page, kv_heads, dim) if layout == "token" else (pages, kv_heads, page, dim)
        c = torch.full((math.prod(shape) + cache_offset,), 3.0, device="cuda").to(kind)[cache_offset:].view(shape)
        caches.append(c if layout == "token" else c.transpose(1, 2))
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].int()
    if tokens > 2:
        slots[0], slots[tokens // 2] = -1, pages * page      # stored nowhere
    q_weight, k_weight = ((torch.rand(dim, generator=g, device="cuda") + 0.5).to(dtype) for _ in range(2))
    e = torch.randint(-6, 2, (2, kv_heads), generator=g, device="cuda", dtype=torch.int32) if exponents else None

    def wanted(y, weight):
        y = y.double().clone()
        if weight is not None:
            y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
        a, b = (torch.arange(pairs) * 2, torch.arange(pairs) * 2 + 1) if interleaved else (torch.arange(pairs), torch.arange(pairs) + pairs)
        angle = positions.double()[torch.tensor(pair_axes, dtype=torch.long)].t() * frequencies.double()
        cos, sin = angle.cos()[:, None], angle.sin()[:, None]
        left, right, length = y[..., a].clone(), y[..., b].clone(), y.abs()
        y[..., a], y[..., b] = left * cos - right * sin, right * cos + left * sin
        length[..., a] = length[..., b] = (left ** 2 + right ** 2).sqrt()
        return y, length * ((dim + 16) * 2.0 ** -24 * (weight is not None) + 2.0 ** -21)

    def stored(y, slack, which):
        """(values, how far they may be off), of all slots"""
        all_, off = (torch.full((pages * page, kv_heads, dim), at, dtype=torch.float64, device="cuda") for at in (3.0, 0.0))
        kept = (slots >= 0) & (slots < pages * page)
        if bits8:
            by = torch.pow(2.0, -e[which].double())[:, None] if e is not None else 1.0
            y, slack = (y * by).clamp(-448, 448), slack * by
            slack = slack * 1.07 + 2.0 ** -4 * y.abs() * 1.001 + 2.0 ** -10
        else:
            slack = slack + UNIT[dtype] * y.abs() * 1.001 + SMALL[dtype]
        all_[slots[kept].long()], off[slots[kept].long()] = y[kept], slack[kept]
        return all_, off

    want_q, slack_q = wanted(q, q_weight if norm else None)
    keys = stored(*wanted(k, k_weight if norm else None), 0)
    values = stored(v.double(), torch.zeros_like(v, dtype=torch.float64), 1)
    before = flat.clone()
    rotation = paged.Rotation(frequencies, pair_axes if axes > 1 else None, interleaved)
    out = paged.norm_rotate_append(rotation, paged.Norm(q_weight, k_weight, eps) if norm else None, q, k, v,
                                   positions[0] if len(positions) == 1 else positions, slots, *caches, exponents=e if bits8 else None,
                                   q_out=q if in_place else None)
    within(out, want_q, UNIT[dtype] * want_q.abs() * 1.001 + slack_q + SMALL[dtype])
    for c, (want, off) in zip(caches, (keys, values)):
        got = c.reshape(pages * page, kv_heads, dim) if kind is not E4M3 else c.float().reshape(pages * page, kv_heads, dim)
        within(got, want, off)
    # a value that only has to be rounded is rounded to the nearest, ties to even
    if bits8 and e is not None:
        nearest = (v.float() * torch.exp2(-e[1].float())[:, None]).clamp(-448, 448).to(E4M3)
        kept = (slots >= 0) & (slots < pages * page)
        got = caches[1].float().reshape(pages * page, kv_heads, dim)[slots[kept].long()]
        assert torch.equal(got, nearest.float()[kept])
    if in_place:
        assert out is q
    else:
        assert torch.equal(flat, before)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (64, 64), (128, 32), (96, 64), (80, 20), (256, 256), (192, 96), (7, 6), (64, 0), (33, 2), (1, 0)])
@pytest.mark.parametrize("bits8,norm", [(True, True), (True, False), (False, True)])
def test_append_dims(dtype, interleaved, dim, rotary, bits8, norm):
    appended(37, 6, 2, dim, rotary, 16, dtype, bits8, norm, interleaved=interleaved)


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 32, 8), (3, 1, 1), (1025, 8, 1), (130, 5, 5), (4, 0, 2), (300, 96, 8)])
@pytest.mark.parametrize("layout,page", [("token", 16), ("head", 5), ("token", 1)])
def test_append_tokens_and_layouts(tokens, heads, kv_heads, layout, page):
    appended(tokens, heads, kv_heads, 64, 64, page, layout=layout)


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_append_whole_blocks(dim, dtype):
    """As many heads as fill blocks, and more tokens than there are blocks."""
    for tokens in (1, 900):
        appended(tokens, 32, 8, dim, dim, 16, dtype)
        appended(tokens, 32, 8, dim, dim, 16, dtype, bits8=False)


@pytest.mark.parametrize("offset,cache_offset", [(0, 0), (1, 0), (0, 3), (8, 8), (4, 4)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_alignment_and_in_place(offset, cache_offset, interleaved):
    """Addresses off the grid of the vectors, of inputs and of the cache."""
    for in_place in (False, True):
        appended(50, 4, 2, 64, 32, 8, offset=offset, cache_offset=cache_offset, interleaved=interleaved, in_place=in_place)
        appended(50, 4, 2, 128, 128, 8, F32, offset=offset, cache_offset=cache_offset, interleaved=interleaved, in_place=in_place)


@pytest.mark.parametrize("axes", [2, 3])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_axes(axes, interleaved):
    appended(200, 8, 2, 128, 96, 16, F16, axes=axes, interleaved=interleaved)


def test_append_saturates_and_small_values():
    """Values over 448, below the normal range, and squares that only eps keeps from 0."""
    appended(64, 4, 2, 128, 128, 16, BF16, norm=False, size=3000.0, exponents=False)
    appended(64, 4, 2, 128, 128, 16, F32, norm=False, size=2.0 ** -9, exponents=False)
    appended(64, 4, 2, 128, 128, 16, F32, size=1e-6, eps=1e-5)


def test_append_values_that_are_not_finite():
    """NaN stays, infinities saturate; exponents count as the nearest of -15..7."""
    cache = [torch.zeros(1, 16, 1, 64, device="cuda").to(E4M3) for _ in range(2)]
    x = torch.zeros(3, 1, 64, device="cuda")
    x[0, 0, 0], x[1, 0, 0], x[2, 0, 1] = math.nan, math.inf, -math.inf
    at = torch.arange(3, dtype=torch.int32, device="cuda")
    rotation = paged.Rotation(torch.zeros(0, device="cuda"))
    paged.norm_rotate_append(rotation, None, x, x, x, at, at, *cache)
    for c in cache:
        got = c.float()[0, :3, 0]
        assert bool(got[0, 0].isnan()) and got[1, 0] == 448 and got[2, 1] == -448 and got.nan_to_num().abs().sum() == 896
    one = torch.ones(1, 1, 64, device="cuda")
    for e, want in ((-15, 448.0), (-100, 448.0), (7, 2.0 ** -7), (100, 2.0 ** -7), (-3, 8.0)):
        paged.norm_rotate_append(rotation, None, one, one, one, at[:1], at[:1], *cache,
                                 exponents=torch.tensor([[e], [0]], dtype=torch.int32, device="cuda"))
        assert cache[0].float()[0, 0, 0, 0] == want and cache[1].float()[0, 0, 0, 0] == 1


def test_append_without_norm_or_8_bits_is_rotate_append():
    g = generator()
    q, k, v = (torch.randn(70, n, 64, generator=g, device="cuda").bfloat16() for n in (8, 2, 2))
    at = torch.randperm(80, generator=g, device="cuda")[:70].int()
    rotation = paged.Rotation(torch.rand(32, generator=g, device="cuda"))
    caches = [[torch.zeros(5, 16, 2, 64, dtype=BF16, device="cuda") for _ in range(2)] for _ in range(2)]
    outs = [paged.rotate_append(rotation, q, k, v, at, at, *caches[0]), paged.norm_rotate_append(rotation, None, q, k, v, at, at, *caches[1])]
    assert torch.equal(*outs) and all(torch.equal(a, b) for a, b in zip(*caches))


def test_append_refuses():
    rotation = paged.Rotation(torch.ones(32, device="cuda"))
    cache = [torch.zeros(4, 16, 2, 64, device="cuda").to(E4M3) for _ in range(2)]
    q, kv, w = torch.zeros(5, 4, 64, device="cuda", dtype=F16), torch.zeros(5, 2, 64, device="cuda", dtype=F16), torch.ones(64, device="cuda", dtype=F16)
    at, e = torch.arange(5, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    norm = paged.Norm(w, w)

    def refused(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            paged.norm_rotate_append(rotation, *args, **kw)

    refused("positions", norm, q, kv, kv, at.long(), at, *cache)
    refused("slots", norm, q, kv, kv, at, at[:4], *cache)
    refused("k:", norm, q, kv.float(), kv, at, at, *cache)
    refused("fit", norm, q, kv[:, :1], kv[:, :1], at, at, *cache)
    refused("v_cache", norm, q, kv, kv, at, at, cache[0], cache[1].half())
    refused("k_cache", norm, q, kv, kv, at, at, cache[0].bfloat16(), cache[1].bfloat16())
    refused("exponents", norm, q, kv, kv, at, at, *cache, exponents=e[:1])
    refused("exponents", norm, q, kv, kv, at, at, *cache, exponents=e.float())
    refused("8-bit", norm, q, kv, kv, at, at, cache[0].half(), cache[1].half(), exponents=e)
    refused("norm", paged.Norm(w.float(), w.float()), q, kv, kv, at, at, *cache)
    refused("norm", paged.Norm(w[:32], w[:32]), q, kv, kv, at, at, *cache)
    refused("q_out", norm, q, kv, kv, at, at, *cache, q_out=q[:4])
    refused("requires grad", paged.Norm(w.clone().requires_grad_(), w), q, kv, kv, at, at, *cache)
    with torch.no_grad():
        paged.norm_rotate_append(rotation, paged.Norm(w.clone().requires_grad_(), w), q, kv, kv, at, at, *cache)
    for args in ((w, w.float()), (w, w[:32]), (w.double(), w.double()), (w, w, -1.0)):
        with pytest.raises(ValueError):
            paged.Norm(*args)


def test_append_writes_are_known_to_autograd():
    rotation = paged.Rotation(torch.ones(32, device="cuda"))
    cache = [torch.zeros(4, 16, 2, 64, device="cuda").to(E4M3) for _ in range(2)]
    q, kv, at = torch.zeros(5, 4, 64, device="cuda"), torch.zeros(5, 2, 64, device="cuda"), torch.arange(5, dtype=torch.int32, device="cuda")
    before = [c._version for c in cache]
    paged.norm_rotate_append(rotation, None, q, kv, kv, at, at, *cache)
    assert [c._version for c in cache] == [b + 1 for b in before]


# ------------------------------------------------------------------ quantised_attention
@pytest.fixture(params=[None, 3])
def ways(request, monkeypatch):
    """Plans for as many CTAs as there are, which little work goes to as few rows, and for a few, which it does not."""
    made = paged.QuantisedPlan.__init__
    monkeypatch.setattr(paged.QuantisedPlan, "__init__", lambda self, *args, **how: made(self, *args, **{"ctas": request.param, **how}))


def make(q_lens, kv_lens, heads, kv_heads, dim, page, dtype=BF16, layout="token", seed=0, size=16.0):
    """Inputs whose cache holds NaN wherever no sequence has a token, and whose table has
    page numbers from nowhere after each sequence's last; and the cache's values."""
    g = generator(seed)
    need = [-(-n // page) for n in kv_lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    table = torch.full((len(kv_lens), max(need + [1]) + 2), -1, dtype=torch.int32)
    table[:, -1] = 2 ** 30
    exponents = torch.randint(-5, -2, (2, kv_heads), generator=g, device="cuda", dtype=torch.int32)
    caches = [torch.full((pages, page, kv_heads, dim), math.nan, device="cuda") for _ in range(2)]
    at = 0
    for s, n in enumerate(kv_lens):
        for i in range(need[s]):
            table[s, i] = order[at]
            rows = min(page, n - i * page)
            for c in caches:
                c[order[at], :rows] = torch.randn(rows, kv_heads, dim, generator=g, device="cuda") * size
            at += 1
    held = []
    for c in caches:
        c = c.to(E4M3) if layout == "token" else c.transpose(1, 2).contiguous().to(E4M3).transpose(1, 2)
        held.append(c)
    q = torch.randn(sum(q_lens), heads, dim, generator=g, device="cuda").to(dtype)
    return q, held[0], held[1], exponents, table.cuda()


def values(cache, exponents):
    return cache.float() * torch.exp2(exponents.float())[:, None]


def wanted(made, q_lens, kv_lens, scale, causal=True, window=None):
    q, k, v, e, table = made
    return definition(q, values(k, e[0]), values(v, e[1]), table, q_lens, kv_lens, scale, causal, window)


def check(q_lens, kv_lens, heads, kv_heads, dim, page, dtype=BF16, layout="token", causal=True, window=None, scale=None, ctas=None, seed=0):
    """With as many CTAs as there are, which little work goes to as few rows, and with a few, which it does not."""
    made = make(q_lens, kv_lens, heads, kv_heads, dim, page, dtype, layout, seed)
    want = wanted(made, q_lens, kv_lens, scale or dim ** -0.5, causal, window)
    for n in (3, ctas):
        plan = paged.QuantisedPlan(q_lens, kv_lens, heads, kv_heads, dim, causal, window, ctas=n)
        out, lse = paged.quantised_attention(plan, *made, scale=scale)
        plan.check()
        close(out, lse, want, UNIT[dtype])
    return plan, made, out, lse


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("layout,page", [("token", 16), ("head", 64), ("token", 8), ("head", 128), ("token", 384), ("head", 8), ("token", 32)])
def test_decode_types_pages_layouts(dim, dtype, layout, page):
    check([1] * 10, [1, 15, 16, 17, 31, 32, 33, 257, 640, 1000], 16, 4, dim, page, dtype, layout)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (6, 2), (5, 1), (40, 8), (16, 1), (128, 1), (65, 1), (9, 1), (33, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_head_groups(heads, kv_heads, dim):
    check([1, 3, 40, 129], [300, 3, 170, 513], heads, kv_heads, dim, 32)


@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 7, 8, 9, 12, 13, 16, 17, 32, 33, 64, 65, 128, 129, 192, 193, 255, 256, 257])
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
def test_rows_around_the_tiles(tokens, dim, dtype):
    """Query rows about 8, 16, 24, 32, 128, 256, 384 and 512, which the ways of computing begin at."""
    check([tokens, 1], [tokens + 100, 70], 4, 2, dim, 16, dtype)


@pytest.mark.parametrize("q_lens,kv_lens", [
    ([128], [128]), ([129], [129]), ([257], [300]), ([1, 200, 1, 31, 64], [900, 200, 1, 600, 65]), ([500, 1, 333], [500, 2000, 777]),
])
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
def test_chunks(q_lens, kv_lens, dim, dtype, page):
    check(q_lens, kv_lens, 8, 4, dim, page, dtype)


@pytest.mark.parametrize("window", [1, 7, 128, 200, 5000])
@pytest.mark.parametrize("dim", [64, 128])
def test_window(window, dim):
    check([1, 300, 5, 129, 20], [1500, 1000, 5, 640, 700], 8, 2, dim, 16, window=window)


@pytest.mark.parametrize("seed", range(24))
def test_random_batches(seed):
    """Decoding, drafts and chunks together: every kernel's sequences in one call."""
    r = random.Random(seed)
    n, kv_heads, group = r.randint(1, 12), r.choice((1, 2, 3, 4, 8)), r.choice((1, 2, 3, 4, 8, 16))
    q_lens = [r.choice((0, 1, 1, 1, r.randint(2, 9), r.randint(10, 40), r.choice((3, 100, 300)))) for _ in range(n)]
    kv_lens = [max(q, r.choice((0, r.randint(1, 200), r.randint(1, 3000)))) if r.random() < 0.9 else q // 2 for q in q_lens]
    check(q_lens, kv_lens, group * kv_heads, kv_heads, r.choice((64, 128)), r.choice((8, 16, 32, 64, 128, 256)), r.choice((BF16, F16)),
          r.choice(("token", "head")), window=r.choice((None, None, r.randint(1, 700))), ctas=r.choice((None, None, 2, 11)), seed=seed)


@pytest.mark.parametrize("dim", [64, 128])
def test_every_token_sees_all(dim):
    check([1, 40, 300, 7], [300, 129, 555, 2000], 8, 2, dim, 32, causal=False)


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_see_nothing(dim):
    """No keys at all, more new tokens than keys, sequences without new tokens."""
    for causal in (True, False):
        _, _, out, lse = check([2, 9, 0, 300, 1], [0, 4, 50, 100, 0], 8, 2, dim, 16, causal=causal)
        assert not out[:2].any() and bool((lse[:2] == -math.inf).all())
        if causal:
            assert not out[2:7].any() and bool((lse[2:7] == -math.inf).all())


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("q_lens,kv_lens,heads,kv_heads", [
    ([1], [20000], 8, 1), ([3], [9000], 8, 8), ([9], [12000], 8, 4), ([1, 90], [40000, 6000], 16, 2), ([16], [30000], 8, 1)])
def test_split_over_keys(dim, dtype, q_lens, kv_lens, heads, kv_heads):
    """Few rows and many keys: parts joined by the last to arrive, the same bits on every
    call, the words left as they were."""
    plan, made, out, lse = check(q_lens, kv_lens, heads, kv_heads, dim, 64, dtype)
    words = plan.words.clone()
    assert plan.scratch.numel() > 0
    for _ in range(5):
        again = paged.quantised_attention(plan, *made)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    assert torch.equal(plan.words, words)


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("heads,kv_heads,tokens", [(32, 8, 1), (6, 6, 2), (20, 4, 3), (8, 1, 4), (5, 5, 9), (3, 3, 24), (64, 16, 1)])
def test_pieces_of_a_warp(heads, kv_heads, tokens, dim, dtype):
    """Work enough that each warp takes a head of its own, in parts that their last joins."""
    kv_lens = [(331 * s) % 1500 + tokens for s in range(60)]
    plan, made, out, lse = check([tokens] * 60, kv_lens, heads, kv_heads, dim, 16, dtype, ctas=3)
    words = plan.words.clone()
    for _ in range(3):
        again = paged.quantised_attention(plan, *made)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    assert torch.equal(plan.words, words)


@pytest.mark.parametrize("ctas", [1, 3, 37])
def test_few_ctas(ctas):
    """Many pieces a CTA, whose copies run ahead from one into the next."""
    q_lens, kv_lens = [1, 150, 1, 1, 300, 2, 20, 0, 1], [800, 150, 3, 0, 650, 129, 1000, 7, 17]
    check(q_lens, kv_lens, 8, 2, 128, 32, ctas=ctas)
    check(q_lens, kv_lens, 8, 2, 64, 32, F16, ctas=ctas)
    check([1] * 40, [17 * s % 333 for s in range(40)], 8, 2, 128, 16, ctas=ctas)


@pytest.mark.usefixtures("ways")
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_that_grow(dim, dtype):
    """The running maximum moves far in every slice, up or down: bases, outputs and sums with it."""
    for direction in (1, -1):
        q_lens, kv_lens = [2, 9, 200], [1500, 700, 900]
        q, k, v, e, table = make(q_lens, kv_lens, 4, 2, dim, 16, dtype)
        q.copy_(q.abs() + 0.5)
        big = k.float().abs()
        for s, n in enumerate(kv_lens):
            j = torch.arange(n, device="cuda")
            pages = table[s, :-(-n // 16)].long()
            big[pages[j // 16], j % 16] *= ((j if direction > 0 else n - j).float() / n * 6)[:, None, None]
        k = big.to(E4M3)
        plan = paged.QuantisedPlan(q_lens, kv_lens, 4, 2, dim)
        out, lse = paged.quantised_attention(plan, q, k, v, e, table, scale=0.5)
        plan.check()
        o, ls, size = wanted((q, k, v, e, table), q_lens, kv_lens, 0.5)
        # scores reach 2^10 (128 terms of 4 x 60 2^-3): sums and products in 32 bits put up to
        # 128 x 2^-24 x 2^10 on the exponent, were all their roundings of one sign
        within(out, o, UNIT[dtype] * (o.abs() + size) * 1.01 + 8e-3 * size + SMALL[dtype])
        assert float((lse.double() - ls).abs().max()) < 8e-3


@pytest.mark.usefixtures("ways")
@pytest.mark.parametrize("dtype,size", [(BF16, 2.0 ** 100), (BF16, 2.0 ** -100), (BF16, 2.0 ** -130), (F16, 60000.0), (F16, 2.0 ** -20)])
def test_queries_of_any_size(dtype, size):
    """The power of two that makes a row of queries f16 comes out of the scores again."""
    q_lens, kv_lens = [1, 5], [200, 77]
    q, k, v, e, table = make(q_lens, kv_lens, 8, 2, 128, 16, dtype)
    q = (q.clamp(-1, 1).double() * size).to(dtype)
    q[0, 3] = 0
    # scores of N(0, 1): what is left of the queries' size
    scale = min(float(128 ** -0.5 / size), 2.0 ** 126)
    plan = paged.QuantisedPlan(q_lens, kv_lens, 8, 2, 128)
    out, lse = paged.quantised_attention(plan, q, k, v, e, table, scale=scale)
    close(out, lse, wanted((q, k, v, e, table), q_lens, kv_lens, float(torch.tensor(scale, dtype=F32))), UNIT[dtype])


@pytest.mark.usefixtures("ways")
def test_queries_of_many_sizes_in_a_row():
    """Components 2^-24 of the largest count for as much as their keys make of them."""
    q_lens, kv_lens = [1, 7], [100, 90]
    q, k, v, e, table = make(q_lens, kv_lens, 8, 2, 64, 16, BF16)
    q[..., 0] = 4096.0
    q[..., 1:] *= 2.0 ** -9
    k = k.float()
    k[..., 0] *= 2.0 ** -12
    k = k.to(E4M3)
    plan = paged.QuantisedPlan(q_lens, kv_lens, 8, 2, 64)
    out, lse = paged.quantised_attention(plan, q, k, v, e, table, scale=4.0)
    close(out, lse, wanted((q, k, v, e, table), q_lens, kv_lens, 4.0), UNIT[BF16])


@pytest.mark.usefixtures("ways")
def test_keys_that_are_not_numbers_concern_the_tokens_that_see_them():
    q_lens, kv_lens = [3, 140], [40, 150]
    q, k, v, e, table = make(q_lens, kv_lens, 4, 2, 64, 16)
    raw = k.view(torch.uint8)
    raw[table[0, 2].long(), 7, 0, 5] = 0x7F          # position 39: the last token's own
    raw[table[1, 9].long(), 4, 1, 0] = 0xFF          # position 148: seen by the last two tokens
    plan = paged.QuantisedPlan(q_lens, kv_lens, 4, 2, 64)
    out, lse = paged.quantised_attention(plan, q, k, v, e, table)
    nan = torch.zeros(143, 4, dtype=torch.bool, device="cuda")
    nan[2, :2], nan[141:, 2:] = True, True
    assert torch.equal(lse.isnan(), nan) and torch.equal(out.isnan().all(-1), nan) and torch.equal(out.isnan().any(-1), nan)


@pytest.mark.usefixtures("ways")
def test_strided_views_and_given_outputs():
    q_lens, kv_lens = [3, 130, 5], [200, 300, 90]
    q, k, v, e, table = make(q_lens, kv_lens, 8, 2, 64, 16)
    n = sum(q_lens)
    joined = torch.randn(n, 12, 64, device="cuda").bfloat16()
    joined[:, 2:10] = q
    wide = torch.full((k.shape[0], 16, 4, 64), math.nan, device="cuda").to(E4M3)
    wide.view(torch.uint8)[:, :, 1:3] = k.view(torch.uint8)
    frame = torch.full((n + 2, 10, 64), 7.0, dtype=q.dtype, device="cuda")
    out, lse = frame[1:-1, 1:9], torch.empty(n, 8, device="cuda")
    wide_table = torch.full((3, table.shape[1] + 5), -9, dtype=torch.int32, device="cuda")
    wide_table[:, :table.shape[1]] = table
    plan = paged.QuantisedPlan(q_lens, kv_lens, 8, 2, 64)
    got = paged.quantised_attention(plan, joined[:, 2:10], wide[:, :, 1:3], v, e, wide_table[:, :table.shape[1]], out=out, lse=lse)
    plan.check()
    assert got[0] is out and got[1] is lse
    close(out, lse, wanted((q, k, v, e, table), q_lens, kv_lens, 0.125), UNIT[q.dtype])
    frame[1:-1, 1:9] = 7.0
    assert bool((frame == 7.0).all())


def test_no_exponents_are_zeros():
    made = list(make([1, 140], [77, 150], 4, 2, 64, 16, size=2.0))
    plan = paged.QuantisedPlan([1, 140], [77, 150], 4, 2, 64)
    made[3] = torch.zeros_like(made[3])
    want = paged.quantised_attention(plan, *made)
    made[3] = None
    got = paged.quantised_attention(plan, *made)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.usefixtures("ways")
@pytest.mark.parametrize("exponent", [-15, 7])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_exponents_at_the_ends(exponent, dtype):
    """Exact in either type: the smallest 8-bit float times 2^-15, the largest times 2^7."""
    q_lens, kv_lens = [1, 140], [77, 150]
    q, k, v, e, table = make(q_lens, kv_lens, 4, 2, 64, 16, dtype, size=1.0)
    e.fill_(exponent)
    k.view(torch.uint8)[table[0, 0].long(), 0, 0, :4] = torch.tensor([1, 0x81, 0x7E, 0xFE], dtype=torch.uint8, device="cuda")
    v.view(torch.uint8)[table[0, 0].long(), 1, 1, :4] = torch.tensor([1, 0x81, 0x7E, 0xFE], dtype=torch.uint8, device="cuda")
    plan = paged.QuantisedPlan(q_lens, kv_lens, 4, 2, 64)
    out, lse = paged.quantised_attention(plan, q, k, v, e, table, scale=2.0 ** -exponent / 8)
    o, ls, size = wanted((q, k, v, e, table), q_lens, kv_lens, 2.0 ** -exponent / 8)
    within(out, o, UNIT[dtype] * (o.abs() + size) * 1.01 + 1e-4 * size + SMALL[dtype])
    assert float((lse.double() - ls).abs().max()) < 1e-4
    # a sequence of one key gives its value as it is
    paged.quantised_attention(paged.QuantisedPlan([1], [1], 4, 2, 64), q[:1], k, v, e, table[:1])
    got = paged.quantised_attention(paged.QuantisedPlan([1], [1], 4, 2, 64), q[:1], k, v, e, table[:1])[0]
    assert torch.equal(got[0].float(), values(v, e[1])[table[0, 0].long(), 0].repeat_interleave(2, 0))


@pytest.mark.usefixtures("ways")
def test_pages_outside_the_cache_read_as_zeros():
    for n in (1, 64):
        q, k, v, e, table = make([n], [64], 4, 2, 64, 16)
        bad = table.clone()
        bad[0, 1], bad[0, 2] = -5, 2 ** 30
        zk, zv = k.clone(), v.clone()
        for z in (zk, zv):
            z.view(torch.uint8)[table[0, 1:3].long()] = 0
        plan = paged.QuantisedPlan([n], [64], 4, 2, 64)
        got = paged.quantised_attention(plan, q, k, v, e, bad)
        want = paged.quantised_attention(plan, q, zk, zv, e, table)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.usefixtures("ways")
@pytest.mark.parametrize("n", [4, 150])
def test_cache_beyond_32_bit_offsets(n):
    page, kv_heads, dim = 64, 8, 128
    pages = 2 ** 32 // (page * kv_heads * dim) + 8
    k, v = (torch.empty(pages, page, kv_heads, dim, dtype=E4M3, device="cuda") for _ in range(2))
    last = torch.tensor([[pages - 2, 1, pages - 1]], dtype=torch.int32, device="cuda")
    slots = torch.cat([torch.arange(p * page, p * page + page) for p in last[0].tolist()])[:150].int().cuda()
    g = generator()
    kn, vn = (torch.randn(150, kv_heads, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(150, 16, dim, generator=g, device="cuda").bfloat16()
    zero = torch.zeros(150, dtype=torch.int32, device="cuda")
    e = torch.full((2, kv_heads), -6, dtype=torch.int32, device="cuda")
    paged.norm_rotate_append(paged.Rotation(torch.zeros(4, device="cuda")), None, q, kn, vn, zero, slots, k, v, exponents=e)
    held = [c.view(torch.uint8)[last[0].long()].view(E4M3) for c in (k, v)]
    assert torch.equal(held[0].float().flatten(0, 1)[:150], (kn.float() * 64).to(E4M3).float())
    plan = paged.QuantisedPlan([n], [150], 16, kv_heads, dim)
    out, lse = paged.quantised_attention(plan, q[:n], k, v, e, last)
    plan.check()
    close(out, lse, wanted((q[:n], *held, e, torch.arange(3, device="cuda")[None]), [n], [150], dim ** -0.5), UNIT[q.dtype])


def test_attention_refuses():
    q, k, v, e, table = make([2], [64], 4, 2, 64, 16)
    plan = paged.QuantisedPlan([2], [64], 4, 2, 64)

    def refused(error, match, *args, **kw):
        with pytest.raises(error, match=match):
            paged.quantised_attention(plan, *args, **kw)

    refused(ValueError, "q:", q.float(), k, v, e, table)
    refused(ValueError, "k_cache", q, k.half(), v, e, table)
    refused(ValueError, "v_cache", q, k, v.to(torch.float8_e5m2), e, table)
    refused(ValueError, "q:", q[:1], k, v, e, table)
    refused(ValueError, "table", q, k, v, e, table.long())
    refused(ValueError, "table", q, k, v, e, table.repeat(2, 1))
    refused(ValueError, "exponents", q, k, v, e[:, :1], table)
    refused(ValueError, "exponents", q, k, v, e.long(), table)
    refused(ValueError, "different shapes", q, k, v[:, :8], e, table)
    refused(native.EmmyError, "does not hold", q, k, v, e, table[:, :3])
    refused(native.EmmyError, "scale", q, k, v, e, table, scale=0.0)
    refused(native.EmmyError, "page_size", q, k[:, :12], v[:, :12], e, table)
    odd = torch.zeros(2, 4, 68, dtype=q.dtype, device="cuda")[..., :64]
    refused(native.EmmyError, "stride", odd, k, v, e, table)
    refused(ValueError, "lse", q, k, v, e, table, lse=torch.empty(4, 2, device="cuda").t())
    refused(ValueError, "requires grad", q.clone().requires_grad_(), k, v, e, table)
    with pytest.raises(ValueError, match="AttentionPlan"):
        paged.attention(plan, q, k.bfloat16(), v.bfloat16(), table)


def test_no_tokens():
    q, k, v, e, table = make([0, 0], [64, 0], 4, 2, 64, 16)
    plan = paged.QuantisedPlan([0, 0], [64, 0], 4, 2, 64)
    out, lse = paged.quantised_attention(plan, q, k, v, e, table)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    plan.check()


@pytest.mark.usefixtures("ways")
def test_streams_and_graphs():
    q_lens, kv_lens = [1, 1, 140, 5], [5000, 77, 640, 300]
    made = make(q_lens, kv_lens, 8, 2, 128, 16)
    want = wanted(made, q_lens, kv_lens, 128 ** -0.5)
    plan = paged.QuantisedPlan(q_lens, kv_lens, 8, 2, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = paged.quantised_attention(plan, *made)
    side.synchronize()
    close(out, lse, want, UNIT[BF16])
    out2, lse2 = torch.empty_like(out), torch.empty_like(lse)
    paged.quantised_attention(plan, *made, out=out2, lse=lse2, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out2, out) and torch.equal(lse2, lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.quantised_attention(plan, *made, out=out2, lse=lse2)
    for _ in range(3):
        out2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out2, out) and torch.equal(lse2, lse)
    plan.check()


# ------------------------------------------------------------------ verify
def tried(counts, vocabulary, dtype=F32, proposed=True, seed=0, sharp=2.5):
    g = generator(seed)
    rows, drafts = sum(counts) + len(counts), sum(counts)
    first = torch.tensor([sum(counts[:s]) + s for s in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
    logits = torch.randn(rows, vocabulary, generator=g, device="cuda") * sharp
    judged = torch.tensor([i for s, m in enumerate(counts) for i in range(int(first[s]), int(first[s]) + m)], dtype=torch.long, device="cuda")
    proposal = (logits[judged] + 0.7 * torch.randn(drafts, vocabulary, generator=g, device="cuda")).softmax(-1)
    drafted = torch.multinomial(proposal, 1, generator=g)[:, 0].int() if drafts else first[:0]
    u, f = torch.rand(drafts, generator=g, device="cuda"), torch.rand(len(counts), generator=g, device="cuda")
    return logits.softmax(-1).to(dtype), proposal.to(dtype) if proposed else None, drafted, u, f, first


def by_definition(target, proposal, drafted, uniforms, finals, first):
    """In 64 bits on the host; the border nearest to a final, relative, as well."""
    p, q = target.double().cpu(), None if proposal is None else proposal.double().cpu()
    drafted, u, f, first = drafted.tolist(), uniforms.tolist(), finals.tolist(), first.tolist()
    accepted, tokens, nearest = [], [], 1.0
    for s, (begin, end) in enumerate(zip(first, first[1:])):
        n, kept = end - begin - 1, 0
        for i in range(n):
            x = drafted[begin - s + i]
            if not (0 <= x < p.shape[1]) or not u[begin - s + i] * (1.0 if q is None else float(q[begin - s + i, x])) < float(p[begin + i, x]):
                break
            kept += 1
        mass = p[begin + kept].nan_to_num(nan=0).clamp(min=0)
        if kept < n:
            rest = mass.clone()
            if q is not None:
                rest = (p[begin + kept] - q[begin - s + kept]).nan_to_num(nan=0).clamp(min=0)
            elif 0 <= drafted[begin - s + kept] < p.shape[1]:
                rest[drafted[begin - s + kept]] = 0
            mass = rest if rest.sum() > 0 else mass
        sums = mass.cumsum(0)
        past = (sums > f[s] * sums[-1]).nonzero()
        token = int(past[0]) if len(past) else (int(mass.nonzero()[-1]) if sums[-1] > 0 else -1)
        if sums[-1] > 0:
            nearest = min(nearest, float((sums / sums[-1] - f[s]).abs().min()))
        accepted.append(kept)
        tokens += drafted[begin - s:begin - s + kept] + [token] + [-1] * (n - kept)
    return accepted, tokens, nearest


def verified(made):
    accepted, tokens = paged.verify(*made)
    want = by_definition(*made)
    # (sums of 2^17 numbers in 64 bits in another order may differ by 2^17 2^-53)
    assert want[2] > 2.0 ** -35, "a final on a border"
    assert accepted.dtype is torch.int32 and accepted.tolist() == want[0]
    assert tokens.dtype is torch.int32 and tokens.tolist() == want[1]
    return accepted, tokens


@pytest.mark.parametrize("counts,vocabulary", [
    ([0], 1), ([1], 1), ([3], 2), ([4], 32000), ([0, 0, 0], 5), ([5, 0, 1, 8, 2], 257), ([2] * 7, 4096), ([1, 3] * 20, 4097), ([3, 1], 131071),
    ([i % 9 for i in range(150)], 1000), ([300, 2], 50), ([2] * 700, 300), ([1] * 80, 20011),
])
@pytest.mark.parametrize("proposed", [True, False])
def test_verify(counts, vocabulary, proposed):
    verified(tried(counts, vocabulary, proposed=proposed, seed=vocabulary))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("proposed", [True, False])
def test_verify_types(dtype, proposed):
    verified(tried([4, 0, 7, 1], 5003, dtype, proposed))


@pytest.mark.parametrize("seed", range(6))
def test_verify_distributions_near_and_far(seed):
    """Drafts that are mostly kept, mostly not, and a row that is one token."""
    verified(tried([5] * 30, 3001, seed=seed, sharp=(0.1, 1.0, 8.0)[seed % 3]))


def test_verify_strided_rows():
    made = list(tried([3, 4, 0], 999))
    for i in (0, 1):
        wide = torch.full((made[i].shape[0], 1203), 0.5, device="cuda")
        wide[:, 7:1006] = made[i]
        made[i] = wide[:, 7:1006]
    verified(made)


def test_verify_borders():
    """A product equal to the probability is not kept; the running sum has to exceed the final."""
    vocabulary = 1024
    p = torch.zeros(4, vocabulary, device="cuda")
    p[:, 3], p[:, 700], p[:, 1023] = 0.25, 0.5, 0.25
    q = torch.zeros(2, vocabulary, device="cuda")
    q[:, 3] = 0.5
    first = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    drafted = torch.tensor([3, 3], dtype=torch.int32, device="cuda")
    u = torch.tensor([0.5, 0.5 - 2.0 ** -25], device="cuda")           # 0.5 x 0.5 is 0.25; the other is below
    for f, want in ((0.0, [700, 3]), (0.25, [700, 700]), (0.75, [1023, 1023]), (2.0 / 3, [1023, 700]), (0.2499, [700, 3]), (1.0, [1023, 1023])):
        accepted, tokens = paged.verify(p, q, drafted, u, torch.tensor([f, f], device="cuda"), first)
        assert accepted.tolist() == [0, 1]
        # the first sequence draws from {700: 1/2, 1023: 1/4}, the second from p (2/3 in 32
        # bits is 2^-25 2/3 more, and 3/4 of it past 1/2)
        assert tokens.tolist() == [want[0], -1, 3, want[1]], f


def test_verify_nothing_left_or_not_a_number():
    vocabulary = 5000
    g = generator()
    p = torch.rand(2, vocabulary, generator=g, device="cuda").softmax(-1)
    first = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    drafted, u, f = torch.tensor([17], dtype=torch.int32, device="cuda"), torch.ones(1, device="cuda"), torch.full((1,), 0.4, device="cuda")
    # the proposal covers the target: drawn from the target
    verified([p, p[:1].clone(), drafted, u, f, first])
    verified([p, p[:1] * 2, drafted, u, f, first])
    # certain, and the whole target
    one = torch.zeros(2, vocabulary, device="cuda")
    one[:, 17] = 1
    verified([one, None, drafted, u, f, first])
    # drafts outside the vocabulary
    for x in (-1, vocabulary, 2 ** 31 - 1):
        verified([p, None, torch.tensor([x], dtype=torch.int32, device="cuda"), u * 0, f, first])
    # nothing to draw from, and values that are not numbers
    accepted, tokens = paged.verify(p * 0, p[:1], drafted, u, f, first)
    assert accepted.tolist() == [0] and tokens.tolist() == [-1, -1]
    broken = p.clone()
    broken[0, ::7] = math.nan
    verified([broken, p[:1], drafted, u, f, first])
    assert paged.verify(p * math.nan, p[:1], drafted, u, f, first)[1].tolist() == [-1, -1]


def test_verify_rows_that_are_not_there():
    """Entries of `first` that are no rows: nothing is read or written for those sequences."""
    made = list(tried([2, 3, 1], 100))
    good = verified(made)
    for change in ([0, 3, 3, 9], [0, 3, 2, 9], [-1, 3, 7, 9], [0, 3, 7, 10], [0, 2 ** 31 - 1, 7, 9], [0, 3, 7, -2 ** 31]):
        first = torch.tensor(change, dtype=torch.int32, device="cuda")
        accepted, _ = paged.verify(*made[:5], first)
        for s, (begin, end) in enumerate(zip(change, change[1:])):
            fine = 0 <= begin < end <= 9 and begin >= s and end - 1 - s <= 6
            assert (accepted[s] >= 0) == fine
        if change[:2] == [0, 3]:
            assert accepted[0] == good[0][0]


def test_verify_streams_and_graphs():
    made = tried([4, 1, 6], 40000)
    want = verified(made)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged.verify(*made)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = paged.verify(*made, stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged.verify(*made)
    for _ in range(3):
        for t in got:
            t.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_verify_refuses():
    p, q, drafted, u, f, first = tried([2, 1], 50)

    def refused(match, *args):
        with pytest.raises(ValueError, match=match):
            paged.verify(*args)

    refused("target", p.double(), q, drafted, u, f, first)
    refused("proposal", p, q.half(), drafted, u, f, first)
    refused("proposal", p, q[:2], drafted, u, f, first)
    refused("drafted", p, q, drafted.long(), u, f, first)
    refused("drafted", p, q, drafted[:2], u[:2], f, first)
    refused("uniforms", p, q, drafted, u[:2], f, first)
    refused("first", p, q, drafted, u, f, first[:2])
    refused("finals", p, q, drafted, u, f.double(), first)
    refused("innermost", p.t().contiguous().t(), q, drafted, u, f, first)
    refused("requires grad", p.clone().requires_grad_(), q, drafted, u, f, first)


def test_verify_no_sequences():
    e = torch.zeros(0, dtype=torch.int32, device="cuda")
    accepted, tokens = paged.verify(torch.zeros(0, 10, device="cuda"), None, e, e.float(), e.float(), torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert accepted.shape == (0,) and tokens.shape == (0,)


# ------------------------------------------------------------------ together
@pytest.mark.usefixtures("ways")
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_a_serving_step_with_drafts(dtype, dim):
    """Prompts into the 8-bit cache, attention of a step with drafts over it, and their
    verification, each on what the one before gave."""
    heads, kv_heads, page, prompts, counts, vocabulary = 8, 2, 16, [37, 150, 8], [3, 0, 5], 700
    g = generator(3)
    kv_lens = [p + n + 1 for p, n in zip(prompts, counts)]
    need = [-(-n // page) for n in kv_lens]
    table = torch.zeros(3, max(need), dtype=torch.int32)
    for s in range(3):
        table[s, :need[s]] = torch.arange(sum(need[:s]), sum(need[:s + 1]))
    table = table.flip(0).contiguous().flip(0).cuda()
    caches = [torch.zeros(sum(need), page, kv_heads, dim, device="cuda").to(E4M3) for _ in range(2)]
    exponents = torch.full((2, kv_heads), -5, dtype=torch.int32, device="cuda")
    rotation = paged.Rotation(10000.0 ** (-torch.arange(dim // 2, device="cuda") / (dim // 2)))
    w = [(torch.rand(dim, generator=g, device="cuda") + 0.5).to(dtype) for _ in range(2)]
    norm = paged.Norm(*w)
    x = [torch.randn(n, heads + 2 * kv_heads, dim, generator=g, device="cuda").to(dtype) for n in kv_lens]

    def append(parts, starts):
        at = torch.cat([torch.arange(b, b + len(y), device="cuda") for y, b in zip(parts, starts)]).int()
        seq = torch.cat([torch.full((len(y),), s, device="cuda") for s, y in enumerate(parts)])
        slots = table[seq, (at // page).long()] * page + at % page
        return paged.norm_rotate_append(rotation, norm, *torch.cat(parts).split([heads, kv_heads, kv_heads], 1), at, slots, *caches, exponents=exponents)

    append([y[:p] for y, p in zip(x, prompts)], [0] * 3)
    q = append([y[p:] for y, p in zip(x, prompts)], prompts)
    q_lens = [n + 1 for n in counts]
    plan = paged.QuantisedPlan(q_lens, kv_lens, heads, kv_heads, dim)
    out, lse = paged.quantised_attention(plan, q, *caches, exponents, table)
    close(out, lse, wanted((q, *caches, exponents, table), q_lens, kv_lens, dim ** -0.5), UNIT[dtype])
    # queries and keys by the formulas
    for s, (y, p) in enumerate(zip(x, prompts)):
        for part, weight, got in ((y[p:, :heads], w[0], q[sum(q_lens[:s]):][:q_lens[s]].double()),
                                  (y[:, heads:heads + kv_heads], w[1], values(caches[0].view(torch.uint8)[table[s, :need[s]].long()].view(E4M3), exponents[0])
                                   .flatten(0, 1)[:kv_lens[s]].double())):
            z = part.double()
            z = z / (z.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
            at = torch.arange(kv_lens[s] - len(z), kv_lens[s], device="cuda").double()[:, None] * rotation.frequencies.double()
            a, b = z.chunk(2, -1)
            cos, sin = at.cos()[:, None], at.sin()[:, None]
            z = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
            u = UNIT[dtype] if part.shape[1] == heads else 2.0 ** -4
            # (of an 8-bit float below its normal range, times 2^-5: 2^-15)
            within(got, z, u * z.abs() * 1.01 + (2.0 ** -15 if u > 0.01 else SMALL[dtype]) + 2.0 ** -16)
    head = (torch.randn(heads * dim, vocabulary, generator=g, device="cuda") * 0.2).to(dtype)
    target = (out.flatten(1) @ head).float().softmax(-1)
    first = torch.tensor([0, 4, 5, 11], dtype=torch.int32, device="cuda")
    drafted = torch.randint(0, vocabulary, (8,), generator=g, device="cuda", dtype=torch.int32)
    proposal = torch.full((8, vocabulary), 1.0 / vocabulary, device="cuda")
    verified([target, proposal, drafted, torch.rand(8, generator=g, device="cuda"), torch.rand(3, generator=g, device="cuda"), first])

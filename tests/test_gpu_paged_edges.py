"""The paged-cache operators on the GPU where their values or arguments are unusual."""
import math

import pytest
import torch

from emmy_b200 import native, paged
from test_gpu_paged import UNIT, close, definition, make

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------- infinite values
@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (64, torch.float16), (128, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("q_lens,kv_lens,heads,kv_heads", [
    ([1], [40], 8, 2), ([1, 1, 1, 1], [129, 300, 1000, 64], 8, 2), ([3, 2], [300, 500], 4, 4), ([20], [400], 8, 2),
    ([90], [700], 8, 2), ([1], [9000], 8, 1), ([1, 300], [640, 900], 6, 2)])
def test_infinite_values(dim, dtype, q_lens, kv_lens, heads, kv_heads):
    """An infinite value that every token of a chunk sees gives an infinite component,
    both signs of it NaN, and no other component, head or sequence is touched.  (Scores
    are within +-8 or so: no weight rounds to 0 in 16 bits.)"""
    q, k, v, table = make(q_lens, kv_lens, heads, kv_heads, dim, 16, dtype)
    for s, (n, length) in enumerate(zip(q_lens, kv_lens)):
        # each value of a component of its own, at keys all over a tile, in the last
        # head of keys; two meet in the last component
        seen = length - n + 1
        for i, j in enumerate(j for j in (0, 5, 33, 37, 64, 70, 96, 127, 128, 250, 299, 639, 8999) if j < seen):
            v[table[s, j // 16].long(), j % 16, -1, 3 * i] = math.inf if i % 2 else -math.inf
        for j, x in ((0, math.inf), (seen - 1, -math.inf)):
            v[table[s, j // 16].long(), j % 16, -1, dim - 1] = x
    plan = paged.AttentionPlan(q_lens, kv_lens, heads, kv_heads, dim)
    out, lse = paged.attention(plan, q, k, v, table)
    plan.check()
    o, ls, size = definition(q, k, v, table, q_lens, kv_lens, dim ** -0.5)
    special = ~o.isfinite()
    assert special.any()
    assert torch.equal(torch.nan_to_num(out.double(), nan=1.0, posinf=2.0, neginf=3.0)[special],
                       torch.nan_to_num(o, nan=1.0, posinf=2.0, neginf=3.0)[special])
    close(out.masked_fill(special, 0.0), lse, (o.masked_fill(special, 0.0), ls, size.masked_fill(special, 0.0)), UNIT[dtype])


@pytest.mark.parametrize("dim", [64, 128])
def test_infinite_values_outside_the_window(dim):
    """A decoding token's window hides them, whatever tile or page they share with it."""
    q_lens, kv_lens = [1, 1, 1], [300, 129, 1000]
    q, k, v, table = make(q_lens, kv_lens, 8, 2, dim, 16)
    for s, n in enumerate(kv_lens):
        for j in range(n - 100):
            for c, x in ((k, math.nan), (v, math.inf)):
                c[table[s, j // 16].long(), j % 16] = x
    plan = paged.AttentionPlan(q_lens, kv_lens, 8, 2, dim, window=100)
    out, lse = paged.attention(plan, q, k, v, table)
    plan.check()
    clean = [torch.nan_to_num(c, nan=0.0, posinf=0.0, neginf=0.0) for c in (k, v)]
    close(out, lse, definition(q, *clean, table, q_lens, kv_lens, dim ** -0.5, window=100), UNIT[q.dtype])


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim", [64, 128])
def test_keys_that_later_tokens_see(what, dim):
    """A key that is not finite spoils the tokens that see it only (their score is NaN
    or infinite), not the others of the chunk."""
    q_lens, kv_lens = [3, 20, 300, 1], [300, 171, 640, 77]
    q, k, v, table = make(q_lens, kv_lens, 8, 2, dim, 16)
    want = definition(q, k, v, table, q_lens, kv_lens, dim ** -0.5)
    clean = torch.ones(len(q), dtype=torch.bool, device="cuda")
    start = 0
    for s, (n, length) in enumerate(zip(q_lens, kv_lens)):
        j = length - 1 - n // 3                                # the last n // 3 + 1 tokens see it
        k[table[s, j // 16].long(), j % 16] = what
        start += n
        clean[start - n // 3 - 1:start] = False
    plan = paged.AttentionPlan(q_lens, kv_lens, 8, 2, dim)
    out, lse = paged.attention(plan, q, k, v, table)
    plan.check()
    close(out[clean], lse[clean], tuple(w[clean] for w in want), UNIT[q.dtype])
    if math.isnan(what):
        assert out[~clean].isnan().all() and lse[~clean].isnan().all()


# ---------------------------------------------------------------- large scores
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, n) for n in (20, 24, 27, 29, 33, 60, 112)] +
                         [(torch.float16, n) for n in (20, 24, 27, 29, 33)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 3, 20, 300, 9], [300, 40, 170, 900, 4]), ([1], [20000])])
@pytest.mark.parametrize("factor", [1.0, 181 / 128])
def test_scores_of_any_size(factor, q_lens, kv_lens, dim, dtype, size, sign):
    """Scores of +-factor * 2^size and half of that before they are scaled: exact, as
    every product of components has 8 bits, so a row's weights are equal over its largest
    ones.  Odd heads have scores of +-8 and so on in the same tiles.

    The logarithm carries the rounding of the scale, of its conversion to base 2, of the
    scaled score and of the way back: 8 roundings of 2^-24 of it."""
    heads, kv_heads = 8, 2
    q, k, v, table = make(q_lens, kv_lens, heads, kv_heads, dim, 16, dtype)
    b = min(12, size // 2)
    q[:, 0::2], q[:, 1::2] = 2.0 ** (size - b) / dim, 2.0 ** (3 - b) / dim
    g = torch.Generator(device="cuda").manual_seed(5)
    half = torch.rand(k.shape[:3], generator=g, device="cuda") < 0.5
    keys = torch.where(half, 2.0 ** (b - 1), 2.0 ** b) * (factor * sign)
    k.copy_(torch.where(k.isnan(), k.float(), keys[..., None]).to(dtype))
    assert q.isfinite().all() and (q > 0).all()
    plan = paged.AttentionPlan(q_lens, kv_lens, heads, kv_heads, dim)
    out, lse = paged.attention(plan, q, k, v, table)
    plan.check()
    o, ls, weighed = definition(q, k, v, table, q_lens, kv_lens, dim ** -0.5)
    assert torch.isfinite(out).all()
    u = UNIT[dtype]
    assert bool(((out.double() - o).abs() <= u * (o.abs() + weighed) * 1.01 + 1e-4 * weighed).all())
    empty = ls == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert bool(((lse.double() - ls).abs() <= 8 * 2.0 ** -24 * ls.abs() + 1e-4)[~empty].all())


# --------------------------------------------------------------------- windows
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 1, 2 ** 32 + 5, 2 ** 63])
@pytest.mark.parametrize("dim", [64, 128])
def test_windows_beyond_every_length(window, dim):
    q_lens, kv_lens = [10, 1, 300, 40], [4, 1000, 100, 640]
    made = make(q_lens, kv_lens, 8, 2, dim, 16)
    got = []
    for w in (None, window):
        plan = paged.AttentionPlan(q_lens, kv_lens, 8, 2, dim, window=w)
        got.append(paged.attention(plan, *made))
        plan.check()
    assert all(torch.equal(a, b) for a, b in zip(*got))
    close(*got[1], definition(*made, q_lens, kv_lens, dim ** -0.5), UNIT[torch.bfloat16])


# --------------------------------------------------------------------- numbers
def test_scales_out_of_range():
    made = make([2], [64], 4, 2, 64, 16)
    plan = paged.AttentionPlan([2], [64], 4, 2, 64)
    for scale in (1e39, 3e38, 1e-60, math.nan):
        with pytest.raises(native.EmmyError, match="scale"):
            paged.attention(plan, *made, scale=scale)
    with pytest.raises(ValueError, match="fit"):
        paged.attention(plan, *made, scale="1")


# ------------------------------------------------------------- nothing to read
@pytest.mark.parametrize("causal", [True, False])
def test_a_batch_without_keys_needs_no_cache(causal):
    q = torch.randn(5, 8, 64, device="cuda").bfloat16()
    plan = paged.AttentionPlan([2, 3], [0, 0], 8, 2, 64, causal=causal)
    for pages in (0, 3):
        cache = torch.zeros(pages, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
        for width in (0, 2):
            out, lse = paged.attention(plan, q, cache, cache, torch.zeros(2, width, dtype=torch.int32, device="cuda"),
                                       out=torch.full_like(q, 7.0))
            plan.check()
            assert not out.any() and bool((lse == -math.inf).all())


# ------------------------------------------------------------------- gave up
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 3], [9000, 70]), ([1, 300], [9000, 900]), ([300], [900])])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_plan_that_gave_up_stays_so(dim, q_lens, kv_lens):
    """Once a wait ran out (here: the word that says so is set), later calls with the plan write nothing."""
    made = make(q_lens, kv_lens, 8, 2, dim, 16)
    plan = paged.AttentionPlan(q_lens, kv_lens, 8, 2, dim)
    plan.words[0] = 2
    words = plan.words.clone()
    out, lse = torch.full_like(made[0], 7.0), torch.full(made[0].shape[:2], 7.0, device="cuda")
    paged.attention(plan, *made, out=out, lse=lse)
    with pytest.raises(native.EmmyError, match="ran out"):
        plan.check()
    assert bool((out == 7.0).all()) and bool((lse == 7.0).all()) and torch.equal(plan.words, words)
    plan.words[0] = 0
    paged.attention(plan, *made, out=out, lse=lse)
    plan.check()
    close(out, lse, definition(*made, q_lens, kv_lens, dim ** -0.5), UNIT[torch.bfloat16])


# ------------------------------------------------------------------ gradients
def _rotate_inputs():
    cache = [torch.zeros(4, 16, 2, 64, device="cuda") for _ in range(2)]
    q, k, v = (torch.randn(5, n, 64, device="cuda") for n in (4, 2, 2))
    at = torch.arange(5, dtype=torch.int32, device="cuda")
    return paged.Rotation(torch.ones(32, device="cuda")), q, k, v, at, at, *cache


@pytest.mark.parametrize("which", [1, 2, 3, 6, 7, "q_out", "frequencies"])
def test_rotate_append_has_no_backward(which):
    args, kw = list(_rotate_inputs()), {}
    if which == "q_out":
        kw["q_out"] = torch.zeros_like(args[1], requires_grad=True)
    elif which == "frequencies":
        args[0].frequencies.requires_grad_()
    else:
        args[which].requires_grad_()
    with pytest.raises(ValueError, match="backward"):
        paged.rotate_append(*args, **kw)
    with torch.no_grad():
        paged.rotate_append(*args, **kw)


@pytest.mark.parametrize("which", [0, 1, 2, "out", "lse"])
def test_attention_has_no_backward(which):
    args, kw = list(make([2], [64], 4, 2, 64, 16, poison=0.0)), {}
    plan = paged.AttentionPlan([2], [64], 4, 2, 64)
    if isinstance(which, str):
        kw[which] = torch.zeros((2, 4, 64) if which == "out" else (2, 4), device="cuda",
                                dtype=torch.bfloat16 if which == "out" else torch.float32, requires_grad=True)
    else:
        args[which].requires_grad_()
    with pytest.raises(ValueError, match="backward"):
        paged.attention(plan, *args, **kw)
    with torch.inference_mode():
        paged.attention(plan, *args, **kw)


# ------------------------------------------------------------------- versions
def test_what_is_written_is_known_to_autograd():
    """A tensor that another operation keeps for its gradient and that is then written here."""
    rotation, q, k, v, at, _, kc, vc = _rotate_inputs()
    for kept in (q, kc, vc):
        w = torch.ones_like(kept, requires_grad=True)
        y = (w * kept).sum()
        paged.rotate_append(rotation, q, k, v, at, at, kc, vc, q_out=q)
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    made = make([2], [64], 4, 2, 64, 16, poison=0.0)
    plan = paged.AttentionPlan([2], [64], 4, 2, 64)
    out, lse = torch.zeros_like(made[0]), torch.zeros(2, 4, device="cuda")
    for kept in (out, lse):
        w = torch.ones_like(kept, requires_grad=True)
        y = (w * kept).sum()
        paged.attention(plan, *made, out=out, lse=lse)
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    with torch.inference_mode():                   # tensors without a version counter
        out = torch.empty_like(made[0])
        paged.attention(plan, *made, out=out)

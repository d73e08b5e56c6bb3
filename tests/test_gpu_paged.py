"""The paged-cache operators on the GPU against their definitions in 64 bits.

Tolerances.  With u the unit roundoff of the 16-bit type (2^-8 bfloat16, 2^-11
float16): a weight rounded to 16 bits moves an output by at most u sum(p|v|)/l, the
final rounding by u|o|; 32-bit scores, exponentials and sums of these lengths stay
below 1e-4 of sum(p|v|)/l and, in the logarithm, below 1e-4.  A weight below
float16's normal range is off by 2^-25 at most where the largest is 2^6, far below
that.  A rotated component is off by u of itself, and by 2^-21 of its pair's
length from 32-bit arithmetic on cosines and sines of an angle reduced in 64."""
import math

import pytest
import torch

from emmy_b200 import native, paged

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


# ------------------------------------------------------------------ attention
def definition(q, k_cache, v_cache, table, q_lens, kv_lens, scale, causal=True, window=None):
    """(out, lse, sum(p|v|)/l) in 64 bits."""
    tokens, heads, dim = q.shape
    page, kv_heads = k_cache.shape[1:3]
    group = heads // kv_heads
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64, device=q.device)
    at = 0
    for s, (n, length) in enumerate(zip(q_lens, kv_lens)):
        if length and n:
            pages = table[s, :-(-length // page)].long()
            k = k_cache[pages].double().flatten(0, 1)[:length].repeat_interleave(group, 1)
            v = v_cache[pages].double().flatten(0, 1)[:length].repeat_interleave(group, 1)
            score = torch.einsum("nhd,khd->hnk", q[at:at + n].double(), k) * scale
            pos = torch.arange(length - n, length, device=q.device)[:, None]
            j = torch.arange(length, device=q.device)
            seen = torch.ones(n, length, dtype=torch.bool, device=q.device)
            if causal:
                seen &= j <= pos
            if window:
                seen &= j > pos - window
            score = score.masked_fill(~seen, -math.inf)
            any_ = seen.any(1)
            p = torch.where(any_[None, :, None], torch.softmax(score, -1), 0.0)
            out[at:at + n] = torch.einsum("hnk,khd->nhd", p, v)
            size[at:at + n] = torch.einsum("hnk,khd->nhd", p, v.abs())
            lse[at:at + n] = torch.logsumexp(score, -1).t()
        at += n
    return out, lse, size


def make(q_lens, kv_lens, heads, kv_heads, dim, page, dtype=torch.bfloat16, layout="token", seed=0, poison=math.nan,
         spare=3):
    """Inputs whose cache holds `poison` wherever no sequence has a token, and
    whose table has page numbers from nowhere after each sequence's last."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in kv_lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    width = max(need + [1]) + 2
    table = torch.full((len(kv_lens), width), -1, dtype=torch.int32)
    table[:, -1] = 2 ** 30
    shape = (pages, page, kv_heads, dim) if layout == "token" else (pages, kv_heads, page, dim)
    caches = []
    for _ in range(2):
        c = torch.full(shape, poison, dtype=dtype, device="cuda")
        caches.append(c if layout == "token" else c.transpose(1, 2))
    at = 0
    for s, n in enumerate(kv_lens):
        for i in range(need[s]):
            table[s, i] = order[at]
            rows = min(page, n - i * page)
            for c in caches:
                c[order[at], :rows] = torch.randn(rows, kv_heads, dim, generator=g, device="cuda").to(dtype)
            at += 1
    q = torch.randn(sum(q_lens), heads, dim, generator=g, device="cuda").to(dtype)
    return q, caches[0], caches[1], table.cuda()


def close(out, lse, want, u):
    o, ls, size = want
    assert torch.isfinite(out).all()
    bad = (out.double() - o).abs() > u * (o.abs() + size) * 1.01 + 1e-4 * size
    assert not bad.any(), (int(bad.sum()), float((out.double() - o).abs().max()))
    empty = ls == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    d = (lse.double() - ls)[~empty].abs()
    assert d.numel() == 0 or float(d.max()) < 1e-4, float(d.max())


def check(q_lens, kv_lens, heads, kv_heads, dim, page, dtype=torch.bfloat16, layout="token", causal=True, window=None,
          scale=None, ctas=None, seed=0, q=None):
    made = make(q_lens, kv_lens, heads, kv_heads, dim, page, dtype, layout, seed)
    q = made[0] if q is None else q
    plan = paged.AttentionPlan(q_lens, kv_lens, heads, kv_heads, dim, causal, window, ctas=ctas)
    out, lse = paged.attention(plan, q, *made[1:], scale=scale)
    plan.check()
    want = definition(q, *made[1:], q_lens, kv_lens, scale or dim ** -0.5, causal, window)
    close(out, lse, want, UNIT[dtype])
    return plan, made, out, lse


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout,page", [("token", 16), ("head", 64), ("token", 8), ("head", 128), ("token", 384)])
def test_decode_types_pages_layouts(dim, dtype, layout, page):
    check([1] * 9, [1, 127, 128, 129, 255, 256, 257, 640, 1000], 16, 4, dim, page, dtype, layout)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (6, 2), (5, 1), (40, 8), (16, 1), (128, 1), (65, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_head_groups(heads, kv_heads, dim):
    check([1, 3, 40, 129], [300, 3, 170, 513], heads, kv_heads, dim, 32)


@pytest.mark.parametrize("q_lens,kv_lens", [
    ([128], [128]), ([129], [129]), ([256], [1024]), ([257], [300]), ([1, 200, 1, 31, 64], [900, 200, 1, 600, 65]),
    ([500, 1, 333], [500, 2000, 777]),
])
@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_chunks(q_lens, kv_lens, dim, dtype):
    check(q_lens, kv_lens, 8, 4, dim, 16, dtype)


@pytest.mark.parametrize("window", [1, 7, 128, 200, 5000])
@pytest.mark.parametrize("dim", [64, 128])
def test_window(window, dim):
    check([1, 300, 5, 129], [1500, 1000, 5, 640], 8, 2, dim, 16, window=window)


@pytest.mark.parametrize("dim", [64, 128])
def test_every_token_sees_all(dim):
    check([1, 40, 300], [300, 129, 555], 8, 2, dim, 32, causal=False)


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_see_nothing(dim):
    """No keys at all, more new tokens than keys, sequences without new tokens."""
    for causal in (True, False):
        _, _, out, lse = check([2, 9, 0, 300, 1], [0, 4, 50, 100, 0], 8, 2, dim, 16, causal=causal)
        assert not out[:2].any() and bool((lse[:2] == -math.inf).all())
        if causal:
            assert not out[2:7].any() and bool((lse[2:7] == -math.inf).all())


@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("q_lens,kv_lens,heads,kv_heads", [
    ([1], [20000], 8, 1), ([3], [9000], 8, 8), ([70], [12000], 8, 4), ([1, 90], [40000, 6000], 16, 2)])
def test_split_over_keys(dim, dtype, q_lens, kv_lens, heads, kv_heads):
    """Few rows and many keys: parts joined by the last to arrive, the same bits
    on every call, the counters left as they were."""
    plan, made, out, lse = check(q_lens, kv_lens, heads, kv_heads, dim, 64, dtype)
    words = plan.words.clone()
    assert plan.scratch.numel() > 0
    for _ in range(5):
        again = paged.attention(plan, *made)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    assert torch.equal(plan.words, words)


@pytest.mark.parametrize("ctas", [1, 3, 37])
def test_few_ctas(ctas):
    """Many units a CTA, wide and narrow ones in turn."""
    check([1, 150, 1, 1, 300, 2, 64], [800, 150, 3, 0, 650, 129, 1000], 8, 2, 128, 32, ctas=ctas)
    check([1, 150, 1, 1, 300, 2, 64], [800, 150, 3, 0, 650, 129, 1000], 8, 2, 64, 32, torch.float16, ctas=ctas)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_that_grow(dim, dtype):
    """The running maximum moves far in every tile, up or down, and the scores
    are large: the base moves, outputs and sums with it."""
    for direction in (1, -1):
        q_lens, kv_lens = [2, 200], [1500, 900]
        q, k, v, table = make(q_lens, kv_lens, 4, 2, dim, 16, dtype)
        q.copy_(q.abs() + 0.5)
        for s, n in enumerate(kv_lens):
            j = torch.arange(n, device="cuda")
            size = (j if direction > 0 else n - j).float() / n * 6
            pages = table[s, :-(-n // 16)].long()
            k[pages[j // 16], j % 16] = (k[pages[j // 16], j % 16].float().abs() * size[:, None, None]).to(dtype)
        plan = paged.AttentionPlan(q_lens, kv_lens, 4, 2, dim)
        out, lse = paged.attention(plan, q, k, v, table, scale=0.5)
        plan.check()
        o, ls, size = definition(q, k, v, table, q_lens, kv_lens, 0.5)
        # scores reach 2^9: 32-bit products and sums put 128 x 2^-24 x 2^9 = 4e-3 on the exponent
        u = UNIT[dtype]
        assert bool(((out.double() - o).abs() <= u * (o.abs() + size) * 1.01 + 8e-3 * size).all())
        assert float((lse.double() - ls).abs().max()) < 8e-3


def test_strided_views_and_given_outputs():
    q_lens, kv_lens = [3, 130], [200, 300]
    q, k, v, table = make(q_lens, kv_lens, 8, 2, 64, 16)
    joined = torch.randn(sum(q_lens), 12, 64, device="cuda").bfloat16()
    joined[:, 2:10] = q
    view = joined[:, 2:10]
    wide_k = torch.full((k.shape[0], k.shape[1], 4, 64), math.nan, dtype=k.dtype, device="cuda")
    wide_k[:, :, 1:3] = k
    frame = torch.full((sum(q_lens) + 2, 10, 64), 7.0, dtype=q.dtype, device="cuda")
    out, lse = frame[1:-1, 1:9], torch.empty(sum(q_lens), 8, device="cuda")
    wide_table = torch.full((2, table.shape[1] + 5), -9, dtype=torch.int32, device="cuda")
    wide_table[:, :table.shape[1]] = table
    plan = paged.AttentionPlan(q_lens, kv_lens, 8, 2, 64)
    got = paged.attention(plan, view, wide_k[:, :, 1:3], v, wide_table[:, :table.shape[1]], out=out, lse=lse)
    plan.check()
    assert got[0] is out and got[1] is lse
    close(out, lse, definition(q, k, v, table, q_lens, kv_lens, 0.125), UNIT[q.dtype])
    frame[1:-1, 1:9] = 7.0
    assert bool((frame == 7.0).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_lens,kv_lens,heads,kv_heads", [
    ([40, 1, 7, 18], [40, 33, 9, 18], 8, 2), ([1, 1, 2, 4], [3, 8, 16, 40], 4, 4), ([40, 40], [40, 40], 10, 2),
])
def test_lse_to_the_last_bits(q_lens, kv_lens, heads, kv_heads, dim, dtype):
    """Components of -2..2, so products and their sums are exact and a row's largest
    weights can stand at any key.  What is left: the exponentials (2^-22 from the unit,
    at most 2.7e-6 where a polynomial forms them), the sum's n roundings, and a few of
    2^-24 of the scores and the result."""
    q, k, v, table = make(q_lens, kv_lens, heads, kv_heads, dim, 16, dtype)
    q, k = (torch.nan_to_num(x).clamp(-2, 2).round() for x in (q, k))
    plan = paged.AttentionPlan(q_lens, kv_lens, heads, kv_heads, dim)
    lse = paged.attention(plan, q, k, v, table)[1]
    want = definition(q, k, torch.nan_to_num(v), table, q_lens, kv_lens, dim ** -0.5)[1]
    most = 4.0 * dim * dim ** -0.5
    assert bool(((lse.double() - want).abs() <= 2.7e-6 + 2.0 ** -22 + (max(kv_lens) + 4 * most + 8) * 2.0 ** -24).all())


def test_streams_and_graphs():
    q_lens, kv_lens = [1, 1, 5], [5000, 77, 640]
    made = make(q_lens, kv_lens, 8, 2, 128, 16)
    want = definition(*made, q_lens, kv_lens, 128 ** -0.5)
    plan = paged.AttentionPlan(q_lens, kv_lens, 8, 2, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = paged.attention(plan, *made)
    side.synchronize()
    close(out, lse, want, UNIT[torch.bfloat16])
    out2, lse2 = torch.empty_like(out), torch.empty_like(lse)
    paged.attention(plan, *made, out=out2, lse=lse2, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out2, out) and torch.equal(lse2, lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attention(plan, *made, out=out2, lse=lse2)
    for _ in range(3):
        out2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out2, out) and torch.equal(lse2, lse)
    plan.check()


@pytest.mark.parametrize("given", [False, True])
def test_memory_of_a_dropped_plan_waits_for_its_stream(given):
    """The allocator's own list says so: nothing is written to memory that a kernel may still use."""
    made = make([1], [20000], 8, 2, 128, 16)
    side = torch.cuda.Stream()
    plan = paged.AttentionPlan([1], [20000], 8, 2, 128)
    rotation = paged.Rotation(torch.ones(32, device="cuda") * 0.5, axes=[0] * 16 + [1] * 16)
    assert plan.scratch.numel()
    used = {t.data_ptr() for t in (plan.scratch, plan.words, rotation.frequencies, rotation.pair_axis)}
    at = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    out, lse = torch.empty_like(made[0]), torch.empty(1, 8, device="cuda")
    turned = torch.empty_like(made[0])
    kv = torch.zeros(1, 2, 128, dtype=made[0].dtype, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.current_stream() if given else side):
        how = dict(stream=side.cuda_stream) if given else {}
        paged.rotate_append(rotation, made[0], kv, kv, at, at[0], made[1], made[2], q_out=turned, **how)
        paged.attention(plan, *made, out=out, lse=lse, **how)
    del plan, rotation
    states = {}
    for segment in torch.cuda.memory_snapshot():
        address = segment["address"]
        for block in segment["blocks"]:
            states[address] = block["state"]
            address += block["size"]
    side.synchronize()
    assert [states.get(a) for a in used] == ["active_pending_free"] * 4


def test_pages_outside_the_cache_read_as_zeros():
    q, k, v, table = make([1], [64], 4, 2, 64, 16)
    bad = table.clone()
    bad[0, 1], bad[0, 2] = -5, 2 ** 30
    zk, zv = k.clone(), v.clone()
    zk[table[0, 1:3].long()], zv[table[0, 1:3].long()] = 0, 0
    plan = paged.AttentionPlan([1], [64], 4, 2, 64)
    got = paged.attention(plan, q, k, v, bad)
    want = paged.attention(plan, q, zk, zv, table)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_cache_beyond_32_bit_offsets():
    """Pages whose elements lie past 2^32 in the cache."""
    page, kv_heads, dim = 64, 8, 128
    pages = (2 ** 32) // (page * kv_heads * dim) + 8
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.empty(pages, page, kv_heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    last = torch.tensor([[pages - 2, 1, pages - 1]], dtype=torch.int32, device="cuda")
    slots = torch.cat([torch.arange(p * page, p * page + page) for p in last[0].tolist()])[:150].int().cuda()
    kn, vn = (torch.randn(150, kv_heads, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(150, 16, dim, generator=g, device="cuda").bfloat16()
    rotation = paged.Rotation(torch.zeros(4, device="cuda"))
    paged.rotate_append(rotation, q, kn, vn, torch.zeros(150, dtype=torch.int32, device="cuda"), slots, k, v)
    assert torch.equal(k[last[0].long()].flatten(0, 1)[:150], kn)
    plan = paged.AttentionPlan([4], [150], 16, kv_heads, dim)
    out, lse = paged.attention(plan, q[:4], k, v, last)
    plan.check()
    close(out, lse, definition(q[:4], k, v, last, [4], [150], dim ** -0.5), UNIT[q.dtype])


def test_attention_refuses():
    q, k, v, table = make([2], [64], 4, 2, 64, 16)
    plan = paged.AttentionPlan([2], [64], 4, 2, 64)

    def refused(error, match, *args, **kw):
        with pytest.raises(error, match=match):
            paged.attention(plan, *args, **kw)

    refused(ValueError, "q:", q.float(), k, v, table)
    refused(ValueError, "k_cache", q, k.half(), v, table)
    refused(ValueError, "q:", q[:1], k, v, table)
    refused(ValueError, "table", q, k, v, table.long())
    refused(ValueError, "table", q, k, v, table.repeat(2, 1))
    refused(ValueError, "innermost", q, k.transpose(2, 3).contiguous().transpose(2, 3), v, table)
    refused(ValueError, "different shapes", q, k, v[:, :8], table)
    refused(native.EmmyError, "does not hold", q, k, v, table[:, :3])
    refused(native.EmmyError, "scale", q, k, v, table, scale=0.0)
    refused(native.EmmyError, "scale", q, k, v, table, scale=math.inf)
    refused(native.EmmyError, "page_size", q, k[:, :12], v[:, :12], table)
    refused(native.EmmyError, "page_size", q, k[:, :4], v[:, :4], table.repeat(1, 8))
    wide = torch.zeros(2 * 4 * 64 + 8, dtype=q.dtype, device="cuda")
    refused(native.EmmyError, "16 bytes", wide[1:513].view(2, 4, 64), k, v, table)
    odd = torch.zeros(2, 4, 68, dtype=q.dtype, device="cuda")[..., :64]
    refused(native.EmmyError, "stride", odd, k, v, table)
    refused(ValueError, "lse", q, k, v, table, lse=torch.empty(4, 2, device="cuda").t())


def test_no_tokens():
    q, k, v, table = make([0, 0], [64, 0], 4, 2, 64, 16)
    plan = paged.AttentionPlan([0, 0], [64, 0], 4, 2, 64)
    out, lse = paged.attention(plan, q, k, v, table)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    plan.check()


# ------------------------------------------------------------------ rotate_append
def turned(x, positions, frequencies, axes, interleaved):
    y = x.double().clone()
    n = len(frequencies)
    a, b = (torch.arange(n) * 2, torch.arange(n) * 2 + 1) if interleaved else (torch.arange(n), torch.arange(n) + n)
    angle = positions.double()[torch.tensor(axes, dtype=torch.long)].t() * frequencies.double()
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    y[..., a] = x.double()[..., a] * cos - x.double()[..., b] * sin
    y[..., b] = x.double()[..., b] * cos + x.double()[..., a] * sin
    length = torch.zeros_like(y)
    length[..., a] = length[..., b] = (x.double()[..., a] ** 2 + x.double()[..., b] ** 2).sqrt()
    return y, length


def rotated(tokens, heads, kv_heads, dim, rotary, page, dtype=torch.bfloat16, layout="token", axes=None, interleaved=False,
            reach=1 << 20, joined=True, offset=0, in_place=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    total = heads + 2 * kv_heads
    flat = torch.randn(tokens * total * dim + offset, generator=g, device="cuda").to(dtype)
    x = flat[offset:].view(tokens, total, dim)
    q, k, v = x.split([heads, kv_heads, kv_heads], 1)
    if not joined:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    freq = 10000.0 ** -(torch.arange(rotary // 2, device="cuda", dtype=torch.float64) / max(1, rotary // 2))
    freq = freq.float()
    pair_axes = [0] * (rotary // 2) if axes is None else [i * axes // (rotary // 2) for i in range(rotary // 2)]
    n_axes = max(pair_axes, default=0) + 1
    positions = torch.randint(-5, reach, (n_axes, tokens), generator=g, device="cuda", dtype=torch.int32)
    pages = tokens // page + 3
    shape = (pages, page, kv_heads, dim) if layout == "token" else (pages, kv_heads, page, dim)
    caches = [torch.full(shape, 3.0, dtype=dtype, device="cuda") for _ in range(2)]
    if layout == "head":
        caches = [c.transpose(1, 2) for c in caches]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].int()
    if tokens > 2:
        slots[0], slots[tokens // 2] = -1, pages * page      # stored nowhere
    want_q, len_q = turned(q, positions, freq, pair_axes, interleaved)
    want_k, len_k = turned(k, positions, freq, pair_axes, interleaved)
    want = [torch.full((pages * page, kv_heads, dim), 3.0, dtype=torch.float64, device="cuda") for _ in range(2)]
    slack = torch.zeros_like(want[0])
    kept = (slots >= 0) & (slots < pages * page)
    at = slots[kept].long()
    want[0][at], slack[at], want[1][at] = want_k[kept], len_k[kept], v[kept].double()
    rotation = paged.Rotation(freq, None if axes is None else pair_axes, interleaved)
    before = x.clone()
    out = paged.rotate_append(rotation, q, k, v, positions[0] if n_axes == 1 else positions, slots, *caches,
                              q_out=q if in_place else None)
    u = UNIT[dtype]
    assert bool(((out.double() - want_q).abs() <= u * want_q.abs() * 1.001 + 2.0 ** -21 * len_q).all())
    got_k, got_v = (c.reshape(pages * page, kv_heads, dim) for c in caches)
    assert bool(((got_k.double() - want[0]).abs() <= u * want[0].abs() * 1.001 + 2.0 ** -21 * slack).all())
    assert torch.equal(got_v.double(), want[1])
    # the components that do not turn, and what no token goes to, to the bit
    if in_place:
        assert out is q
    else:
        assert torch.equal(x, before)
    assert torch.equal(out[..., rotary:].double(), want_q[..., rotary:])
    assert torch.equal(got_k[..., rotary:].double(), want[0][..., rotary:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (64, 64), (128, 32), (96, 64), (80, 20), (7, 6), (64, 0), (33, 2), (1, 0)])
def test_rotation_dims(dtype, interleaved, dim, rotary):
    rotated(37, 6, 2, dim, rotary, 16, dtype, interleaved=interleaved)


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 32, 8), (3, 1, 1), (1025, 8, 1), (130, 5, 5)])
@pytest.mark.parametrize("layout,page", [("token", 16), ("head", 5), ("token", 1)])
def test_rotation_tokens_and_layouts(tokens, heads, kv_heads, layout, page):
    rotated(tokens, heads, kv_heads, 64, 64, page, layout=layout)


@pytest.mark.parametrize("axes", [2, 3])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_axes(axes, interleaved):
    rotated(200, 8, 2, 128, 96, 16, torch.float16, axes=axes, interleaved=interleaved)


@pytest.mark.parametrize("offset", [0, 1, 4])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_alignment_and_in_place(offset, interleaved):
    """Addresses off the 16-byte grid, with a joint projection's strides."""
    rotated(50, 4, 2, 64, 32, 8, offset=offset, interleaved=interleaved)
    rotated(50, 4, 2, 64, 32, 8, offset=offset, interleaved=interleaved, in_place=True)
    rotated(50, 4, 2, 64, 32, 8, offset=offset, interleaved=interleaved, joined=False)


def test_rotation_far_positions():
    rotated(64, 2, 1, 64, 64, 16, torch.float32, reach=2 ** 31 - 1)


def test_rotation_streams_and_nothing_to_do():
    rotation = paged.Rotation(torch.ones(32, device="cuda"))
    cache = [torch.zeros(4, 16, 2, 64, device="cuda") for _ in range(2)]
    empty = torch.zeros(0, 4, 64, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert paged.rotate_append(rotation, empty, empty[:, :2], empty[:, :2], none, none, *cache).shape == (0, 4, 64)
    q, kv = torch.randn(5, 4, 64, device="cuda"), torch.randn(5, 2, 64, device="cuda")
    at = torch.arange(5, dtype=torch.int32, device="cuda")
    want = paged.rotate_append(rotation, q, kv, kv, at, at, *cache)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(q)
    paged.rotate_append(rotation, q, kv, kv, at, at, *cache, q_out=out, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, want)


def test_rotate_append_refuses():
    freq = torch.ones(32, device="cuda")
    rotation = paged.Rotation(freq, axes=[0] * 16 + [1] * 16)
    cache = [torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.float16) for _ in range(2)]
    q, kv = (torch.zeros(5, n, 64, device="cuda", dtype=torch.float16) for n in (4, 2))
    pos, at = torch.zeros(2, 5, dtype=torch.int32, device="cuda"), torch.arange(5, dtype=torch.int32, device="cuda")

    def refused(error, match, *args, **kw):
        with pytest.raises(error, match=match):
            paged.rotate_append(*args, **kw)

    refused(ValueError, "positions", rotation, q, kv, kv, pos[0], at, *cache)
    refused(ValueError, "positions", rotation, q, kv, kv, pos.long(), at, *cache)
    refused(ValueError, "slots", rotation, q, kv, kv, pos, at[:4], *cache)
    refused(ValueError, "k:", rotation, q, kv.float(), kv, pos, at, *cache)
    refused(ValueError, "fit", rotation, q, kv[:, :1], kv[:, :1], pos, at, *cache)
    refused(ValueError, "q:", rotation, q.double(), kv, kv, pos, at, *cache)
    refused(ValueError, "k_cache", rotation, q, kv, kv, pos, at, cache[0].cpu(), cache[1])
    refused(ValueError, "q_out", rotation, q, kv, kv, pos, at, *cache, q_out=q[:4])
    refused(native.EmmyError, "rotary_dim", paged.Rotation(torch.ones(33, device="cuda")), q, kv, kv, pos, at, *cache)
    with pytest.raises(ValueError, match="entries"):
        paged.Rotation(freq, axes=[0] * 31 + [16])
    with pytest.raises(ValueError, match="32 pairs"):
        paged.Rotation(freq, axes=[0])

"""The 8-bit cache's operators where calls, streams, graphs and caches meet."""
import math

import pytest
import torch

from emmy_b200 import native, paged
from test_gpu_paged import UNIT, close
from test_gpu_paged_streams import PENDING, states
from test_gpu_quantised import BF16, E4M3, F16, make, wanted, ways  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

# few query rows of a key head (of 2 each), those that are widened, and those read back
FEW, MIDDLE, MANY = [5], [30], [200]


def plan_and_inputs(q_lens, kv_lens, dim=128, heads=8, kv_heads=2, page=16, dtype=BF16, seed=0, **how):
    return paged.QuantisedPlan(q_lens, kv_lens, heads, kv_heads, dim, **how), make(q_lens, kv_lens, heads, kv_heads, dim, page, dtype, seed=seed)


@pytest.mark.parametrize("dim,kv_heads,dtype", [(128, 8, BF16), (64, 16, F16)])
@pytest.mark.parametrize("window", [None, 16500])
def test_every_kernel_in_one_call(dim, kv_heads, dtype, window):
    """Sequences of more than the 32 MiB that go with those read back: few rows, more, many; in a graph as well."""
    q_lens, kv_lens = [1, 20, 300, 2, 0], [17000, 17001, 900, 2500, 40]
    made = make(q_lens, kv_lens, 2 * kv_heads, kv_heads, dim, 64, dtype)
    plan = paged.QuantisedPlan(q_lens, kv_lens, 2 * kv_heads, kv_heads, dim, window=window)
    want = wanted(made, q_lens, kv_lens, dim ** -0.5, True, window)
    out, lse = paged.quantised_attention(plan, *made)
    close(out, lse, want, UNIT[dtype])
    out2, lse2 = torch.empty_like(out), torch.empty_like(lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.quantised_attention(plan, *made, out=out2, lse=lse2)
    for _ in range(3):
        out2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out2, out) and torch.equal(lse2, lse)
    plan.check()


@pytest.mark.parametrize("q_lens", [FEW, MIDDLE, MANY])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_plan_that_gave_up_stays_so(q_lens, dim):
    """Once a wait ran out (here: the word that says so is set), later calls with the plan write nothing."""
    group = 2
    plan, made = plan_and_inputs(q_lens, [2000], dim, 2 * group, 2, ctas=3)      # (too few for all to be few)
    status = 3 if q_lens is FEW else 16       # its own, or the first word of the other kernel's plan behind it
    plan.words[status] = 2
    out, lse = torch.full_like(made[0], 7.0), torch.full(made[0].shape[:2], 7.0, device="cuda")
    paged.quantised_attention(plan, *made, out=out, lse=lse)
    with pytest.raises(native.EmmyError, match="ran out"):
        plan.check()
    assert bool((out == 7.0).all()) and bool((lse == 7.0).all())
    plan.words[status] = 0
    paged.quantised_attention(plan, *made, out=out, lse=lse)
    plan.check()
    close(out, lse, wanted(made, q_lens, [2000], dim ** -0.5), UNIT[BF16])


@pytest.mark.parametrize("heads,kv_heads,tokens", [(127, 1, 4), (127, 1, 5), (127, 1, 30), (96, 1, 7), (100, 2, 6), (100, 2, 9), (39, 3, 40), (3, 1, 900)])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_rows_of_little_work(heads, kv_heads, tokens, dim):
    """Groups that are no powers of two, whose rows are many."""
    for n in (tokens, tokens + 200):
        plan, made = plan_and_inputs([tokens], [n], dim, heads, kv_heads)
        close(*paged.quantised_attention(plan, *made), wanted(made, [tokens], [n], dim ** -0.5), UNIT[BF16])


@pytest.mark.usefixtures("ways")
@pytest.mark.parametrize("q_lens", [[1] * 3, [30, 25, 20], [300, 200, 1]])
@pytest.mark.parametrize("dim", [64, 128])
def test_sequences_that_share_pages(q_lens, dim):
    """A common beginning, its pages in every sequence's row."""
    kv_lens, page = [700, 900, 640], 32
    plan, (q, k, v, e, table) = plan_and_inputs(q_lens, kv_lens, dim, 8, 2, page)
    table[1:, :18] = table[0, :18]
    made = (q, k, v, e, table)
    close(*paged.quantised_attention(plan, *made), wanted(made, q_lens, kv_lens, dim ** -0.5), UNIT[BF16])


@pytest.mark.usefixtures("ways")
@pytest.mark.parametrize("tokens", [1, 20, 200])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [8, 64])
def test_pages_before_the_window_may_be_anything(tokens, dim, page):
    """Given back to the cache and taken by others: not numbers, or page numbers from nowhere."""
    n, window = 3000, 500
    plan, (q, k, v, e, table) = plan_and_inputs([tokens], [n], dim, 8, 2, page, window=window)
    want = wanted((q, k, v, e, table), [tokens], [n], dim ** -0.5, True, window)
    gone = (n - tokens - window + 1) // page              # whole pages that no token sees
    assert gone > 2
    for c in (k, v):
        c.view(torch.uint8)[table[0, : gone - 1].long()] = 0x7f
    table[0, gone - 1] = 2 ** 29
    table[0, 0] = -7
    close(*paged.quantised_attention(plan, q, k, v, e, table), want, UNIT[BF16])


@pytest.mark.usefixtures("ways")
def test_two_plans_on_two_streams():
    """Graphs of two plans replayed at once, and exponents that change between replays."""
    shapes = [([1, 9, 70], [9000, 3000, 400]), ([200, 1], [1200, 7000])]
    cases = [plan_and_inputs(q, n, 128, 8, 2, 16, seed=i) for i, (q, n) in enumerate(shapes)]
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [(torch.empty_like(made[0]), torch.empty(made[0].shape[:2], device="cuda")) for _, made in cases]
    graphs = []
    for (plan, made), (out, lse) in zip(cases, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged.quantised_attention(plan, *made, out=out, lse=lse)
        graphs.append(graph)
    for step in range(3):
        for _, made in cases:
            made[3].sub_(step)
        torch.cuda.synchronize()
        for _ in range(4):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for (q_lens, kv_lens), (plan, made), (out, lse) in zip(shapes, cases, outs):
            close(out, lse, wanted(made, q_lens, kv_lens, 128 ** -0.5), UNIT[BF16])
            plan.check()


@pytest.mark.usefixtures("ways")
def test_results_are_the_same_every_time():
    for q_lens in ([1] * 20, [9] * 20, [40] * 20, [200] * 4):
        kv_lens = [2000 + 300 * i for i in range(len(q_lens))]
        plan, made = plan_and_inputs(q_lens, kv_lens, 128, 8, 2, 32)
        out, lse = paged.quantised_attention(plan, *made)
        for _ in range(5):
            again = paged.quantised_attention(plan, *made)
            assert torch.equal(again[0], out) and torch.equal(again[1], lse)


def test_a_slot_of_two_tokens():
    """Either token's keys and values, 8 components at a time."""
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(64, n, 128, generator=g, device="cuda").bfloat16() for n in (8, 2, 2))
    rotation, at = paged.Rotation(torch.ones(32, device="cuda")), torch.zeros(64, dtype=torch.int32, device="cuda")
    once, twice = ([torch.zeros(4, 16, 2, 128, device="cuda").to(E4M3) for _ in range(2)] for _ in range(2))
    paged.norm_rotate_append(rotation, None, q, k, v, at, torch.arange(64, dtype=torch.int32, device="cuda"), *once)
    paged.norm_rotate_append(rotation, None, q, k, v, at, torch.arange(64, dtype=torch.int32, device="cuda") // 2, *twice)
    for a, b in zip(once, twice):
        a, b = (t.view(torch.uint8).view(64, 2, 16, 8) for t in (a, b))
        assert bool(((b[:32] == a[0::2]).all(-1) | (b[:32] == a[1::2]).all(-1)).all())
        assert not b[32:].any()


# ------------------------------------------------------------------ memory, autograd
def test_memory_of_what_is_dropped_waits_for_the_other_stream():
    """A plan and a norm, made under one stream, used on the other, dropped."""
    plan, made = plan_and_inputs([1], [20000])
    assert plan.scratch.numel()
    weights = [torch.ones(128, dtype=BF16, device="cuda") for _ in range(2)]
    norm, rotation = paged.Norm(*weights), paged.Rotation(torch.ones(64, device="cuda"))
    q, kv, at = made[0], torch.ones(1, 2, 128, dtype=BF16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse, turned = torch.empty_like(q), torch.empty(1, 8, device="cuda"), torch.empty_like(q)
    used = {t.data_ptr() for t in (plan.scratch, plan.words, *weights)}
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        paged.norm_rotate_append(rotation, norm, q, kv, kv, at, at, made[1], made[2], q_out=turned)
        paged.quantised_attention(plan, *made, out=out, lse=lse)
    del plan, norm, weights
    got = states()
    torch.cuda.synchronize()
    assert [got.get(a) for a in used] == [PENDING] * 4


def test_what_is_written_is_known_to_autograd():
    """A tensor that another operation keeps for its gradient and that is then written here."""
    plan, made = plan_and_inputs([2], [64], 64, 4, 2)
    out, lse = torch.zeros_like(made[0]), torch.zeros(2, 4, device="cuda")
    for kept in (out, lse):
        w = torch.ones_like(kept, requires_grad=True)
        y = (w * kept).sum()
        paged.quantised_attention(plan, *made, out=out, lse=lse)
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    with torch.inference_mode():                   # tensors without a version counter
        out = torch.empty_like(made[0])
        paged.quantised_attention(plan, *made, out=out)


# ------------------------------------------------------------------ verify
def test_verify_many_sequences_of_small_vocabularies():
    """More sequences than CTAs that fit, vocabularies of one to a warp's worth, against the running sums in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for vocabulary in (1, 2, 31, 33, 300):
        n = 3000
        first = torch.arange(n + 1, dtype=torch.int32, device="cuda")
        target = torch.rand(n, vocabulary, generator=g, device="cuda")
        finals = torch.rand(n, generator=g, device="cuda")
        none_i, none_f = first[:0], finals[:0]
        accepted, tokens = paged.verify(target, None, none_i, none_f, finals, first)
        sums = target.double().cumsum(1)
        goal = finals.double() * sums[:, -1]
        want = (sums <= goal[:, None]).sum(1).clamp(max=vocabulary - 1)
        near = ((sums - goal[:, None]).abs().min(1)[0] < 1e-12 * sums[:, -1])
        assert not accepted.any() and bool(((tokens == want) | near).all()) and int(near.sum()) < 5


def test_verify_the_same_row_for_all():
    """Rows of stride 0: one distribution for every sequence."""
    p = torch.tensor([[0.25, 0.0, 0.5, 0.25]], device="cuda").expand(6, 4)
    finals = torch.tensor([0.0, 0.2, 0.25, 0.5, 0.75, 0.9999], device="cuda")
    first = torch.arange(7, dtype=torch.int32, device="cuda")
    _, tokens = paged.verify(p, None, first[:0], finals[:0], finals, first)
    assert tokens.tolist() == [0, 0, 2, 2, 3, 3] and math.isclose(float(p[0].sum()), 1.0)

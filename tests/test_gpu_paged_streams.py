"""Memory of the paged-cache operators on more than one stream, by the allocator's own
list: what a call may still use on one stream is not handed out on another."""
import pytest
import torch

from emmy_b200 import paged

pytestmark = pytest.mark.gpu

PENDING = "active_pending_free"


def states():
    """Address -> state of every block of the allocator."""
    got = {}
    for segment in torch.cuda.memory_snapshot():
        address = segment["address"]
        for block in segment["blocks"]:
            got[address] = block["state"]
            address += block["size"]
    return got


class Case:
    """Inputs and outputs of both operators, on the default stream."""

    def __init__(self):
        g = torch.Generator(device="cuda").manual_seed(0)
        self.frequencies = torch.rand(32, generator=g, device="cuda")
        self.q = torch.randn(1, 8, 128, generator=g, device="cuda").bfloat16()
        self.kv = torch.randn(1, 2, 128, generator=g, device="cuda").bfloat16()
        self.caches = [torch.randn(1250, 16, 2, 128, generator=g, device="cuda").bfloat16() for _ in range(2)]
        self.table = torch.arange(1250, dtype=torch.int32, device="cuda")[None]
        self.at = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
        self.slots = torch.full((1,), 19999, dtype=torch.int32, device="cuda")
        self.turned, self.out, self.lse = torch.empty_like(self.q), torch.empty_like(self.q), torch.empty(1, 8, device="cuda")
        torch.cuda.synchronize()

    def made(self):
        """A plan with split rows and a rotation of two axes."""
        plan = paged.AttentionPlan([1], [20000], 8, 2, 128)
        assert plan.scratch.numel()
        return plan, paged.Rotation(self.frequencies.clone(), axes=[0] * 16 + [1] * 16)

    def call(self, plan, rotation, given=True, **how):
        results = dict(q_out=self.turned) if given else {}
        turned = paged.rotate_append(rotation, self.q, self.kv, self.kv, self.at, self.slots, *self.caches, **results, **how)
        results = dict(out=self.out, lse=self.lse) if given else {}
        return turned, *paged.attention(plan, turned, *self.caches, self.table, **results, **how)


def memory(plan, rotation):
    return {t.data_ptr() for t in (plan.scratch, plan.words, rotation.frequencies, rotation.pair_axis)}


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("made_on_default", [False, True])
def test_memory_of_what_is_dropped_waits_for_the_other_stream(made_on_default, given):
    """Made under one stream, used on the other (as the current one, or by its handle), dropped."""
    case, side = Case(), torch.cuda.Stream()
    maker, user = (torch.cuda.default_stream(), side) if made_on_default else (side, torch.cuda.default_stream())
    with torch.cuda.stream(maker):
        plan, rotation = case.made()
        used = memory(plan, rotation)
    torch.cuda.synchronize()
    if given:
        with torch.cuda.stream(maker):
            case.call(plan, rotation, stream=user.cuda_stream)
    else:
        with torch.cuda.stream(user):
            case.call(plan, rotation)
    del plan, rotation
    got = states()
    torch.cuda.synchronize()
    assert [got.get(a) for a in used] == [PENDING] * 4


def test_memory_of_one_stream_is_free_at_once():
    case = Case()
    plan, rotation = case.made()
    used = memory(plan, rotation)
    case.call(plan, rotation)
    del plan, rotation
    got = states()
    torch.cuda.synchronize()
    assert PENDING not in [got.get(a) for a in used]


@pytest.mark.parametrize("given", [False, True])
def test_frequencies_of_another_stream(given):
    """Allocated on one stream; the rotation made and used under another, both dropped."""
    case, side = Case(), torch.cuda.Stream()
    frequencies = case.frequencies.clone()
    address = frequencies.data_ptr()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        rotation = paged.Rotation(frequencies)
        paged.rotate_append(rotation, case.q, case.kv, case.kv, case.at[0], case.slots, *case.caches, q_out=case.turned,
                            **(dict(stream=side.cuda_stream) if given else {}))
    del rotation, frequencies
    got = states()
    torch.cuda.synchronize()
    assert got.get(address) == PENDING


@pytest.mark.parametrize("side_is_current", [False, True])
def test_results_for_a_given_stream_are_of_its_memory(side_is_current):
    """What the current stream has let go of, and may still use, is not written by another;
    results that are dropped wait for the current stream, which may have read them."""
    case, side = Case(), torch.cuda.Stream()
    current, user = (side, torch.cuda.default_stream()) if side_is_current else (torch.cuda.default_stream(), side)
    with torch.cuda.stream(current):
        plan, rotation = case.made()
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        held = [torch.empty_like(t) for t in (case.turned, case.out, case.lse)]
        torch.cuda._sleep(1_000_000)
        for t in held:
            t.zero_()
        freed = {t.data_ptr() for t in held}
        del held, t
        got = case.call(plan, rotation, given=False, stream=user.cuda_stream)
        mine = {t.data_ptr() for t in got}
        assert not mine & freed
        current.wait_stream(user)
        want = case.call(plan, rotation)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del got
        now = states()
        torch.cuda.synchronize()
        assert [now.get(a) for a in mine] == [PENDING] * 3


@pytest.mark.parametrize("given", [False, True])
def test_check_waits_for_calls_on_other_streams(given):
    case, side = Case(), torch.cuda.Stream()
    plan, rotation = case.made()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        if not given:
            case.call(plan, rotation)
    if given:
        case.call(plan, rotation, stream=side.cuda_stream)
    plan.check()
    assert side.query()

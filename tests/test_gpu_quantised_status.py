"""A plan of the attention over an 8-bit cache whose sequences go to several kernels, after one gave up."""
import pytest
import torch

from emmy_b200 import native, paged
from test_gpu_paged import UNIT, close
from test_gpu_quantised import BF16, make, wanted

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,kv_heads", [(128, 8), (64, 16)])
def test_every_kernel_stops_when_one_gave_up(dim, kv_heads):
    """The word that says so (set here) is the whole batch's: nothing is written, read back or joined, until it is
    taken away."""
    # more than the 32 MiB that go with those read back: each kernel has a sequence, and some have parts
    q_lens, kv_lens = [1, 20, 300, 2, 0], [17000, 17001, 900, 2500, 40]
    plan = paged.QuantisedPlan(q_lens, kv_lens, 2 * kv_heads, kv_heads, dim)
    made = make(q_lens, kv_lens, 2 * kv_heads, kv_heads, dim, 64)
    want = wanted(made, q_lens, kv_lens, dim ** -0.5)
    plan.words[3] = 1
    plan.scratch.fill_(0xA5)
    out, lse = torch.full_like(made[0], 7.0), torch.full(made[0].shape[:2], 7.0, device="cuda")
    words = plan.words.clone()
    for _ in range(2):
        paged.quantised_attention(plan, *made, out=out, lse=lse)
        with pytest.raises(native.EmmyError, match="ran out"):
            plan.check()
    assert bool((out == 7.0).all()) and bool((lse == 7.0).all()) and bool((plan.scratch == 0xA5).all())
    assert torch.equal(plan.words, words)
    plan.words[3] = 0
    paged.quantised_attention(plan, *made, out=out, lse=lse)
    plan.check()
    close(out, lse, want, UNIT[BF16])

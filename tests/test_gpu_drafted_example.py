"""The example of serving from an 8-bit cache with drafted tokens on the GPU: the logits that
tokens were drawn from are those of the computation without a cache, whatever was drafted and
rejected before.

Tolerance.  As for the 16-bit example, below 1e-2 of the largest logit: both sides hold keys
and values as the same 8-bit floats.  A key or value so near to the middle of two of them that
32 and 64 bits round it apart (one in 2^20 or so) is off by 2^-3 of itself, with its weight among
many."""
import sys

import pytest

from conftest import REPO

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompts,drafts,tokens", [([37, 150, 8], 4, 24), ([1], 8, 40), ([300, 5, 16, 129], 1, 10), ([20, 33], 0, 7)])
def test_serving_with_drafts_matches_whole_sequences(prompts, drafts, tokens):
    sys.path.insert(0, str(REPO / "examples"))
    import drafted_serving
    texts, (tried, kept), worst = drafted_serving.serve(prompts, drafts, tokens)
    assert all(n + tokens <= len(t) <= n + tokens + drafts for t, n in zip(texts, prompts))
    assert 0 <= kept <= tried and (tried > 0) == (drafts > 0 and tokens > 7)
    assert worst < 1e-2, worst

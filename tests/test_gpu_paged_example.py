"""The serving example on the GPU: prompts read in chunks of any size give the
logits of the computation without a cache, whatever the chunking.

Tolerance.  Rounding to bfloat16 (2^-8) of the weights and of the mixed values
moves a component of the layer's output by at most 2 x 2^-8 of the mixed values'
size; merged and added to the embedding, which is as large or larger, and compared
with the largest logit, that stays below 1e-2."""
import sys

import pytest

from conftest import REPO

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompts,chunk", [([37, 150, 8], 64), ([1], 1), ([300, 5, 16, 129], 300), ([20, 33], 7)])
def test_serving_matches_whole_sequences(prompts, chunk):
    sys.path.insert(0, str(REPO / "examples"))
    import paged_serving
    texts, worst = paged_serving.serve(prompts, chunk, steps=4)
    assert [len(t) for t in texts] == [n + 4 for n in prompts]
    assert worst < 1e-2, worst

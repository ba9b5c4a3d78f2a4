"""The serving example: prompts read in one packed pass and tokens decoded over the
paged cache in a graph give the logits of the whole text without a cache."""

import os
import sys

import pytest

pytestmark = pytest.mark.gpu

EXAMPLES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples")


@pytest.mark.parametrize("steps,layers,prompts", [(12, 2, (37, 5, 120, 64, 1)), (20, 1, (200,))])
def test_serving_example(steps, layers, prompts):
    sys.path.insert(0, EXAMPLES)
    try:
        import serve
    finally:
        sys.path.remove(EXAMPLES)
    # Both sides work in bf16 (unit roundoff 2^-8) outside the attention.  Where their
    # attention outputs round differently (at most one unit each), the difference passes
    # `layers` residual additions, norms and two products, each of which may round a
    # value one way on one side and the other way on the other: 8 roundings a layer and
    # 4 at the end, in the worst case all of the size of the largest logit.
    bound = (8 * layers + 4) * 2.0 ** -8
    assert serve.main(steps, layers, prompts) <= bound


@pytest.mark.parametrize("steps", [1, 2, 3])
def test_serving_example_of_few_steps(steps):
    """One step: the prompts' own logits.  Two: a single run of the graph."""
    test_serving_example(steps, 2, (37, 5, 120, 64, 1))


def test_serving_example_needs_a_step():
    sys.path.insert(0, EXAMPLES)
    try:
        import serve
    finally:
        sys.path.remove(EXAMPLES)
    for steps, prompts in [(0, (3, 4)), (2, (3, 0))]:
        with pytest.raises(ValueError):
            serve.main(steps, 1, prompts)

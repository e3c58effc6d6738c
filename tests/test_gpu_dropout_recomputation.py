"""GPU: the layer's masks when a forward pass is run again in the backward pass."""
import pytest

import dropout_recomputed as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("capturable", [False, True])
def test_recomputation(built, reentrant, capturable):
    R.the_gradients_mask_is_the_outputs("cuda", reentrant, capturable)
    R.segments_and_calls_in_any_order("cuda", reentrant, capturable)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_state_that_is_not_preserved(built, reentrant):
    R.a_state_that_is_not_preserved_is_refused("cuda", reentrant)


def test_the_same_seed_of_torch_twice(built):
    R.the_same_seed_of_torch_twice_makes_two_masks("cuda")

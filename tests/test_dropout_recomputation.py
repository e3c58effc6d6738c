"""CPU: the layer's masks when a forward pass is run again in the backward pass, with a stand-in for the kernel."""
import pytest

import dropout_recomputed as R
import dropout_stand_in


@pytest.fixture(autouse=True)
def stand_in(built, monkeypatch):
    dropout_stand_in.place(monkeypatch)


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("capturable", [False, True])
def test_recomputation(reentrant, capturable):
    R.the_gradients_mask_is_the_outputs("cpu", reentrant, capturable)
    R.segments_and_calls_in_any_order("cpu", reentrant, capturable)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_state_that_is_not_preserved(reentrant):
    R.a_state_that_is_not_preserved_is_refused("cpu", reentrant)


def test_the_same_seed_of_torch_twice():
    R.the_same_seed_of_torch_twice_makes_two_masks("cpu")


def test_what_is_remembered_ends(monkeypatch):
    """Calls long past are forgotten, and not copied or saved with the layer."""
    import copy
    import torch
    import tf_approximate_b200 as ax
    layer = ax.Dropout(0.5, seed=3)
    monkeypatch.setattr(ax.Dropout, "REMEMBERED", 10)
    x = torch.ones(8)
    for _ in range(25):
        layer(x)
    assert len(layer._recent) == 10 and sorted(layer._recent.values()) == list(range(15, 25))
    assert not copy.deepcopy(layer)._recent and copy.deepcopy(layer).calls == 25

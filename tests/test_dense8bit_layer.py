"""CPU: the layer that answers in 8 bits, with a stand-in for its kernels."""
import pytest

import dense8bit_layer as D
import dense8bit_stand_in


@pytest.fixture(autouse=True)
def stand_in(built, monkeypatch):
    dense8bit_stand_in.place(monkeypatch)


def test_gradients_are_refused():
    D.gradients_are_refused("cpu")


def test_casts_of_a_network():
    D.casts_of_a_network_leave_the_operands("cpu")


def test_types():
    D.answers_have_the_types_that_the_dense_layers_have("cpu")

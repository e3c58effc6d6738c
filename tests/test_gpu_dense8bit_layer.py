"""GPU: the layer that answers in 8 bits, around its kernels."""
import pytest

import dense8bit_layer as D

pytestmark = pytest.mark.gpu


def test_gradients_are_refused(built):
    D.gradients_are_refused("cuda")


def test_casts_of_a_network(built):
    D.casts_of_a_network_leave_the_operands("cuda")

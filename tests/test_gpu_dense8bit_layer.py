"""GPU: the layer that answers in 8 bits, around its kernels."""
import pytest

import dense8bit_layer as D

pytestmark = pytest.mark.gpu


def test_gradients_are_refused(built):
    D.gradients_are_refused("cuda")


def test_casts_of_a_network(built):
    D.casts_of_a_network_leave_the_operands("cuda")


def test_types(built):
    D.answers_have_the_types_that_the_dense_layers_have("cuda")

"""
The shapes of tile that the grouped and 8-bit products are made of, each by name: sizes at which the choice falls on it,
checked to have run, against 64-bit forms.
"""

import pytest
import torch

import attorch_b200 as attorch
from attorch_b200 import _lib
from tests.expert_helpers import grouped64, offsets_of
from tests.test_grouped_linear_gpu import integer_case

pytestmark = pytest.mark.gpu

PAIR = 256 | _lib.TILE_PAIR


@pytest.fixture(autouse=True)
def backward_in_this_thread():
    """What ran last is noted per host thread."""
    with torch.autograd.set_multithreading_enabled(False):
        yield


def tile():
    return _lib.load().ab200_last_tile()


# Rows of the groups, K, N, and the tiles of the forward product, dX and dW.
FP32_SHAPES = [([700, 300, 0, 600], 136, 1800, PAIR, 128, 128), ([390, 0, 1000, 170], 1032, 1800, PAIR, 128, PAIR),
               ([1201, 400, 700, 0, 600, 99, 1], 1000, 1416, PAIR, PAIR, PAIR), ([1] * 64, 72, 2048, 128, 128, 128),
               ([300], 136, 4104, 128, 128, 128)]


@pytest.mark.parametrize('counts,k,n,forward,dx,dw', FP32_SHAPES)
def test_fp32_products_run_the_shape_that_was_chosen(counts, k, n, forward, dx, dw):
    """fp32 has pairs and 128 columns: the choice is made between them, and a width it does not have is never costed."""
    x, w, _, dy = integer_case(counts, 0, k, n, torch.float32)
    y64, (dx64, dw64, _) = grouped64(x, counts, w, None, None, dy)
    for leaf, expected, shape in ((x, dx64, dx), (w, dw64, dw)):
        leaf.requires_grad_()
        y = attorch.grouped_linear(x, offsets_of(counts), w)
        assert tile() == forward and torch.equal(y.double(), y64)
        grad, = torch.autograd.grad(y, leaf, dy)
        assert tile() == shape and torch.equal(grad.double(), expected)
        leaf.requires_grad_(False)
    attorch.check_status()

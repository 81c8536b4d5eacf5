"""Forward-mode tangents: the operators have no such derivative and say so, whether or not a gradient is recorded."""

import pytest
import torch
from torch.autograd import forward_ad

import attorch_b200 as attorch
from tests.expert_helpers import offsets_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('grad', [False, True])
def test_tangents_are_refused_and_not_dropped(grad):
    x, logits = torch.randn(6, 8, device='cuda'), torch.randn(6, 4, device='cuda')
    routing = attorch.route(logits, 2)
    rows = attorch.dispatch(x, routing)
    w, b, offsets = torch.randn(4, 8, 16, device='cuda'), torch.randn(4, 16, device='cuda'), routing.offsets
    held, scale = attorch.quantize_weight(w[0])
    stack, scales = attorch.quantize_weight(w)
    router = attorch.Router(8, 4, 2)

    def dual(t):
        return forward_ad.make_dual(t, torch.ones_like(t))

    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        for call in (lambda: attorch.route(dual(logits), 2),
                     lambda: attorch.dispatch(dual(x), routing),
                     lambda: attorch.combine(dual(rows), routing),
                     lambda: attorch.combine(rows, routing._replace(weights=dual(routing.weights))),
                     lambda: attorch.grouped_linear(dual(rows), offsets, w, b),
                     lambda: attorch.grouped_linear(rows, offsets, dual(w), b),
                     lambda: attorch.grouped_linear(rows, offsets, w, dual(b)),
                     lambda: router(dual(x)),
                     lambda: attorch.Float8Linear(8, 16)(dual(x)),
                     lambda: attorch.float8_linear(dual(x), held, scale),
                     lambda: attorch.float8_linear(x, held, dual(scale)),
                     lambda: attorch.float8_grouped_linear(rows, offsets, stack, scales, dual(b))):
            with pytest.raises(NotImplementedError, match='jvp|forward-mode'):
                call()
        # Without a tangent the calls work inside a dual level too.
        inside = attorch.grouped_linear(attorch.dispatch(x, attorch.route(logits, 2)), offsets, w, b)
        y = attorch.combine(inside, routing)
        eight = attorch.float8_linear(x, held, scale)
    assert torch.equal(inside, attorch.grouped_linear(rows, offsets, w, b)) and torch.equal(y, attorch.combine(inside, routing))
    assert torch.equal(eight, attorch.float8_linear(x, held, scale))

"""Plans that a caller edits or makes: what may be changed in place, holes, and values that padding holds."""

import pytest
import torch

import attorch_b200 as attorch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('tokens', [20, 500])
def test_plan_can_be_edited_before_backward(tokens):
    """The gradient of the weights reads the logits, the weights and the chosen experts, not the plan."""
    g = torch.Generator(device='cuda').manual_seed(1)
    logits = torch.randn(tokens, 6, generator=g, device='cuda', requires_grad=True)
    grad = torch.randn(tokens, 2, generator=g, device='cuda')
    expected, = torch.autograd.grad(attorch.route(logits, 2).weights, logits, grad)
    routing = attorch.route(logits, 2)
    routing.token_row[routing.token_row > 30] = -1
    routing.row_token.fill_(-1)
    routing.offsets.clamp_(max=31)
    got, = torch.autograd.grad(routing.weights, logits, grad)
    assert torch.equal(got, expected)
    # Each tensor has a version counter of its own: rows that were moved by one part of a plan may outlive edits of another.
    routing = attorch.route(logits, 2)
    x = torch.randn(tokens, 8, device='cuda', requires_grad=True)
    rows = attorch.dispatch(x, routing)
    routing.experts.zero_()
    routing.row_token.zero_()
    rows.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2.0))

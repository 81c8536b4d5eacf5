"""The router's gate: its gradient in a data-parallel bucket, the type of its logits, what padding may hold."""

import pytest
import torch

import attorch_b200 as attorch
from attorch_b200.dp import GradientBuckets

pytestmark = pytest.mark.gpu


def gate_step(router, x, dweights):
    """One backward pass through the router's weights; the gradient of the input."""
    x = x.clone().requires_grad_()
    router(x).weights.backward(dweights)
    return x.grad


@pytest.mark.parametrize('grad_dtype', [None, torch.bfloat16])
def test_gate_writes_its_gradient_into_a_bucket(grad_dtype):
    """Several steps with the bucket's contract (nothing is cleared between them) give the last step's gradient each."""
    torch.manual_seed(1)
    plain, bucketed = (attorch.Router(64, 8, 2) for _ in range(2))
    bucketed.load_state_dict(plain.state_dict())
    other = attorch.Linear(64, 64)
    layers = [m for m in torch.nn.ModuleList([other, bucketed]).modules() if isinstance(m, attorch.Linear)]
    assert layers == [other, bucketed.gate]
    buckets = GradientBuckets(layers, grad_dtype=grad_dtype)
    for step in range(3):
        x, dweights = torch.randn(48, 64, device='cuda'), torch.randn(48, 2, device='cuda')
        plain.gate.weight.grad = None
        with torch.autocast('cuda', dtype=torch.bfloat16, enabled=grad_dtype is not None):
            expected = gate_step(plain, x, dweights)
            buckets.zero_grad()
            got = gate_step(bucketed, x, dweights)
        buckets.finish()
        # dW and dX are Linear's: their pieces may be added in another order.
        torch.testing.assert_close(got, expected, rtol=1e-4, atol=1e-4)
        tolerance = 1e-4 if grad_dtype is None else 2.0 ** -8
        torch.testing.assert_close(bucketed.gate.weight.grad, plain.gate.weight.grad, rtol=tolerance, atol=tolerance)
        assert bucketed.gate.weight.grad.data_ptr() == (buckets.flat_grad[buckets._offsets[1]:]).data_ptr()
    attorch.check_status()


def test_gate_tells_the_exchange_and_puts_its_input_gradient_off():
    """Every block of dW is announced once, in order, after it has been enqueued; dX runs when the caller says so."""
    torch.manual_seed(2)
    router = attorch.Router(64, 8, 2, 'sigmoid')
    x, dweights = torch.randn(40, 64, device='cuda'), torch.randn(40, 2, device='cuda')
    expected = gate_step(router, x, dweights)
    weight_grad = router.gate.weight.grad.clone()
    router.gate.weight.grad = None
    told, put_off = [], []
    out = torch.zeros_like(router.gate.weight)

    def ready(block, blocks):
        told.append((block, blocks, out[block * 16:(block + 1) * 16].clone()))

    router.gate.weight_grad_out, router.gate.grad_ready, router.gate.dw_chunks = out, ready, 4
    router.gate.defer_input_grad = put_off.append
    got = gate_step(router, x, dweights)
    assert [t[:2] for t in told] == [(i, 4) for i in range(4)] and router.gate.weight.grad is None
    torch.testing.assert_close(torch.cat([t[2] for t in told]), weight_grad, rtol=1e-4, atol=1e-4)
    launch, = put_off
    launch(0, 13)
    launch(13)
    torch.testing.assert_close(got, expected, rtol=1e-4, atol=1e-4)
    router.gate.weight.requires_grad_(False)
    told.clear()
    gate_step(router, x, dweights)
    assert [t[:2] for t in told] == [(0, 1)]
    attorch.check_status()

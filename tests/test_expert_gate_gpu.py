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


def test_gate_tells_the_exchange():
    """Every block of dW is announced once, in order, after it has been enqueued."""
    torch.manual_seed(2)
    router = attorch.Router(64, 8, 2, 'sigmoid')
    x, dweights = torch.randn(40, 64, device='cuda'), torch.randn(40, 2, device='cuda')
    expected = gate_step(router, x, dweights)
    weight_grad = router.gate.weight.grad.clone()
    router.gate.weight.grad = None
    told = []
    out = torch.zeros_like(router.gate.weight)

    def ready(block, blocks):
        told.append((block, blocks, out[block * 16:(block + 1) * 16].clone()))

    router.gate.weight_grad_out, router.gate.grad_ready, router.gate.dw_chunks = out, ready, 4
    got = gate_step(router, x, dweights)
    assert [t[:2] for t in told] == [(i, 4) for i in range(4)] and router.gate.weight.grad is None
    torch.testing.assert_close(torch.cat([t[2] for t in told]), weight_grad, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(got, expected, rtol=1e-4, atol=1e-4)
    router.gate.weight.requires_grad_(False)
    told.clear()
    gate_step(router, x, dweights)
    assert [t[:2] for t in told] == [(0, 1)]
    attorch.check_status()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('tokens,dim,experts', [(3, 64, 8), (300, 100, 12), (40, 4096, 130)])
def test_logits_are_fp32(dtype, tokens, dim, experts):
    """Products of 16-bit operands summed in fp32 and not rounded: off by at most dim 2^-23 of the sum of magnitudes."""
    from attorch_b200.expert_routing_layer import GateAutoGrad
    g = torch.Generator(device='cuda').manual_seed(dim)
    x = torch.randn(tokens, dim, generator=g, device='cuda').to(dtype).requires_grad_()
    w = torch.randn(dim, experts, generator=g, device='cuda').to(dtype).requires_grad_()
    logits = GateAutoGrad.apply(x, w)
    expected, size = x.detach().double() @ w.detach().double(), x.detach().double().abs() @ w.detach().double().abs()
    assert logits.dtype is torch.float32 and ((logits.double() - expected).abs() <= dim * 2.0 ** -23 * size).all()
    dlogits = torch.randn(tokens, experts, generator=g, device='cuda').to(dtype)      # exact in the operands' type
    dx, dw = torch.autograd.grad(logits, (x, w), dlogits.float())
    eps = torch.finfo(dtype).eps / 2
    for got, left, right in ((dx, dlogits, w.detach().T), (dw, x.detach().T, dlogits)):
        exact, size = left.double() @ right.double(), left.double().abs() @ right.double().abs()
        assert got.dtype is dtype
        assert ((got.double() - exact).abs() <= eps * exact.abs() + 1.1 * left.shape[1] * 2.0 ** -23 * size + 2.0 ** -25).all()


@pytest.mark.parametrize('dtype,gap', [(torch.bfloat16, 2.0 ** -10), (torch.float16, 2.0 ** -13), (torch.float32, 2.0 ** -9)], ids=str)
def test_near_ties_go_to_the_larger_logit(dtype, gap):
    """1 and 1 + gap are one number in 16 bits; the second expert's logit is larger."""
    router = attorch.Router(16, 4, 1, dtype=dtype)
    with torch.no_grad():
        router.gate.weight.zero_()
        router.gate.weight[0, :3] = 1.0
        router.gate.weight[1, 1] = 1.0
        x = torch.zeros(5, 16, device='cuda', dtype=dtype)
        x[:, 0], x[:, 1] = 1.0, gap
        assert (router(x).experts == 1).all()

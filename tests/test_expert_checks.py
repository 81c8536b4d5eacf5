"""What the expert block's operators and the 8-bit products check on the host, before any address is taken."""

import pytest
import torch

import attorch_b200 as attorch
from attorch_b200 import expert_routing_layer as routing_layer

CPU = torch.device('cpu')


@pytest.mark.parametrize('offsets', [torch.zeros(0, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32),
                                     torch.tensor(3, dtype=torch.int32), torch.zeros(3), torch.zeros(6, dtype=torch.int32)[::2]])
def test_plans_without_an_end_are_refused(offsets):
    """The end of the last expert's rows is read from the last entry: there has to be one."""
    plan = torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(AssertionError, match='offsets'):
        routing_layer._check_plan(attorch.Routing(torch.zeros(4, 2), plan, offsets, plan.flatten(), plan), CPU, 4)
    routing_layer._check_plan(attorch.Routing(torch.zeros(4, 2), plan, torch.zeros(1, dtype=torch.int32), plan.flatten(), plan), CPU, 4)


def test_gate_refuses_weights_of_another_device():
    """The kernel gets both addresses on the input's device."""
    router = attorch.Router(8, 4, 2, device='meta')
    with pytest.raises(AssertionError, match='weights are on meta'):
        router(torch.zeros(3, 8))


def test_buckets_refuse_layers_that_do_not_write_into_them():
    """Their .grad would be a view of a bucket that nothing of theirs is written to, exchanged or cleared in."""
    from attorch_b200.dp import GradientBuckets
    linear = attorch.Linear(4, 6, device='cpu')
    with pytest.raises(TypeError, match='GroupedLinear'):
        GradientBuckets([linear, attorch.GroupedLinear(2, 4, 6, device='cpu')])
    with pytest.raises(TypeError, match='Float8Linear'):
        GradientBuckets([attorch.Float8Linear(4, 6, device='cpu')])
    assert linear.weight_grad_out is None and linear.weight.grad is None       # refused before anything was changed
    gate = attorch.Router(4, 6, 2, device='cpu').gate
    buckets = GradientBuckets([linear, gate])
    assert gate.weight.grad.data_ptr() == gate.weight_grad_out.data_ptr() == buckets.flat[30:].data_ptr()


def test_frozen_copies_leave_the_trained_layer_alone(monkeypatch):
    """The 8-bit form of a layer in training is a snapshot: the layer's parameters still train, and do not reach the copy."""
    from attorch_b200 import float8_linear_layer

    def snapshot(weight):
        return weight.detach().transpose(-1, -2).contiguous().to(torch.float8_e4m3fn), torch.ones(*weight.shape[:-2], 1, 1)

    monkeypatch.setattr(float8_linear_layer, 'quantize_weight', snapshot)
    linear = attorch.Linear(16, 32, device='cpu')
    frozen = attorch.Float8Linear.from_linear(linear).freeze()
    grouped = attorch.GroupedLinear(2, 16, 32, device='cpu')
    eight = attorch.Float8GroupedLinear.from_grouped(grouped)
    for source, copy in ((linear, frozen), (grouped, eight)):
        assert source.weight.requires_grad and source.bias.requires_grad and not copy.bias.requires_grad
        before = copy.bias.clone()
        assert torch.equal(before, source.bias)
        with torch.no_grad():
            source.bias.add_(1.0)
        assert torch.equal(copy.bias, before)


def test_fp32_output_excludes_a_kept_pre_activation():
    from attorch_b200 import _lib
    from attorch_b200 import build as builder
    builder.build()
    a = 0x1000
    for dtype in (_lib.F32, _lib.F16, _lib.BF16):
        assert _lib.load().ab200_grouped_linear_forward(a, a, None, None, a, a, 0, 1, 8, 8, 8, 0, 8, 8, 8, dtype, 0, 0, 0.0, a, None,
                                                        _lib.FLAG_OUTPUT_FP32) == -3
        assert _lib.load().ab200_grouped_linear_forward(a, a, None, None, None, a, 0, 1, 8, 8, 8, 0, 8, 8, 8, dtype, 0, 0, 0.0, a, None,
                                                        _lib.FLAG_OUTPUT_FP32) == 0


def test_gate_refuses_to_put_its_input_gradient_off():
    """Its input also goes to dispatch: autograd would add a gradient that has not been computed yet."""
    from attorch_b200.dp import GradientBuckets
    router = attorch.Router(4, 6, 2, device='cpu')
    GradientBuckets([router.gate], defer_first_input_grad=True)
    with pytest.raises(RuntimeError, match='put off'):
        router(torch.zeros(3, 4, requires_grad=True))
    with pytest.raises(RuntimeError, match='no CPU fallback'):      # nothing to put off
        router(torch.zeros(3, 4))

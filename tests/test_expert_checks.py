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

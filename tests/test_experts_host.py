"""
What the expert block's operators and the 8-bit products refuse, and the sizes their entry points ask for: checks
of the host, before anything is launched.
"""

import ctypes

import pytest
import torch

import attorch_b200 as attorch
from attorch_b200 import _lib
from attorch_b200 import build as builder
from attorch_b200.grouped_linear_layer import _check_offsets, _check_operands


@pytest.fixture(scope='module')
def lib():
    builder.build()
    return _lib.load()


FAKE, ODD = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1008)


def test_grouped_entry_points_reject(lib):
    def forward(x=FAKE, w=FAKE, off=FAKE, pre=None, out=FAKE, rows=4, groups=2, K=8, N=8, ld_x=8, wg=64, ld_w=8, ld_pre=8, ld_out=8,
                dtype=2, bias=None, bias_dtype=0, act=0, status=FAKE, flags=0):
        return lib.ab200_grouped_linear_forward(x, w, bias, off, pre, out, rows, groups, K, N, ld_x, wg, ld_w, ld_pre, ld_out, dtype,
                                                bias_dtype, act, 0.0, status, None, flags)
    assert forward(rows=0) == 0 and forward(N=0) == 0
    assert forward(rows=-1) == -2 and forward(groups=0) == -2 and forward(K=-1) == -2
    assert forward(groups=513) == -9 and forward(rows=2 ** 31) == -9
    assert forward(dtype=3) == -3 and forward(bias=FAKE, bias_dtype=9) == -3
    assert forward(act=22) == -4
    for name in ('x', 'w', 'off', 'out', 'status'):
        assert forward(**{name: None}) == -1, name
    assert forward(ld_x=7) == -5 and forward(ld_w=7) == -5 and forward(ld_out=7) == -5 and forward(pre=FAKE, ld_pre=7) == -5
    assert forward(wg=0) == -5
    assert forward(x=ODD, flags=_lib.FLAG_FORCE_TCGEN05) == -5

    def dx(dz=FAKE, w=FAKE, off=FAKE, out=FAKE, rows=4, groups=2, K=8, N=8, ld_dz=8, ld_dx=8, dtype=2, status=FAKE):
        return lib.ab200_grouped_linear_backward_input(dz, w, off, out, rows, groups, K, N, ld_dz, 64, 8, ld_dx, dtype, 2, status, None, 0)
    assert dx(rows=0) == 0 and dx(rows=-1) == -2 and dx(dtype=5) == -3 and dx(ld_dz=4) == -5 and dx(ld_dx=4) == -5
    for name in ('dz', 'w', 'off', 'out', 'status'):
        assert dx(**{name: None}) == -1, name

    def dw(x=FAKE, dz=FAKE, off=FAKE, out=FAKE, rows=4, groups=2, K=8, N=8, ld_x=8, ld_dz=8, dtype=2, status=FAKE):
        return lib.ab200_grouped_linear_backward_weight(x, dz, off, out, rows, groups, K, N, ld_x, ld_dz, dtype, 2, status, None, 0)
    assert dw(K=0) == 0 and dw(groups=-1) == -2 and dw(dtype=5) == -3 and dw(ld_x=4) == -5 and dw(ld_dz=4) == -5
    for name in ('x', 'dz', 'off', 'out', 'status'):
        assert dw(**{name: None}) == -1, name

    def db(dy=FAKE, z=None, dz=None, out=FAKE, off=FAKE, rows=4, groups=2, N=8, ld=8, act=0, ws=FAKE, nbytes=1 << 20):
        return lib.ab200_grouped_act_backward(dy, z, dz, out, off, rows, groups, N, ld, ld, ld, 2, 2, act, 0.0, ws, nbytes, None)
    assert db(dz=None, out=None) == 0 and db(rows=-1) == -2 and db(act=24) == -4 and db(act=5) == -1 and db(ld=4) == -5
    assert db(nbytes=95) == -6 and db(ws=None) == -6 and db(dy=None) == -1 and db(off=None) == -1
    assert lib.ab200_grouped_act_backward_workspace_bytes(4, 2, 8) == (1 + 2) * 8 * 4
    assert lib.ab200_grouped_act_backward_workspace_bytes(129, 2, 8) == (2 + 2) * 8 * 4
    assert lib.ab200_grouped_act_backward_workspace_bytes(0, 2, 8) == 0


def test_routing_entry_points_reject(lib):
    def forward(logits=FAKE, weights=FAKE, chosen=FAKE, off=FAKE, row=FAKE, tok=FAKE, tokens=4, experts=8, k=2, ld=8, dtype=0, ws=None, nbytes=0):
        return lib.ab200_route_forward(logits, None, weights, chosen, None, off, row, tok, tokens, experts, k, ld, dtype, 0, 1, ws, nbytes, None)
    assert forward(tokens=-1) == -2 and forward(k=0) == -2 and forward(k=9) == -2 and forward(experts=0) == -2
    assert forward(experts=513, ld=513) == -9 and forward(k=33, experts=64, ld=64) == -9 and forward(tokens=2 ** 31) == -9
    assert forward(tokens=2 ** 30, k=2) == -9                       # 2^31 rows
    assert forward(dtype=3) == -3 and forward(ld=7) == -5
    for name in ('logits', 'weights', 'chosen', 'off', 'row', 'tok'):
        assert forward(**{name: None}) == -1, name
    assert forward(tokens=300) == -6 and forward(tokens=300, ws=FAKE, nbytes=95) == -6
    assert lib.ab200_route_workspace_bytes(256, 8) == 0
    assert lib.ab200_route_workspace_bytes(300, 8) == 3 * 8 * 4
    assert lib.ab200_route_workspace_bytes(16384, 128) == 128 * 128 * 4
    assert lib.ab200_route_workspace_bytes(1 << 20, 64) == 512 * 64 * 4

    def backward(k=2, stats=FAKE, dtype=0, ld=8, tokens=4):
        return lib.ab200_route_backward(FAKE, FAKE, FAKE, stats, FAKE, FAKE, tokens, 8, k, ld, dtype, 0, 1, None)
    assert backward(tokens=0) == 0 and backward(k=9) == -2 and backward(stats=None) == -1 and backward(dtype=4) == -3 and backward(ld=7) == -5

    assert lib.ab200_expert_dispatch(FAKE, FAKE, FAKE, FAKE, 4, 33, 8, 8, 8, 0, None) == -9
    assert lib.ab200_expert_dispatch(FAKE, FAKE, FAKE, FAKE, 4, 2, 8, 8, 7, 0, None) == -5
    assert lib.ab200_expert_dispatch(None, FAKE, FAKE, FAKE, 4, 2, 8, 8, 8, 0, None) == -1
    assert lib.ab200_expert_dispatch(FAKE, FAKE, FAKE, FAKE, 4, 2, 0, 8, 8, 0, None) == 0
    assert lib.ab200_expert_combine(FAKE, FAKE, None, FAKE, 4, 2, 8, 8, 7, 0, None) == -5
    assert lib.ab200_expert_combine(FAKE, None, None, FAKE, 4, 2, 8, 8, 8, 0, None) == -1
    assert lib.ab200_expert_combine(FAKE, FAKE, None, FAKE, 4, 2, 8, 8, 8, 7, None) == -3
    assert lib.ab200_expert_combine_backward(FAKE, FAKE, FAKE, None, FAKE, FAKE, None, 4, 2, 8, 8, 8, 8, 0, None) == -1
    assert lib.ab200_expert_combine_backward(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 4, 2, 8, 8, 4, 8, 0, None) == -5
    assert lib.ab200_expert_combine_backward(FAKE, FAKE, FAKE, FAKE, FAKE, None, None, 4, 2, 8, 8, 8, 8, 0, None) == 0


def test_float8_entry_points_reject(lib):
    def rows(x=FAKE, q=FAKE, s=FAKE, m=4, k=20, ld_x=20, ld_q=32, ld_s=4, dtype=2):
        return lib.ab200_float8_quantize_rows(x, q, s, m, k, ld_x, ld_q, ld_s, dtype, None)
    assert rows(m=0) == 0 and rows(m=-1) == -2 and rows(k=2 ** 31) == -9 and rows(dtype=4) == -3
    assert rows(x=None) == -1 and rows(q=None) == -1 and rows(s=None) == -1
    assert rows(ld_x=19) == -5 and rows(ld_q=20) == -5 and rows(ld_s=3) == -5 and rows(q=ODD) == -5

    def weight(q=FAKE, q_t=FAKE, k=20, n=24, ld=24, ld_q=32, ld_t=32, dtype=2, s=FAKE):
        return lib.ab200_float8_quantize_weight(FAKE, q, q_t, s, 1, k, n, 0, ld, ld_q, ld_t, dtype, None)
    assert weight(k=0) == 0 and weight(k=-1) == -2 and weight(dtype=8) == -3 and weight(s=None) == -1 and weight(q=None, q_t=None) == -1
    assert weight(ld=23) == -5 and weight(ld_q=24) == -5 and weight(ld_t=20) == -5 and weight(q_t=ODD) == -5

    def product(x=FAKE, xs=FAKE, w=FAKE, ws=FAKE, off=None, out=FAKE, m=4, groups=1, k=32, n=8, ld_x=32, ld_xs=4, wg=256, ld_w=32, ld_out=8,
                dtype=2, act=0, status=FAKE):
        return lib.ab200_float8_product(x, xs, w, ws, None, off, None, out, m, groups, k, n, ld_x, ld_xs, wg, ld_w, 1, 1, 1, 8, ld_out, dtype,
                                        0, act, 0.0, status, None, 0)
    assert product(m=0) == 0 and product(n=0) == 0 and product(k=0) == -2 and product(m=-1) == -2 and product(groups=513, off=FAKE) == -9
    assert product(dtype=4) == -3 and product(act=23) == -4 and product(groups=2) == -1
    for name in ('x', 'xs', 'w', 'ws', 'out', 'status'):
        assert product(**{name: None}) == -1, name
    assert product(ld_x=40) == -5 and product(ld_w=24) == -5 and product(ld_xs=3) == -5 and product(ld_out=7) == -5 and product(x=ODD) == -5
    assert product(groups=2, off=FAKE, wg=0) == -5 and product(groups=2, off=FAKE, wg=250) == -5


def test_layers_reject():
    x, w, offsets = torch.zeros(6, 8), torch.zeros(2, 8, 16), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        attorch.grouped_linear(x, offsets, w)
    with pytest.raises(AssertionError, match='Incompatible input'):
        attorch.grouped_linear(x, offsets, torch.zeros(2, 9, 16))
    with pytest.raises(AssertionError, match='must be 3D'):
        attorch.grouped_linear(x, offsets, torch.zeros(8, 16))
    with pytest.raises(AssertionError, match='must be 2D'):
        attorch.grouped_linear(torch.zeros(2, 3, 8), offsets, w)
    with pytest.raises(AssertionError, match='bias'):
        attorch.grouped_linear(x, offsets, w, torch.zeros(16))
    with pytest.raises(AssertionError, match='512'):
        _check_operands(x, torch.zeros(513, 8, 16), None)
    with pytest.raises(AssertionError, match='one entry per group'):
        _check_offsets(torch.zeros(2, dtype=torch.int32), 2, x)
    with pytest.raises(AssertionError, match='integers'):
        _check_offsets(torch.zeros(3), 2, x)
    with pytest.raises(ValueError):
        attorch.GroupedLinear(2, 8, 16, act_func='swish', device='cpu')
    with pytest.raises(RuntimeError, match='groups'):
        attorch.GroupedLinear(0, 8, 16, device='cpu')
    layer = attorch.GroupedLinear(2, 8, 16, device='cpu')
    assert layer.weight.shape == (2, 8, 16) and layer.bias.shape == (2, 16) and set(layer.state_dict()) == {'weight', 'bias'}
    assert float(layer.weight.detach().abs().max()) <= 8 ** -0.5 and 'num_groups=2' in repr(layer)

    logits = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        attorch.route(logits, 2)
    with pytest.raises(ValueError, match='score_func'):
        attorch.route(logits, 2, 'relu')
    with pytest.raises(AssertionError, match='top_k'):
        attorch.route(logits, 9)
    with pytest.raises(AssertionError, match='2D'):
        attorch.route(torch.zeros(2, 2, 8), 1)
    with pytest.raises(AssertionError, match='experts'):
        attorch.route(torch.zeros(2, 513), 1)
    with pytest.raises(RuntimeError, match='top|experts'):
        attorch.Router(8, 4, 5, device='cpu')
    with pytest.raises(ValueError, match='score_func'):
        attorch.Router(8, 4, 2, 'tanh', device='cpu')
    plan = torch.zeros(4, 2, dtype=torch.int32)
    routing = attorch.Routing(torch.zeros(4, 2), plan, offsets, plan.flatten(), plan)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        attorch.dispatch(torch.zeros(4, 8), routing)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        attorch.combine(torch.zeros(8, 8), routing)
    block = attorch.MixtureOfExperts(8, 16, 4, 2, gated=True, device='cpu')
    assert block.up.weight.shape == (4, 8, 32) and block.down.weight.shape == (4, 16, 8)

    with pytest.raises(AssertionError, match='float8_e4m3fn'):
        attorch.float8_linear(x, torch.zeros(16, 8), torch.zeros(1, 1))
    held = torch.zeros(16, 8, dtype=torch.float8_e4m3fn)
    with pytest.raises(AssertionError, match='Scales'):
        attorch.float8_linear(x, held, torch.zeros(1, 2))
    with pytest.raises(AssertionError, match='Incompatible input'):
        attorch.float8_linear(torch.zeros(6, 9), held, torch.zeros(1, 1))
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        attorch.float8_linear(x, held, torch.zeros(1, 1))
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        attorch.Float8Linear(8, 16, device='cpu')(x)
    linear = attorch.Linear(8, 16, device='cpu')
    assert attorch.Float8Linear.from_linear(linear).weight is linear.weight


@pytest.mark.gpu
def test_rejections_that_need_a_device():
    x = torch.zeros(6, 8, device='cuda')
    offsets = torch.zeros(3, dtype=torch.int32, device='cuda')
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        attorch.grouped_linear(x, offsets.cpu(), torch.zeros(2, 8, 16, device='cuda'))
    with pytest.raises(TypeError, match='Unsupported dtype'):
        attorch.grouped_linear(x.double(), offsets, torch.zeros(2, 8, 16, device='cuda', dtype=torch.float64))
    with pytest.raises(AssertionError, match='boolean'):
        attorch.route(x, 2, mask=torch.ones(6, device='cuda'))
    with pytest.raises(AssertionError, match='one entry per token'):
        attorch.route(x, 2, mask=torch.ones(5, dtype=torch.bool, device='cuda'))
    routing = attorch.route(x, 2)
    with pytest.raises(AssertionError, match='tokens'):
        attorch.dispatch(x[:5], routing)
    with pytest.raises(AssertionError, match='rows'):
        attorch.combine(x, routing)
    with pytest.raises(TypeError, match='Unsupported dtype'):
        attorch.dispatch(x.double(), routing)
    with pytest.raises(AssertionError, match='fp32'):
        attorch.combine(torch.zeros(12, 8, device='cuda'), routing._replace(weights=routing.weights.half()))
    held, scale = attorch.quantize_weight(torch.zeros(8, 16, device='cuda'))
    with pytest.raises(RuntimeError, match='no gradient'):
        attorch.float8_linear(x.requires_grad_(), held, scale)

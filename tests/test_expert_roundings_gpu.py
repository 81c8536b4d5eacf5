"""
Where the experts' and the 8-bit products round, and where they must not: act'(Z), the bias gradient, the gate's logits, what
forward keeps for backward.
"""

import pytest
import torch

import attorch_b200 as attorch
from attorch_b200 import _lib
from tests.expert_helpers import act64, offsets_of

pytestmark = pytest.mark.gpu


def fractions(shape, steps, size, generator):
    """Multiples of 1 / steps within +-size."""
    return torch.randint(-size * steps, size * steps + 1, shape, generator=generator, device='cuda') / steps


def kept_slope(y):
    """What a call kept of act'(Z): its last saved tensor."""
    return y.grad_fn.saved_tensors[3]


@pytest.mark.parametrize('act', ['gelu', 'silu', 'sigmoid'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('rows,n,flags', [(70, 40, 0), (1500, 1032, 0), (70, 40, _lib.FLAG_FORCE_GENERIC), (70, 39, 0)])
def test_derivative_is_taken_at_the_unrounded_value(act, dtype, rows, n, flags):
    """
    Z is a multiple of 2^-11 within +-4, exact in fp32 and not in 16 bits.  What is kept of act'(Z) is rounded to fp16 (half
    a step: 2^-11 of it) and evaluated in fp32 (a few 1e-6); act' of a rounded Z would be off by up to 2^-9 |Z| |act''|.
    """
    g = torch.Generator(device='cuda').manual_seed(rows)
    x = fractions((rows, 8), 16, 1, g).to(dtype)
    w = fractions((2, 8, n), 64, 1, g).to(dtype) / 2
    counts = [rows // 3, rows - rows // 3]
    z64 = torch.cat([x[:counts[0]].double() @ w[0].double(), x[counts[0]:].double() @ w[1].double()])
    previous = attorch.set_gemm_flags(flags)
    try:
        y = attorch.grouped_linear(x, offsets_of(counts), w.requires_grad_(), None, act)
    finally:
        attorch.set_gemm_flags(previous)
    slope = act64(z64, act)[1]
    assert kept_slope(y).dtype is torch.float16
    assert ((kept_slope(y).double() - slope).abs() <= 2.0 ** -11 * slope.abs() + 4e-6).all()


@pytest.mark.parametrize('act', ['gelu', 'silu'])
@pytest.mark.parametrize('rows,n', [(70, 40), (1500, 2056)])
def test_derivative_of_8_bit_products_is_taken_at_the_unrounded_value(act, rows, n):
    """The same; multiples of 1/8 within +-1 (four significant bits at most) are held exactly by e4m3."""
    g = torch.Generator(device='cuda').manual_seed(rows)
    size = torch.exp2(-torch.randint(0, 5, (rows, 1), generator=g, device='cuda').float())
    x = (fractions((rows, 24), 8, 1, g) * size).bfloat16()
    w = (fractions((24, n), 8, 1, g) / 2).bfloat16()
    z64 = x.double() @ w.double()
    y = attorch.Float8LinearAutoGrad.apply(x, w.requires_grad_(), None, act)
    slope = act64(z64, act)[1]
    assert kept_slope(y).dtype is torch.float16
    assert ((kept_slope(y).double() - slope).abs() <= 2.0 ** -11 * slope.abs() + 4e-6).all()


@pytest.mark.parametrize('n', [40, 39])
@pytest.mark.parametrize('counts', [[256, 0, 64], [3, 1000]])
def test_bias_gradient_sums_unrounded_values(counts, n):
    """
    dZ = 129/128 * 3/4 = 387/512 lies halfway between two bf16 numbers.  Its sum over a group's rows is a multiple of 1/512
    below 2^11, exact in fp32; a sum of rounded values would be off by a 387th.
    """
    rows = sum(counts)
    x = torch.ones(rows, 8, device='cuda', dtype=torch.bfloat16)
    w = torch.full((len(counts), 8, n), -1.0, device='cuda', dtype=torch.bfloat16)
    b = torch.zeros(len(counts), n, device='cuda', requires_grad=True)
    y = attorch.grouped_linear(x, offsets_of(counts), w, b, 'leaky_relu_0.75')
    db, = torch.autograd.grad(y, b, torch.full_like(y, 129 / 128))
    expected = torch.tensor(counts, device='cuda')[:, None] * (387 / 512)
    assert db.dtype is torch.float32 and torch.equal(db, expected.expand(-1, n))


@pytest.mark.parametrize('act', ['gelu', 'leaky_relu_0.01'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize('rows,n', [(70, 40), (1400, 1032)])
@pytest.mark.parametrize('eight', [False, True])
def test_pre_activation_is_kept_where_the_caller_asks(act, dtype, rows, n, eight):
    """
    ``set_save_derivative(False)``: Z is kept in the layer's type instead of act'(Z), as in ``Linear``.  Whole numbers, exact
    in every type, so that dZ is off by its own rounding and the evaluation of act' (a few 1e-6), and dW by those times the
    rows (x is 0 or +-1) and its own rounding.
    """
    g = torch.Generator(device='cuda').manual_seed(rows)
    x = torch.randint(-1, 2, (rows, 8), generator=g, device='cuda').to(dtype)
    w = torch.randint(-1, 2, (2, 8, n), generator=g, device='cuda').to(dtype)
    dy = torch.randn(rows, n, generator=g, device='cuda').to(dtype)
    counts = [rows] if eight else [rows // 3, rows - rows // 3]
    leaf = (w[0] if eight else w).clone().requires_grad_()
    previous = attorch.set_save_derivative(False)
    try:
        y = attorch.Float8LinearAutoGrad.apply(x, leaf, None, act) if eight else \
            attorch.grouped_linear(x, offsets_of(counts), leaf, None, act)
    finally:
        attorch.set_save_derivative(previous)
    stack = leaf.detach().double().view(len(counts), 8, n)
    groups = [(e, r) for e, r in enumerate(torch.arange(rows, device='cuda').split(counts))]
    z64 = torch.cat([x[r].double() @ stack[e] for e, r in groups])
    kept = y.grad_fn.saved_tensors[3]
    assert kept.dtype is dtype and torch.equal(kept.double(), z64)
    dw, = torch.autograd.grad(y, leaf, dy)
    # fp32 operands are multiplied as TF32, which keeps 10 bits (a whole step of 2^-10 where they are cut off).
    eps = 2.0 ** -10 if dtype is torch.float32 else torch.finfo(dtype).eps / 2
    dz = dy.double() * act64(z64, act)[1]
    size = dz.abs() * eps + dy.double().abs() * 4e-6 + 2.0 ** -25
    expected = torch.stack([x[r].double().T @ dz[r] for _, r in groups]).view_as(leaf)
    bound = torch.stack([x[r].double().abs().T @ (size[r] + rows * 2.0 ** -23 * dz[r].abs()) for _, r in groups]).view_as(leaf)
    assert ((dw.double() - expected).abs() <= bound + eps * (expected.abs() + bound)).all()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('rows,k,n', [(70, 256, 136), (33, 100, 72)])
def test_frozen_layer_gives_the_trained_ones_bits_under_autocast(dtype, rows, k, n):
    """Both quantise the fp32 input itself; so the training form is right with respect to its held value too."""
    from tests.expert_helpers import held_as_e4m3
    torch.manual_seed(1)
    layer = attorch.Float8Linear(k, n, act_func='silu')
    x = torch.randn(rows, k, device='cuda')
    wide = torch.randn(rows, k + 3, device='cuda')
    for xx in (x, wide[:, 3:], x.T.contiguous().T):
        with torch.autocast('cuda', dtype=dtype):
            trained = layer(xx.clone().requires_grad_() if xx is x else xx)
            with torch.no_grad():
                evaluated = layer(xx)
                weight, scale = attorch.quantize_weight(layer.weight)
                served = attorch.float8_linear(xx, weight, scale, layer.bias, 'silu')
        assert trained.dtype is dtype and torch.equal(trained, served) and torch.equal(evaluated, served)
    z = held_as_e4m3(x, 1)[0] @ held_as_e4m3(layer.weight.detach(), 128)[0]
    size = held_as_e4m3(x, 1)[0].abs() @ held_as_e4m3(layer.weight.detach(), 128)[0].abs()
    with torch.autocast('cuda', dtype=dtype), torch.no_grad():
        plain = attorch.Float8LinearAutoGrad.apply(x, layer.weight, None, None)
    assert ((plain.double() - z).abs() <= torch.finfo(dtype).eps / 2 * z.abs() + k * 2.0 ** -23 * size + 2.0 ** -25).all()

"""
The 8-bit products on a GPU: the held values bit for bit, whole-number products exactly, any scales, gradients,
strides, values that are not finite.
"""

import pytest
import torch

import attorch_b200 as attorch
from attorch_b200 import _lib
from attorch_b200.float8_linear_layer import _quantize_rows, _quantize_weight
from tests.expert_helpers import act64, grouped64, held_as_e4m3, offsets_of, relative_error, small_integers

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def stream():
    return torch.cuda.current_stream().cuda_stream


def wild(shape, dtype, seed):
    """Values of very different sizes per block, with zeros, subnormals and exact powers of two."""
    g = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randn(shape, generator=g, device='cuda')
    x = x * torch.exp2(torch.randint(-12, 8, (*shape[:-1], 1), generator=g, device='cuda').float())
    x[torch.rand(shape, generator=g, device='cuda') < 0.05] = 0.0
    flat = x.view(-1, shape[-1])
    flat[0] = 0.0
    if flat.shape[0] > 4:
        flat[1] = torch.exp2(torch.randint(-20, 3, (shape[-1],), generator=g, device='cuda').float())
        flat[2] *= 2.0 ** -130 if dtype is not torch.float16 else 2.0 ** -14
        flat[3] = 448.0
        flat[4] = 449.0
    return x.to(dtype)


@pytest.mark.parametrize('rows,cols', [(1, 1), (1, 128), (5, 127), (16, 129), (17, 1000), (100, 4096), (3, 8), (513, 136)])
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_quantized_rows_bit_for_bit(rows, cols, dtype):
    x = wild((rows, cols), dtype, rows)
    q, scale = _quantize_rows(x, stream())
    held, scale64 = held_as_e4m3(x, 1)
    assert torch.equal(scale.T.double(), scale64)
    back = q.double() * scale.T.double().repeat_interleave(128, 1)[:, :cols]
    assert torch.equal(back, held)


@pytest.mark.parametrize('groups,rows,cols', [(0, 128, 128), (0, 1, 1), (0, 130, 255), (3, 64, 200), (2, 300, 136), (0, 1000, 513)])
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_quantized_weights_bit_for_bit(groups, rows, cols, dtype):
    w = wild((groups, rows, cols) if groups else (rows, cols), dtype, cols)
    q, q_t, scale = _quantize_weight(w, True, True, stream())
    only, public_scale = attorch.quantize_weight(w)
    assert torch.equal(only.float(), q_t.float()) and torch.equal(public_scale, scale)
    for e in range(max(groups, 1)):
        part = (lambda t: t[e]) if groups else (lambda t: t)
        held, scale64 = held_as_e4m3(part(w), 128)
        assert torch.equal(part(scale).T.double(), scale64)
        spread = part(scale).double().repeat_interleave(128, 0)[:cols].repeat_interleave(128, 1)[:, :rows]
        assert torch.equal(part(q_t).double() * spread, held.T)
        assert torch.equal(part(q).double() * spread.T, held)


def test_not_finite_blocks_become_nan():
    x = torch.ones(4, 300, device='cuda')
    x[1, 5] = float('inf')
    x[2, 200] = float('nan')
    q, scale = _quantize_rows(x, stream())
    assert torch.isfinite(scale).all()
    nan = q.float().isnan()
    assert nan[1, :128].all() and nan[2, 128:256].all() and int(nan.sum()) == 256
    w, s = attorch.quantize_weight(torch.ones(300, 40, device='cuda'))
    y = attorch.float8_linear(x, w, s)
    assert y[[1, 2]].isnan().all() and torch.equal(y[[0, 3]], torch.full((2, 40), 300.0, device='cuda'))


def exact_case(rows, k, n, dtype, groups=0, seed=0):
    """Whole numbers within +-4 that e4m3 holds exactly under power-of-two scales; sums stay below 256."""
    g = torch.Generator(device='cuda').manual_seed(seed)
    density = min(0.5, 2.0 / max(k, 1) ** 0.5)
    x = small_integers((rows, k), dtype, density, g) * torch.randint(1, 5, (rows, 1), generator=g, device='cuda').to(dtype)
    w = small_integers(((groups,) if groups else ()) + (k, n), dtype, density, g)
    b = small_integers(((groups,) if groups else ()) + (n,), dtype, 1.0, g)
    return x, w, b


@pytest.mark.parametrize('rows,k,n', [(1, 128, 128), (1, 4096, 1000), (3, 200, 33), (5, 16, 1), (33, 1000, 520), (128, 384, 256), (129, 130, 300),
                                      (300, 1, 8), (700, 2048, 2304), (1000, 520, 4104), (4, 8192, 40)])
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_products_are_exact(rows, k, n, dtype):
    x, w, b = exact_case(rows, k, n, dtype)
    expected = x.double() @ w.double() + b.double()
    assert float(expected.abs().max()) <= 256
    weight, scale = attorch.quantize_weight(w)
    y = attorch.float8_linear(x, weight, scale, b)
    assert y.dtype is dtype and torch.equal(y.double(), expected)
    attorch.check_status()


@pytest.mark.parametrize('counts,unused', [([0, 5, 0, 130, 1], 0), ([64, 65, 31], 9), ([1 if i % 2 else 0 for i in range(70)], 3), ([600, 0, 777], 40)])
@pytest.mark.parametrize('k,n', [(264, 200), (1000, 1032)])
def test_grouped_products_are_exact(counts, unused, k, n):
    rows = sum(counts) + unused
    x, w, b = exact_case(rows, k, n, torch.bfloat16, len(counts))
    weight, scale = attorch.quantize_weight(w)
    y64, _ = grouped64(x, counts, w, b, None)
    y = attorch.float8_grouped_linear(x, offsets_of(counts), weight, scale, b)
    assert torch.equal(y.double(), y64)
    attorch.check_status()


@pytest.mark.parametrize('flag', [_lib.FLAG_NO_PAIR, _lib.FLAG_NO_TMA_STORE])
def test_kernel_choices_agree(flag):
    x, w, b = exact_case(900, 520, 2056, torch.bfloat16)
    weight, scale = attorch.quantize_weight(w)
    previous = attorch.set_gemm_flags(flag)
    try:
        assert torch.equal(attorch.float8_linear(x, weight, scale, b).double(), x.double() @ w.double() + b.double())
    finally:
        attorch.set_gemm_flags(previous)


def product_bound(x, w, b, act, eps):
    """64-bit value and the most the roundings can be off: fp32 sums (k terms, then k / 128 scaled ones, products with two scales)."""
    z = x @ w + (0 if b is None else b.double())
    size = x.abs() @ w.abs() + (0 if b is None else b.double().abs())
    y = act64(z, act)[0]
    return y, eps * y.abs() + 1.2 * (x.shape[1] + 12) * 2.0 ** -23 * size + 1e-6 * (1 + z.abs())


@pytest.mark.parametrize('act', [None, 'gelu', 'silu', 'relu'])
@pytest.mark.parametrize('rows,k,n', [(1, 1024, 300), (70, 384, 130), (800, 640, 2100)])
def test_any_scales_and_activations(act, rows, k, n):
    """Stored weights with scales that are no powers of two, of very different sizes."""
    g = torch.Generator(device='cuda').manual_seed(7)
    weight = torch.randn(n, k, generator=g, device='cuda').to(torch.float8_e4m3fn)
    scale = torch.exp(torch.randn(-(-n // 128), -(-k // 128), generator=g, device='cuda')) / k ** 0.5
    x = torch.randn(rows, k, generator=g, device='cuda').bfloat16()
    b = torch.randn(n, generator=g, device='cuda').bfloat16()
    held, _ = held_as_e4m3(x, 1)
    spread = scale.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    expected, bound = product_bound(held, (weight.double() * spread).T, b, act, 2.0 ** -9 * 2)
    y = attorch.float8_linear(x, weight, scale, b, act)
    assert ((y.double() - expected).abs() <= bound).all()
    assert relative_error(y, expected) <= 2.0 ** -8


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('rows,k,n', [(1, 256, 136), (200, 264, 392), (130, 33, 70)])
def test_training_gradients(rows, k, n, dtype):
    """dX uses the held values of dY and W, dW and db the unquantised X and dY."""
    g = torch.Generator(device='cuda').manual_seed(8)
    x = torch.randn(rows, k, generator=g, device='cuda').to(dtype).requires_grad_()
    w = (torch.randn(k, n, generator=g, device='cuda') / k ** 0.5).to(dtype).requires_grad_()
    b = torch.randn(n, generator=g, device='cuda').to(dtype).requires_grad_()
    dy = torch.randn(rows, n, generator=g, device='cuda').to(dtype)
    y = attorch.Float8LinearAutoGrad.apply(x, w, b, None)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    eps = torch.finfo(dtype).eps / 2
    xq, wq, dq = held_as_e4m3(x.detach(), 1)[0], held_as_e4m3(w.detach(), 128)[0], held_as_e4m3(dy, 1)[0]
    tiny = 2.0 ** -25 if dtype is torch.float16 else 0.0
    for what, a, left, right, bias in (('y', y, xq, wq, b.detach()), ('dx', dx, dq, wq.T, None),
                                       ('dw', dw, x.detach().double().T, dy.double(), None)):
        expected, bound = product_bound(left, right, bias, None, eps)
        assert ((a.double() - expected).abs() <= bound + tiny).all(), what
    db64 = dy.double().sum(0)
    assert ((db.double() - db64).abs() <= eps * db64.abs() + rows * 2.0 ** -23 * dy.double().abs().sum(0) + tiny).all()


@pytest.mark.parametrize('act', ['gelu', 'silu'])
def test_training_with_an_activation(act):
    """Against the formula on the held operands; dZ is rounded to bf16, so near a border its held value may be the next one:
    dX is off by a share of e4m3's step."""
    g = torch.Generator(device='cuda').manual_seed(9)
    x = torch.randn(300, 256, generator=g, device='cuda').bfloat16().requires_grad_()
    w = (torch.randn(256, 384, generator=g, device='cuda') / 16).bfloat16().requires_grad_()
    dy = torch.randn(300, 384, generator=g, device='cuda').bfloat16()
    y = attorch.Float8LinearAutoGrad.apply(x, w, None, act)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    xq, wq = held_as_e4m3(x.detach(), 1)[0], held_as_e4m3(w.detach(), 128)[0]
    value, slope = act64(xq @ wq, act)
    dz = dy.double() * slope
    assert relative_error(y, value) <= 2.0 ** -8
    assert relative_error(dw, x.detach().double().T @ dz) <= 2.0 ** -7
    assert relative_error(dx, held_as_e4m3(dz.bfloat16(), 1)[0] @ wq.T) <= 2.0 ** -4 / 2


def test_layers():
    """Float8Linear trains from its parameters, shares them with a Linear, and serves from its frozen form."""
    torch.manual_seed(1)
    linear = attorch.Linear(200, 320, act_func='gelu', dtype=torch.bfloat16)
    layer = attorch.Float8Linear.from_linear(linear)
    assert layer.weight is linear.weight and set(layer.state_dict()) == set(linear.state_dict())
    x = torch.randn(2, 30, 200, device='cuda').bfloat16()
    y = layer(x)
    y.sum().backward()
    assert linear.weight.grad is not None and linear.bias.grad is not None and y.shape == (2, 30, 320)
    with torch.no_grad():
        expected = layer(x)
        assert torch.equal(expected, y)
        assert relative_error(expected, linear(x)) <= 2 * 2.0 ** -4 / 3 ** 0.5
        layer.freeze()
        assert layer.weight is None and torch.equal(layer(x), expected)
        assert torch.equal(layer(x, residual=expected), expected + expected)
    with pytest.raises(RuntimeError, match='no gradient'):
        layer(x.clone().requires_grad_())
    assert set(layer.state_dict()) == {'weight_float8', 'weight_scale', 'bias'}       # a frozen layer can be saved
    bucketed = attorch.Float8Linear.from_linear(linear)
    bucketed.weight_grad_out = torch.empty_like(linear.weight)
    with pytest.raises(RuntimeError, match='bucket'):
        bucketed(x)
    grouped = attorch.GroupedLinear(3, 128, 256, act_func='silu', dtype=torch.bfloat16)
    eight = attorch.Float8GroupedLinear.from_grouped(grouped)
    rows = torch.randn(50, 128, device='cuda').bfloat16()
    with torch.no_grad():
        a, e = eight(rows, offsets_of([20, 0, 25])), grouped(rows, offsets_of([20, 0, 25]))
    assert not a[45:].any() and relative_error(a, e) <= 2 * 2.0 ** -4 / 3 ** 0.5


def test_strides_autocast_and_empty():
    x, w, b = exact_case(60, 100, 72, torch.float32)
    weight, scale = attorch.quantize_weight(w)
    expected = x.double() @ w.double() + b.double()
    tight = weight.clone()                                   # rows of 100 bytes: not on 16-byte boundaries
    wide = torch.zeros(60, 130, device='cuda')
    wide[:, 3:103] = x
    for xx in (x, wide[:, 3:103], x.T.contiguous().T):
        for ww in (weight, tight):
            assert torch.equal(attorch.float8_linear(xx, ww, scale.T.contiguous().T, b).double(), expected)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        y = attorch.float8_linear(x, weight, scale, b)
    assert y.dtype is torch.bfloat16 and torch.equal(y.double(), expected)
    assert attorch.float8_linear(x[:0], weight, scale).shape == (0, 72)
    empty = x[:0].clone().requires_grad_()
    weight_leaf = w.clone().requires_grad_()
    y = attorch.Float8LinearAutoGrad.apply(empty, weight_leaf, None, None)
    dx, dw = torch.autograd.grad(y, (empty, weight_leaf), torch.empty(0, 72, device='cuda'))
    assert dx.shape == (0, 100) and not dw.any()


def test_captured_and_on_another_stream():
    x, w, b = exact_case(40, 256, 384, torch.float16)
    weight, scale = attorch.quantize_weight(w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = attorch.float8_linear(x, weight, scale, b)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = attorch.float8_linear(x, weight, scale, b)
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first.double(), -x.double() @ w.double() + b.double())
    assert torch.equal(y.double(), x.double() @ w.double() + b.double())
    attorch.check_status()

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


@pytest.mark.parametrize('act', [None, 'gelu', 'silu'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('counts,unused,k,n,forward,dx,dw', [
    ([700, 300, 0, 600], 0, 136, 1800, PAIR, 64, PAIR),                  # the second CTA of a group's last pair has few or no rows
    ([390, 0, 1000, 163], 7, 1032, 1800, PAIR, PAIR, 256),
    ([1] * 63 + [2], 0, 264, 2056, 256, 256, 256),                       # few rows each: one CTA, 256 columns
    ([70, 0, 130, 60], 5, 136, 264, 64, 64, 64)])
def test_activations_and_gradients_by_shape(act, dtype, counts, unused, k, n, forward, dx, dw):
    """Values, bias, activation, saved derivative and gradients within the bounds of their roundings."""
    from tests.test_grouped_linear_gpu import bounds
    g = torch.Generator(device='cuda').manual_seed(k)
    rows = sum(counts) + unused
    x = torch.randn(rows, k, generator=g, device='cuda').to(dtype)
    w = (torch.randn(len(counts), k, n, generator=g, device='cuda') / k ** 0.5).to(dtype)
    b = torch.randn(len(counts), n, generator=g, device='cuda').to(dtype)
    dy = torch.randn(rows, n, generator=g, device='cuda').to(dtype)
    expected, limits = bounds(x, counts, w, b, act, dy, torch.finfo(dtype).eps / 2, 2.0 ** -11)
    for leaves, shape, picked in (((x,), dx, (1,)), ((w, b), dw, (2, 3))):
        for t in leaves:
            t.requires_grad_()
        y = attorch.grouped_linear(x, offsets_of(counts), w, b, act)
        assert tile() == forward
        got = (y, *torch.autograd.grad(y, leaves, dy))
        assert tile() == shape
        for t in leaves:
            t.requires_grad_(False)
        for i, a in zip((0, *picked), got):
            # Below its smallest normal number a type's half step is absolute: fp16 values under 2^-14 are 2^-24 apart.
            limit = limits[i] + (2.0 ** -25 if dtype is torch.float16 else 0.0)
            assert ((a.double() - expected[i]).abs() <= limit).all(), ('y', 'dx', 'dw', 'db')[i]
    attorch.check_status()


def stored(groups, n, k, g):
    """8-bit weights and scales that are no powers of two and differ from block to block by up to e^6; in 64 bits."""
    lead = (groups,) if groups else ()
    weight = torch.randn(*lead, n, k, generator=g, device='cuda').to(torch.float8_e4m3fn)
    scale = torch.exp(1.5 * torch.randn(*lead, -(-n // 128), -(-k // 128), generator=g, device='cuda')) / k ** 0.5
    spread = scale.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]
    return weight, scale, (weight.double() * spread).transpose(-1, -2)


@pytest.mark.parametrize('act', [None, 'gelu', 'silu'])
@pytest.mark.parametrize('counts,unused,k,n,shape,alone', [
    ([1000], 0, 520, 4104, PAIR, 128), ([900], 0, 640, 4104, PAIR, 128),
    ([700, 300, 0, 600], 0, 136, 1800, PAIR, 128), ([260, 0, 1000, 233], 107, 1032, 1800, PAIR, 128), ([513, 255, 732], 0, 264, 2056, PAIR, 128),
    ([1] * 63 + [2], 0, 264, 2056, 128, 128), ([4], 0, 4104, 520, 32, 32), ([300, 0, 41], 9, 200, 2056, 64, 64)])
def test_8_bit_products_by_shape(act, counts, unused, k, n, shape, alone):
    """One weight and a stack, scales of every block its own, ragged ends; with the pair and without."""
    from tests.expert_helpers import held_as_e4m3
    from tests.test_float8_gpu import product_bound
    g = torch.Generator(device='cuda').manual_seed(n)
    groups, rows = len(counts), sum(counts) + unused
    single = groups == 1
    weight, scale, w64 = stored(0 if single else groups, n, k, g)
    x = torch.randn(rows, k, generator=g, device='cuda').bfloat16()
    b = torch.randn(n, generator=g, device='cuda').bfloat16() if single else torch.randn(groups, n, generator=g, device='cuda').bfloat16()
    held, at, parts = held_as_e4m3(x, 1)[0], 0, []
    for e, count in enumerate(counts):
        parts.append(product_bound(held[at:at + count], w64 if single else w64[e], b if single else b[e], act, 2.0 ** -8))
        at += count
    expected, limit = (torch.cat(p) for p in zip(*parts))
    for flags, picked in ((0, shape), (_lib.FLAG_NO_PAIR, alone), (_lib.FLAG_NO_TMA_STORE, shape)):
        previous = attorch.set_gemm_flags(flags)
        try:
            y = attorch.float8_linear(x, weight, scale, b, act) if single else \
                attorch.float8_grouped_linear(x, offsets_of(counts), weight, scale, b, act)
        finally:
            attorch.set_gemm_flags(previous)
        assert tile() == picked and not y[at:].any()
        assert ((y[:at].double() - expected).abs() <= limit).all()
    attorch.check_status()


@pytest.mark.parametrize('act', [None, 'silu', 'gelu'])
@pytest.mark.parametrize('rows,k,n,forward,dx', [(1000, 520, 4104, PAIR, 32), (1000, 4104, 520, 32, PAIR), (1500, 2056, 2056, PAIR, PAIR)])
def test_8_bit_training_by_shape(act, rows, k, n, forward, dx):
    """Weights whose blocks differ in size by powers of two up to 2^6: a scale of another block would be seen."""
    from tests.expert_helpers import act64, held_as_e4m3, relative_error
    from tests.test_float8_gpu import product_bound
    g = torch.Generator(device='cuda').manual_seed(k)
    x = torch.randn(rows, k, generator=g, device='cuda').bfloat16().requires_grad_()
    size = torch.exp2(torch.randint(-3, 4, (-(-k // 128), -(-n // 128)), generator=g, device='cuda').float())
    w = torch.randn(k, n, generator=g, device='cuda') / k ** 0.5
    w = (w * size.repeat_interleave(128, 0)[:k].repeat_interleave(128, 1)[:, :n]).bfloat16()
    dy = torch.randn(rows, n, generator=g, device='cuda').bfloat16()
    y = attorch.Float8LinearAutoGrad.apply(x, w, None, act)
    assert tile() == forward
    kept = y.grad_fn.saved_tensors[3]
    grad, = torch.autograd.grad(y, x, dy)
    assert tile() == dx
    wq, xq = held_as_e4m3(w, 128)[0], held_as_e4m3(x.detach(), 1)[0]
    expected, limit = product_bound(xq, wq, None, act, 2.0 ** -8)
    assert ((y.double() - expected).abs() <= limit).all()
    if act is None:
        expected, limit = product_bound(held_as_e4m3(dy, 1)[0], wq.T, None, None, 2.0 ** -8)
        assert ((grad.double() - expected).abs() <= limit).all()
    else:
        slope = act64(xq @ wq, act)[1]
        magnitude = xq.abs() @ wq.abs()
        # Half a step of fp16, the evaluation, and Z's own error in front of |act''| <= 1.2.
        assert ((kept.double() - slope).abs() <= 2.0 ** -11 * slope.abs() + 4e-6 + 1.2 * 1.2 * (k + 12) * 2.0 ** -23 * magnitude).all()
        dz = (dy.double() * kept.double()).bfloat16()            # what backward multiplies, rounding included
        expected, limit = product_bound(held_as_e4m3(dz, 1)[0], wq.T, None, None, 2.0 ** -8)
        assert ((grad.double() - expected).abs() <= limit).all() and relative_error(grad, (dy.double() * slope) @ wq.T) <= 2.0 ** -4
    attorch.check_status()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize('k,n', [(33, 57), (1, 1), (130, 66), (64, 65)])
def test_unaligned_operands_from_c(dtype, k, n):
    """Rows at odd distances, bases off 16 bytes: the CUDA-core kernel, which the Python layers pad their way around."""
    counts, unused = [70, 0, 129, 3], 5
    x, w, b, dy = integer_case(counts, unused, k, n, dtype)
    y64, (dx64, dw64, _) = grouped64(x, counts, w, b, None, dy)
    lib, rows, groups, offsets = _lib.load(), sum(counts) + unused, len(counts), offsets_of(counts)
    dt = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}[dtype]
    stream = torch.cuda.current_stream().cuda_stream
    status = torch.zeros(1, dtype=torch.int32, device='cuda')

    def shifted(t, pitch):
        """One element behind a 16-byte boundary, rows `pitch` elements apart."""
        held = torch.zeros(1 + t.shape[:-1].numel() * pitch, dtype=t.dtype, device='cuda')[1:].view(*t.shape[:-1], pitch)[..., :t.shape[-1]]
        return held.copy_(t)

    px, pn = k + 1 + k % 2, n + 1 + n % 2                                # odd pitches
    xs, ws, dys = shifted(x, px), shifted(w, pn), shifted(dy, pn)
    out, pre = (torch.full((rows, n), 7.0, dtype=dtype, device='cuda') for _ in range(2))
    _lib.check(lib.ab200_grouped_linear_forward(
        xs.data_ptr(), ws.data_ptr(), b.data_ptr(), offsets.data_ptr(), pre.data_ptr(), out.data_ptr(), rows, groups, k, n, px, k * pn, pn,
        n, n, dt, dt, 4, 0.0, status.data_ptr(), stream, 0), 'forward')        # 4: relu
    assert lib.ab200_last_path() == _lib.PATH_GENERIC and tile() == 0
    live = sum(counts)
    assert torch.equal(pre.double(), y64) and torch.equal(out.double(), y64.clamp(min=0)) and not out[live:].any()
    dx = torch.full((rows, k), 7.0, dtype=dtype, device='cuda')
    _lib.check(lib.ab200_grouped_linear_backward_input(
        dys.data_ptr(), ws.data_ptr(), offsets.data_ptr(), dx.data_ptr(), rows, groups, k, n, pn, k * pn, pn, k, dt, dt,
        status.data_ptr(), stream, 0), 'dx')
    assert lib.ab200_last_path() == _lib.PATH_GENERIC and torch.equal(dx.double(), dx64)
    dw = torch.full((groups, k, n), 7.0, dtype=dtype, device='cuda')
    _lib.check(lib.ab200_grouped_linear_backward_weight(
        xs.data_ptr(), dys.data_ptr(), offsets.data_ptr(), dw.data_ptr(), rows, groups, k, n, px, pn, dt, dt, status.data_ptr(), stream, 0),
        'dw')
    assert lib.ab200_last_path() == _lib.PATH_GENERIC and torch.equal(dw.double(), dw64) and not status.any()

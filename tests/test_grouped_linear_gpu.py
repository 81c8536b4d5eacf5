"""
The grouped linear layer on a GPU: whole-number inputs, whose results are exact in every type, over group sizes,
widths and kernels; activations and gradients against a 64-bit form; strides, offsets of other types and values,
streams, graphs.
"""

import pytest
import torch

import attorch_b200 as attorch
from attorch_b200 import _lib
from tests.expert_helpers import grouped64, offsets_of, relative_error, small_integers

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]

# Group sizes: none, one, odd, around tile borders (32, 64, 128, 256), and rows that belong to no group.
COUNTS = {
    'one row': ([1], 0),
    'single group': ([300], 0),
    'empty between': ([0, 5, 0, 0, 130, 1, 0], 0),
    'all empty': ([0, 0, 0], 7),
    'borders': ([31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257], 0),
    'unused rows': ([17, 0, 90], 41),
    'many': ([i % 4 for i in range(130)], 3),
    'most': ([1 if i % 3 else 0 for i in range(512)], 0),
}


def integer_case(counts, unused, k, n, dtype, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    rows = sum(counts) + unused
    # Sums of at most `k` (rows, n) products; the density keeps them well below 256, where bf16 is exact.
    density = min(1.0, 6.0 / max(k, n, max(counts) if counts else 1) ** 0.5)
    x = small_integers((rows, k), dtype, density, g)
    w = small_integers((len(counts), k, n), dtype, density, g)
    b = small_integers((len(counts), n), dtype, 1.0, g)
    dy = small_integers((rows, n), dtype, density, g)
    return x, w, b, dy


def check_exact(counts, unused, k, n, dtype, bias=True):
    x, w, b, dy = integer_case(counts, unused, k, n, dtype)
    b = b if bias else None
    y64, (dx64, dw64, db64) = grouped64(x, counts, w, b, None, dy)
    for t in (x, w) + ((b,) if bias else ()):
        t.requires_grad_()
    y = attorch.grouped_linear(x, offsets_of(counts), w, b)
    got = torch.autograd.grad(y, (x, w) + ((b,) if bias else ()), dy)
    for what, a, e in zip(('y', 'dx', 'dw', 'db'), (y, *got), (y64, dx64, dw64, db64)):
        assert a.dtype is dtype and float(e.abs().max() if e.numel() else 0) <= 256, what
        assert torch.equal(a.double(), e), f'{what}: {int((a.double() != e).sum())} of {e.numel()} differ'
    attorch.check_status()


@pytest.mark.parametrize('name', COUNTS)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_group_sizes_are_exact(name, dtype):
    counts, unused = COUNTS[name]
    check_exact(counts, unused, 96, 72, dtype)


@pytest.mark.parametrize('k,n', [(8, 8), (64, 256), (72, 264), (200, 520), (1000, 136), (24, 2048), (1, 1), (7, 9), (130, 33), (65, 64)])
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_widths_are_exact(k, n, dtype):
    """Widths that end inside a tile, a stage and a 16-byte unit (those run on the CUDA-core kernel)."""
    check_exact([70, 0, 129, 3], 5, k, n, dtype)


@pytest.mark.parametrize('counts', [[600, 0, 700, 260], [256, 512, 257, 255], [1500, 33]])
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_pairs_are_exact(counts, dtype):
    """Sizes that run as CTA pairs, whose second CTA has some or no rows of a group's last tile."""
    check_exact(counts, 0, 1032, 1800, dtype, bias=False)
    check_exact(counts, 150, 520, 2056, dtype)


@pytest.mark.parametrize('flag', [_lib.FLAG_NO_PAIR, _lib.FLAG_FORCE_GENERIC, _lib.FLAG_NO_TMA_STORE, 40 << _lib.FLAG_RESERVE_SMS_SHIFT])
def test_kernel_choices_agree(flag):
    previous = attorch.set_gemm_flags(flag)
    try:
        check_exact([600, 0, 700, 261], 30, 264, 1032, torch.bfloat16)
    finally:
        attorch.set_gemm_flags(previous)


def bounds(x, counts, w, b, act, dy, eps, slope_eps):
    """
    Largest errors the roundings can make, element by element (eps: half a step of the type, slope_eps: of the type act' is
    held in).  A sum of n products in fp32 is off by at most n 2^-23 of the sum of magnitudes.  dZ has the rounding of act',
    act' taken at Z rounded to the type (|act''| <= 1.2 for these activations), and its own.
    """
    y64, _ = grouped64(x, counts, w, b, act, dy)
    xa, wa = x.double().abs(), w.double().abs()
    size, _ = grouped64(xa, counts, wa, None if b is None else b.abs(), None)
    z64, _ = grouped64(x, counts, w, b, None)
    by = eps * y64.abs() + 1.2 * (x.shape[1] + 8) * 2.0 ** -23 * size + 1e-6 * (1 + z64.abs())
    slope = torch.ones_like(z64)
    dslope = torch.zeros_like(z64)
    if act is not None:
        from tests.expert_helpers import act64
        slope = act64(z64, act)[1]
        dslope = slope_eps * slope.abs() + 1.2 * eps * z64.abs() + 1.2 * (x.shape[1] + 8) * 2.0 ** -23 * size + 2e-6
    dz = (dy.double() * slope).abs()
    ddz = dy.double().abs() * dslope
    ddz = ddz + eps * (dz + ddz) * (act is not None)
    bx, bw, bb = torch.zeros_like(xa), torch.zeros_like(wa), torch.zeros(w.shape[0], w.shape[2], dtype=torch.float64, device=x.device)
    at = 0
    for e, c in enumerate(counts):
        r = slice(at, at + c)
        at += c
        total = dz[r] + ddz[r]
        bx[r] = (ddz[r] + w.shape[2] * 2.0 ** -23 * total) @ wa[e].T
        bw[e] = xa[r].T @ (ddz[r] + c * 2.0 ** -23 * total)
        bb[e] = (ddz[r] + c * 2.0 ** -23 * total).sum(0)
    _, (dx64, dw64, db64) = grouped64(x, counts, w, b, act, dy)
    return (y64, dx64, dw64, db64), (by, bx + eps * (dx64.abs() + bx), bw + eps * (dw64.abs() + bw), bb + eps * (db64.abs() + bb))


@pytest.mark.parametrize('act', [None, 'relu', 'gelu', 'silu', 'sigmoid', 'leaky_relu_0.01'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('k,n', [(256, 384), (136, 40), (33, 57)])
def test_activations_and_gradients(act, dtype, k, n):
    counts, unused = [129, 0, 40, 300, 1], 11
    g = torch.Generator(device='cuda').manual_seed(3)
    rows = sum(counts) + unused
    x = torch.randn(rows, k, generator=g, device='cuda').to(dtype)
    w = (torch.randn(len(counts), k, n, generator=g, device='cuda') / k ** 0.5).to(dtype)
    b = torch.randn(len(counts), n, generator=g, device='cuda').to(dtype)
    dy = torch.randn(rows, n, generator=g, device='cuda').to(dtype)
    eps = torch.finfo(dtype).eps / 2
    slope_eps = 2.0 ** -11
    expected, bound = bounds(x, counts, w, b, act, dy, eps, slope_eps)
    for t in (x, w, b):
        t.requires_grad_()
    y = attorch.GroupedLinearAutoGrad.apply(x, offsets_of(counts), w, b, act)
    got = (y, *torch.autograd.grad(y, (x, w, b), dy))
    for what, a, e, limit in zip(('y', 'dx', 'dw', 'db'), got, expected, bound):
        # Below its smallest normal number a type's half step is absolute: fp16 values under 2^-14 are 2^-24 apart.
        limit = limit + (2.0 ** -25 if dtype is torch.float16 else 0.0)
        if act in ('relu', 'leaky_relu_0.01') and what != 'y':
            continue            # a pre-activation within rounding of 0 may fall on either side: the norm below bounds it
        over = (a.double() - e).abs() - limit
        assert (over <= 0).all(), f'{what}: {float(over.max())} over its bound'
    # At most four roundings of half a step each, independent: rms below 4 / sqrt(3) half steps.
    for what, a, e in zip(('y', 'dx', 'dw', 'db'), got, expected):
        assert relative_error(a, e) <= 4 / 3 ** 0.5 * eps + (5e-3 if 'relu' in (act or '') else 0.0), what
    attorch.check_status()


@pytest.mark.parametrize('k,n', [(264, 200), (130, 66)])
def test_fp32_is_multiplied_as_tf32(k, n):
    """Half a step of TF32 is 2^-11 per operand (hardware may truncate: a whole step, 2^-10)."""
    counts = [70, 0, 190]
    g = torch.Generator(device='cuda').manual_seed(4)
    x = torch.randn(260, k, generator=g, device='cuda')
    w = torch.randn(3, k, n, generator=g, device='cuda')
    dy = torch.randn(260, n, generator=g, device='cuda')
    y64, grads64 = grouped64(x, counts, w, None, None, dy)
    x.requires_grad_()
    w.requires_grad_()
    y = attorch.grouped_linear(x, offsets_of(counts), w)
    for a, e in zip((y, *torch.autograd.grad(y, (x, w), dy)), (y64, *grads64)):
        assert a.dtype is torch.float32 and relative_error(a, e) <= 2 * 2.0 ** -10


def test_gradient_against_differences():
    """Whole-number inputs and an odd polynomial of the output: central differences of step 1 are exact to the last digit."""
    counts = [3, 0, 5]
    g = torch.Generator(device='cuda').manual_seed(5)
    x = small_integers((8, 16), torch.float32, 0.7, g)
    w = small_integers((3, 16, 8), torch.float32, 0.7, g)
    offsets = offsets_of(counts)
    scale = torch.arange(64, device='cuda', dtype=torch.float32).view(8, 8) - 30

    def loss(xx, ww):
        return (attorch.grouped_linear(xx, offsets, ww) * scale).sum()

    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(loss(xg, wg), (xg, wg))
    for i, j in [(0, 0), (2, 7), (3, 1), (7, 15)]:
        step = torch.zeros_like(x)
        step[i, j] = 1.0
        assert float(dx[i, j]) == float(loss(x + step, w) - loss(x - step, w)) / 2
    for e, i, j in [(0, 0, 0), (1, 3, 3), (2, 15, 7)]:
        step = torch.zeros_like(w)
        step[e, i, j] = 1.0
        assert float(dw[e, i, j]) == float(loss(x, w + step) - loss(x, w - step)) / 2


def test_other_groups_values_do_not_leak():
    """NaN and infinities in the rows, weights and gradients of one group stay in that group."""
    counts = [70, 50, 90]
    x, w, b, dy = integer_case(counts, 20, 200, 136, torch.bfloat16)
    y64, (dx64, dw64, db64) = grouped64(x, counts, w, b, None, dy)
    x[70:120] = float('nan')
    w[1] = float('inf')
    dy[70:120] = float('nan')
    x[210:] = float('nan')
    dy[210:] = float('inf')
    for t in (x, w, b):
        t.requires_grad_()
    y = attorch.grouped_linear(x, offsets_of(counts), w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    rows = torch.cat([torch.arange(70), torch.arange(120, 230)]).cuda()
    assert torch.equal(y[rows].double(), y64[rows]) and torch.equal(dx[rows].double(), dx64[rows])
    assert torch.equal(dw[[0, 2]].double(), dw64[[0, 2]]) and torch.equal(db[[0, 2]].double(), db64[[0, 2]])
    assert not dw[1].isfinite().any() and not db[1].isfinite().any()


@pytest.mark.parametrize('offsets', [[0, 3, 1, 9], [5, 9, 12, 20], [0, 4, 40, 50], [0, -3, 7, 2 ** 31 - 1]])
def test_bad_offsets_stay_in_bounds(offsets):
    """Descending, late, too large: clamped and made ascending, as the operator says."""
    x, w, _, dy = integer_case([20, 0, 0], 0, 64, 72, torch.bfloat16)
    ends, last = [0], 0
    for v in offsets[1:]:
        last = max(last, min(max(v, 0), 20))
        ends.append(last)
    counts = [b - a for a, b in zip(ends, ends[1:])]
    y64, (dx64, dw64, _) = grouped64(x, counts, w, None, None, dy)
    x.requires_grad_()
    w.requires_grad_()
    y = attorch.grouped_linear(x, torch.tensor(offsets, dtype=torch.int64, device='cuda'), w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(y.double(), y64) and torch.equal(dx.double(), dx64) and torch.equal(dw.double(), dw64)


def test_strides_and_layouts():
    """Row views, transposed and expanded operands, stacks with gaps and a gradient that is an expanded scalar."""
    counts = [40, 60]
    x, w, b, _ = integer_case(counts, 0, 64, 96, torch.float16)
    y64, _ = grouped64(x, counts, w, b, None)
    offsets = offsets_of(counts)
    wide = torch.zeros(100, 200, dtype=x.dtype, device='cuda')
    wide[:, 8:72] = x
    odd = torch.zeros(100, 67, dtype=x.dtype, device='cuda')
    odd[:, 1:65] = x
    stack = torch.zeros(2, 80, 104, dtype=w.dtype, device='cuda')
    stack[:, :64, :96] = w
    for xx in (wide[:, 8:72], odd[:, 1:65], x.T.contiguous().T):
        for ww in (w, stack[:, :64, :96], w.transpose(1, 2).contiguous().transpose(1, 2)):
            assert torch.equal(attorch.grouped_linear(xx, offsets, ww, b.T.contiguous().T).double(), y64)
    same = w[:1].expand(2, -1, -1)
    assert torch.equal(attorch.grouped_linear(x, offsets, same, None).double(), x.double() @ w[0].double())
    xg = x.clone().requires_grad_()
    attorch.grouped_linear(xg, offsets, w, b).sum().backward()
    _, (dx64, _, _) = grouped64(x, counts, w, b, None, torch.ones(100, 96, device='cuda'))
    assert torch.equal(xg.grad.double(), dx64)


def test_shared_weight_gets_the_sum_of_its_gradients():
    """One matrix expanded over the groups: its gradient is the sum over them."""
    counts = [40, 60]
    x, w, _, dy = integer_case(counts, 0, 64, 96, torch.float32)
    shared = w[0].clone().requires_grad_()
    attorch.grouped_linear(x, offsets_of(counts), shared.expand(2, -1, -1)).backward(dy)
    assert torch.equal(shared.grad.double(), x.double().T @ dy.double())


def test_autocast_and_mixed_parameter_types():
    """fp32 parameters under autocast: 16-bit operands, 32-bit parameter gradients."""
    counts = [33, 0, 200]
    x, w, b, dy = integer_case(counts, 3, 128, 144, torch.float32)
    y64, (dx64, dw64, db64) = grouped64(x, counts, w, b, None, dy)
    layer = attorch.GroupedLinear(3, 128, 144)
    with torch.no_grad():
        layer.weight.copy_(w)
        layer.bias.copy_(b)
    x.requires_grad_()
    for dtype in (torch.float16, torch.bfloat16):
        x.grad = layer.weight.grad = layer.bias.grad = None
        with torch.autocast('cuda', dtype=dtype):
            y = layer(x, offsets_of(counts))
        assert y.dtype is dtype and torch.equal(y.double(), y64)
        y.backward(dy.to(dtype))
        for a, e in ((x.grad, dx64), (layer.weight.grad, dw64), (layer.bias.grad, db64)):
            assert a.dtype is torch.float32 and torch.equal(a.double(), e)


def test_only_the_asked_gradients():
    counts = [33, 20]
    x, w, b, dy = integer_case(counts, 0, 64, 64, torch.bfloat16)
    _, grads64 = grouped64(x, counts, w, b, None, dy)
    for i in range(3):
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        y = attorch.grouped_linear(leaves[0], offsets_of(counts), leaves[1], leaves[2])
        grad, = torch.autograd.grad(y, leaves[i], dy)
        assert torch.equal(grad.double(), grads64[i])


def test_no_rows_and_no_features():
    w = torch.randn(3, 32, 48, device='cuda', requires_grad=True)
    b = torch.randn(3, 48, device='cuda', requires_grad=True)
    x = torch.empty(0, 32, device='cuda', requires_grad=True)
    y = attorch.grouped_linear(x, offsets_of([0, 0, 0]), w, b, 'gelu')
    assert y.shape == (0, 48)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 48, device='cuda'))
    assert dx.shape == (0, 32) and not dw.any() and not db.any()
    # No input features: the bias is all there is.
    y = attorch.grouped_linear(torch.empty(5, 0, device='cuda'), offsets_of([2, 3]), torch.empty(2, 0, 16, device='cuda'),
                               torch.arange(32.0, device='cuda').view(2, 16))
    assert torch.equal(y, torch.arange(32.0, device='cuda').view(2, 16)[[0, 0, 1, 1, 1]])


def test_two_streams_and_a_captured_step():
    """Calls on two streams at once, and a captured forward and backward replayed with other group sizes."""
    x, w, b, dy = integer_case([100, 0, 156], 0, 128, 96, torch.bfloat16)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    plans = [[100, 0, 156], [7, 200, 49]]
    outs = []
    torch.cuda.synchronize()
    for stream, counts in zip(side, plans):
        offsets = offsets_of(counts)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            outs.append(attorch.grouped_linear(x, offsets, w, b))
    torch.cuda.synchronize()
    for counts, y in zip(plans, outs):
        assert torch.equal(y.double(), grouped64(x, counts, w, b, None)[0])

    offsets = offsets_of(plans[0])
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        y = attorch.grouped_linear(leaves[0], offsets, leaves[1], leaves[2], 'silu')
        torch.autograd.grad(y, leaves, dy)
    torch.cuda.current_stream().wait_stream(warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=warm):
        y = attorch.grouped_linear(leaves[0], offsets, leaves[1], leaves[2], 'silu')
        grads = torch.autograd.grad(y, leaves, dy)
    for counts in plans:
        offsets.copy_(offsets_of(counts))
        graph.replay()
        torch.cuda.synchronize()
        eager = attorch.grouped_linear(leaves[0], offsets_of(counts), leaves[1], leaves[2], 'silu')
        expected = torch.autograd.grad(eager, leaves, dy)
        for a, e in zip((y, *grads), (eager, *expected)):
            assert torch.equal(a, e)
    attorch.check_status()


def test_results_repeat():
    counts = [300, 11, 0, 513]
    g = torch.Generator(device='cuda').manual_seed(6)
    x = torch.randn(824, 512, generator=g, device='cuda').bfloat16().requires_grad_()
    w = torch.randn(4, 512, 768, generator=g, device='cuda').bfloat16().requires_grad_()
    b = torch.randn(4, 768, generator=g, device='cuda').bfloat16().requires_grad_()
    dy = torch.randn(824, 768, generator=g, device='cuda').bfloat16()
    runs = []
    for _ in range(2):
        y = attorch.grouped_linear(x, offsets_of(counts), w, b, 'gelu')
        runs.append((y, *torch.autograd.grad(y, (x, w, b), dy)))
    for a, e in zip(*runs):
        assert torch.equal(a, e)

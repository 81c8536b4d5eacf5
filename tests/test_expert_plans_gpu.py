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


def drop(routing, share, seed):
    """The plan with a share of its choices dropped, and which choices are left."""
    g = torch.Generator(device='cuda').manual_seed(seed)
    keep = (torch.rand(routing.token_row.shape, generator=g, device='cuda') >= share) & (routing.token_row >= 0)
    return routing._replace(token_row=torch.where(keep, routing.token_row, -1)), keep


def poison(*shape, dtype):
    """Memory that is handed out next holds NaN."""
    torch.full(shape, float('nan'), dtype=dtype, device='cuda')


@pytest.mark.parametrize('tokens,k,dim', [(1, 1, 8), (8, 4, 264), (33, 2, 7), (700, 3, 40), (9000, 8, 16), (1100000, 8, 1)])
@pytest.mark.parametrize('share', [0.0, 0.3, 1.0])
def test_dropped_choices_leave_zeros(tokens, k, dim, share):
    g = torch.Generator(device='cuda').manual_seed(tokens)
    logits = torch.randn(tokens, max(k, 8), generator=g, device='cuda')
    mask = torch.rand(tokens, generator=g, device='cuda') >= 0.1
    routing, keep = drop(attorch.route(logits, k, mask=mask), share, 2)
    x = torch.randn(tokens, dim, generator=g, device='cuda').bfloat16().requires_grad_()
    token, row = keep.nonzero()[:, 0], routing.token_row[keep].long()
    expected = torch.zeros(tokens * k, dim, dtype=x.dtype, device='cuda')
    expected[row] = x.detach()[token]
    poison(tokens * k, dim, dtype=x.dtype)
    rows = attorch.dispatch(x, routing)
    assert torch.equal(rows, expected)
    drows = torch.randn(tokens * k, dim, generator=g, device='cuda').bfloat16()
    poison(tokens, dim, dtype=x.dtype)
    dx, = torch.autograd.grad(rows, x, drows)
    total = torch.zeros(tokens, dim, dtype=torch.float64, device='cuda').index_add_(0, token, drows[row].double())
    size = torch.zeros(tokens, dim, dtype=torch.float64, device='cuda').index_add_(0, token, drows[row].double().abs())
    assert ((dx.double() - total).abs() <= 2.0 ** -9 * 2 * total.abs() + k * 2.0 ** -23 * size).all()

    h = torch.randn(tokens * k, dim, generator=g, device='cuda').bfloat16().requires_grad_()
    weights = routing.weights.detach().requires_grad_()
    dy = torch.randn(tokens, dim, generator=g, device='cuda').bfloat16()
    y = attorch.combine(h, routing._replace(weights=weights))
    poison(tokens * k, dim, dtype=x.dtype)
    dh, dw = torch.autograd.grad(y, (h, weights), dy)
    # A weight times a gradient is rounded to fp32 before it is stored: two roundings.
    dh64 = torch.zeros(tokens * k, dim, dtype=torch.float64, device='cuda')
    dh64[row] = weights.detach()[keep].double()[:, None] * dy[token].double()
    assert ((dh.double() - dh64).abs() <= (2.0 ** -9 * 2 + 2.0 ** -23) * dh64.abs()).all()
    products = h.detach()[row].double() * dy[token].double()
    assert not dw[~keep].any()
    assert ((dw[keep].double() - products.sum(1)).abs() <= dim * 2.0 ** -23 * products.abs().sum(1)).all()


def test_rows_behind_the_end_are_zeros_whatever_names_them():
    """A plan cut off at a smaller end: no entry reaches behind it."""
    routing = attorch.route(torch.randn(300, 4, device='cuda'), 2)
    routing.offsets.clamp_(max=201)
    x = torch.randn(300, 64, device='cuda')
    for _ in range(20):
        rows = attorch.dispatch(x, routing)
        assert not rows[201:].any() and torch.equal(rows[:201], x[routing.row_token[:201].long()])
        h = torch.ones(600, 64, device='cuda', requires_grad=True)
        attorch.combine(h, routing).sum().backward()
        assert not h.grad[201:].any() and (h.grad[:201] > 0).all()


def test_block_trains_with_dropped_choices():
    """Choices over a capacity dropped between routing and the experts: as if their rows did not exist."""
    torch.manual_seed(3)
    block = attorch.MixtureOfExperts(64, 96, 4, 2, 'silu', dtype=torch.bfloat16)
    x = torch.randn(400, 64, device='cuda').bfloat16()
    poisoned = []
    for again in range(2):
        routing, keep = drop(block.router(x), 0.4, 4)
        if again:
            for width in (64, 96):
                poison(800, width, dtype=x.dtype)
        rows = block.down(block.up(attorch.dispatch(x, routing), routing.offsets), routing.offsets)
        y = attorch.combine(rows, routing)
        if again:
            for width in (64, 96):
                poison(800, width, dtype=x.dtype)
        poisoned.append((y, *torch.autograd.grad(y, [block.up.weight, block.up.bias, block.down.weight, block.down.bias], torch.ones_like(y))))
    assert all(torch.isfinite(t).all() for t in poisoned[0]) and int((~keep).sum()) > 200
    for a, b in zip(*poisoned):
        assert torch.equal(a, b)


@pytest.mark.parametrize('gated', [False, True])
@pytest.mark.parametrize('held', [float('nan'), float('inf')])
@pytest.mark.parametrize('dim', [64, 60])
def test_padding_may_hold_anything(gated, held, dim):
    """Fully masked attention rows are NaN: as padding they change no output, gradient or parameter's gradient."""
    torch.manual_seed(5)
    block = attorch.MixtureOfExperts(dim, 96, 4, 2, 'gelu', gated=gated, dtype=torch.bfloat16)
    x = torch.randn(4, 50, dim, device='cuda').bfloat16()
    mask = torch.rand(4, 50, device='cuda') >= 0.3
    dy = torch.randn(4, 50, dim, device='cuda').bfloat16()
    results = []
    for value in (0.0, held):
        xx = torch.where(mask[..., None], x, value).requires_grad_()
        y = block(xx, mask)
        results.append((y, *torch.autograd.grad(y, [xx, *block.parameters()], dy)))
    names = ('y', 'x', *(name for name, _ in block.named_parameters()))
    for name, a, b in zip(names, *results):
        assert torch.isfinite(b).all(), name
        if name in ('x', 'router.gate.weight'):        # Linear's products: their pieces may be added in another order
            torch.testing.assert_close(a, b, rtol=2.0 ** -7, atol=2.0 ** -7)
        else:
            assert torch.equal(a, b), name
    assert not results[1][0][~mask].any() and not results[1][1][~mask].any()
    attorch.check_status()


def test_mask_buffer_can_be_reused_before_backward():
    """Two batches in flight with one mask buffer: each backward uses what its forward was given."""
    torch.manual_seed(6)
    block = attorch.MixtureOfExperts(32, 48, 4, 2, 'relu', dtype=torch.bfloat16)
    params = list(block.parameters())
    xs = [torch.randn(60, 32, device='cuda').bfloat16() for _ in range(2)]
    masks = [torch.rand(60, device='cuda') >= 0.3 for _ in range(2)]
    for x, mask in zip(xs, masks):
        x[~mask] = float('nan')
    expected = [torch.autograd.grad(block(x, mask).float().sum(), params) for x, mask in zip(xs, masks)]
    buffer = torch.empty(60, dtype=torch.bool, device='cuda')
    losses = [block(x, buffer.copy_(mask)).float().sum() for x, mask in zip(xs, masks)]
    for loss, gradients in zip(losses, expected):
        for (name, _), a, b in zip(block.named_parameters(), torch.autograd.grad(loss, params), gradients):
            assert torch.isfinite(a).all() and (torch.equal(a, b) or name == 'router.gate.weight'), name
            torch.testing.assert_close(a, b, rtol=2.0 ** -7, atol=2.0 ** -7)


@pytest.mark.parametrize('gated', [False, True])
@pytest.mark.parametrize('shape,live', [((0, 64), 0), ((3, 0, 64), 0), ((1, 64), 1), ((1, 64), 0), ((2, 5, 64), 0), ((300, 64), 0)])
def test_block_with_no_or_only_padded_tokens(gated, shape, live):
    """Zero rows anywhere: outputs of the right shape, zero gradients of every parameter, none left as allocated."""
    torch.manual_seed(7)
    block = attorch.MixtureOfExperts(64, 96, 4, 2, 'silu', gated=gated, dtype=torch.bfloat16)
    x = torch.randn(shape, device='cuda').bfloat16().requires_grad_()
    mask = torch.full(shape[:-1], bool(live), device='cuda')
    poison(4, 64, 192, dtype=x.dtype)
    y = block(x, mask)
    grads = torch.autograd.grad(y, [x, *block.parameters()], torch.ones_like(y))
    assert y.shape == x.shape and grads[0].shape == x.shape
    if live:
        assert all(torch.isfinite(t).all() for t in (y, *grads)) and y.any() and grads[0].any()
    else:
        assert not y.any() and not any(t.any() for t in grads)
    with torch.no_grad():
        assert torch.equal(block(x, mask), y)
        assert block.to_float8()(x, mask).shape == y.shape and (live or not block(x, mask).any())
    attorch.check_status()

"""
Routing, dispatch and combine on a GPU against token-by-token 64-bit forms: ties, masks, infinities, NaN, sizes around
the kernels' borders, gradients, and the whole mixture-of-experts block.
"""

import math

import pytest
import torch

import attorch_b200 as attorch
from tests.expert_helpers import grouped64, offsets_of, relative_error, route64, small_integers

pytestmark = pytest.mark.gpu


def check_plan(routing, expected):
    for what, a, e in zip(('experts', 'offsets', 'row_token', 'token_row'), routing[1:], expected[1:5]):
        assert a.dtype is torch.int32 and torch.equal(a.cpu(), e), what


def check_weights(weights, expected):
    # exp, a sum of up to 512 terms in a tree over 32 lanes (16 + 5 additions) and a division, all in fp32: at most
    # 2 + 21 + 1 roundings of 2^-24 and exp's own 2 ulp, relative; the exponent's rounding |x| 2^-24 <= 40 2^-24.
    assert weights.dtype is torch.float32
    torch.testing.assert_close(weights.cpu().double(), expected, rtol=80 * 2.0 ** -24, atol=1e-30, equal_nan=True)


@pytest.mark.parametrize('tokens,experts,k', [(1, 1, 1), (1, 64, 8), (3, 4, 4), (31, 33, 5), (33, 8, 2), (255, 100, 7), (256, 128, 8),
                                              (257, 16, 3), (1000, 160, 6), (70, 512, 32), (4099, 8, 1), (300, 257, 9)])
@pytest.mark.parametrize('score_func,renormalize', [('softmax', True), ('softmax', False), ('sigmoid', True), ('sigmoid', False)])
def test_route_and_gradient(tokens, experts, k, score_func, renormalize):
    g = torch.Generator().manual_seed(tokens + experts)
    logits = (torch.randn(tokens, experts, generator=g) * 2).cuda().requires_grad_()
    grad = torch.randn(tokens, k, generator=g)
    expected = route64(logits.detach(), k, score_func, renormalize, None, grad)
    routing = attorch.route(logits, k, score_func, renormalize)
    check_plan(routing, expected)
    check_weights(routing.weights.detach(), expected[0])
    dlogits, = torch.autograd.grad(routing.weights, logits, grad.cuda())
    # The gradient's differences cancel: relative to the largest of its row's terms, a few dozen roundings.
    assert dlogits.dtype is torch.float32 and relative_error(dlogits.cpu(), expected[5]) <= 200 * 2.0 ** -24 + 1e-7


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_route_16_bit_logits_and_ties(dtype):
    """Rounded logits tie often: the lowest index comes first.  -0 and +0 tie too."""
    g = torch.Generator().manual_seed(1)
    logits = (torch.randint(-3, 4, (513, 40), generator=g) / 2).to(dtype)
    logits[5] = 0.0
    logits[5, ::2] = -0.0
    grad = torch.randn(513, 6, generator=g)
    expected = route64(logits, 6, 'softmax', True, None, grad)
    x = logits.cuda().requires_grad_()
    routing = attorch.route(x, 6)
    check_plan(routing, expected)
    check_weights(routing.weights.detach(), expected[0])
    dlogits, = torch.autograd.grad(routing.weights, x, grad.cuda())
    assert dlogits.dtype is dtype and relative_error(dlogits.cpu(), expected[5]) <= torch.finfo(dtype).eps / 2


@pytest.mark.parametrize('tokens', [40, 400])
@pytest.mark.parametrize('score_func,renormalize', [('softmax', True), ('softmax', False), ('sigmoid', True)])
def test_route_masks(tokens, score_func, renormalize):
    """Padded tokens, rows of -inf, rows with fewer experts than top_k, masks made of the type's lowest value."""
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(tokens, 24, generator=g)
    mask = torch.rand(tokens, generator=g) < 0.8
    logits[3] = -math.inf
    logits[4, 3:] = -math.inf
    logits[5, 2:] = torch.finfo(torch.float32).min
    logits[6] = torch.finfo(torch.float32).min
    mask[:7] = True
    mask[0] = False
    logits[0, 0] = math.nan                                  # what padding holds does not matter
    grad = torch.randn(tokens, 4, generator=g)
    expected = route64(logits, 4, score_func, renormalize, mask, grad)
    x = logits.cuda().requires_grad_()
    routing = attorch.route(x, 4, score_func, renormalize, mask.cuda())
    check_plan(routing, expected)
    check_weights(routing.weights.detach(), expected[0])
    dlogits, = torch.autograd.grad(routing.weights, x, grad.cuda())
    assert torch.isfinite(dlogits).all() and not dlogits[0].any() and not dlogits[3].any()
    live = [t for t in range(tokens) if t != 0]
    assert relative_error(dlogits.cpu()[live], expected[5][live]) <= 200 * 2.0 ** -24 + 1e-7
    everyone = attorch.route(x.detach(), 4, score_func, renormalize, torch.zeros(tokens, dtype=torch.bool, device='cuda'))
    assert not everyone.weights.any() and not everyone.offsets.any() and (everyone.row_token == -1).all() and (everyone.token_row == -1).all()


def test_route_nan_and_infinity():
    logits = torch.zeros(3, 8)
    logits[0, 3] = math.nan
    logits[1, 5] = math.inf
    routing = attorch.route(logits.cuda(), 2)
    assert routing.weights[0].isnan().all() and routing.weights[1].isnan().all() and torch.equal(routing.weights[2].cpu(), torch.tensor([0.5, 0.5]))
    assert routing.experts[0].tolist() == [3, 0] and routing.experts[1].tolist() == [5, 0]
    assert int(routing.offsets[-1]) == 6


def test_route_strides_and_no_tokens():
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(50, 100, generator=g)
    for logits in (wide[:, 10:42], wide.T[:50, :32], wide[:1].expand(50, 100)[:, :32], wide[::2, ::3]):
        routing = attorch.route(logits.cuda() if logits.is_contiguous() else _strided(logits), 3)
        check_plan(routing, route64(logits, 3, 'softmax', True, None))
    routing = attorch.route(torch.empty(0, 16, device='cuda'), 2)
    assert routing.weights.shape == (0, 2) and routing.offsets.tolist() == [0] * 17 and routing.row_token.numel() == 0


def _strided(t):
    """The same strides on the GPU."""
    out = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device='cuda')
    if 0 in t.stride():
        return t[:1].cuda().expand(t.shape)
    return out.copy_(t)


def plan_of(tokens, k, experts, g, share=0.1):
    chosen = torch.rand(tokens, experts, generator=g).argsort(1)[:, :k].int()
    logits = torch.full((tokens, experts), -math.inf)
    logits.scatter_(1, chosen.long(), torch.rand(tokens, k, generator=g) + 0.1)
    mask = torch.rand(tokens, generator=g) >= share
    return attorch.route(logits.cuda(), k, mask=mask.cuda())


@pytest.mark.parametrize('tokens,k,dim', [(1, 1, 1), (1, 8, 4096), (7, 2, 8), (130, 3, 100), (64, 32, 264), (500, 4, 1027), (1000, 5, 2048), (9, 6, 8192)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_dispatch_and_combine(tokens, k, dim, dtype):
    g = torch.Generator().manual_seed(tokens)
    routing = plan_of(tokens, k, max(k, 9), g)
    weights = torch.rand(tokens, k, generator=g).cuda().requires_grad_()
    routing = attorch.Routing(weights, *routing[1:])
    x = torch.randn(tokens, dim, generator=g).cuda().to(dtype).requires_grad_()
    h = torch.randn(tokens * k, dim, generator=g).cuda().to(dtype).requires_grad_()
    drows = torch.randn(tokens * k, dim, generator=g).cuda().to(dtype)
    dy = torch.randn(tokens, dim, generator=g).cuda().to(dtype)
    rows = attorch.dispatch(x, routing)
    y = attorch.combine(h, routing)
    dx, dh, dw = torch.autograd.grad((rows, y), (x, h, weights), (drows, dy))

    at = routing.token_row.long()
    live = (at >= 0).double()[..., None]
    gathered = h.detach().double()[at.clamp(min=0)] * live
    row_token = routing.row_token.long()
    used = (row_token >= 0)[:, None]
    assert torch.equal(rows.detach(), torch.where(used, x.detach()[row_token.clamp(min=0)], 0))
    eps = torch.finfo(dtype).eps / 2
    w64 = weights.detach().double()[..., None]
    expected = (gathered * w64).sum(1)
    size = (gathered * w64).abs().sum(1)
    tiny = 2.0 ** -25 if dtype is torch.float16 else 0.0
    assert ((y.double() - expected).abs() <= eps * expected.abs() + k * 2.0 ** -23 * size + tiny).all()
    back = drows.double()[at.clamp(min=0)] * live
    assert ((dx.double() - back.sum(1)).abs() <= eps * back.sum(1).abs() + k * 2.0 ** -23 * back.abs().sum(1) + tiny).all()
    dh64 = torch.zeros_like(h, dtype=torch.float64)
    dh64[at[at >= 0]] = (w64 * dy.double()[:, None, :])[at >= 0]
    assert ((dh.double() - dh64).abs() <= (eps + 2.0 ** -24) * dh64.abs() + tiny).all()
    products = gathered * dy.double()[:, None, :]
    assert ((dw.double() - products.sum(2)).abs() <= dim * 2.0 ** -23 * products.abs().sum(2)).all()
    assert dw.dtype is torch.float32


def test_moves_take_strided_rows_and_expanded_gradients():
    g = torch.Generator().manual_seed(9)
    routing = plan_of(60, 3, 10, g)
    wide = torch.randn(60, 90, generator=g).cuda()
    for x in (wide[:, 3:67], wide[:, :64], wide.T.contiguous().T[:, :64], wide[:1].expand(60, 90)):
        want = torch.where((routing.row_token >= 0)[:, None], x[routing.row_token.long().clamp(min=0)], 0)
        assert torch.equal(attorch.dispatch(x, routing), want)
        rows = want.clone().requires_grad_()
        attorch.combine(rows, routing).sum().backward()
        total = torch.zeros(180, device='cuda')
        live = routing.token_row >= 0
        total[routing.token_row[live].long()] = routing.weights[live]
        assert torch.equal(rows.grad, total[:, None].expand_as(rows))
    y = attorch.combine(torch.zeros(180, 8, device='cuda').expand(180, 8).T.contiguous().T, routing)
    assert not y.any()


def test_moves_ignore_rows_outside():
    """A plan whose entries lie outside the rows is skipped, not followed."""
    token_row = torch.tensor([[0, 7], [-5, 2 ** 30], [3, 1]], dtype=torch.int32, device='cuda')
    routing = attorch.Routing(torch.ones(3, 2, device='cuda'), token_row, torch.tensor([0, 99], dtype=torch.int32, device='cuda'), None, token_row)
    x = torch.arange(24.0, device='cuda').view(3, 8)
    rows = attorch.dispatch(x, routing)
    assert torch.equal(rows[[0, 3, 1]], x[[0, 2, 2]])
    y = attorch.combine(torch.ones(6, 8, device='cuda'), routing)
    assert torch.equal(y[:, 0].cpu(), torch.tensor([1.0, 0.0, 2.0]))


@pytest.mark.parametrize('gated', [False, True])
def test_mixture_of_experts_block(gated):
    """The whole block against the formula, gradients included, with padded tokens, and replayed from a graph."""
    torch.manual_seed(4)
    dim, hidden, experts, k, tokens = 96, 64, 6, 2, 75
    block = attorch.MixtureOfExperts(dim, hidden, experts, k, 'silu', gated=gated)
    x = torch.randn(3, 25, dim, device='cuda', requires_grad=True)
    mask = torch.ones(3, 25, dtype=torch.bool, device='cuda')
    mask[1, 20:] = False
    mask[2, 5:] = False
    dy = torch.randn(3, 25, dim, device='cuda')
    y = block(x, mask)
    params = list(block.parameters())
    got = torch.autograd.grad(y, [x, *params], dy)
    assert y.shape == x.shape and not y[~mask].any() and not got[0][~mask].any()

    x64 = x.detach().double().flatten(0, 1).requires_grad_()
    p64 = {n: p.detach().double().requires_grad_() for n, p in block.named_parameters()}
    logits = x64 @ p64['router.gate.weight']
    chosen = block.router(x.detach().flatten(0, 1), mask.flatten()).experts.long()          # TF32 logits decide
    picked = torch.softmax(logits, 1).gather(1, chosen.clamp(min=0))
    weights = picked / picked.sum(1, keepdim=True)
    out = torch.zeros_like(x64)
    for e in range(experts):
        for j in range(k):
            at = (chosen[:, j] == e).nonzero().flatten()
            z = x64[at] @ p64['up.weight'][e] + p64['up.bias'][e]
            z = z[:, :hidden] * torch.nn.functional.silu(z[:, hidden:]) if gated else torch.nn.functional.silu(z)
            out = out.index_add(0, at, weights[at, j, None] * (z @ p64['down.weight'][e] + p64['down.bias'][e]))
    expected = torch.autograd.grad(out, [x64, *(p64[n] for n, _ in block.named_parameters())], dy.double().flatten(0, 1))
    # TF32 products (a step of 2^-10 per operand at most), two of them in a row and up to four behind a gradient.
    for what, a, e in zip(('y', 'x', *(n for n, _ in block.named_parameters())), (y.flatten(0, 1), *got), (out, *expected)):
        assert relative_error(a.reshape(e.shape), e) <= 8 * 2.0 ** -10, what
    attorch.check_status()


def test_block_under_autocast_and_8_bit_weights():
    """bf16 under autocast stays near fp32; its 8-bit form is off by e4m3's half step of 2^-4 per operand and product."""
    torch.manual_seed(5)
    block = attorch.MixtureOfExperts(256, 384, 8, 2, 'gelu')
    x = torch.randn(70, 256, device='cuda')
    with torch.no_grad():
        plan = block.router(x)
        full = attorch.combine(block.down(block.up(attorch.dispatch(x, plan), plan.offsets), plan.offsets), plan)
        with torch.autocast('cuda', dtype=torch.bfloat16):
            rows = block.up(attorch.dispatch(x, plan), plan.offsets)
            half = attorch.combine(block.down(rows, plan.offsets), plan)
        assert half.dtype is torch.bfloat16 and relative_error(half, full) <= 8 * 2.0 ** -8
        block.to_float8()
        eight = attorch.combine(block.down(block.up(attorch.dispatch(x, plan), plan.offsets), plan.offsets), plan)
        # Four rounded operands of relative rms at most 2^-4 / sqrt(3) each, independent.
        assert relative_error(eight, full) <= 2 * 2.0 ** -4 / 3 ** 0.5 + 8 * 2.0 ** -10
        again = block(x)
        assert torch.equal(again, eight)


def test_block_step_in_a_graph():
    """A captured forward and backward replays with new tokens, which go to other experts."""
    torch.manual_seed(6)
    block = attorch.MixtureOfExperts(64, 96, 5, 2, 'relu', dtype=torch.bfloat16)
    x = torch.randn(300, 64, device='cuda').bfloat16()
    params = list(block.parameters())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(block(x).float().square().sum(), params)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = block(x)
        grads = torch.autograd.grad(y.float().square().sum(), params)
    for seed in (1, 2):
        x.copy_(torch.randn(300, 64, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda').bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        eager = block(x)
        assert torch.equal(y, eager)
        for (name, _), a, e in zip(block.named_parameters(), grads, torch.autograd.grad(eager.float().square().sum(), params)):
            # The gate's weight gradient is Linear's: its pieces are added in any order, then rounded to bf16.
            assert torch.equal(a, e) or (name == 'router.gate.weight' and relative_error(a, e) <= 2.0 ** -8), name
    attorch.check_status()


def test_first_call_of_a_stream_inside_a_capture():
    """The status word of a stream whose first call is captured is valid before the graph has run."""
    block = attorch.MixtureOfExperts(32, 32, 4, 2, 'relu', dtype=torch.bfloat16)
    x = torch.randn(20, 32, device='cuda').bfloat16()
    with torch.no_grad():
        expected = block(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            y = block(x)
        attorch.check_status()
        graph.replay()
        torch.cuda.synchronize()
    assert torch.equal(y, expected)
    attorch.check_status()


def test_two_graphs_of_one_stream_replayed_together():
    """Graphs captured on one stream share no workspace: replayed at once on two, both give their own results."""
    block = attorch.MixtureOfExperts(64, 128, 8, 2, 'silu', dtype=torch.bfloat16)
    xs = [torch.randn(600, 64, device='cuda').bfloat16() for _ in range(2)]
    stream = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.no_grad():
        for x in xs:
            block(x)
        torch.cuda.synchronize()
        for x in xs:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(block(x))
            graphs.append(graph)
        replay = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(20):
            for graph, s in zip(graphs, replay):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(xs, outs):
            assert torch.equal(y, block(x))
    attorch.check_status()

"""
The experts' and 8-bit operators on tensors of more than 2^31 elements.  Operands are outer products of small whole numbers, so
that every element of a result is known without a second product of that size.
"""

import pytest
import torch

import attorch_b200 as attorch
from tests.expert_helpers import offsets_of

pytestmark = pytest.mark.gpu

LIMIT = 1 << 31


@pytest.fixture(autouse=True)
def free_memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def signs(n, seed, keep=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    s = torch.randint(0, 2, (n,), generator=g, device='cuda') * 2 - 1
    return (s * (torch.rand(n, generator=g, device='cuda') < keep)).double()


def outer(a, b, dtype=torch.bfloat16):
    return a.to(dtype)[:, None] * b.to(dtype)[None, :]


def equal_outer(got, a, b):
    """got[r] == a[r] * b[e] for runs of rows with one b each, in pieces."""
    at = 0
    for rows, row in b:
        for r0 in range(at, at + rows, 8192):
            r1 = min(r0 + 8192, at + rows)
            if not torch.equal(got[r0:r1], (a[r0:r1, None] * row[None, :]).to(got.dtype)):
                return False
        at += rows
    return not got[at:].any()


def test_rows_of_many_features():
    """Output, dY and dZ of 70000 x 32768, the last group and the rows behind it above 2^31 elements."""
    counts, unused, k, n = [40000, 27000, 2900], 100, 64, 32768
    rows = sum(counts) + unused
    assert rows * n > LIMIT and (rows - unused - 2900) * n > LIMIT
    a, c, a2, d = signs(rows, 1), signs(k, 2, 0.3), signs(rows, 3), signs(n, 4, 0.01)
    w = torch.stack([outer(signs(k, 5 + e, 0.5), signs(n, 9 + e)) for e in range(3)])
    x, w, b = outer(a, c).requires_grad_(), w.requires_grad_(), torch.zeros(3, n, dtype=torch.bfloat16, device='cuda', requires_grad=True)
    y = attorch.grouped_linear(x, offsets_of(counts), w, b)
    assert equal_outer(y.detach(), a, [(count, c @ w[e].detach().double()) for e, count in enumerate(counts)])
    dx, dw, db = torch.autograd.grad(y, (x, w, b), outer(a2, d))
    del y
    assert equal_outer(dx, a2, [(count, d @ w[e].detach().double().T) for e, count in enumerate(counts)])
    at = 0
    for e, count in enumerate(counts):
        r = slice(at, at + count)
        at += count
        assert torch.equal(dw[e], ((a[r] @ a2[r]) * c[:, None] * d[None, :]).bfloat16())
        assert torch.equal(db[e], (a2[r].sum() * d).bfloat16())
    attorch.check_status()


@pytest.mark.parametrize('eight', [False, True])
def test_stack_of_many_weights(eight):
    """Weights of 260 x 4096 x 2056; rows only in the last experts."""
    groups, k, n = 260, 4096, 2056
    assert (groups - 3) * k * n > LIMIT
    counts = [0] * (groups - 3) + [5, 130, 1]
    rows = sum(counts)
    c = signs(k, 2, 0.02)
    w = torch.zeros(groups, k, n, dtype=torch.bfloat16, device='cuda')
    for e in range(groups - 3, groups):
        w[e] = outer(signs(k, 5 + e, 0.5), signs(n, 9 + e))
    a = signs(rows, 1)
    x = outer(a, c)
    expected = [(counts[e], c @ w[e].double()) for e in range(groups - 3, groups)]
    if eight:
        weight, scale = attorch.quantize_weight(w)
        assert torch.equal(weight[-1].double() * scale[-1].double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k],
                           w[-1].double().T)
        del w
        assert equal_outer(attorch.float8_grouped_linear(x, offsets_of(counts), weight, scale), a, expected)
    else:
        a2, d = signs(rows, 3), signs(n, 4, 0.02)
        x.requires_grad_()
        w.requires_grad_()
        y = attorch.grouped_linear(x, offsets_of(counts), w)
        assert equal_outer(y.detach(), a, expected)
        dx, dw = torch.autograd.grad(y, (x, w), outer(a2, d))
        assert equal_outer(dx, a2, [(counts[e], d @ w[e].detach().double().T) for e in range(groups - 3, groups)])
        at = 0
        for e in range(groups - 3, groups):
            r = slice(at, at + counts[e])
            at += counts[e]
            assert torch.equal(dw[e], ((a[r] @ a2[r]) * c[:, None] * d[None, :]).bfloat16())
        assert not dw[:groups - 3].any()
    attorch.check_status()


def test_8_bit_rows():
    """Activations of 530000 x 4104, held in 8 bits in the call, and a dY as large."""
    rows, k, n = 530000, 4104, 64
    assert rows * k > LIMIT
    a, c = signs(rows, 1), signs(k, 2, 0.02)
    w = outer(signs(k, 3, 0.5), signs(n, 4))
    weight, scale = attorch.quantize_weight(w)
    x = outer(a, c)
    assert equal_outer(attorch.float8_linear(x, weight, scale), a, [(rows, c @ w.double())])
    # The other way round: dY is the large one, and the output of the forward product.
    x, w = outer(a, signs(n, 5)).requires_grad_(), outer(signs(n, 6), signs(k, 7, 0.5))
    y = attorch.Float8LinearAutoGrad.apply(x, w, None, None)
    assert equal_outer(y.detach(), a, [(rows, signs(n, 5) @ w.double())])
    a2, d = signs(rows, 8), signs(k, 9, 0.02)
    dx, = torch.autograd.grad(y, x, outer(a2, d))
    assert equal_outer(dx, a2, [(rows, d @ w.double().T)])
    attorch.check_status()


def test_moves_of_many_rows():
    """Expert-sorted rows of 528000 x 4160, some choices dropped."""
    tokens, k, dim = 66000, 8, 4160
    assert tokens * k * dim > LIMIT
    g = torch.Generator(device='cuda').manual_seed(1)
    mask = torch.rand(tokens, generator=g, device='cuda') >= 0.02
    routing = attorch.route(torch.randn(tokens, 16, generator=g, device='cuda'), k, mask=mask)
    keep = (torch.rand(tokens, k, generator=g, device='cuda') >= 0.1) & (routing.token_row >= 0)
    routing = routing._replace(token_row=torch.where(keep, routing.token_row, -1), weights=torch.where(keep, 0.5, 0.0).requires_grad_())
    a, c = signs(tokens, 2), signs(dim, 3)
    token, row = keep.nonzero()[:, 0], routing.token_row[keep].long()
    per_row = torch.zeros(tokens * k, dtype=torch.float64, device='cuda')
    per_row[row] = a[token]
    rows = attorch.dispatch(outer(a, c), routing)
    assert equal_outer(rows, per_row, [(tokens * k, c)])
    rows.requires_grad_()
    y = attorch.combine(rows, routing)
    share = keep.sum(1).double() * 0.5
    assert equal_outer(y.detach(), a * share, [(tokens, c)])
    a2 = signs(tokens, 4)
    drows, dweights = torch.autograd.grad(y, (rows, routing.weights), outer(a2, c))
    per_row[row] = 0.5 * a2[token]
    assert equal_outer(drows, per_row, [(tokens * k, c)])
    assert torch.equal(dweights.double(), torch.where(keep, (a * a2 * dim)[:, None], 0.0))
    attorch.check_status()

"""Plain 64-bit forms of the expert block's operators and of the 8-bit product, and the inputs of their tests."""

import math

import torch


def offsets_of(counts, device='cuda', dtype=torch.int32):
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    return torch.tensor(ends, dtype=dtype, device=device)


def small_integers(shape, dtype, density, generator, device='cuda'):
    """-1, 0, 1: products and their sums are whole numbers, exact in every type while they stay small."""
    sign = torch.randint(0, 2, shape, generator=generator, device=device) * 2 - 1
    keep = torch.rand(shape, generator=generator, device=device) < density
    return (sign * keep).to(dtype)


def act64(z, act):
    """act(z), act'(z) in 64 bits for the activations the tests use."""
    if act is None:
        return z, torch.ones_like(z)
    if act == 'relu':
        return z.clamp(min=0), (z > 0).double()
    if act == 'sigmoid':
        p = torch.sigmoid(z)
        return p, p * (1 - p)
    if act == 'silu':
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if act == 'gelu':
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    assert act == 'leaky_relu_0.01'
    return torch.where(z > 0, z, 0.01 * z), torch.where(z > 0, 1.0, 0.01).double()


def grouped64(x, counts, w, b, act, dy=None):
    """y and, with dy, (dx, dw, db) of the grouped linear layer; rows behind the last group are zero."""
    x, w = x.double(), w.double()
    y = torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64, device=x.device)
    grads = None
    if dy is not None:
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        db = torch.zeros(w.shape[0], w.shape[2], dtype=torch.float64, device=x.device)
        grads = (dx, dw, db)
    at = 0
    for e, count in enumerate(counts):
        rows = slice(at, at + count)
        at += count
        if count == 0:
            continue
        z = x[rows] @ w[e] + (0 if b is None else b[e].double())
        y[rows], slope = act64(z, act)
        if dy is not None:
            dz = dy[rows].double() * slope
            dx[rows] = dz @ w[e].T
            dw[e] = x[rows].T @ dz
            db[e] = dz.sum(0)
    return y, grads


def held_as_e4m3(x, rows):
    """The values blocks of rows x 128 of a matrix are held as, and their scales [row blocks, column blocks], in 64 bits."""
    m, n = x.shape
    pad = torch.zeros(-(-m // rows) * rows, -(-n // 128) * 128, dtype=torch.float64, device=x.device)
    pad[:m, :n] = x.double()
    view = pad.view(-1, rows, pad.shape[1] // 128, 128)
    amax = view.abs().amax((1, 3), keepdim=True)
    scale = torch.ones_like(amax)
    for power in range(-126, 128):                       # the smallest power of two with amax <= 448 s
        s = 2.0 ** power
        scale = torch.where((amax > 448 * s / 2) & ((amax <= 448 * s) | (s == 2.0 ** 127)), s, scale)
    scale = torch.where((amax > 0) & (amax <= 448 * 2.0 ** -126), 2.0 ** -126, scale)
    held = (view / scale).float().to(torch.float8_e4m3fn).double() * scale
    return held.reshape(pad.shape)[:m, :n], scale[:, 0, :, 0]


def route64(logits, k, score_func, renormalize, mask, grad=None):
    """(weights, experts, offsets, row_token, token_row[, dlogits]) worked out token by token."""
    rows = logits.double().cpu()
    tokens, experts = rows.shape
    weights = torch.zeros(tokens, k, dtype=torch.float64)
    chosen = torch.full((tokens, k), -1, dtype=torch.int32)
    dlogits = torch.zeros_like(rows)
    for t in range(tokens):
        row = rows[t]
        if mask is not None and not bool(mask[t]):
            continue
        order = sorted((e for e in range(experts) if row[e] != -math.inf), key=lambda e: (-row[e], e))[:k]
        if not order:
            continue
        p = torch.softmax(row, 0) if score_func == 'softmax' else torch.sigmoid(row)
        picked = p[order]
        total = picked.sum() if renormalize else torch.tensor(1.0, dtype=torch.float64)
        w = picked / total if total > 0 else torch.zeros_like(picked)
        weights[t, :len(order)] = w
        chosen[t, :len(order)] = torch.tensor(order, dtype=torch.int32)
        if grad is not None:
            g = grad[t, :len(order)].double().cpu()
            if renormalize:
                g = (g - (g * w).sum()) / total if total > 0 else torch.zeros_like(g)
            dp = torch.zeros(experts, dtype=torch.float64)
            dp[order] = g
            dlogits[t] = p * (dp - (dp * p).sum()) if score_func == 'softmax' else dp * p * (1 - p)
    pairs = sorted((int(chosen[t, j]), t, j) for t in range(tokens) for j in range(k) if chosen[t, j] >= 0)
    counts = [0] * experts
    row_token = torch.full((tokens * k,), -1, dtype=torch.int32)
    token_row = torch.full((tokens, k), -1, dtype=torch.int32)
    for row, (e, t, j) in enumerate(pairs):
        counts[e] += 1
        row_token[row] = t
        token_row[t, j] = row
    out = (weights, chosen, offsets_of(counts, 'cpu'), row_token, token_row)
    return out if grad is None else (*out, dlogits)


def relative_error(actual, expected):
    """2-norm of the difference over the 2-norm of what was expected."""
    actual, expected = actual.detach().double(), expected.detach().double()
    norm = float(expected.norm())
    return float((actual - expected).norm()) / norm if norm > 0 else float(actual.norm())

"""
The operators of a mixture-of-experts block and of the 8-bit product, as cases to be measured: the sizes, what a
program has in hand before a call, the operator in elementary torch operations, and the call a user makes of this
package (``own``).

Kinds of case
    route     logits -> the k experts of every token, their weights and the expert-sorted row plan (and d logits)
    mix       token rows -> expert-sorted rows (dispatch) and back as a weighted sum (combine) (and their gradients)
    experts   y[r] = act(x[r] W_e + b_e) over ragged runs of rows (and dX, dW, db)
    float8    y = act(x W^T + b) with e4m3 operands and one scale per block of 128, for one weight or per expert
              (and dX, dW, db for one weight)
"""
import math
import random

import torch

own = False

TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
BLOCK = 128


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One new token of a chat: the smallest call, all latency.
        dict(name='route-one-token', kind='route', tokens=1, experts=64, k=8, dtype='bf16', score='softmax',
             renormalize=True, masked=0.0, grad=False),
        # A training batch with padding at the end of its sequences, scores not renormalised, gradient of the logits.
        dict(name='route-training', kind='route', tokens=16384, experts=128, k=8, dtype='fp32', score='softmax',
             renormalize=False, masked=0.06, grad=True),
        # Eight sequences decoding.
        dict(name='mix-decode', kind='mix', tokens=8, k=4, experts=16, dim=4096, dtype='fp16', masked=0.0, grad=False),
        # One GPU's share of a training batch, with padded tokens.
        dict(name='mix-training', kind='mix', tokens=8192, k=4, experts=32, dim=4096, dtype='bf16', masked=0.05, grad=True),
        # Eight tokens, eight experts each: most experts have one row or none, the call reads weights.
        dict(name='experts-decode', kind='experts', rows=64, experts=64, k_dim=4096, n_dim=2048, dtype='fp16',
             act='silu', bias=False, grad=False),
        # Small, odd and ragged, an expert without rows: a fine-tuning step.
        dict(name='experts-ragged', kind='experts', rows=3001, experts=7, k_dim=1000, n_dim=1416, dtype='bf16',
             act='gelu', bias=True, grad=True),
        # A training step of the up-projection of 32 experts.
        dict(name='experts-training', kind='experts', rows=32768, experts=32, k_dim=4096, n_dim=2048, dtype='bf16',
             act='silu', bias=True, grad=True),
        # One token through a wide output projection with stored 8-bit weights.
        dict(name='float8-one-token', kind='float8', rows=1, experts=0, k_dim=8192, n_dim=28672, dtype='fp16',
             act=None, bias=False, grad=False),
        # A prompt through a square projection with stored 8-bit weights.
        dict(name='float8-prompt', kind='float8', rows=8192, experts=0, k_dim=4096, n_dim=4096, dtype='bf16',
             act='gelu', bias=True, grad=False),
        # A training step of an up-projection: weights quantised in the call, gradients of all three.
        dict(name='float8-training', kind='float8', rows=16384, experts=0, k_dim=4096, n_dim=14336, dtype='bf16',
             act=None, bias=True, grad=True),
        # The decode step of 'experts-decode' with stored 8-bit weights.
        dict(name='float8-experts-decode', kind='float8', rows=64, experts=64, k_dim=4096, n_dim=2048, dtype='bf16',
             act=None, bias=False, grad=False),
        # A prompt through 32 experts with stored 8-bit weights.
        dict(name='float8-experts-prompt', kind='float8', rows=16384, experts=32, k_dim=4096, n_dim=2048,
             dtype='bf16', act='silu', bias=True, grad=False),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A feature size: mostly a multiple of 64 or 8, now and then any number."""
    n = _log_int(rng, low, high)
    step = rng.choice([64, 64, 64, 8, 8, 1])
    return max(step, n // step * step)


def draw(rng):
    kind = rng.choice(['route', 'mix', 'experts', 'experts', 'float8', 'float8'])
    grad = rng.random() < 0.5
    dtype = rng.choice(['bf16', 'bf16', 'fp16'])
    if kind == 'route':
        experts = _log_int(rng, 4, 256)
        return dict(kind=kind, tokens=_log_int(rng, 1, 16384), experts=experts, k=rng.randint(1, min(8, experts)),
                    dtype=rng.choice(['bf16', 'fp16', 'fp32']), score=rng.choice(['softmax', 'sigmoid']),
                    renormalize=rng.random() < 0.5, masked=rng.choice([0.0, 0.1]), grad=grad)
    if kind == 'mix':
        k = rng.randint(1, 8)
        dim = _width(rng, 64, 8192)
        tokens = min(_log_int(rng, 1, 8192), max(1, 8192 * 4 * 4096 // (k * dim)))
        return dict(kind=kind, tokens=tokens, k=k, experts=rng.randint(k, 64), dim=dim, dtype=dtype,
                    masked=rng.choice([0.0, 0.1]), grad=grad)
    k_dim, n_dim = _width(rng, 128, 8192), _width(rng, 128, 8192)
    experts = _log_int(rng, 2, 64) if kind == 'experts' or rng.random() < 0.4 else 0
    if experts:
        # Stacked weights of at most the largest listed case's size.
        experts = max(2, min(experts, 64 * 4096 * 2048 // (k_dim * n_dim)))
    if kind == 'float8':
        grad = grad and not experts
    cost = (6.0 if grad else 2.0) * k_dim * n_dim
    rows = min(_log_int(rng, 1, 32768), max(1, int((6.0 * 32768 * 4096 * 2048 if experts else 6.0 * 16384 * 4096 * 14336) / 2 / cost)))
    # The gradient of an 8-bit product quantises dZ; with an activation in between, dZ is itself a rounded value.
    act = None if kind == 'float8' and grad else rng.choice([None, 'gelu', 'silu', 'relu', 'sigmoid'])
    return dict(kind=kind, rows=rows, experts=experts, k_dim=k_dim, n_dim=n_dim, dtype=dtype, act=act,
                bias=rng.random() < 0.5, grad=grad)


def _counts(case):
    """Rows of every expert: uneven, some without any, the same for every seed (their order is not)."""
    rng = random.Random('%d %d' % (case['rows'], case['experts']))
    share = [0.0 if rng.random() < 0.08 else rng.lognormvariate(0.0, 0.5) for _ in range(case['experts'])]
    share[rng.randrange(len(share))] += 0.5
    total = sum(share)
    counts = [int(case['rows'] * s / total) for s in share]
    alive = [e for e, s in enumerate(share) if s > 0]
    for i in range(case['rows'] - sum(counts)):
        counts[alive[(i * 7919 + 3) % len(alive)]] += 1
    return counts


def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    if case['kind'] == 'route':
        t, e, k = case['tokens'], case['experts'], case['k']
        return {'bytes': t * e * size * (3 if case['grad'] else 1) + t * k * (20 if case['grad'] else 16) + 4 * e + t,
                'flops': t * e * (8 if case['grad'] else 4)}
    if case['kind'] == 'mix':
        t, k, d = case['tokens'], case['k'], case['dim']
        token, rows = t * d * size, t * k * d * size
        # dispatch reads tokens, writes rows; combine the reverse; backward again both, and combine's reads the rows too.
        return {'bytes': 2 * (token + rows) + (2 * (token + rows) + rows if case['grad'] else 0) + 16 * t * k,
                'flops': 2 * t * k * d * (4 if case['grad'] else 1)}
    m, k, n, e = case['rows'], case['k_dim'], case['n_dim'], case['experts']
    used = sum(c > 0 for c in _counts(case)) if e else 1
    total = max(e, 1)
    wsize = 1 if case['kind'] == 'float8' and not case['grad'] else size
    data = m * (k + n) * size + used * k * n * wsize + (used * n * size if case['bias'] else 0)
    if case['grad']:
        data += m * (k + n) * size + total * k * n * size + (total * n * size if case['bias'] else 0)
    return {'bytes': data, 'flops': 2.0 * m * k * n * (3 if case['grad'] else 1)}


# ------------------------------------------------------------------------------------------------ inputs
def _plan(experts, num_experts):
    """[tokens, k] expert of every choice (-1: none) -> offsets, row_token, token_row of the expert-sorted order."""
    tokens, k = experts.shape
    flat = torch.where(experts < 0, num_experts, experts).reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    per = torch.zeros(num_experts + 1, dtype=torch.int64, device=flat.device).index_add_(0, flat, torch.ones_like(flat))
    offsets = torch.zeros(num_experts + 1, dtype=torch.int32, device=flat.device)
    offsets[1:] = torch.cumsum(per[:num_experts], 0)
    row = torch.arange(tokens * k, device=flat.device)
    used = row < offsets[-1]
    row_token = torch.where(used, order // k, -1).int()
    token_row = torch.empty(tokens * k, dtype=torch.int32, device=flat.device)
    token_row[order] = torch.where(used, row, -1).int()
    return offsets, row_token, token_row.view(tokens, k)


def _block_scales(amax):
    """The smallest power of two s with amax <= 448 s (1 where amax is 0)."""
    mantissa, exponent = torch.frexp(amax)                      # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    shift = torch.where(mantissa > 0.875, exponent - 8, exponent - 9).clamp(min=-126)
    power = ((shift + 127) << 23).to(torch.int32).view(torch.float32)           # 2^shift, exactly
    return torch.where(amax > 0, power, 1.0)


def _blocks(x, rows, cols):
    """[..., M, N] -> [..., M / rows, rows, N / cols, cols], padded with zeros."""
    m, n = x.shape[-2:]
    x = torch.nn.functional.pad(x, (0, -n % cols, 0, -m % rows))
    return x.unflatten(-1, (-1, cols)).unflatten(-3, (-1, rows))


def _stored_weight(w):
    """[..., N, K] fp32 -> e4m3 values (row pitch a multiple of 16) and one fp32 scale per 128 x 128 block, as a checkpoint holds them."""
    n, k = w.shape[-2:]
    blocks = _blocks(w, BLOCK, BLOCK)
    scale = (blocks.abs().amax(dim=(-3, -1)) / 448).clamp(min=1e-30)
    q = (blocks / scale[..., :, None, :, None]).flatten(-2).flatten(-3, -2)[..., :n, :k].to(torch.float8_e4m3fn)
    held = torch.zeros(*w.shape[:-1], -(-k // 16) * 16, dtype=torch.float8_e4m3fn, device=w.device)
    held.view(torch.uint8)[..., :k] = q.contiguous().view(torch.uint8)
    return held[..., :k], scale.contiguous()


def prepare(case, seed):
    device = 'cuda'
    g = torch.Generator(device=device).manual_seed(seed)
    host = random.Random(seed)
    dtype, grad = TYPES[case['dtype']], case['grad']

    def normal(*shape, std=1.0, to=dtype):
        return (torch.randn(*shape, generator=g, device=device) * std).to(to)

    state = {'case': case}
    if case['kind'] == 'route':
        t, e = case['tokens'], case['experts']
        # A gate's logits: experts differ in how often they are chosen.
        state['logits'] = (normal(t, e, std=1.5, to=torch.float32) + normal(1, e, std=0.5, to=torch.float32)).to(dtype).requires_grad_(grad)
        state['mask'] = torch.rand(t, generator=g, device=device) >= case['masked'] if case['masked'] else None
        state['dweights'] = normal(t, case['k'], to=torch.float32) if grad else None
    elif case['kind'] == 'mix':
        t, k, d, e = case['tokens'], case['k'], case['dim'], case['experts']
        chosen = torch.rand(t, e, generator=g, device=device).argsort(dim=1)[:, :k].int()
        if case['masked']:
            chosen[torch.rand(t, generator=g, device=device) < case['masked']] = -1
        offsets, row_token, token_row = _plan(chosen, e)
        weights = torch.rand(t, k, generator=g, device=device) + 0.05
        weights = torch.where(chosen < 0, 0.0, weights / weights.sum(1, keepdim=True))
        state.update(x=normal(t, d).requires_grad_(grad), rows=normal(t * k, d).requires_grad_(grad),
                     weights=weights.requires_grad_(grad), experts=chosen, offsets=offsets, row_token=row_token,
                     token_row=token_row)
        if grad:
            state.update(drows=normal(t * k, d), dy=normal(t, d))
    else:
        m, k, n, e = case['rows'], case['k_dim'], case['n_dim'], case['experts']
        # Activations with a few channels larger than the others.
        channel = 1.0 + 7.0 * (torch.rand(k, generator=g, device=device) < 0.01).float()
        state['x'] = (torch.randn(m, k, generator=g, device=device) * channel).to(dtype).requires_grad_(grad)
        lead = (e,) if e else ()
        if e:
            counts = _counts(case)
            host.shuffle(counts)
            ends = [0]
            for c in counts:
                ends.append(ends[-1] + c)
            state['offsets'] = torch.tensor(ends, dtype=torch.int32, device=device)
            state['most'] = max(counts)         # a bound on an expert's rows, for the padded plain form
        if case['kind'] == 'float8' and not grad:
            state['weight'], state['scale'] = _stored_weight(normal(*lead, n, k, std=k ** -0.5, to=torch.float32))
        else:
            state['weight'] = normal(*lead, k, n, std=k ** -0.5).requires_grad_(grad)
        state['bias'] = normal(*lead, n, std=0.1).requires_grad_(grad) if case['bias'] else None
        if grad:
            state['dy'] = normal(m, n, std=0.01)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state['case']
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        if case['kind'] == 'route':
            return _route_plain(case, state)
        if case['kind'] == 'mix':
            return _mix_plain(case, state)
        if case['kind'] == 'experts':
            return _experts_plain(case, state)
        return _float8_plain(case, state)


def _run_own(case, s):
    import attorch_b200 as attorch
    grad = case['grad']
    with torch.set_grad_enabled(grad):
        if case['kind'] == 'route':
            routing = attorch.route(s['logits'], case['k'], case['score'], case['renormalize'], s['mask'])
            out = dict(zip(('weights', 'experts', 'offsets', 'row_token', 'token_row'), routing))
            if grad:
                out['dlogits'], = torch.autograd.grad(routing.weights, s['logits'], s['dweights'])
            return out
        if case['kind'] == 'mix':
            routing = attorch.Routing(s['weights'], s['experts'], s['offsets'], s['row_token'], s['token_row'])
            rows = attorch.dispatch(s['x'], routing)
            y = attorch.combine(s['rows'], routing)
            out = {'rows': rows, 'y': y}
            if grad:
                out['dx'], out['drows'], out['dweights'] = torch.autograd.grad(
                    (rows, y), (s['x'], s['rows'], s['weights']), (s['drows'], s['dy']))
            return out
        act = case['act']
        if case['kind'] == 'experts':
            y = attorch.grouped_linear(s['x'], s['offsets'], s['weight'], s['bias'], act)
        elif grad:
            y = attorch.Float8LinearAutoGrad.apply(s['x'], s['weight'], s['bias'], act)
        elif case['experts']:
            return {'y': attorch.float8_grouped_linear(s['x'], s['offsets'], s['weight'], s['scale'], s['bias'], act)}
        else:
            return {'y': attorch.float8_linear(s['x'], s['weight'], s['scale'], s['bias'], act)}
        out = {'y': y}
        if grad:
            leaves = [s['x'], s['weight']] + ([s['bias']] if s['bias'] is not None else [])
            out.update(zip(('dx', 'dweight', 'dbias'), torch.autograd.grad(y, leaves, s['dy'])))
        return out


# ------------------------------------------------------------------------------------------------ plain forms
def _act(z, act):
    """act(z) and act'(z)."""
    if act is None:
        return z, torch.ones_like(z)
    if act == 'relu':
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if act == 'gelu':
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    p = torch.sigmoid(z)
    if act == 'sigmoid':
        return p, p * (1 - p)
    return z * p, p * (1 + z * (1 - p))                          # silu


def _route_plain(case, s):
    logits, k = s['logits'].float(), case['k']
    num_experts = logits.shape[1]
    if s['mask'] is not None:
        logits = logits.masked_fill(~s['mask'][:, None], -math.inf)
    top, chosen = torch.sort(logits, dim=1, descending=True, stable=True)
    top, chosen = top[:, :k], chosen[:, :k]
    valid = top > -math.inf
    if case['score'] == 'softmax':
        score = torch.exp(logits - logits.amax(1, keepdim=True).clamp(min=-3e38))
        score = score / score.sum(1, keepdim=True).clamp(min=1e-30)
    else:
        score = torch.sigmoid(logits)
    picked = torch.where(valid, score.gather(1, chosen), 0.0)
    total = picked.sum(1, keepdim=True)
    weights = picked / torch.where(total > 0, total, 1.0) if case['renormalize'] else picked
    experts = torch.where(valid, chosen, -1).int()
    offsets, row_token, token_row = _plan(experts, num_experts)
    out = {'weights': weights, 'experts': experts, 'offsets': offsets, 'row_token': row_token, 'token_row': token_row}
    if case['grad']:
        d = s['dweights']
        if case['renormalize']:
            d = (d - (d * weights).sum(1, keepdim=True)) / torch.where(total > 0, total, 1.0)
        d = torch.where(valid, d, 0.0)
        dscore = torch.zeros_like(logits).scatter_(1, chosen, d)
        if case['score'] == 'softmax':
            dlogits = score * (dscore - (dscore * score).sum(1, keepdim=True))
        else:
            dlogits = dscore * score * (1 - score)
        out['dlogits'] = dlogits.to(s['logits'].dtype)
    return out


def _mix_plain(case, s):
    dtype = s['x'].dtype
    used = (s['row_token'] >= 0)[:, None]
    token = s['row_token'].clamp(min=0).long()
    valid = (s['token_row'] >= 0)[..., None]
    row = s['token_row'].clamp(min=0).long()
    rows = torch.where(used, s['x'][token], 0)
    gathered = torch.where(valid, s['rows'][row].float(), 0)                                  # [tokens, k, dim]
    weights = s['weights'].float()
    out = {'rows': rows, 'y': (gathered * weights[..., None]).sum(1).to(dtype)}
    if case['grad']:
        out['dx'] = torch.where(valid, s['drows'][row].float(), 0).sum(1).to(dtype)
        dy = s['dy'].float()
        drows = torch.zeros(rows.shape, dtype=torch.float32, device=rows.device)
        drows[row[valid[..., 0]]] = (weights[..., None] * dy[:, None, :])[valid[..., 0]]
        out['drows'] = drows.to(dtype)
        out['dweights'] = (gathered * dy[:, None, :]).sum(2)
    return out


def _pad(x, offsets, most):
    """Expert-sorted rows [R, D] -> [E, most, D] with zeros, and where each row went."""
    experts = offsets.numel() - 1
    row = torch.arange(x.shape[0], device=x.device)
    group = torch.searchsorted(offsets[1:].contiguous(), row.int(), right=True)
    at = group * most + row - offsets[group]
    padded = torch.zeros(experts * most, x.shape[1], dtype=x.dtype, device=x.device)
    padded[at] = x
    return padded.view(experts, most, -1), at


def _experts_plain(case, s):
    dtype = s['x'].dtype
    x, at = _pad(s['x'].float(), s['offsets'], s['most'])
    w = s['weight'].float()
    z = torch.bmm(x, w)
    if s['bias'] is not None:
        z = z + s['bias'].float()[:, None, :]
    y, slope = _act(z, case['act'])
    out = {'y': y.flatten(0, 1)[at].to(dtype)}
    if case['grad']:
        dz = _pad(s['dy'].float(), s['offsets'], s['most'])[0] * slope
        out['dx'] = torch.bmm(dz, w.transpose(1, 2)).flatten(0, 1)[at].to(dtype)
        out['dweight'] = torch.bmm(x.transpose(1, 2), dz).to(dtype)
        if s['bias'] is not None:
            out['dbias'] = dz.sum(1).to(dtype)
    return out


def _through_float8(x, rows, cols):
    """The e4m3 values with power-of-two block scales that x is held as, in fp32."""
    blocks = _blocks(x.float(), rows, cols)
    scale = _block_scales(blocks.abs().amax(dim=(-3, -1)))[..., :, None, :, None]
    held = (blocks / scale).to(torch.float8_e4m3fn).float() * scale
    return held.flatten(-2).flatten(-3, -2)[..., :x.shape[-2], :x.shape[-1]]


def _spread(q, scale):
    """Stored 8-bit weights times their block scales, in fp32."""
    n, k = q.shape[-2:]
    return q.float() * scale.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _float8_plain(case, s):
    dtype = s['x'].dtype
    x = _through_float8(s['x'], 1, BLOCK)
    w = _through_float8(s['weight'], BLOCK, BLOCK) if case['grad'] else _spread(s['weight'], s['scale']).transpose(-1, -2)
    if case['experts']:
        x, at = _pad(x, s['offsets'], s['most'])
    z = torch.matmul(x, w)
    if s['bias'] is not None:
        z = z + s['bias'].float().unsqueeze(-2)
    y = _act(z, case['act'])[0]
    out = {'y': (y.flatten(0, 1)[at] if case['experts'] else y).to(dtype)}
    if case['grad']:
        dz = s['dy']
        out['dx'] = torch.matmul(_through_float8(dz, 1, BLOCK), w.T).to(dtype)
        out['dweight'] = torch.matmul(s['x'].float().T, dz.float()).to(dtype)
        if s['bias'] is not None:
            out['dbias'] = dz.float().sum(0).to(dtype)
    return out


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        return {'route': _route_exact, 'mix': _mix_exact, 'experts': _experts_exact, 'float8': _float8_exact}[case['kind']](case, s)


def _route_exact(case, s):
    logits = s['logits'].double()
    tokens, k = logits.shape[0], case['k']
    alive = torch.ones(tokens, dtype=torch.bool, device=logits.device) if s['mask'] is None else s['mask']
    p = torch.softmax(logits, 1) if case['score'] == 'softmax' else 1 / (1 + torch.exp(-logits))
    left, picks = logits.clone(), []
    for _ in range(k):
        best = torch.eq(left, left.amax(1, keepdim=True)).int().argmax(1)          # first of the largest
        picks.append(best)
        left.scatter_(1, best[:, None], -math.inf)
    picks = torch.stack(picks, 1)
    chosen = torch.zeros_like(p).scatter_(1, picks, 1.0) * alive[:, None]
    norm = (p * chosen).sum(1, keepdim=True).clamp(min=1e-300) if case['renormalize'] else torch.ones_like(p[:, :1])
    out = {'weights': (p * chosen / norm).gather(1, picks), 'experts': None, 'offsets': None, 'row_token': None, 'token_row': None}
    if case['grad']:
        g = torch.zeros_like(p).scatter_(1, picks, s['dweights'].double()) * chosen
        if case['renormalize']:
            g = chosen * (g - (g * p * chosen / norm).sum(1, keepdim=True)) / norm
        out['dlogits'] = (p * (g - (g * p).sum(1, keepdim=True)) if case['score'] == 'softmax' else g * p * (1 - p)) * alive[:, None]
    return out


def _mix_exact(case, s):
    tokens, k = s['token_row'].shape
    dim = s['x'].shape[1]
    x, rows, w = s['x'].double(), s['rows'].double(), s['weights'].double()
    out = {'rows': torch.zeros_like(rows), 'y': torch.zeros_like(x)}
    if case['grad']:
        out.update(dx=torch.zeros_like(x), drows=torch.zeros_like(rows), dweights=torch.zeros_like(w))
        drows, dy = s['drows'].double(), s['dy'].double()
    for j in range(k):
        live = (s['token_row'][:, j] >= 0).nonzero().flatten()
        at = s['token_row'][live, j].long()
        out['rows'][at] = x[live]
        out['y'][live] += w[live, j, None] * rows[at]
        if case['grad']:
            out['dx'][live] += drows[at]
            out['drows'][at] = w[live, j, None] * dy[live]
            out['dweights'][live, j] = (rows[at] * dy[live]).sum(1)
    return out


def _experts_exact(case, s):
    ends = s['offsets'].tolist()
    m, n = s['x'].shape[0], case['n_dim']
    y = torch.zeros(m, n, dtype=torch.float64, device=s['x'].device)
    out = {'y': y}
    if case['grad']:
        out.update(dx=torch.zeros(s['x'].shape, dtype=torch.float64, device=y.device),
                   dweight=torch.zeros(s['weight'].shape, dtype=torch.float64, device=y.device))
        if s['bias'] is not None:
            out['dbias'] = torch.zeros(s['bias'].shape, dtype=torch.float64, device=y.device)
    for e in range(len(ends) - 1):
        at = slice(ends[e], ends[e + 1])
        x, w = s['x'][at].double(), s['weight'][e].double()
        z = x @ w + (s['bias'][e].double() if s['bias'] is not None else 0.0)
        value, slope = _act(z, case['act'])
        y[at] = value
        if case['grad']:
            dz = s['dy'][at].double() * slope
            out['dx'][at] = dz @ w.T
            out['dweight'][e] = x.T @ dz
            if s['bias'] is not None:
                out['dbias'][e] = dz.sum(0)
    return out


def _power_exact(exponent):
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _held_exact(x, rows):
    """What blocks of `rows` x 128 are held as, in fp64: the grid of e4m3 around every value, worked out from its definition."""
    m, k = x.shape
    pad = torch.zeros(-(-m // rows) * rows, -(-k // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    pad[:m, :k] = x.double()
    view = pad.view(-1, rows, pad.shape[1] // BLOCK, BLOCK)
    amax = view.abs().amax((1, 3), keepdim=True)
    scale = _power_exact(torch.ceil(torch.log2(amax.clamp(min=2.0 ** -126) / 448)))
    scale = torch.where(amax > 448 * scale, 2 * scale, torch.where(2 * amax <= 448 * scale, scale / 2, scale))
    scale = torch.where(amax > 0, scale.clamp(min=2.0 ** -126), 1.0)
    v = view / scale
    step = _power_exact(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)    # 3 mantissa bits, down to 2^-9
    return (torch.round(v / step) * step * scale).reshape(pad.shape)[:m, :k]


def _float8_exact(case, s):
    x = _held_exact(s['x'], 1)
    bias = s['bias'].double() if s['bias'] is not None else None
    if case['experts']:
        ends = s['offsets'].tolist()
        y = torch.zeros(x.shape[0], case['n_dim'], dtype=torch.float64, device=x.device)
        for e in range(case['experts']):
            at = slice(ends[e], ends[e + 1])
            z = x[at] @ _spread_exact(s['weight'][e], s['scale'][e]).T
            y[at] = _act(z + bias[e] if bias is not None else z, case['act'])[0]
        return {'y': y}
    w = _held_exact(s['weight'], BLOCK) if case['grad'] else _spread_exact(s['weight'], s['scale']).T
    z = x @ w
    out = {'y': _act(z + bias if bias is not None else z, case['act'])[0]}
    if case['grad']:
        dz = s['dy']
        out['dx'] = _held_exact(dz, 1) @ w.T
        out['dweight'] = s['x'].double().T @ dz.double()
        if bias is not None:
            out['dbias'] = dz.double().sum(0)
    return out


def _spread_exact(q, scale):
    n, k = q.shape
    row = torch.arange(n, device=q.device) // BLOCK
    col = torch.arange(k, device=q.device) // BLOCK
    return q.to(torch.float32).double() * scale.double()[row][:, col]

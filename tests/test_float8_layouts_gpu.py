"""The 8-bit quantisers on buffers wider than their operand, and the 8-bit product's narrowest tile."""

import pytest
import torch

from attorch_b200 import _lib
from tests.expert_helpers import held_as_e4m3

pytestmark = pytest.mark.gpu

MARK = 0x55


def stream():
    return torch.cuda.current_stream().cuda_stream


def check_bytes(held, first, cols, what):
    """Columns [first, first + cols) hold values, then zeros up to a multiple of 8, and nothing else was written."""
    end = first + -(-cols // 8) * 8
    assert not held[:, first + cols:end].any(), what
    assert (held[:, :first] == MARK).all() and (held[:, end:] == MARK).all(), what


@pytest.mark.parametrize('rows,cols', [(5, 64), (33, 20), (16, 129), (3, 8)])
@pytest.mark.parametrize('first', [0, 192])
def test_quantized_rows_leave_a_wider_buffer_alone(rows, cols, first):
    g = torch.Generator(device='cuda').manual_seed(cols)
    x = torch.randn(rows, cols, generator=g, device='cuda').bfloat16()
    held = torch.full((rows + 1, 512), MARK, dtype=torch.uint8, device='cuda')
    scale = torch.empty(-(-cols // 128), rows, device='cuda')
    _lib.check(_lib.load().ab200_float8_quantize_rows(x.data_ptr(), held.data_ptr() + first, scale.data_ptr(), rows, cols, cols, 512,
                                                      rows, _lib.BF16, stream()), 'quantize')
    assert (held[rows] == MARK).all()
    check_bytes(held[:rows], first, cols, 'rows')
    back = held[:rows, first:first + cols].contiguous().view(torch.float8_e4m3fn).double()
    assert torch.equal(back * scale.T.double().repeat_interleave(128, 1)[:, :cols], held_as_e4m3(x, 1)[0])


@pytest.mark.parametrize('k,n', [(64, 40), (20, 129), (130, 12)])
def test_quantized_weights_leave_a_wider_buffer_alone(k, n):
    g = torch.Generator(device='cuda').manual_seed(n)
    w = torch.randn(k, n, generator=g, device='cuda')
    q = torch.full((k + 1, 512), MARK, dtype=torch.uint8, device='cuda')
    q_t = torch.full((n + 1, 512), MARK, dtype=torch.uint8, device='cuda')
    scale = torch.empty(-(-n // 128), -(-k // 128), device='cuda')
    _lib.check(_lib.load().ab200_float8_quantize_weight(w.data_ptr(), q.data_ptr() + 16, q_t.data_ptr() + 16, scale.data_ptr(), 1, k, n, 0,
                                                        n, 512, 512, _lib.F32, stream()), 'quantize')
    assert (q[k] == MARK).all() and (q_t[n] == MARK).all()
    check_bytes(q[:k], 16, n, 'as stored')
    check_bytes(q_t[:n], 16, k, 'transposed')
    a, b = (t.contiguous().view(torch.float8_e4m3fn).float() for t in (q[:k, 16:16 + n], q_t[:n, 16:16 + k]))
    assert torch.equal(a, b.T)


@pytest.mark.parametrize('rows', [1, 33, 100])
@pytest.mark.parametrize('k,n', [(16384, 64), (8192, 1000), (128, 96)])
def test_narrow_products_repeat(rows, k, n):
    """
    Few columns: tiles of 32, whose upper four epilogue warps only hand the accumulators back.  Long reductions, many
    times over: every phase of the four accumulators is waited for by all lanes before it can be reused.
    """
    import attorch_b200 as attorch
    g = torch.Generator(device='cuda').manual_seed(rows)
    keep = 2.0 / k ** 0.5
    x = (torch.randint(-1, 2, (rows, k), generator=g, device='cuda') * (torch.rand(rows, k, generator=g, device='cuda') < keep)).bfloat16()
    w = (torch.randint(-1, 2, (k, n), generator=g, device='cuda') * (torch.rand(k, n, generator=g, device='cuda') < keep)).bfloat16()
    weight, scale = attorch.quantize_weight(w)
    expected = x.double() @ w.double()
    for _ in range(50):
        y = attorch.float8_linear(x, weight, scale)
    assert float(expected.abs().max()) <= 256 and torch.equal(y.double(), expected)
    attorch.check_status()

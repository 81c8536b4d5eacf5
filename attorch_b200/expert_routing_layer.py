"""
Routing of tokens to experts and the moves between token order and expert order: ``route`` (the ``top_k``
experts of every token, their weights, and the plan of the expert-sorted rows), ``dispatch`` (token rows to
expert-sorted rows) and ``combine`` (expert-sorted rows to token rows, as a weighted sum), with their
gradients; ``Router`` is the gate projection and ``route`` as a layer.

No counterpart in the reference.  The device work runs in the library's kernels (``ab200_route_*``,
``ab200_expert_*``); no value of a plan is read by the host, so nothing here synchronises.
"""

from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor, nn

from . import _lib
from ._launch import on, recorded, status_of, stream_of
from .grouped_linear_layer import _pitch, _rows_operand
from .linear_layer import (Linear, _cached_size, _dtype_id, _flags_for, _ptr, _require_cuda,
                           get_output_dtype)

MAX_EXPERTS, MAX_TOP_K = 512, 32


class Routing(NamedTuple):
    """
    Where every token goes.

    weights:   ``[tokens, top_k]`` fp32, largest first; 0 where a token had no expert left to choose.
    experts:   ``[tokens, top_k]`` int32, -1 where there was none.
    offsets:   ``[num_experts + 1]`` int32: first expert-sorted row of every expert, and the end of the last.
    row_token: ``[tokens * top_k]`` int32: the token of every row, -1 from ``offsets[-1]`` on.
    token_row: ``[tokens, top_k]`` int32: the row of every choice, -1 where there was none.

    ``dispatch`` and ``combine`` read ``token_row``, the weights and the end of ``offsets``; a plan of the caller's own needs
    those, with no row named twice.  A choice whose ``token_row`` is set to -1 (over an expert's capacity, say) is dropped: its
    row stays the expert's, holds zeros, and adds nothing to the token or to a gradient of the weights behind it.
    """
    weights: Tensor
    experts: Tensor
    offsets: Tensor
    row_token: Tensor
    token_row: Tensor


def _inner_unit(tensor: Tensor) -> Tensor:
    """The 2-D tensor itself if its rows are contiguous and do not overlap, else a contiguous copy."""
    rows, cols = tensor.shape
    if (cols <= 1 or tensor.stride(1) == 1) and (rows <= 1 or tensor.stride(0) >= cols):
        return tensor
    return tensor.contiguous()


_SCORE_FUNCS = {'softmax': 0, 'sigmoid': 1}


def _check_mask(mask: Optional[Tensor], tokens: int, device: torch.device) -> None:
    if mask is not None:
        assert mask.shape == (tokens,), f'The mask must have one entry per token ({tokens}), received shape {mask.shape}'
        assert mask.dtype is torch.bool, f'The mask must be boolean, received {mask.dtype}'
        assert mask.device == device, f'The mask is on {mask.device}, the tokens on {device}'


def _route(logits: Tensor, top_k: int, score_func: str, renormalize: bool, mask: Optional[Tensor], needs_grad: bool):
    assert logits.ndim == 2, f'Logits must be 2D, received shape {logits.shape}'
    tokens, experts = logits.shape
    if score_func not in _SCORE_FUNCS:
        raise ValueError(f"score_func must be 'softmax' or 'sigmoid', received {score_func!r}")
    assert 1 <= experts <= MAX_EXPERTS, f'1 to {MAX_EXPERTS} experts are supported, received {experts}'
    assert 1 <= top_k <= min(experts, MAX_TOP_K), \
        f'top_k must be 1 to {min(experts, MAX_TOP_K)} for {experts} experts, received {top_k}'
    _require_cuda(logits, 'logits')
    device = logits.device
    _check_mask(mask, tokens, device)
    if mask is not None:
        mask = mask if mask.is_contiguous() else mask.contiguous()
    dtype = _dtype_id(logits.dtype)
    logits = _inner_unit(logits)
    lib = _lib.load()
    with on(device):
        stream = stream_of(device)
        weights = torch.empty((tokens, top_k), dtype=torch.float32, device=device)
        # Tensors of their own, not parts of one: parts share a version counter, and a caller who edits the plan in place would
        # then seem to have changed `chosen`, which backward reads.
        chosen = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
        token_row = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
        row_token = torch.empty(tokens * top_k, dtype=torch.int32, device=device)
        offsets = torch.empty(experts + 1, dtype=torch.int32, device=device)
        stats = torch.empty((tokens, 2), dtype=torch.float32, device=device) if needs_grad else None
        ws_bytes = _cached_size('ab200_route_workspace_bytes', tokens, experts)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
        _lib.check(lib.ab200_route_forward(
            _ptr(logits), _ptr(mask), _ptr(weights), _ptr(chosen), _ptr(stats), _ptr(offsets), _ptr(row_token), _ptr(token_row),
            tokens, experts, top_k, _pitch(logits), dtype, _SCORE_FUNCS[score_func], int(bool(renormalize)), _ptr(workspace),
            ws_bytes, stream), 'ab200_route_forward')
    return (weights, chosen, offsets, row_token, token_row), logits, stats


class RouteAutoGrad(torch.autograd.Function):
    """``apply(logits, top_k, score_func, renormalize, mask)`` -> the five tensors of a ``Routing``."""
    @staticmethod
    def forward(ctx, logits: Tensor, top_k: int, score_func: str, renormalize: bool, mask: Optional[Tensor]):
        routing, logits, stats = _route(logits, top_k, score_func, renormalize, mask, True)
        ctx.mark_non_differentiable(*routing[1:])
        ctx.set_materialize_grads(False)
        ctx.score_func, ctx.renormalize = _SCORE_FUNCS[score_func], int(bool(renormalize))
        ctx.save_for_backward(logits, routing[0], routing[1], stats)
        return routing

    @staticmethod
    def backward(ctx, weights_grad: Optional[Tensor], *_) -> Tuple[Optional[Tensor], ...]:
        if weights_grad is None:
            return None, None, None, None, None
        logits, weights, chosen, stats = ctx.saved_tensors
        tokens, experts = logits.shape
        lib = _lib.load()
        with on(logits.device):
            stream = stream_of(logits.device)
            grad = weights_grad.float().contiguous()
            logits_grad = torch.empty((tokens, experts), dtype=logits.dtype, device=logits.device)
            _lib.check(lib.ab200_route_backward(
                _ptr(logits), _ptr(weights), _ptr(chosen), _ptr(stats), _ptr(grad), _ptr(logits_grad), tokens, experts,
                weights.shape[1], _pitch(logits), _dtype_id(logits.dtype), ctx.score_func, ctx.renormalize, stream),
                'ab200_route_backward')
        return logits_grad, None, None, None, None


def route(logits: Tensor, top_k: int, score_func: str = 'softmax', renormalize: bool = True,
          mask: Optional[Tensor] = None) -> Routing:
    """
    Chooses the ``top_k`` experts of every token and plans the expert-sorted rows.

    Args:
        logits: ``[tokens, num_experts]``.  The largest are chosen, equal ones by lowest index; -inf is never chosen,
            so a token with fewer finite logits than ``top_k`` goes to fewer experts.  NaN makes a token's weights NaN.
        top_k: Experts a token, at most 32.
        score_func: 'softmax' (over all experts) or 'sigmoid': the weight of a chosen expert.
        renormalize: Flag for dividing a token's weights by their sum.
        mask: Optional ``[tokens]`` boolean; False (padding) sends a token to no expert, whatever its logits are.
    """
    if recorded(logits):
        return Routing(*RouteAutoGrad.apply(logits, top_k, score_func, renormalize, mask))
    return Routing(*_route(logits, top_k, score_func, renormalize, mask, False)[0])


def _check_plan(routing: Routing, device: torch.device, tokens: Optional[int]) -> None:
    assert routing.token_row.ndim == 2 and routing.token_row.dtype is torch.int32 and routing.token_row.is_contiguous() and \
        routing.token_row.device == device, 'token_row must be a contiguous 2D int32 tensor on the device of the rows'
    assert routing.offsets.ndim == 1 and routing.offsets.shape[0] >= 1 and routing.offsets.dtype is torch.int32 and \
        routing.offsets.is_contiguous() and routing.offsets.device == device, \
        'offsets must be a contiguous 1D int32 tensor with an end of the last expert, on the device of the rows'
    assert tokens is None or routing.token_row.shape[0] == tokens, \
        f'The routing has {routing.token_row.shape[0]} tokens, the input {tokens}'


def _row_end(routing_offsets: Tensor) -> int:
    """Address of the end of the last expert's rows."""
    return routing_offsets.data_ptr() + 4 * (routing_offsets.shape[0] - 1)


def _dispatch(input: Tensor, token_row: Tensor, offsets: Tensor) -> Tensor:
    tokens, top_k = token_row.shape
    x = _inner_unit(input)
    lib = _lib.load()
    with on(x.device):
        stream = stream_of(x.device)
        rows = torch.empty((tokens * top_k, x.shape[1]), dtype=x.dtype, device=x.device)
        _lib.check(lib.ab200_expert_dispatch(_ptr(x), _ptr(token_row), _row_end(offsets), _ptr(rows), tokens, top_k,
                                             tokens * top_k, x.shape[1], _pitch(x), _dtype_id(x.dtype), stream),
                   'ab200_expert_dispatch')
    return rows


def _combine(rows: Tensor, token_row: Tensor, weights: Optional[Tensor]) -> Tensor:
    tokens, top_k = token_row.shape
    rows = _inner_unit(rows)
    lib = _lib.load()
    with on(rows.device):
        stream = stream_of(rows.device)
        output = torch.empty((tokens, rows.shape[1]), dtype=rows.dtype, device=rows.device)
        _lib.check(lib.ab200_expert_combine(_ptr(rows), _ptr(token_row), _ptr(weights), _ptr(output), tokens, top_k,
                                            rows.shape[0], rows.shape[1], _pitch(rows), _dtype_id(rows.dtype), stream),
                   'ab200_expert_combine')
    return output


class DispatchAutoGrad(torch.autograd.Function):
    """``apply(input, token_row, offsets)``: rows[token_row[t, j]] = input[t]."""
    @staticmethod
    def forward(ctx, input: Tensor, token_row: Tensor, offsets: Tensor) -> Tensor:
        ctx.save_for_backward(token_row)
        return _dispatch(input, token_row, offsets)

    @staticmethod
    def backward(ctx, rows_grad: Tensor) -> Tuple[Optional[Tensor], ...]:
        token_row, = ctx.saved_tensors
        return _combine(rows_grad, token_row, None), None, None


class CombineAutoGrad(torch.autograd.Function):
    """``apply(rows, weights, token_row, offsets)``: output[t] = sum_j weights[t, j] * rows[token_row[t, j]]."""
    @staticmethod
    def forward(ctx, rows: Tensor, weights: Tensor, token_row: Tensor, offsets: Tensor) -> Tensor:
        ctx.needs = (rows.requires_grad, weights.requires_grad)
        ctx.save_for_backward(rows, weights, token_row, offsets)
        return _combine(rows, token_row, weights)

    @staticmethod
    def backward(ctx, output_grad: Tensor) -> Tuple[Optional[Tensor], ...]:
        rows, weights, token_row, offsets = ctx.saved_tensors
        tokens, top_k = token_row.shape
        lib = _lib.load()
        with on(rows.device):
            stream = stream_of(rows.device)
            grad = _inner_unit(output_grad)
            rows = _inner_unit(rows)
            num_rows, dim = rows.shape
            rows_grad = torch.empty((num_rows, dim), dtype=rows.dtype, device=rows.device) if ctx.needs[0] else None
            weights_grad = torch.empty((tokens, top_k), dtype=torch.float32, device=rows.device) if ctx.needs[1] else None
            _lib.check(lib.ab200_expert_combine_backward(
                _ptr(grad), _ptr(rows), _ptr(token_row), _ptr(weights), _row_end(offsets), _ptr(rows_grad), _ptr(weights_grad),
                tokens, top_k, num_rows, dim, _pitch(grad), _pitch(rows), _dtype_id(rows.dtype), stream),
                'ab200_expert_combine_backward')
        return rows_grad, weights_grad, None, None


def dispatch(input: Tensor, routing: Routing) -> Tensor:
    """
    Copies every token's row to its experts: ``[tokens, dim]`` -> ``[tokens * top_k, dim]`` in expert order, zeros in
    all rows that ``routing.token_row`` does not name and in those from ``routing.offsets[-1]`` on.
    """
    assert input.ndim == 2, f'Inputs must be 2D, received shape {input.shape}'
    _require_cuda(input, 'input')
    _dtype_id(input.dtype)
    _check_plan(routing, input.device, input.shape[0])
    if recorded(input):
        return DispatchAutoGrad.apply(input, routing.token_row, routing.offsets)
    return _dispatch(input, routing.token_row, routing.offsets)


def combine(rows: Tensor, routing: Routing) -> Tensor:
    """
    Sums every token's expert outputs by its weights: ``[tokens * top_k, dim]`` in expert order -> ``[tokens, dim]``,
    in fp32, rounded once.  A token without experts gets zeros.
    """
    assert rows.ndim == 2, f'Rows must be 2D, received shape {rows.shape}'
    _require_cuda(rows, 'rows')
    _dtype_id(rows.dtype)
    _check_plan(routing, rows.device, None)
    assert rows.shape[0] == routing.token_row.numel(), \
        f'The routing has {routing.token_row.numel()} rows, received {rows.shape[0]}'
    weights = routing.weights
    assert weights.shape == routing.token_row.shape and weights.dtype is torch.float32 and weights.device == rows.device, \
        'weights must be fp32, one per choice, on the device of the rows'
    if not weights.is_contiguous():
        weights = weights.contiguous()
    if recorded(rows, weights):
        return CombineAutoGrad.apply(rows, weights, routing.token_row, routing.offsets)
    return _combine(rows, routing.token_row, weights)


class GateAutoGrad(torch.autograd.Function):
    """
    ``apply(input, weight)``: ``input @ weight`` with the bits of a row independent of timing.  ``Linear`` shares the
    reduction of a product this narrow out over all SMs and adds the pieces atomically, in an order that changes
    from call to call; a token whose logits nearly tie could then change its experts.  The grouped kernel with one
    group sums every output in one place.  The logits are fp32 whatever type is multiplied (fp32 as TF32, as in ``Linear``):
    rounded to 16 bits, near ties would become ties, which the lowest index wins.  Backward is ``Linear``'s, but rows where
    ``mask`` is False stay out of ``dW`` whatever they hold (their logits have no gradient, and zero times NaN is NaN).  The
    optional trailing arguments are those of ``LinearAutoGrad`` for data-parallel training: where ``dW`` goes and who is told of it.
    """
    @staticmethod
    def forward(ctx, input: Tensor, weight: Tensor, mask: Optional[Tensor] = None, weight_grad_out: Optional[Tensor] = None,
                grad_ready=None, dw_chunks: int = 1) -> Tensor:
        assert input.ndim == 2 and input.shape[1] == weight.shape[0], \
            f'Incompatible input ({input.shape}) and weights ({weight.shape}) shape'
        assert weight.device == input.device, f'The weights are on {weight.device}, the input on {input.device}'
        _check_mask(mask, input.shape[0], input.device)
        _require_cuda(input, 'input')
        _require_cuda(weight, 'weight')
        rows, in_dim = input.shape
        experts = weight.shape[1]
        dtype = get_output_dtype(input.dtype)
        lib = _lib.load()
        with on(input.device):
            stream = stream_of(input.device)
            x_op = _rows_operand(input, dtype, stream)
            w_op = _rows_operand(weight, dtype, stream)
            output = torch.empty((rows, experts), dtype=torch.float32, device=input.device)
            _lib.check(lib.ab200_grouped_linear_forward(
                _ptr(x_op), _ptr(w_op), None, None, None, _ptr(output), rows, 1, in_dim, experts, _pitch(x_op), 0, _pitch(w_op),
                experts, experts, _dtype_id(dtype), 0, _lib.ACT_NONE, 0.0, status_of(input.device), stream,
                _flags_for(input.device) | _lib.FLAG_OUTPUT_FP32), 'ab200_grouped_linear_forward')
        ctx.dtypes = (input.dtype, weight.dtype)
        ctx.needs = (input.requires_grad, weight.requires_grad)
        ctx.weight_grad_out, ctx.grad_ready, ctx.dw_chunks = weight_grad_out, grad_ready, int(dw_chunks)
        # The padded rows as they are now: the caller may fill the mask's buffer for the next batch before backward.
        ctx.save_for_backward(x_op, w_op, ~mask[:, None] if mask is not None and weight.requires_grad else None)
        return output

    @staticmethod
    def backward(ctx, output_grad: Tensor) -> Tuple[Optional[Tensor], ...]:
        x_op, w_op, padded = ctx.saved_tensors
        rows, in_dim = x_op.shape
        experts, dtype, device = w_op.shape[1], x_op.dtype, x_op.device
        input_grad = weight_grad = None
        with on(device):
            # The gradient of the logits is rounded to the operands' type here, for the tensor cores.
            dy = _rows_operand(output_grad, dtype, stream_of(device))
            if ctx.needs[1]:
                if padded is not None:
                    x_op = _rows_operand(x_op.masked_fill(padded, 0), dtype, stream_of(device))
                weight_grad = ctx.weight_grad_out if ctx.weight_grad_out is not None else \
                    torch.empty((in_dim, experts), dtype=ctx.dtypes[1], device=device)
                # Blocks of rows of dW, each handed to the gradient exchange as soon as it is enqueued.
                blocks = ctx.dw_chunks if ctx.grad_ready is not None and ctx.dw_chunks > 1 and in_dim % (ctx.dw_chunks * 8) == 0 else 1
                size = in_dim // blocks
                for block in range(blocks):
                    _gate_weight_grad(x_op[:, block * size:(block + 1) * size], dy, weight_grad[block * size:(block + 1) * size])
                    if ctx.grad_ready is not None:
                        ctx.grad_ready(block, blocks)
            elif ctx.grad_ready is not None:
                ctx.grad_ready(0, 1)
            if ctx.needs[0]:
                input_grad = torch.empty((rows, in_dim), dtype=ctx.dtypes[0], device=device)
                workspace, nbytes = _gemm_workspace(device, rows, in_dim, experts)
                _lib.check(_lib.load().ab200_linear_backward_input(
                    _ptr(dy), _ptr(w_op), _ptr(input_grad), rows, in_dim, experts, _pitch(dy), 1, _pitch(w_op), 1, in_dim,
                    _dtype_id(dtype), _dtype_id(input_grad.dtype), _ptr(workspace), nbytes, status_of(device), stream_of(device),
                    _flags_for(device)), 'ab200_linear_backward_input')
        # A gradient that went to the caller's buffer is not returned as well: autograd would add it to ``.grad``.
        return input_grad, None if ctx.weight_grad_out is not None else weight_grad, None, None, None, None


def _gemm_workspace(device: torch.device, *shape: int) -> Tuple[Optional[Tensor], int]:
    nbytes = _cached_size('ab200_gemm_workspace_bytes', *shape)
    return (torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None), nbytes


def _gate_weight_grad(x: Tensor, dy: Tensor, out: Tensor) -> None:
    """out = x^T dy."""
    (rows, in_dim), experts = x.shape, dy.shape[1]
    workspace, nbytes = _gemm_workspace(x.device, in_dim, experts, rows)
    _lib.check(_lib.load().ab200_linear_backward_weight(
        _ptr(x), _ptr(dy), _ptr(out), rows, in_dim, experts, _pitch(x), 1, _pitch(dy), 1, experts, _dtype_id(x.dtype),
        _dtype_id(out.dtype), _ptr(workspace), nbytes, status_of(x.device), stream_of(x.device), _flags_for(x.device)),
        'ab200_linear_backward_weight')


class Router(nn.Module):
    """
    The gate of a mixture-of-experts block: a projection to one logit per expert, and ``route``.

    Args:
        dim: Number of input features.
        num_experts: Number of experts, at most 512.
        top_k: Experts a token, at most 32.
        score_func: 'softmax' or 'sigmoid', as ``route``.
        renormalize: Flag for dividing a token's weights by their sum.
        device: Device to use.
        dtype: Dtype of layer.
    """
    def __init__(self, dim: int, num_experts: int, top_k: int, score_func: str = 'softmax', renormalize: bool = True,
                 device='cuda', dtype: torch.dtype = torch.float32) -> None:
        super().__init__()
        if not 1 <= num_experts <= MAX_EXPERTS or not 1 <= top_k <= min(num_experts, MAX_TOP_K):
            raise RuntimeError(f'1 to {MAX_EXPERTS} experts and 1 to {MAX_TOP_K} of them a token are supported, received '
                               f'{num_experts} and {top_k}.')
        if score_func not in _SCORE_FUNCS:
            raise ValueError(f"score_func must be 'softmax' or 'sigmoid', received {score_func!r}")
        self.top_k, self.score_func, self.renormalize = top_k, score_func, renormalize
        self.gate = Linear(dim, num_experts, bias=False, device=device, dtype=dtype)

    def forward(self, input: Tensor, mask: Optional[Tensor] = None) -> Routing:
        """``input``: ``[tokens, dim]``; ``mask``: see ``route``."""
        gate = self.gate
        if gate.defer_input_grad is not None and input.requires_grad:
            raise RuntimeError("The input gradient of a router's gate cannot be put off: autograd adds it to that of the dispatched "
                               'rows. Let another layer be the first of the bucket.')
        padding = mask if torch.is_grad_enabled() else None          # the gate needs it for its gradient only
        logits = GateAutoGrad.apply(input, gate.weight, padding, gate.weight_grad_out, gate.grad_ready, gate.dw_chunks)
        return route(logits, self.top_k, self.score_func, self.renormalize, mask)

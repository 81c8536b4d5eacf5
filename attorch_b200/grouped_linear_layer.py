"""
``GroupedLinear``: one ``Linear`` per group of rows (the experts of a mixture-of-experts block) as one
layer.  ``Y[r] = act(X[r] @ W[e] + b[e])`` for the rows ``r`` in ``[offsets[e], offsets[e + 1])``; forward and
backward (``dX``, ``dW``, ``db``) over groups of any size, none included.  ``offsets`` stays on the device: the
group sizes are never read by the host, so a step has no synchronisation and can be captured in a CUDA graph.

It has no counterpart in the reference, whose transformer block has one MLP (examples/wikitext-2/gpt.py:30-37);
constructor, weight layout ``[in_features, out_features]`` per expert, activation strings, autocast and dtype
rules are those of ``Linear`` (attorch/linear_layer.py:164-205).  The device work runs in the library's
kernels (``ab200_grouped_linear_*``, ``ab200_grouped_act_backward``); there is no CPU path.
"""

import math
from typing import Optional, Tuple

import torch
from torch import Tensor, nn

from . import _lib
from . import linear_layer as _layer
from ._launch import on, recorded, status_of, stream_of
from .acts import act_id, parse_act_func
from .linear_layer import _cached_size, _dtype_id, _flags_for, _ptr, _require_cuda, get_output_dtype

MAX_GROUPS = 512


def _pitch(tensor: Tensor) -> int:
    """Row pitch in elements (the stride of a single row may mean nothing)."""
    rows, cols = tensor.shape
    return tensor.stride(0) if rows > 1 or tensor.stride(0) >= cols else cols


def _rows_operand(tensor: Tensor, dtype: torch.dtype, stream: int) -> Tensor:
    """
    A 2-D operand of ``dtype`` that TMA can address (unit inner stride, base and row pitch on 16-byte boundaries): the
    tensor itself, or a converted copy, whose rows are padded where their length is no multiple of 16 bytes.  Such a copy
    costs one pass over the operand; on the CUDA-core kernel a step of 3000 rows through 8 experts of 1001 x 1003 took 963 us
    instead of 244.
    """
    rows, cols = tensor.shape
    unit = 16 // dtype.itemsize
    if tensor.dtype is dtype and (cols <= 1 or tensor.stride(1) == 1):
        pitch = _pitch(tensor)
        if pitch >= cols and pitch % unit == 0 and tensor.data_ptr() % 16 == 0:
            return tensor
    if cols % unit:
        out = torch.empty((rows, -(-cols // unit) * unit), dtype=dtype, device=tensor.device)[:, :cols]
        return out.copy_(tensor)
    out = torch.empty((rows, cols), dtype=dtype, device=tensor.device)
    if out.numel():
        _lib.check(_lib.load().ab200_cast_2d(tensor.data_ptr(), out.data_ptr(), rows, cols, tensor.stride(0), tensor.stride(1),
                                             _dtype_id(tensor.dtype), _dtype_id(dtype), stream), 'ab200_cast_2d')
    return out


def _stack_operand(weight: Tensor, dtype: torch.dtype, stream: int) -> Tensor:
    """The same for a stack of matrices, which also lie a whole number of rows apart."""
    groups, rows, cols = weight.shape
    unit = 16 // dtype.itemsize
    if weight.dtype is dtype and (cols <= 1 or weight.stride(2) == 1) and weight.stride(1) >= max(cols, 1) and \
            weight.stride(1) % unit == 0 and weight.data_ptr() % 16 == 0 and \
            (groups == 1 or (weight.stride(0) >= rows * weight.stride(1) and weight.stride(0) % weight.stride(1) == 0)):
        return weight
    if cols % unit or not weight.is_contiguous():
        out = torch.empty((groups, rows, -(-cols // unit) * unit), dtype=dtype, device=weight.device)[..., :cols]
        return out.copy_(weight)
    return _rows_operand(weight.view(groups * rows, cols), dtype, stream).view(groups, rows, cols)


def _check_offsets(offsets: Tensor, groups: int, input: Tensor) -> Tensor:
    assert offsets.ndim == 1 and offsets.shape[0] == groups + 1, \
        f'Offsets must have one entry per group and one more ({groups + 1}), received shape {offsets.shape}'
    assert not offsets.is_floating_point(), f'Offsets must be integers, received {offsets.dtype}'
    _require_cuda(offsets, 'offsets')
    assert offsets.device == input.device, f'Offsets are on {offsets.device}, the input on {input.device}'
    return offsets if offsets.dtype is torch.int32 and offsets.is_contiguous() else offsets.int().contiguous()


def _check_operands(input: Tensor, weight: Tensor, bias: Optional[Tensor]) -> None:
    assert weight.ndim == 3, f'Weights must be 3D, received shape {weight.shape}'
    assert input.ndim == 2, f'Inputs must be 2D (expert-sorted rows), received shape {input.shape}'
    assert input.shape[1] == weight.shape[1], \
        f'Incompatible input ({input.shape}) and weights ({weight.shape}) shape'
    assert 1 <= weight.shape[0] <= MAX_GROUPS, f'1 to {MAX_GROUPS} groups are supported, received {weight.shape[0]}'
    assert bias is None or bias.shape == (weight.shape[0], weight.shape[2]), \
        f'Incompatible weights ({weight.shape}) and bias shape'
    for name, tensor in (('input', input), ('weight', weight), ('bias', bias)):
        if tensor is not None:
            _require_cuda(tensor, name)
            assert tensor.device == input.device, f'{name} is on {tensor.device}, the input on {input.device}'


def _kept_for_backward(name: Optional[str], param: Optional[float], dtype: torch.dtype, shape: Tuple[int, int],
                       device: torch.device, needs_grad: bool):
    """
    What a forward call keeps of its activation, as ``set_save_derivative`` says: (the tensor or None, flags of the call, the
    activation id and parameter that backward multiplies dY with).  act'(Z) in a bf16 layer is held as fp16, as
    ``Linear`` holds it: the same size and three more bits; Z has the layer's type.
    """
    if name is None or not needs_grad:
        return None, 0, (_lib.ACT_NONE, 0.0)
    if not _layer._save_derivative:
        return torch.empty(shape, dtype=dtype, device=device), 0, (act_id(name), 0.0 if param is None else param)
    fp16 = dtype is torch.bfloat16
    return (torch.empty(shape, dtype=torch.float16 if fp16 else dtype, device=device),
            _lib.FLAG_SAVE_DERIVATIVE | (_lib.FLAG_DERIVATIVE_FP16 if fp16 else 0),
            (_lib.ACT_SAVED_DERIVATIVE_F16 if fp16 else _lib.ACT_SAVED_DERIVATIVE, 0.0))


def _forward(input: Tensor, offsets: Tensor, weight: Tensor, bias: Optional[Tensor], act_func: Optional[str],
             needs_grad: bool):
    """
    (output, saved, backward_act) where saved is what backward needs: operands, offsets, and act'(Z) or Z; backward_act is the
    activation id and parameter that turn the last of them into the factor of dY.
    """
    _check_operands(input, weight, bias)
    name, param = parse_act_func(act_func)
    groups, in_dim, out_dim = weight.shape
    offsets = _check_offsets(offsets, groups, input)
    rows = input.shape[0]
    out_dtype = get_output_dtype(input.dtype)
    lib = _lib.load()
    with on(input.device):
        stream = stream_of(input.device)
        status = status_of(input.device)
        x_op = _rows_operand(input, out_dtype, stream)
        w_op = _stack_operand(weight, out_dtype, stream)
        bias_op = bias if bias is None or bias.is_contiguous() else bias.contiguous()
        output = torch.empty((rows, out_dim), dtype=out_dtype, device=input.device)
        kept, keep_flags, backward_act = _kept_for_backward(name, param, out_dtype, (rows, out_dim), input.device, needs_grad)
        _lib.check(lib.ab200_grouped_linear_forward(
            _ptr(x_op), _ptr(w_op), _ptr(bias_op), _ptr(offsets), _ptr(kept), _ptr(output), rows, groups, in_dim, out_dim,
            _pitch(x_op), w_op.stride(0), w_op.stride(1), out_dim, out_dim, _dtype_id(out_dtype),
            _dtype_id(bias_op.dtype) if bias_op is not None else 0, act_id(name), 0.0 if param is None else param, status,
            stream, _flags_for(input.device) | keep_flags), 'ab200_grouped_linear_forward')
    return output, (x_op, w_op, offsets, kept), backward_act


class GroupedLinearAutoGrad(torch.autograd.Function):
    """``apply(input, offsets, weight, bias, act_func)``: the function behind ``GroupedLinear``."""
    @staticmethod
    def forward(ctx, input: Tensor, offsets: Tensor, weight: Tensor, bias: Optional[Tensor] = None,
                act_func: Optional[str] = None) -> Tensor:
        ctx.needs = (input.requires_grad, weight.requires_grad, bias is not None and bias.requires_grad)
        output, saved, ctx.backward_act = _forward(input, offsets, weight, bias, act_func, any(ctx.needs))
        ctx.dtypes = (input.dtype, weight.dtype, None if bias is None else bias.dtype)
        if any(ctx.needs):
            ctx.save_for_backward(*saved)
        return output

    @staticmethod
    def backward(ctx, output_grad: Tensor) -> Tuple[Optional[Tensor], ...]:
        x_op, w_op, offsets, kept = ctx.saved_tensors
        groups, in_dim, out_dim = w_op.shape
        rows, device, dtype = x_op.shape[0], x_op.device, x_op.dtype
        dt = _dtype_id(dtype)
        lib = _lib.load()
        input_grad = weight_grad = bias_grad = None
        with on(device):
            stream = stream_of(device)
            status = status_of(device)
            flags = _flags_for(device)
            dy = _rows_operand(output_grad, dtype, stream)
            dz = dy
            if kept is not None or ctx.needs[2]:
                if kept is not None:
                    # In the operands' type, which the tensor cores multiply: with it dX and dW are off by sqrt(2) of their own
                    # rounding (bf16 training steps: 2.4e-3 of their size instead of 1.7e-3).  db is summed before it.
                    unit = 16 // dtype.itemsize
                    dz = torch.empty((rows, -(-out_dim // unit) * unit), dtype=dtype, device=device)[:, :out_dim]
                ws_bytes = 0
                workspace = None
                if ctx.needs[2]:
                    bias_grad = torch.empty((groups, out_dim), dtype=ctx.dtypes[2], device=device)
                    ws_bytes = _cached_size('ab200_grouped_act_backward_workspace_bytes', rows, groups, out_dim)
                    workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
                _lib.check(lib.ab200_grouped_act_backward(
                    _ptr(dy), _ptr(kept), _ptr(dz) if kept is not None else None, _ptr(bias_grad), _ptr(offsets), rows, groups,
                    out_dim, _pitch(dy), out_dim, _pitch(dz), dt, _dtype_id(bias_grad.dtype) if bias_grad is not None else 0,
                    *ctx.backward_act, _ptr(workspace), ws_bytes, stream), 'ab200_grouped_act_backward')
            if ctx.needs[1]:
                weight_grad = torch.empty((groups, in_dim, out_dim), dtype=ctx.dtypes[1], device=device)
                _lib.check(lib.ab200_grouped_linear_backward_weight(
                    _ptr(x_op), _ptr(dz), _ptr(offsets), _ptr(weight_grad), rows, groups, in_dim, out_dim, _pitch(x_op), _pitch(dz),
                    dt, _dtype_id(weight_grad.dtype), status, stream, flags), 'ab200_grouped_linear_backward_weight')
            if ctx.needs[0]:
                input_grad = torch.empty((rows, in_dim), dtype=ctx.dtypes[0], device=device)
                _lib.check(lib.ab200_grouped_linear_backward_input(
                    _ptr(dz), _ptr(w_op), _ptr(offsets), _ptr(input_grad), rows, groups, in_dim, out_dim, _pitch(dz),
                    w_op.stride(0), w_op.stride(1), in_dim, dt, _dtype_id(input_grad.dtype), status, stream, flags),
                    'ab200_grouped_linear_backward_input')
        return input_grad, None, weight_grad, bias_grad, None


def grouped_linear(input: Tensor, offsets: Tensor, weight: Tensor, bias: Optional[Tensor] = None,
                   act_func: Optional[str] = None) -> Tensor:
    """
    ``act(input[r] @ weight[e] + bias[e])`` for the rows ``r`` in ``[offsets[e], offsets[e + 1])``; zeros in the rows
    from ``offsets[-1]`` on.

    Args:
        input: Expert-sorted rows ``[rows, in_features]``.
        offsets: First row of every group and the end of the last, ``[groups + 1]`` integers on the device,
            ascending from 0.
        weight: ``[groups, in_features, out_features]``.
        bias: ``[groups, out_features]`` or None.
        act_func: Activation, as ``Linear``.
    """
    if recorded(input, weight, bias):
        return GroupedLinearAutoGrad.apply(input, offsets, weight, bias, act_func)
    return _forward(input, offsets, weight, bias, act_func, False)[0]


class GroupedLinear(nn.Module):
    """
    A ``Linear`` per group of rows.

    Args:
        num_groups: Number of groups (experts), at most 512.
        in_features: Number of input features.
        out_features: Number of output features.
        bias: Flag for additive bias.
        act_func: Name of the activation to fuse, as ``Linear``.
        device: Device to use.
        dtype: Dtype of layer.
    """
    def __init__(self, num_groups: int, in_features: int, out_features: int, bias: bool = True,
                 act_func: Optional[str] = None, device='cuda', dtype: torch.dtype = torch.float32) -> None:
        super().__init__()
        if not 1 <= num_groups <= MAX_GROUPS:
            raise RuntimeError(f'1 to {MAX_GROUPS} groups are supported, received {num_groups}.')
        parse_act_func(act_func)
        self.num_groups, self.in_features, self.out_features, self.act_func = num_groups, in_features, out_features, act_func
        self.weight = nn.Parameter(torch.empty(num_groups, in_features, out_features, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.empty(num_groups, out_features, device=device, dtype=dtype)) if bias else None
        self.reset_parameters()

    def reset_parameters(self) -> None:
        """Every expert as ``Linear`` initialises itself: uniform within 1 / sqrt(in_features)."""
        bound = 1.0 / math.sqrt(self.in_features) if self.in_features > 0 else 0.0
        nn.init.uniform_(self.weight, -bound, bound)
        if self.bias is not None:
            nn.init.uniform_(self.bias, -bound, bound)

    def forward(self, input: Tensor, offsets: Tensor) -> Tensor:
        return grouped_linear(input, offsets, self.weight, self.bias, self.act_func)

    def extra_repr(self) -> str:
        return (f'num_groups={self.num_groups}, in_features={self.in_features}, out_features={self.out_features}, '
                f'bias={self.bias is not None}, act_func={self.act_func!r}')

"""
The linear layer with 8-bit operands: ``Y = act(X @ W + b)`` where ``X`` is held as e4m3 with one scale per row
and 128 features and ``W`` as e4m3 with one scale per block of 128 x 128; products are summed in fp32.

    Float8Linear         a ``Linear`` that multiplies in 8 bits (training, and serving from its parameters)
    Float8GroupedLinear  stored 8-bit weights of a ``GroupedLinear`` (serving)
    float8_linear, float8_grouped_linear
                         the products on weights that are already held as e4m3 and scales (a checkpoint's)
    quantize_weight      e4m3 values and scales of a weight

Scales that this module makes are powers of two (the smallest that keeps a block within e4m3's 448), so that
dividing by them is exact; the products take any fp32 scales.  No counterpart in the reference.  The device work runs in
the library's kernels (``ab200_float8_*``); there is no CPU path.
"""

from typing import Optional, Tuple

import torch
from torch import Tensor, nn

from . import _lib
from ._launch import has_tangent, on, status_of, stream_of
from .acts import act_id, parse_act_func
from .grouped_linear_layer import MAX_GROUPS, GroupedLinear, _check_offsets, _kept_for_backward, _pitch, _rows_operand
from .linear_layer import Linear, _cached_size, _dtype_id, _flags_for, _ptr, _require_cuda, get_output_dtype

BLOCK = 128


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _padded(n: int) -> int:
    """Row pitch of e4m3 values: whole 16-byte units."""
    return -(-n // 16) * 16


def _empty_float8(*shape: int, device) -> Tensor:
    """e4m3 tensor whose rows start on 16-byte boundaries."""
    held = torch.empty((*shape[:-1], _padded(shape[-1])), dtype=torch.float8_e4m3fn, device=device)
    return held if held.shape[-1] == shape[-1] else held[..., :shape[-1]]


def _quantize_rows(x: Tensor, stream: int) -> Tuple[Tensor, Tensor]:
    """e4m3 values of ``x`` [rows, cols] and their scales [blocks of 128 columns, rows]."""
    rows, cols = x.shape
    if (cols > 1 and x.stride(1) != 1) or (rows > 1 and x.stride(0) < cols):
        x = x.contiguous()
    q = _empty_float8(rows, cols, device=x.device)
    scale = torch.empty((_blocks(cols), rows), dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().ab200_float8_quantize_rows(_ptr(x), _ptr(q), _ptr(scale), rows, cols, _pitch(x), _padded(cols), rows,
                                                      _dtype_id(x.dtype), stream), 'ab200_float8_quantize_rows')
    return q, scale


def _quantize_weight(weight: Tensor, stored: bool, transposed: bool, stream: int):
    """(as stored [.., in, out], transposed [.., out, in], scales [.., out blocks, in blocks]); absent ones None."""
    stack = weight if weight.ndim == 3 else weight.unsqueeze(0)
    groups, rows, cols = stack.shape
    if (cols > 1 and stack.stride(2) != 1) or (rows > 1 and stack.stride(1) < cols):
        stack = stack.contiguous()
    device = weight.device
    lead = weight.shape[:-2]
    q = _empty_float8(*lead, rows, cols, device=device) if stored else None
    q_t = _empty_float8(*lead, cols, rows, device=device) if transposed else None
    scale = torch.empty((*lead, _blocks(cols), _blocks(rows)), dtype=torch.float32, device=device)
    _lib.check(_lib.load().ab200_float8_quantize_weight(
        _ptr(stack), _ptr(q), _ptr(q_t), _ptr(scale), groups, rows, cols, stack.stride(0) if groups > 1 else 0,
        stack.stride(1) if rows > 1 else cols, _padded(cols), _padded(rows), _dtype_id(weight.dtype), stream),
        'ab200_float8_quantize_weight')
    return q, q_t, scale


def quantize_weight(weight: Tensor) -> Tuple[Tensor, Tensor]:
    """
    e4m3 values ``[..., out_features, in_features]`` and fp32 scales ``[..., out blocks, in blocks]`` of a weight in
    ``Linear``'s (or ``GroupedLinear``'s) layout ``[..., in_features, out_features]``, as ``float8_linear`` and
    ``float8_grouped_linear`` take them.
    """
    assert weight.ndim in (2, 3), f'Weights must be 2D or 3D, received shape {weight.shape}'
    _require_cuda(weight, 'weight')
    with torch.no_grad(), on(weight.device):
        _, q_t, scale = _quantize_weight(weight.detach(), False, True, stream_of(weight.device))
    return q_t, scale


def _addressable(weight: Tensor) -> Tensor:
    """The e4m3 weight itself if its rows start on 16-byte boundaries at even distances, else an aligned copy."""
    rows, cols = weight.shape[-2:]
    pitch = weight.stride(-2) if rows > 1 else _padded(cols)
    ok = (cols <= 1 or weight.stride(-1) == 1) and pitch % 16 == 0 and pitch >= cols and weight.data_ptr() % 16 == 0
    if weight.ndim == 3 and weight.shape[0] > 1:
        ok = ok and weight.stride(0) >= rows * pitch and weight.stride(0) % pitch == 0
    if ok:
        return weight
    held = _empty_float8(*weight.shape, device=weight.device)
    held.view(torch.uint8).copy_(weight.view(torch.uint8))
    return held


def _product(xq: Tensor, x_scale: Tensor, wq: Tensor, w_scale: Tensor, scale_strides: Tuple[int, int, int], bias: Optional[Tensor],
             offsets: Optional[Tensor], pre_act: Optional[Tensor], out: Tensor, act: int, param: float, stream: int, extra_flags: int = 0) -> None:
    """out = act(xq wq^T scaled + bias); wq: [n, k] or [groups, n, k]; scale_strides: (group, n block, k block)."""
    rows, k = xq.shape
    n = wq.shape[-2]
    device = xq.device
    pitch = wq.stride(-2) if n > 1 else _padded(k)
    grouped = wq.ndim == 3
    _lib.check(_lib.load().ab200_float8_product(
        _ptr(xq), _ptr(x_scale), _ptr(wq), _ptr(w_scale), _ptr(bias), _ptr(offsets), _ptr(pre_act), _ptr(out), rows,
        wq.shape[0] if grouped else 1, k, n, _padded(k), x_scale.shape[1], wq.stride(0) if grouped and wq.shape[0] > 1 else n * pitch,
        pitch, *scale_strides, n, n, _dtype_id(out.dtype), _dtype_id(bias.dtype) if bias is not None else 0, act, param,
        status_of(device), stream, _flags_for(device) | extra_flags), 'ab200_float8_product')


def _check_stored(input: Tensor, weight: Tensor, scale: Tensor, bias: Optional[Tensor], ndim: int) -> None:
    assert weight.ndim == ndim and weight.dtype is torch.float8_e4m3fn, \
        f'Stored weights must be {ndim}D float8_e4m3fn, received {weight.dtype} of shape {weight.shape}'
    assert input.shape[-1] == weight.shape[-1], f'Incompatible input ({input.shape}) and weights ({weight.shape}) shape'
    assert weight.shape[-1] > 0, 'Stored weights must have input features'
    expected = (*weight.shape[:-2], _blocks(weight.shape[-2]), _blocks(weight.shape[-1]))
    assert scale.dtype is torch.float32 and scale.shape == expected, \
        f'Scales must be float32 of shape {expected}, received {scale.dtype} of shape {tuple(scale.shape)}'
    assert bias is None or bias.shape == (*weight.shape[:-2], weight.shape[-2]), f'Incompatible weights ({weight.shape}) and bias shape'
    for name, tensor in (('input', input), ('weight', weight), ('scale', scale), ('bias', bias)):
        if tensor is not None:
            _require_cuda(tensor, name)
            assert tensor.device == input.device, f'{name} is on {tensor.device}, the input on {input.device}'
    if torch.is_grad_enabled() and (input.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError('Products with stored 8-bit weights have no gradient: train with Float8Linear, or call them under '
                           'torch.no_grad().')
    if has_tangent(input, scale, bias):
        raise NotImplementedError('Products with stored 8-bit weights have no forward-mode derivative.')


def _stored(input: Tensor, offsets: Optional[Tensor], weight: Tensor, scale: Tensor, bias: Optional[Tensor],
            act_func: Optional[str]) -> Tensor:
    name, param = parse_act_func(act_func)
    n = weight.shape[-2]
    flat = input.flatten(0, -2)
    out_dtype = get_output_dtype(input.dtype)
    _dtype_id(input.dtype)
    with on(input.device):
        stream = stream_of(input.device)
        output = torch.empty((flat.shape[0], n), dtype=out_dtype, device=input.device)
        if output.numel():
            xq, x_scale = _quantize_rows(flat, stream)
            if not scale.is_contiguous():
                scale = scale.contiguous()
            if bias is not None and not bias.is_contiguous():
                bias = bias.contiguous()
            blocks_n, blocks_k = scale.shape[-2:]
            _product(xq, x_scale, _addressable(weight), scale, (blocks_n * blocks_k, blocks_k, 1), bias, offsets, None, output,
                     act_id(name), 0.0 if param is None else param, stream)
    return output.view(*input.shape[:-1], n)


def float8_linear(input: Tensor, weight: Tensor, scale: Tensor, bias: Optional[Tensor] = None,
                  act_func: Optional[str] = None) -> Tensor:
    """
    ``act(input @ W^T + bias)`` with a stored 8-bit weight: ``W[n, k] = weight[n, k] * scale[n // 128, k // 128]``.
    The input is quantised in the call.  Forward only.

    Args:
        input: ``[..., in_features]`` fp32, fp16 or bf16; the output has its dtype (or autocast's).
        weight: ``[out_features, in_features]`` float8_e4m3fn.  Rows that do not start on 16-byte boundaries
            (in_features no multiple of 16 in a contiguous tensor) are copied to ones that do, in every call.
        scale: ``[ceil(out_features / 128), ceil(in_features / 128)]`` float32.
        bias: ``[out_features]`` or None.
        act_func: Activation, as ``Linear``.
    """
    _check_stored(input, weight, scale, bias, 2)
    return _stored(input, None, weight, scale, bias, act_func)


def float8_grouped_linear(input: Tensor, offsets: Tensor, weight: Tensor, scale: Tensor, bias: Optional[Tensor] = None,
                          act_func: Optional[str] = None) -> Tensor:
    """
    ``grouped_linear`` with stored 8-bit weights ``[groups, out_features, in_features]`` and scales ``[groups,
    ceil(out_features / 128), ceil(in_features / 128)]``; ``bias`` ``[groups, out_features]``.  Forward only.
    """
    assert input.ndim == 2, f'Inputs must be 2D (expert-sorted rows), received shape {input.shape}'
    _check_stored(input, weight, scale, bias, 3)
    assert 1 <= weight.shape[0] <= MAX_GROUPS, f'1 to {MAX_GROUPS} groups are supported, received {weight.shape[0]}'
    return _stored(input, _check_offsets(offsets, weight.shape[0], input), weight, scale, bias, act_func)


class Float8LinearAutoGrad(torch.autograd.Function):
    """
    ``apply(input, weight, bias, act_func)`` with ``weight`` ``[in_features, out_features]``: both operands are quantised in
    the call.  Backward quantises ``dZ`` per row and 128 output features and multiplies it with the same 8-bit
    weight for ``dX``; ``dW`` and ``db`` come from the unquantised ``X`` and ``dZ`` (their reduction runs over rows,
    where neither has scales).
    """
    @staticmethod
    def forward(ctx, input: Tensor, weight: Tensor, bias: Optional[Tensor] = None, act_func: Optional[str] = None) -> Tensor:
        assert weight.ndim == 2, f'Weights must be 2D, received shape {weight.shape}'
        assert input.shape[-1] == weight.shape[0] and weight.shape[0] > 0, \
            f'Incompatible input ({input.shape}) and weights ({weight.shape}) shape'
        assert bias is None or bias.shape == (weight.shape[1],), f'Incompatible weights ({weight.shape}) and bias shape'
        for what, tensor in (('input', input), ('weight', weight), ('bias', bias)):
            if tensor is not None:
                _require_cuda(tensor, what)
                assert tensor.device == input.device, f'{what} is on {tensor.device}, the input on {input.device}'
        name, param = parse_act_func(act_func)
        ctx.needs = (input.requires_grad, weight.requires_grad, bias is not None and bias.requires_grad)
        flat = input.flatten(0, -2)
        rows, in_dim = flat.shape
        out_dim = weight.shape[1]
        out_dtype = get_output_dtype(input.dtype)
        with on(input.device):
            stream = stream_of(input.device)
            x_op = _rows_operand(flat, out_dtype, stream) if ctx.needs[1] else None
            output = torch.empty((rows, out_dim), dtype=out_dtype, device=input.device)
            wq = scale = kept = None
            ctx.backward_act = (_lib.ACT_NONE, 0.0)
            if output.numel():
                # From the values as they came, like a stored weight's product: rounded to 16 bits first (under autocast), some
                # would be held as a neighbour, and the frozen layer would differ from the one that was trained.
                xq, x_scale = _quantize_rows(x_op if x_op is not None and flat.dtype is out_dtype else flat, stream)
                wq, wq_t, scale = _quantize_weight(weight, ctx.needs[0], True, stream)
                kept, flags, ctx.backward_act = _kept_for_backward(name, param, out_dtype, (rows, out_dim), input.device, any(ctx.needs))
                bias_op = bias if bias is None or bias.is_contiguous() else bias.contiguous()
                _product(xq, x_scale, wq_t, scale, (0, scale.shape[1], 1), bias_op, None, kept, output, act_id(name),
                         0.0 if param is None else param, stream, flags)
        ctx.shapes = (input.shape, rows, in_dim, out_dim)
        ctx.dtypes = (input.dtype, weight.dtype, None if bias is None else bias.dtype)
        if any(ctx.needs):
            ctx.save_for_backward(x_op, wq, scale, kept)
        return output.view(*input.shape[:-1], out_dim)

    @staticmethod
    def backward(ctx, output_grad: Tensor) -> Tuple[Optional[Tensor], ...]:
        x_op, wq, scale, kept = ctx.saved_tensors
        shape, rows, in_dim, out_dim = ctx.shapes
        device, dtype = output_grad.device, output_grad.dtype
        lib = _lib.load()
        input_grad = weight_grad = bias_grad = None
        with on(device):
            stream = stream_of(device)
            status = status_of(device)
            dt = _dtype_id(dtype)
            dy = _rows_operand(output_grad.reshape(rows, out_dim), dtype, stream)
            dz = dy
            if ctx.needs[2]:
                bias_grad = torch.empty(out_dim, dtype=ctx.dtypes[2], device=device)
            if (kept is not None or ctx.needs[2]) and out_dim:
                if kept is not None:
                    unit = 16 // dtype.itemsize
                    dz = torch.empty((rows, -(-out_dim // unit) * unit), dtype=dtype, device=device)[:, :out_dim]
                ws_bytes = _cached_size('ab200_act_backward_workspace_bytes', rows, out_dim) if ctx.needs[2] else 0
                workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
                _lib.check(lib.ab200_act_backward(
                    _ptr(dy), _ptr(kept), _ptr(dz) if kept is not None else None, _ptr(bias_grad), rows, out_dim, _pitch(dy),
                    out_dim, _pitch(dz), dt, _dtype_id(bias_grad.dtype) if bias_grad is not None else 0, *ctx.backward_act,
                    _ptr(workspace), ws_bytes, stream), 'ab200_act_backward')
            if ctx.needs[1]:
                weight_grad = torch.empty((in_dim, out_dim), dtype=ctx.dtypes[1], device=device)
                ws_bytes = _cached_size('ab200_gemm_workspace_bytes', in_dim, out_dim, rows)
                workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
                _lib.check(lib.ab200_linear_backward_weight(
                    _ptr(x_op), _ptr(dz), _ptr(weight_grad), rows, in_dim, out_dim, _pitch(x_op), 1, _pitch(dz), 1, out_dim, dt,
                    _dtype_id(weight_grad.dtype), _ptr(workspace), ws_bytes, status, stream, _flags_for(device)),
                    'ab200_linear_backward_weight')
            if ctx.needs[0]:
                input_grad = torch.empty((rows, in_dim), dtype=ctx.dtypes[0], device=device)
                if input_grad.numel() and out_dim:
                    dzq, dz_scale = _quantize_rows(dz, stream)
                    # Output columns are input features, the reduction runs over output features: scale strides swap.
                    _product(dzq, dz_scale, wq, scale, (0, 1, scale.shape[1]), None, None, None, input_grad, _lib.ACT_NONE, 0.0, stream)
                else:
                    input_grad.zero_()
                input_grad = input_grad.view(shape)
        return input_grad, weight_grad, bias_grad, None


class Float8Linear(Linear):
    """
    ``Linear`` whose products run on 8-bit operands; same constructor, parameters and state_dict.  Weights are
    quantised from the parameters in every training forward.  ``freeze()`` lays them out once for serving: from then
    on the layer holds 8-bit weights instead of parameters and has no gradient.

    Args:
        in_features: Number of input features.
        out_features: Number of output features.
        bias: Flag for additive bias.
        act_func: Name of the activation to fuse, as ``Linear``.
        device: Device to use.
        dtype: Dtype of the parameters.
    """
    writes_into_buckets = False         # see dp.GradientBuckets

    def __init__(self, in_features: int, out_features: int, bias: bool = True, act_func: Optional[str] = None,
                 device='cuda', dtype: torch.dtype = torch.float32) -> None:
        super().__init__(in_features, out_features, bias, act_func, device, dtype)
        self.register_buffer('weight_float8', None)
        self.register_buffer('weight_scale', None)

    @classmethod
    def from_linear(cls, linear: Linear) -> 'Float8Linear':
        """The layer with the parameters of ``linear`` (shared, not copied)."""
        layer = cls(linear.in_features, linear.out_features, linear.bias is not None, linear.act_func, 'meta', linear.weight.dtype)
        layer.weight, layer.bias = linear.weight, linear.bias
        return layer

    def freeze(self) -> 'Float8Linear':
        """
        Replaces the weight by its 8-bit form (half of bf16's memory) and the bias by a constant copy; returns the layer.  A
        layer that shares the parameters keeps them as they are.
        """
        if self.weight is None:
            return self
        self.weight_float8, self.weight_scale = quantize_weight(self.weight)
        self.weight = None
        if self.bias is not None:
            # A snapshot like the weight's: the parameter may be another layer's too (from_linear), which goes on training it.
            self.bias = nn.Parameter(self.bias.detach().clone(), requires_grad=False)
        return self

    def forward(self, input: Tensor, residual: Optional[Tensor] = None) -> Tensor:
        if self.weight_grad_out is not None or self.grad_ready is not None or self.defer_input_grad is not None:
            raise RuntimeError('Float8Linear does not write its gradients into a data-parallel bucket; use Linear, or reduce '
                               '.grad after backward.')
        if self.weight is None:
            output = float8_linear(input, self.weight_float8, self.weight_scale, self.bias, self.act_func)
        else:
            output = Float8LinearAutoGrad.apply(input, self.weight, self.bias, self.act_func)
        return output if residual is None else output + residual


class Float8GroupedLinear(nn.Module):
    """
    Stored 8-bit weights of a ``GroupedLinear``, for serving.

    Args:
        weight: ``[groups, out_features, in_features]`` float8_e4m3fn.
        scale: ``[groups, ceil(out_features / 128), ceil(in_features / 128)]`` float32.
        bias: ``[groups, out_features]`` or None.
        act_func: Activation, as ``Linear``.
    """
    def __init__(self, weight: Tensor, scale: Tensor, bias: Optional[Tensor] = None, act_func: Optional[str] = None) -> None:
        super().__init__()
        parse_act_func(act_func)
        self.act_func = act_func
        self.register_buffer('weight', _addressable(weight))
        self.register_buffer('scale', scale)
        self.register_buffer('bias', None if bias is None else bias.detach())

    @classmethod
    def from_grouped(cls, grouped: GroupedLinear) -> 'Float8GroupedLinear':
        """The 8-bit form of a ``GroupedLinear``."""
        weight, scale = quantize_weight(grouped.weight)
        return cls(weight, scale, None if grouped.bias is None else grouped.bias.detach().clone(), grouped.act_func)

    def forward(self, input: Tensor, offsets: Tensor) -> Tensor:
        return float8_grouped_linear(input, offsets, self.weight, self.scale, self.bias, self.act_func)

    def extra_repr(self) -> str:
        groups, out_dim, in_dim = self.weight.shape
        return (f'num_groups={groups}, in_features={in_dim}, out_features={out_dim}, bias={self.bias is not None}, '
                f'act_func={self.act_func!r}')

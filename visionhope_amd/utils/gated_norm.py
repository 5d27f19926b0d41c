"""LayerNorm of token rows with an optional SiLU gate (native, ``csrc/row_norm.hip``).

    y = ((x - mean) / sqrt(var + eps) * weight + bias) * silu(gate)

over the last dimension (biased variance).  Statistics and sums are FP32; y and the
gradients of x and gate are rounded once to x's dtype, those of weight and bias are summed in
FP32 in a fixed order.  ``utils/layer_norm_cuda.py`` is the LayerNorm of ``[B, C, H, W]`` maps.
"""

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import hip
from .cuda import on_tensor_device
from .token_lines import (IO_DTYPES, address, check_like, check_param, differentiated, fp32_param, note_stream,
                          refuse_held_leaves)

MAX_CHANNELS = 8192


def _rows(t):
    """``t`` as rows a fixed number of elements apart: ``(tensor, stride)``.  Leading dimensions
    that do not fold into one are copied."""
    channels = t.shape[-1]
    if t.is_contiguous():
        return t, channels
    if t.ndim == 1:
        t = t[None]
    if t.stride(-1) != 1 and channels > 1:
        t = t.contiguous()
    # the stride of the innermost leading dimension of more than one row, which the others must
    # continue
    stride, expected = None, None
    for size, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if stride is None:
            stride, expected = step, step * size
        elif step != expected:
            return t.contiguous(), channels
        else:
            expected = step * size
    return t, channels if stride is None else stride


def _forward(x, weight, bias, gate, eps, keep):
    channels = x.shape[-1]
    rows = x.numel() // channels
    x, x_row = _rows(x)
    gate_row = 0
    if gate is not None:
        gate, gate_row = _rows(gate)
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    stats, mean, rstd = None, None, None   # mean of every row, then rstd of every row
    if keep:
        stats = torch.empty((2, rows), device=x.device, dtype=torch.float32)
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    hip.check(hip.load_library().vh_gated_layernorm_forward(
        address(x), x_row, address(gate), gate_row, hip.dtype_code(x.dtype), address(weight), address(bias),
        address(y), mean, rstd, rows, channels, float(eps), hip.stream_of(x)),
        "vh_gated_layernorm_forward")
    return y, stats


class _GatedLayerNormFunction(Function):
    @staticmethod
    @on_tensor_device
    def forward(ctx, x, weight, bias, gate, eps):
        weight32, bias32 = fp32_param(weight), fp32_param(bias)
        y, stats = _forward(x, weight32, bias32, gate, eps, True)
        note_stream(ctx, hip.stream_of(x))
        ctx.save_for_backward(x, weight32, bias32, gate, stats)
        ctx.param_dtypes = (weight.dtype, bias.dtype)
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return _GatedLayerNormFunction._gradients(*ctx.saved_tensors, ctx, dy)

    @staticmethod
    @on_tensor_device
    def _gradients(x, weight, bias, gate, stats, ctx, dy):
        refuse_held_leaves("visionhope_gated_layernorm", ctx, torch.cuda.is_current_stream_capturing())
        shape, channels = x.shape, x.shape[-1]
        rows = x.numel() // channels
        # saved-tensor hooks may return other strides than were saved
        weight, bias, stats = weight.contiguous(), bias.contiguous(), stats.contiguous()
        need = ctx.needs_input_grad
        x, x_row = _rows(x)
        dy, dy_row = _rows(dy.to(x.dtype))
        gate_row, dgate = 0, None
        if gate is not None:
            gate, gate_row = _rows(gate)
            dgate = torch.empty(shape, device=x.device, dtype=x.dtype)
        dx = torch.empty(shape, device=x.device, dtype=x.dtype)
        dweight = torch.empty(channels, device=x.device, dtype=torch.float32) if need[1] else None
        dbias = torch.empty(channels, device=x.device, dtype=torch.float32) if need[2] else None
        lib = hip.load_library()
        ws = hip.workspace(lib.vh_gated_layernorm_backward_workspace_bytes(rows, channels), x.device)
        hip.check(lib.vh_gated_layernorm_backward(
            address(dy), dy_row, address(x), x_row, address(gate), gate_row, hip.dtype_code(x.dtype), address(weight),
            address(bias), stats.data_ptr(), stats.data_ptr() + 4 * rows, address(dx), address(dgate), address(dweight), address(dbias),
            rows, channels, address(ws), ws.numel() * 4, hip.stream_of(x)), "vh_gated_layernorm_backward")
        return (dx, dweight.to(ctx.param_dtypes[0]) if need[1] else None,
                dbias.to(ctx.param_dtypes[1]) if need[2] else None, dgate, None)


def visionhope_gated_layernorm(x, weight, bias, eps=1e-6, *, gate=None):
    """LayerNorm of ``x`` ``[..., C]`` over its last dimension (C of up to 8192), times
    ``silu(gate)`` with a gate of x's shape and dtype (module docstring).  ``weight`` and ``bias``
    ``[C]``.  ``x`` and ``gate`` may be slices of wider tensors; y is dense, in x's dtype."""
    name = "visionhope_gated_layernorm"
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{name} expects CUDA tensors")
    if x.dtype not in IO_DTYPES:
        raise TypeError(f"{name} supports FP16, BF16 and FP32 tensors, got {x.dtype}")
    if x.ndim < 1 or x.numel() == 0:
        raise ValueError(f"{name} expects nonempty rows, got shape {tuple(x.shape)}")
    channels = x.shape[-1]
    if channels > MAX_CHANNELS:
        raise ValueError(f"{name} supports at most {MAX_CHANNELS} channels, got {channels}")
    check_param(name, "weight", weight, (channels,), x.device)
    check_param(name, "bias", bias, (channels,), x.device)
    if gate is not None:
        check_like(name, "gate", gate, x.shape, x.dtype, x.device)
    if differentiated(x, weight, bias, gate):
        return _GatedLayerNormFunction.apply(x, weight, bias, gate, float(eps))
    return _no_grad_forward(x, weight, bias, gate, eps)


@on_tensor_device
def _no_grad_forward(x, weight, bias, gate, eps):
    return _forward(x, fp32_param(weight), fp32_param(bias), gate, eps, False)[0].view(x.shape)

"""Group norm of channels-last maps with an activation (native, ``csrc/group_norm.hip``).

    y = f((x - mean) / sqrt(var + eps) * weight + bias)

with the mean and the (biased) variance over the channels of a group and all pixels of an image,
and f the identity, SiLU or the exact GELU.  Statistics and sums are FP32 or wider; y and the
gradient of x are rounded once to x's dtype, the gradients of weight and bias are summed in FP32 in
a fixed order.  ``utils/layer_norm_cuda.py`` normalises each pixel.
"""

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import hip
from .cuda import on_tensor_device
from .token_lines import address, check_io, check_param, differentiated, fp32_param, note_stream, refuse_held_leaves

MAX_GROUP_CHANNELS = 1024
ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}


def _sizes(x, groups):
    batch, channels, height, width = x.shape
    return batch, height * width, channels, groups


def _forward(x, groups, weight, bias, eps, activation, keep):
    sizes, code = _sizes(x, groups), hip.dtype_code(x.dtype)
    lib = hip.load_library()
    y = torch.empty_like(x, memory_format=torch.channels_last)
    stats = torch.empty((3, sizes[0], groups), device=x.device, dtype=torch.float32) if keep else None
    nbytes = lib.vh_group_norm_workspace_bytes(*sizes, code)
    ws = hip.workspace(nbytes, x.device) if nbytes else None
    hip.check(lib.vh_group_norm_forward(
        x.data_ptr(), code, weight.data_ptr(), bias.data_ptr(), activation, y.data_ptr(), address(stats), *sizes, eps,
        address(ws), nbytes, hip.stream_of(x)), "vh_group_norm_forward")
    return y, stats


class _GroupNormFunction(Function):
    @staticmethod
    @on_tensor_device
    def forward(ctx, x, weight, bias, groups, eps, activation):
        weight32, bias32 = fp32_param(weight), fp32_param(bias)
        y, stats = _forward(x, groups, weight32, bias32, eps, activation, True)
        note_stream(ctx, hip.stream_of(x))
        ctx.save_for_backward(x, weight32, bias32, stats)
        ctx.groups, ctx.activation = groups, activation
        ctx.param_dtypes = (weight.dtype, bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return _GroupNormFunction._gradients(*ctx.saved_tensors, ctx, dy)

    @staticmethod
    @on_tensor_device
    def _gradients(x, weight, bias, stats, ctx, dy):
        refuse_held_leaves("visionhope_group_norm", ctx, torch.cuda.is_current_stream_capturing())
        # saved-tensor hooks may return other strides than were saved
        x = x.contiguous(memory_format=torch.channels_last)
        weight, bias, stats = weight.contiguous(), bias.contiguous(), stats.contiguous()
        dy = dy.to(x.dtype).contiguous(memory_format=torch.channels_last)
        sizes, code, need = _sizes(x, ctx.groups), hip.dtype_code(x.dtype), ctx.needs_input_grad
        dx = torch.empty_like(x, memory_format=torch.channels_last)
        dweight, dbias = (torch.empty(sizes[2], device=x.device, dtype=torch.float32) if want else None for want in need[1:3])
        lib = hip.load_library()
        nbytes = lib.vh_group_norm_backward_workspace_bytes(*sizes, code)
        ws = hip.workspace(nbytes, x.device)
        hip.check(lib.vh_group_norm_backward(
            dy.data_ptr(), x.data_ptr(), code, weight.data_ptr(), bias.data_ptr(), ctx.activation, stats.data_ptr(),
            dx.data_ptr(), address(dweight), address(dbias), *sizes, ws.data_ptr(), nbytes, hip.stream_of(x)),
            "vh_group_norm_backward")
        dweight, dbias = (None if t is None else t.to(d) for t, d in zip((dweight, dbias), ctx.param_dtypes))
        return dx, dweight, dbias, None, None, None


def visionhope_group_norm(x, groups, weight, bias, eps=1e-5, *, activation=None):
    """Group norm of ``x`` ``[B, C, H, W]`` in ``groups`` equal runs of channels (up to 1024 each),
    then ``activation`` (None, ``"silu"`` or ``"gelu"``); ``weight`` and ``bias`` ``[C]``.  The
    kernels run on channels-last storage: other inputs are copied to it first.  y is channels-last,
    in x's dtype.  Differentiable in x, weight and bias."""
    name = "visionhope_group_norm"
    check_io(name, x, 4)
    channels, groups = x.shape[1], int(groups)
    if groups < 1 or channels % groups:
        raise ValueError(f"{name}: {channels} channels do not divide into {groups} groups")
    if channels // groups > MAX_GROUP_CHANNELS:
        raise ValueError(f"{name} supports groups of at most {MAX_GROUP_CHANNELS} channels, got {channels // groups}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"{name}: activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    check_param(name, "weight", weight, (channels,), x.device)
    check_param(name, "bias", bias, (channels,), x.device)
    x = x.contiguous(memory_format=torch.channels_last)
    code = ACTIVATIONS[activation]
    if differentiated(x, weight, bias):
        return _GroupNormFunction.apply(x, weight, bias, groups, float(eps), code)
    return _no_grad_forward(x, weight, bias, groups, float(eps), code)


@on_tensor_device
def _no_grad_forward(x, weight, bias, groups, eps, activation):
    return _forward(x, groups, fp32_param(weight), fp32_param(bias), eps, activation, False)[0]

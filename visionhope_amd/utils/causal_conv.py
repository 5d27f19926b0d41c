"""Short causal depthwise convolution of token lines (native, ``csrc/causal_conv.hip``).

    y[b, t, c] = f(bias[c] + sum_k weight[c, k] * x[b, t - K + 1 + k, c])

with f the identity or SiLU, K = 2 .. 8 taps, and the K - 1 inputs before the first token
taken from a state (zero without one).  Prompts run through ``visionhope_causal_conv``
(differentiable), single tokens through ``visionhope_causal_conv_step`` on the state that the
prompt returned.  Sums are FP32; outputs are rounded once to the input's dtype.
"""

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import hip
from .cuda import on_tensor_device
from .token_lines import (address, check_io, check_like, check_param, dense_channels, differentiated,
                          fp32_param, line_lengths, moved_on, note_stream, refuse_gradients, refuse_held_leaves)

MAX_TAPS = 8


def _forward(x, weight, bias, silu, state, lengths, return_state):
    batch, length, channels = x.shape
    taps = weight.shape[-1]
    y = torch.empty((batch, length, channels), device=x.device, dtype=x.dtype)
    new_state = (torch.empty((batch, taps - 1, channels), device=x.device, dtype=x.dtype)
                 if return_state else None)
    hip.check(hip.load_library().vh_causal_conv_forward(
        address(x), x.stride(0), x.stride(1), hip.dtype_code(x.dtype), address(weight), address(bias), int(silu),
        address(state), address(lengths), address(y), address(new_state), batch, length, channels, taps,
        hip.stream_of(x)), "vh_causal_conv_forward")
    return y, new_state


class _CausalConvFunction(Function):
    @staticmethod
    @on_tensor_device
    def forward(ctx, x, weight, bias, state, silu, lengths, return_state):
        weight32, bias32 = fp32_param(weight).reshape(x.shape[-1], -1), fp32_param(bias)
        y, new_state = _forward(x, weight32, bias32, silu, state, lengths, return_state)
        note_stream(ctx, hip.stream_of(x))
        ctx.save_for_backward(x, weight32, bias32, state, lengths)
        ctx.silu = silu
        ctx.weight_like = (weight.shape, weight.dtype)
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        return (y, new_state) if return_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dnew_state=None):
        x, weight, bias, state, lengths = ctx.saved_tensors
        return _CausalConvFunction._gradients(x, weight, bias, state, lengths, ctx, dy, dnew_state)

    @staticmethod
    @on_tensor_device
    def _gradients(x, weight, bias, state, lengths, ctx, dy, dnew_state):
        refuse_held_leaves("visionhope_causal_conv", ctx, torch.cuda.is_current_stream_capturing())
        if dy is None and dnew_state is None:
            return (None,) * 7
        # saved-tensor hooks may return other strides than were saved
        x, weight = dense_channels(x), weight.contiguous()
        bias, state, lengths = (None if t is None else t.contiguous() for t in (bias, state, lengths))
        batch, length, channels = x.shape
        taps = weight.shape[1]
        dy = torch.zeros_like(x, memory_format=torch.contiguous_format) if dy is None else dense_channels(dy.to(x.dtype))
        if dnew_state is not None:
            dnew_state = dnew_state.to(x.dtype).contiguous()
        need = ctx.needs_input_grad
        dx = torch.empty((batch, length, channels), device=x.device, dtype=x.dtype)
        dweight = torch.empty((channels, taps), device=x.device, dtype=torch.float32) if need[1] else None
        dbias = torch.empty((channels,), device=x.device, dtype=torch.float32) if need[2] else None
        dstate = torch.empty_like(state) if need[3] else None
        lib = hip.load_library()
        ws = hip.workspace(lib.vh_causal_conv_backward_workspace_bytes(batch, length, channels, taps), x.device)
        hip.check(lib.vh_causal_conv_backward(
            address(dy), dy.stride(0), dy.stride(1), address(x), x.stride(0), x.stride(1), hip.dtype_code(x.dtype),
            address(weight), address(bias), int(ctx.silu), address(state), address(lengths), address(dnew_state),
            address(dx), address(dweight), address(dbias), address(dstate), batch, length, channels, taps, address(ws),
            ws.numel() * 4, hip.stream_of(x)), "vh_causal_conv_backward")
        if dweight is not None:
            dweight = dweight.view(ctx.weight_like[0]).to(ctx.weight_like[1])
        if dbias is not None:
            dbias = dbias.to(ctx.bias_dtype)
        return dx if need[0] else None, dweight, dbias, dstate, None, None, None


def _check_weight(name, weight, bias, channels, device):
    """``[C, K]``, or ``[C, 1, K]`` as a depthwise ``nn.Conv1d`` keeps it; returns K."""
    if not isinstance(weight, torch.Tensor) or weight.ndim not in (2, 3) or (weight.ndim == 3 and weight.shape[1] != 1):
        raise ValueError(f"{name}: weight must be [C, K] or [C, 1, K]")
    taps = weight.shape[-1]
    if not 2 <= taps <= MAX_TAPS:
        raise ValueError(f"{name}: supports 2 to {MAX_TAPS} taps, got {taps}")
    check_param(name, "weight", weight, (channels, taps) if weight.ndim == 2 else (channels, 1, taps), device)
    if bias is not None:
        check_param(name, "bias", bias, (channels,), device)
    return taps


def visionhope_causal_conv(x, weight, bias=None, *, silu=False, state=None, lengths=None, return_state=False):
    """Causal depthwise convolution of ``x`` ``[B, N, C]`` (module docstring).

    ``weight`` ``[C, K]`` or ``[C, 1, K]``, ``bias`` ``[C]``; ``state`` ``[B, K - 1, C]`` in x's
    dtype holds the inputs before the first token (oldest first).  With ``lengths`` ``[B]``
    (int32 or int64, values clamped to 0 .. N) outputs and gradients at and behind a
    sequence's end are zero.  Returns y, or ``(y, new_state)`` with ``return_state``: the last
    K - 1 inputs of every sequence, for the next call.  ``x`` may be a slice of a wider tensor
    (any batch and token strides); the outputs are dense.
    """
    name = "visionhope_causal_conv"
    check_io(name, x, 3)
    batch, _, channels = x.shape
    taps = _check_weight(name, weight, bias, channels, x.device)
    if state is not None:
        check_like(name, "state", state, (batch, taps - 1, channels), x.dtype, x.device)
        state = state.contiguous()
    lengths = line_lengths(name, lengths, batch, x.device)
    x = dense_channels(x)
    if differentiated(x, weight, bias, state):
        return _CausalConvFunction.apply(x, weight, bias, state, bool(silu), lengths, bool(return_state))
    y, new_state = _no_grad_forward(x, weight, bias, silu, state, lengths, return_state)
    return (y, new_state) if return_state else y


@on_tensor_device
def _no_grad_forward(x, weight, bias, silu, state, lengths, return_state):
    return _forward(x, fp32_param(weight).reshape(x.shape[-1], -1), fp32_param(bias), silu, state, lengths,
                    return_state)


@on_tensor_device
def visionhope_causal_conv_step(x, state, weight, bias=None, *, silu=False, new_state=None):
    """One token of every sequence: ``x`` ``[B, C]``, ``state`` ``[B, K - 1, C]`` (dense, x's
    dtype) as ``visionhope_causal_conv`` returns it.  Returns y ``[B, C]``; the state is moved on
    in place, or written to ``new_state`` (same shape, no overlap) and left as it was.
    Inference only."""
    name = "visionhope_causal_conv_step"
    check_io(name, x, 2)
    batch, channels = x.shape
    taps = _check_weight(name, weight, bias, channels, x.device)
    check_like(name, "state", state, (batch, taps - 1, channels), x.dtype, x.device)
    refuse_gradients(name, x, state, weight, bias, new_state)
    if new_state is None:
        new_state = state
    else:
        check_like(name, "new_state", new_state, state.shape, x.dtype, x.device)
    if not state.is_contiguous() or not new_state.is_contiguous():
        raise ValueError(f"{name}: states must be contiguous")
    x = dense_channels(x)
    weight, bias = fp32_param(weight), fp32_param(bias)   # [C, K] and [C, 1, K] are the same memory
    y = torch.empty((batch, channels), device=x.device, dtype=x.dtype)
    hip.check(hip.load_library().vh_causal_conv_step(
        address(x), x.stride(0), hip.dtype_code(x.dtype), address(weight), address(bias), int(silu), address(state),
        address(new_state), address(y), batch, channels, taps, hip.stream_of(x)), "vh_causal_conv_step")
    moved_on(new_state)
    return y

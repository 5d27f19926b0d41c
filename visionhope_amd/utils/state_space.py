"""Selective state space scan of token lines (native, ``csrc/state_space.hip``).

For every sequence and channel c, with S states in FP32:

    step[t] = softplus(dt[t] + dt_bias)                      (or dt[t] + dt_bias)
    h[t, n] = exp(step[t] * A[c, n]) * h[t-1, n] + step[t] * x[t] * B[t, n]
    y[t]    = (sum_n C[t, n] * h[t, n] + D * x[t]) * silu(gate[t])

Prompts run through ``visionhope_state_space_scan`` (differentiable), single tokens through
``visionhope_state_space_step`` on the states that the prompt returned.  B and C are shared by
all channels, or by the channels of a group (the four scan orders of a map as four groups of
one line, for instance).  ``models/srnl_core`` holds the framework's other recurrence.
"""

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from . import hip
from .cuda import on_tensor_device
from .token_lines import (check_io, check_like, check_param, dense_channels, fp32_param, line_lengths,
                          refuse_gradients)

MAX_STATES = 32


def _padded_states(states):
    """The state count that the prompt kernels are built for."""
    return 8 if states <= 8 else 16 if states <= 16 else 32


def _in_place(t):
    """Whether the scan can read ``t`` ``[B, N, G, S]`` where it stands: its states and groups
    dense, rows of whole words."""
    groups, states = t.shape[2:]
    size = t.element_size()
    return (t.dtype in (torch.float32, torch.bfloat16) and states == _padded_states(states) and t.stride(3) == 1
            and (groups == 1 or t.stride(2) == states) and t.data_ptr() % 4 == 0
            and t.stride(0) * size % 4 == 0 and t.stride(1) * size % 4 == 0)


def _state_maps(b, c):
    """B and C as the scan reads them: as given, or padded FP32 copies of both."""
    if _in_place(b) and _in_place(c):
        return b, c
    pad = _padded_states(b.shape[-1]) - b.shape[-1]
    return tuple(F.pad(t.float(), (0, pad)).contiguous() for t in (b, c))


def _pad_last(t, pad):
    return None if t is None else F.pad(t, (0, pad)) if pad else t


def _aligned(t):
    """``t`` dense and 16-byte aligned (the states are moved in 16-byte pieces)."""
    if t is None:
        return None
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _strides(t):
    return (None, 0, 0) if t is None else (hip.ptr(t), t.stride(0), t.stride(1))


def _forward(x, dt, A, b, c, D, gate, dt_bias, state, softplus, lengths, return_state, keep):
    """The native call on prepared operands; returns y, the states (padded) and what the
    backward starts from."""
    batch, length, channels = x.shape
    groups, states = b.shape[2:]
    lib = hip.load_library()
    y = torch.empty((batch, length, channels), device=x.device, dtype=x.dtype)
    new_state = torch.empty((batch, channels, states), device=x.device, dtype=torch.float32) if return_state else None
    sizes = (batch, length, channels, groups, states)
    kept = hip.workspace(lib.vh_state_space_kept_bytes(*sizes), x.device) if keep else None
    nbytes = lib.vh_state_space_workspace_bytes(*sizes)
    ws = hip.workspace(nbytes, x.device) if nbytes else None
    hip.check(lib.vh_state_space_forward(
        *_strides(x), *_strides(dt), *_strides(gate), hip.dtype_code(x.dtype), *_strides(b), *_strides(c),
        hip.dtype_code(b.dtype), hip.ptr(A), hip.ptr(D), hip.ptr(dt_bias), int(softplus), hip.ptr(state),
        hip.ptr(lengths), hip.ptr(y), hip.ptr(new_state), hip.ptr(kept), *sizes, hip.ptr(ws), nbytes,
        hip.stream_of(x)), "vh_state_space_forward")
    return y, new_state, kept


def _prepare(A, b, c, D, dt_bias, state):
    b, c = _state_maps(b, c)
    pad = b.shape[-1] - A.shape[-1]
    return (_aligned(_pad_last(fp32_param(A), pad)), b, c, fp32_param(D), fp32_param(dt_bias),
            _aligned(_pad_last(state, pad)))


class _StateSpaceScanFunction(Function):
    @staticmethod
    @on_tensor_device
    def forward(ctx, x, dt, A, b, c, D, gate, dt_bias, state, softplus, lengths, return_state):
        states = A.shape[1]
        A32, b32, c32, D32, bias32, state32 = _prepare(A, b.detach(), c.detach(), D, dt_bias,
                                                       None if state is None else state.detach())
        y, new_state, kept = _forward(x, dt, A32, b32, c32, D32, gate, bias32, state32, softplus, lengths, return_state,
                                      True)
        ctx.save_for_backward(x, dt, A32, b32, c32, D32, gate, bias32, lengths, kept)
        ctx.softplus, ctx.states = softplus, states
        ctx.dtypes = tuple(None if t is None else t.dtype for t in (A, b, c, D, dt_bias))
        ctx.has_state = state is not None
        ctx.set_materialize_grads(False)
        if not return_state:
            return y
        return y, new_state if new_state.shape[-1] == states else new_state[..., :states].contiguous()

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dnew_state=None):
        return _StateSpaceScanFunction._gradients(*ctx.saved_tensors, ctx, dy, dnew_state)

    @staticmethod
    @on_tensor_device
    def _gradients(x, dt, A, b, c, D, gate, dt_bias, lengths, kept, ctx, dy, dnew_state):
        if dy is None and dnew_state is None:
            return (None,) * 12
        batch, length, channels = x.shape
        groups, padded = b.shape[2:]
        states = ctx.states
        need = ctx.needs_input_grad
        dy = torch.zeros_like(x, memory_format=torch.contiguous_format) if dy is None else dense_channels(dy.to(x.dtype))
        if dnew_state is not None:
            dnew_state = _aligned(_pad_last(dnew_state.float(), padded - states))

        def out(*shape, dtype=torch.float32):
            return torch.empty(shape, device=x.device, dtype=dtype)

        dx, ddt = out(*x.shape, dtype=x.dtype), out(*x.shape, dtype=x.dtype)
        dgate = out(*x.shape, dtype=x.dtype) if gate is not None else None
        db = out(batch, length, groups, padded, dtype=x.dtype)
        dc = out(batch, length, groups, padded, dtype=x.dtype)
        dA = out(channels, padded) if need[2] else None
        dD = out(channels) if need[5] else None
        dbias = out(channels) if need[7] else None
        dstate = out(batch, channels, padded) if need[8] else None
        lib = hip.load_library()
        sizes = (batch, length, channels, groups, padded)
        nbytes = lib.vh_state_space_backward_workspace_bytes(*sizes)
        ws = hip.workspace(nbytes, x.device)
        hip.check(lib.vh_state_space_backward(
            *_strides(dy), *_strides(x), *_strides(dt), *_strides(gate), hip.dtype_code(x.dtype), *_strides(b),
            *_strides(c), hip.dtype_code(b.dtype), hip.ptr(A), hip.ptr(D), hip.ptr(dt_bias), int(ctx.softplus),
            hip.ptr(lengths), hip.ptr(kept), hip.ptr(dnew_state), hip.ptr(dx), hip.ptr(ddt), hip.ptr(dgate),
            hip.ptr(db), hip.ptr(dc), hip.ptr(dA), hip.ptr(dD), hip.ptr(dbias), hip.ptr(dstate), *sizes, hip.ptr(ws),
            nbytes, hip.stream_of(x)), "vh_state_space_backward")

        def shaped(t, dtype=None):
            if t is None:
                return None
            if padded != states:
                t = t[..., :states]
            return t if dtype is None else t.to(dtype)

        dtypes = ctx.dtypes
        return (dx, ddt, shaped(dA, dtypes[0]), shaped(db), shaped(dc), None if dD is None else dD.to(dtypes[3]), dgate,
                None if dbias is None else dbias.to(dtypes[4]), shaped(dstate), None, None, None)


def _check_recurrence(name, x, dt, A, B, C, D, gate, dt_bias):
    """Checks shared by the scan and the step; returns ``(states, groups)``."""
    lead, channels = x.shape[:-1], x.shape[-1]
    if not isinstance(A, torch.Tensor) or A.ndim != 2:
        raise ValueError(f"{name}: A must be [C, S]")
    states = A.shape[1]
    if not 1 <= states <= MAX_STATES:
        raise ValueError(f"{name}: supports 1 to {MAX_STATES} states, got {states}")
    check_param(name, "A", A, (channels, states), x.device)
    check_like(name, "dt", dt, x.shape, x.dtype, x.device)
    if gate is not None:
        check_like(name, "gate", gate, x.shape, x.dtype, x.device)
    if not isinstance(B, torch.Tensor) or B.ndim not in (len(lead) + 1, len(lead) + 2):
        raise ValueError(f"{name}: B must be [..., S] or [..., groups, S] with x's leading dimensions")
    groups = 1 if B.ndim == len(lead) + 1 else B.shape[-2]
    if groups < 1 or channels % groups:
        raise ValueError(f"{name}: {channels} channels do not divide into {groups} groups")
    shape = (*lead, states) if B.ndim == len(lead) + 1 else (*lead, groups, states)
    check_like(name, "B", B, shape, x.dtype, x.device)
    check_like(name, "C", C, shape, x.dtype, x.device)
    for what, t in (("D", D), ("dt_bias", dt_bias)):
        if t is not None:
            check_param(name, what, t, (channels,), x.device)
    return states, groups


def visionhope_state_space_scan(x, dt, A, B, C, D=None, *, gate=None, dt_bias=None, softplus=True, state=None,
                                lengths=None, return_state=False):
    """The selective scan of ``x`` ``[B, N, C]`` (module docstring).

    ``dt`` and ``gate`` like ``x``; ``A`` ``[C, S]`` with S of up to 32 (negative rates decay);
    ``B`` and ``C`` ``[B, N, S]``, or ``[B, N, groups, S]`` with the channels in ``groups`` equal
    runs; ``D`` and ``dt_bias`` ``[C]``; ``state`` ``[B, C, S]`` FP32, the states before the first
    token (zero without).  With ``lengths`` ``[B]`` (int32 or int64, values clamped to 0 .. N)
    outputs and gradients at and behind a sequence's end are zero, whatever stands there.
    Returns y in x's dtype, or ``(y, new_state)`` with ``return_state``.  x, dt, gate, B and C may
    be slices of wider tensors; results are dense.  Differentiable in every tensor but lengths.
    """
    name = "visionhope_state_space_scan"
    check_io(name, x, 3)
    batch, _, channels = x.shape
    states, _ = _check_recurrence(name, x, dt, A, B, C, D, gate, dt_bias)
    if state is not None:
        check_like(name, "state", state, (batch, channels, states), torch.float32, x.device)
    lengths = line_lengths(name, lengths, batch, x.device)
    if B.ndim == 3:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    x, dt = dense_channels(x), dense_channels(dt)
    gate = None if gate is None else dense_channels(gate)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (x, dt, A, B, C, D, gate, dt_bias, state)):
        return _StateSpaceScanFunction.apply(x, dt, A, B, C, D, gate, dt_bias, state, bool(softplus), lengths,
                                             bool(return_state))
    return _no_grad_forward(x, dt, A, B, C, D, gate, dt_bias, state, softplus, lengths, return_state)


@on_tensor_device
def _no_grad_forward(x, dt, A, b, c, D, gate, dt_bias, state, softplus, lengths, return_state):
    states = A.shape[1]
    A, b, c, D, dt_bias, state = _prepare(A, b, c, D, dt_bias, state)
    y, new_state, _ = _forward(x, dt, A, b, c, D, gate, dt_bias, state, softplus, lengths, return_state, False)
    if not return_state:
        return y
    return y, new_state if new_state.shape[-1] == states else new_state[..., :states].contiguous()


@on_tensor_device
def visionhope_state_space_step(x, dt, A, B, C, state, D=None, *, gate=None, dt_bias=None, softplus=True,
                                new_state=None):
    """One token of every sequence: ``x``, ``dt``, ``gate`` ``[B, C]``, ``B`` and ``C`` ``[B, S]`` or
    ``[B, groups, S]``, ``state`` ``[B, C, S]`` (FP32, dense) as ``visionhope_state_space_scan``
    returns it.  Returns y ``[B, C]``; the state is moved on in place, or written to ``new_state``
    (same shape, no overlap) and left as it was.  Inference only."""
    name = "visionhope_state_space_step"
    check_io(name, x, 2)
    batch, channels = x.shape
    states, groups = _check_recurrence(name, x, dt, A, B, C, D, gate, dt_bias)
    refuse_gradients(name, x, dt, A, B, C, state, D, gate, dt_bias)
    check_like(name, "state", state, (batch, channels, states), torch.float32, x.device)
    if new_state is None:
        new_state = state
    else:
        check_like(name, "new_state", new_state, state.shape, torch.float32, x.device)
    if not state.is_contiguous() or not new_state.is_contiguous():
        raise ValueError(f"{name}: states must be contiguous")
    if B.ndim == 3 and (groups > 1 and B.stride(1) != states or states > 1 and B.stride(2) != 1):
        B = B.contiguous()
    if C.ndim == 3 and (groups > 1 and C.stride(1) != states or states > 1 and C.stride(2) != 1):
        C = C.contiguous()
    x, dt, B, C = (dense_channels(t) for t in (x, dt, B, C))
    gate = None if gate is None else dense_channels(gate)
    A, D, dt_bias = fp32_param(A), fp32_param(D), fp32_param(dt_bias)
    y = torch.empty((batch, channels), device=x.device, dtype=x.dtype)
    hip.check(hip.load_library().vh_state_space_step(
        hip.ptr(x), x.stride(0), hip.ptr(dt), dt.stride(0), hip.ptr(gate), 0 if gate is None else gate.stride(0),
        hip.dtype_code(x.dtype), hip.ptr(B), B.stride(0), hip.ptr(C), C.stride(0), hip.ptr(A), hip.ptr(D),
        hip.ptr(dt_bias), int(softplus), hip.ptr(state), hip.ptr(new_state), hip.ptr(y), batch, channels, groups, states,
        hip.stream_of(x)), "vh_state_space_step")
    return y

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

from . import hip
from .cuda import on_tensor_device
from .token_lines import (address, check_io, check_like, check_param, dense_channels, differentiated,
                          fp32_param, line_lengths, moved_on, note_stream, refuse_gradients, refuse_held_leaves,
                          rows_of)

MAX_STATES = 32


def _dense_maps(t):
    """B or C ``[..., G, S]`` with the groups and states of a token dense."""
    groups, states = t.shape[-2:]
    if (states == 1 or t.stride(-1) == 1) and (groups == 1 or t.stride(-2) == states):
        return t
    return t.contiguous()


def _forward(x, dt, A, b, c, D, gate, dt_bias, state, softplus, lengths, return_state, keep):
    """The native call; returns y, the states and what the backward starts from."""
    batch, length, channels = x.shape
    sizes = (batch, length, channels, b.shape[2], A.shape[1])
    lib = hip.load_library()
    y = torch.empty((batch, length, channels), device=x.device, dtype=x.dtype)
    new_state = (torch.empty((batch, channels, sizes[4]), device=x.device, dtype=torch.float32)
                 if return_state else None)
    kept = hip.workspace(lib.vh_state_space_kept_bytes(*sizes), x.device) if keep else None
    nbytes = lib.vh_state_space_workspace_bytes(*sizes)
    ws = hip.workspace(nbytes, x.device)
    hip.check(lib.vh_state_space_forward(
        *rows_of(x), *rows_of(dt), *rows_of(gate), hip.dtype_code(x.dtype), *rows_of(b), *rows_of(c), address(A),
        address(D), address(dt_bias), softplus, address(state), address(lengths), address(y), address(new_state),
        address(kept), *sizes, address(ws), nbytes, hip.stream_of(x)), "vh_state_space_forward")
    return y, new_state, kept


class _StateSpaceScanFunction(Function):
    @staticmethod
    @on_tensor_device
    def forward(ctx, x, dt, A, b, c, D, gate, dt_bias, state, softplus, lengths, return_state):
        A32, D32, bias32 = fp32_param(A), fp32_param(D), fp32_param(dt_bias)
        y, new_state, kept = _forward(x, dt, A32, b, c, D32, gate, bias32, state, softplus, lengths, return_state,
                                      any(ctx.needs_input_grad))
        note_stream(ctx, hip.stream_of(x))
        ctx.save_for_backward(x, dt, A32, b, c, D32, gate, bias32, lengths, kept)
        ctx.softplus = softplus
        ctx.param_dtypes = tuple(None if t is None else t.dtype for t in (A, D, dt_bias))
        ctx.set_materialize_grads(False)
        return (y, new_state) if return_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dnew_state=None):
        return _StateSpaceScanFunction._gradients(*ctx.saved_tensors, ctx, dy, dnew_state)

    @staticmethod
    @on_tensor_device
    def _gradients(x, dt, A, b, c, D, gate, dt_bias, lengths, kept, ctx, dy, dnew_state):
        refuse_held_leaves("visionhope_state_space_scan", ctx, torch.cuda.is_current_stream_capturing())
        if dy is None and dnew_state is None:
            return (None,) * 12
        # saved-tensor hooks may return other strides than were saved
        x, dt, b, c = dense_channels(x), dense_channels(dt), _dense_maps(b), _dense_maps(c)
        gate = None if gate is None else dense_channels(gate)
        A, D, dt_bias, lengths, kept = (None if t is None else t.contiguous() for t in (A, D, dt_bias, lengths, kept))
        shape, device, dtype = x.shape, x.device, x.dtype
        sizes = (*shape, b.shape[2], A.shape[1])
        need = ctx.needs_input_grad
        dy = torch.zeros(shape, device=device, dtype=dtype) if dy is None else dense_channels(dy.to(dtype))
        if dnew_state is not None:
            dnew_state = dnew_state.float().contiguous()

        def fp32(want, *shape):
            return torch.empty(shape, device=device, dtype=torch.float32) if want else None

        dx, ddt = torch.empty(shape, device=device, dtype=dtype), torch.empty(shape, device=device, dtype=dtype)
        dgate = torch.empty(shape, device=device, dtype=dtype) if gate is not None else None
        db, dc = torch.empty(b.shape, device=device, dtype=dtype), torch.empty(b.shape, device=device, dtype=dtype)
        channels, states = A.shape
        dA, dD, dbias = fp32(need[2], channels, states), fp32(need[5], channels), fp32(need[7], channels)
        dstate = fp32(need[8], shape[0], channels, states)
        lib = hip.load_library()
        nbytes = lib.vh_state_space_backward_workspace_bytes(*sizes)
        ws = hip.workspace(nbytes, device)
        hip.check(lib.vh_state_space_backward(
            *rows_of(dy), *rows_of(x), *rows_of(dt), *rows_of(gate), hip.dtype_code(dtype), *rows_of(b), *rows_of(c),
            address(A), address(D), address(dt_bias), ctx.softplus, address(lengths), address(kept),
            address(dnew_state), address(dx), address(ddt), address(dgate), address(db), address(dc), address(dA),
            address(dD), address(dbias), address(dstate), *sizes, address(ws), nbytes, hip.stream_of(x)),
            "vh_state_space_backward")
        dA, dD, dbias = (None if t is None else t.to(d) for t, d in zip((dA, dD, dbias), ctx.param_dtypes))
        return dx, ddt, dA, db, dc, dD, dgate, dbias, dstate, None, None, None


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
    x, dt, B, C = dense_channels(x), dense_channels(dt), _dense_maps(B), _dense_maps(C)
    gate = None if gate is None else dense_channels(gate)
    state = None if state is None else state.contiguous()
    if differentiated(x, dt, A, B, C, D, gate, dt_bias, state):
        return _StateSpaceScanFunction.apply(x, dt, A, B, C, D, gate, dt_bias, state, int(bool(softplus)), lengths,
                                             bool(return_state))
    return _no_grad_forward(x, dt, A, B, C, D, gate, dt_bias, state, int(bool(softplus)), lengths, return_state)


@on_tensor_device
def _no_grad_forward(x, dt, A, b, c, D, gate, dt_bias, state, softplus, lengths, return_state):
    y, new_state, _ = _forward(x, dt, fp32_param(A), b, c, fp32_param(D), gate, fp32_param(dt_bias), state, softplus,
                               lengths, return_state, False)
    return (y, new_state) if return_state else y


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
    check_like(name, "state", state, (batch, channels, states), torch.float32, x.device)
    refuse_gradients(name, x, dt, A, B, C, state, D, gate, dt_bias, new_state)
    if new_state is None:
        new_state = state
    else:
        check_like(name, "new_state", new_state, state.shape, torch.float32, x.device)
    if not state.is_contiguous() or not new_state.is_contiguous():
        raise ValueError(f"{name}: states must be contiguous")
    B, C = (_dense_maps(t if t.ndim == 3 else t[:, None]) for t in (B, C))
    x, dt = dense_channels(x), dense_channels(dt)
    gate = None if gate is None else dense_channels(gate)
    A, D, dt_bias = fp32_param(A), fp32_param(D), fp32_param(dt_bias)
    y = torch.empty((batch, channels), device=x.device, dtype=x.dtype)
    hip.check(hip.load_library().vh_state_space_step(
        x.data_ptr(), x.stride(0), dt.data_ptr(), dt.stride(0), address(gate), 0 if gate is None else gate.stride(0),
        hip.dtype_code(x.dtype), B.data_ptr(), B.stride(0), C.data_ptr(), C.stride(0), A.data_ptr(), address(D),
        address(dt_bias), int(bool(softplus)), state.data_ptr(), new_state.data_ptr(), y.data_ptr(), batch, channels,
        groups, states, hip.stream_of(x)), "vh_state_space_step")
    moved_on(new_state)
    return y

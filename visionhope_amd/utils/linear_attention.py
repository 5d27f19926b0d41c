"""Linear attention of token lines with a decay for each head (native, ``csrc/linear_attention.hip``).

For every sequence and head, with a state S of key_dim x value_dim FP32 values:

    S[t] = exp(log_decay) * S[t-1] + k[t] v[t]^T
    o[t] = scale * q[t]^T S[t]

Prompts run through ``visionhope_linear_attention`` (differentiable), in chunks on the matrix
cores; single tokens through ``visionhope_linear_attention_step`` on the states that the prompt
returned.  ``utils/state_space.py`` is the recurrence whose decay each token chooses.
"""

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import hip
from .cuda import on_tensor_device
from .token_lines import (address, check_io, check_like, check_param, dense_channels, differentiated, fp32_param,
                          line_lengths, moved_on, note_stream, refuse_gradients, refuse_held_leaves)

MAX_HEAD_DIM = 128


def _lines(t):
    """``t`` with dense heads and tokens less than 2^24 elements apart, as the kernels take it."""
    return t.contiguous() if t.stride(1) >= 1 << 24 and t.shape[1] > 1 else dense_channels(t)


def _heads_of(t):
    """Native arguments of ``[B, N, H, D]``: address and element strides of sequence, token, head."""
    return t.data_ptr(), t.stride(0), 0 if t.shape[1] == 1 else t.stride(1), t.stride(2)


def _forward(q, k, v, log_decay, scale, state, lengths, return_state):
    batch, length, heads, key_dim = q.shape
    sizes = (batch, length, heads, key_dim, v.shape[3])
    lib = hip.load_library()
    out = torch.empty((batch, length, heads, sizes[4]), device=q.device, dtype=q.dtype)
    new_state = (torch.empty((batch, heads, key_dim, sizes[4]), device=q.device, dtype=torch.float32)
                 if return_state else None)
    code = hip.dtype_code(q.dtype)
    nbytes = lib.vh_linear_attention_workspace_bytes(*sizes, code)
    ws = hip.workspace(nbytes, q.device) if nbytes else None
    hip.check(lib.vh_linear_attention_forward(
        *_heads_of(q), *_heads_of(k), *_heads_of(v), code, address(log_decay), scale, address(state), address(lengths),
        address(out), address(new_state), *sizes, address(ws), nbytes, hip.stream_of(q)), "vh_linear_attention_forward")
    return out, new_state, ws   # the workspace: states that the backward starts from


class _LinearAttentionFunction(Function):
    @staticmethod
    @on_tensor_device
    def forward(ctx, q, k, v, log_decay, state, scale, lengths, return_state):
        decay32 = fp32_param(log_decay)
        out, new_state, kept = _forward(q, k, v, decay32, scale, state, lengths, return_state)
        note_stream(ctx, hip.stream_of(q))
        ctx.save_for_backward(q, k, v, decay32, state, lengths, kept)
        ctx.scale, ctx.decay_dtype = scale, log_decay.dtype
        ctx.set_materialize_grads(False)
        return (out, new_state) if return_state else out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dnew_state=None):
        return _LinearAttentionFunction._gradients(*ctx.saved_tensors, ctx, dout, dnew_state)

    @staticmethod
    @on_tensor_device
    def _gradients(q, k, v, log_decay, state, lengths, kept, ctx, dout, dnew_state):
        refuse_held_leaves("visionhope_linear_attention", ctx, torch.cuda.is_current_stream_capturing())
        if dout is None and dnew_state is None:
            return (None,) * 8
        # saved-tensor hooks may return other strides than were saved
        q, k, v = _lines(q), _lines(k), _lines(v)
        log_decay, state, lengths, kept = (None if t is None else t.contiguous()
                                           for t in (log_decay, state, lengths, kept))
        batch, length, heads, key_dim = q.shape
        value_dim, device, dtype = v.shape[3], q.device, q.dtype
        sizes, need = (batch, length, heads, key_dim, value_dim), ctx.needs_input_grad
        dout = (torch.zeros(v.shape, device=device, dtype=dtype) if dout is None else _lines(dout.to(dtype)))
        if dnew_state is not None:
            dnew_state = dnew_state.float().contiguous()
        dq, dk = (torch.empty(q.shape, device=device, dtype=dtype) for _ in range(2))
        dv = torch.empty(v.shape, device=device, dtype=dtype)
        dstate = torch.empty((batch, heads, key_dim, value_dim), device=device, dtype=torch.float32) if need[4] else None
        ddecay = torch.empty(heads, device=device, dtype=torch.float32) if need[3] else None
        lib, code = hip.load_library(), hip.dtype_code(dtype)
        nbytes = lib.vh_linear_attention_backward_workspace_bytes(*sizes, code, int(need[3]))
        ws = hip.workspace(nbytes, device) if nbytes else None
        hip.check(lib.vh_linear_attention_backward(
            *_heads_of(dout), *_heads_of(q), *_heads_of(k), *_heads_of(v), code, address(log_decay), ctx.scale,
            address(state), address(lengths), address(kept), address(dnew_state), address(dq), address(dk),
            address(dv), address(dstate), address(ddecay), *sizes, address(ws), nbytes, hip.stream_of(q)),
            "vh_linear_attention_backward")
        return dq, dk, dv, None if ddecay is None else ddecay.to(ctx.decay_dtype), dstate, None, None, None


def _check_heads(name, q, k, v, log_decay):
    """Checks shared by the prompt form and the step; returns heads, key_dim and value_dim."""
    lead, (heads, key_dim) = q.shape[:-2], q.shape[-2:]
    check_like(name, "k", k, q.shape, q.dtype, q.device)
    if not isinstance(v, torch.Tensor) or v.ndim != q.ndim or v.shape[-1] < 1:
        raise ValueError(f"{name}: v must be {tuple((*lead, heads))} with a nonempty last dimension")
    value_dim = v.shape[-1]
    check_like(name, "v", v, (*lead, heads, value_dim), q.dtype, q.device)
    if key_dim > MAX_HEAD_DIM or value_dim > MAX_HEAD_DIM:
        raise ValueError(f"{name} supports heads of up to {MAX_HEAD_DIM}, got {key_dim} and {value_dim}")
    check_param(name, "log_decay", log_decay, (heads,), q.device)
    return heads, key_dim, value_dim


def visionhope_linear_attention(q, k, v, log_decay, *, scale=None, state=None, lengths=None, return_state=False):
    """Linear attention of ``q`` and ``k`` ``[B, N, H, key_dim]`` and ``v`` ``[B, N, H, value_dim]``
    (module docstring), heads of up to 128.

    ``log_decay`` ``[H]`` is the logarithm of each head's decay, at most zero (minus infinity
    forgets at every token); ``scale`` defaults to ``key_dim ** -0.5``; ``state``
    ``[B, H, key_dim, value_dim]`` FP32 is the state before the first token (zero without).  With
    ``lengths`` ``[B]`` (int32 or int64, values clamped to 0 .. N) outputs and gradients at and behind
    a sequence's end are zero, whatever stands there.  Returns o in q's dtype, or
    ``(o, new_state)`` with ``return_state``.  q, k and v may be slices of wider tensors or expanded
    over heads (keys and values that heads share); results are dense.  Differentiable in every
    tensor but lengths.  Values within a sequence must be finite: a key or value that is not
    reaches, in its head, every later output through the state and earlier ones of its chunk of 64.
    """
    name = "visionhope_linear_attention"
    check_io(name, q, 4)
    heads, key_dim, value_dim = _check_heads(name, q, k, v, log_decay)
    batch = q.shape[0]
    if state is not None:
        check_like(name, "state", state, (batch, heads, key_dim, value_dim), torch.float32, q.device)
        state = state.contiguous()
    lengths = line_lengths(name, lengths, batch, q.device)
    scale = key_dim ** -0.5 if scale is None else float(scale)
    q, k, v = _lines(q), _lines(k), _lines(v)
    if differentiated(q, k, v, log_decay, state):
        return _LinearAttentionFunction.apply(q, k, v, log_decay, state, scale, lengths, bool(return_state))
    return _no_grad_forward(q, k, v, log_decay, state, scale, lengths, return_state)


@on_tensor_device
def _no_grad_forward(q, k, v, log_decay, state, scale, lengths, return_state):
    out, new_state, _ = _forward(q, k, v, fp32_param(log_decay), scale, state, lengths, return_state)
    return (out, new_state) if return_state else out


@on_tensor_device
def visionhope_linear_attention_step(q, k, v, log_decay, state, *, scale=None, new_state=None):
    """One token of every sequence: ``q`` and ``k`` ``[B, H, key_dim]``, ``v`` ``[B, H, value_dim]``,
    ``state`` ``[B, H, key_dim, value_dim]`` (FP32, dense) as ``visionhope_linear_attention`` returns
    it.  Returns o ``[B, H, value_dim]``; the state is moved on in place, or written to ``new_state``
    (same shape, no overlap) and left as it was.  Inference only."""
    name = "visionhope_linear_attention_step"
    check_io(name, q, 3)
    heads, key_dim, value_dim = _check_heads(name, q, k, v, log_decay)
    batch = q.shape[0]
    check_like(name, "state", state, (batch, heads, key_dim, value_dim), torch.float32, q.device)
    refuse_gradients(name, q, k, v, log_decay, state, new_state)
    if new_state is None:
        new_state = state
    else:
        check_like(name, "new_state", new_state, state.shape, torch.float32, q.device)
    if not state.is_contiguous() or not new_state.is_contiguous():
        raise ValueError(f"{name}: states must be contiguous")
    q, k, v = dense_channels(q), dense_channels(k), dense_channels(v)
    log_decay = fp32_param(log_decay)
    out = torch.empty((batch, heads, value_dim), device=q.device, dtype=q.dtype)
    hip.check(hip.load_library().vh_linear_attention_step(
        q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
        v.stride(1), hip.dtype_code(q.dtype), log_decay.data_ptr(), key_dim ** -0.5 if scale is None else float(scale),
        state.data_ptr(), new_state.data_ptr(), out.data_ptr(), batch, heads, key_dim, value_dim, hip.stream_of(q)),
        "vh_linear_attention_step")
    moved_on(new_state)
    return out

"""Argument handling shared by the operators of token lines ``[B, N, C]``."""

from weakref import WeakValueDictionary

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .cuda import on_tensor_device

IO_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def check_io(name, x, ndim):
    """``x`` is a CUDA tensor of a supported type with ``ndim`` nonempty dimensions."""
    if isinstance(x, torch.Tensor) and x.is_cuda and x.dtype in IO_DTYPES and x.ndim == ndim and x.numel():
        return
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{name} expects CUDA tensors")
    if x.dtype not in IO_DTYPES:
        raise TypeError(f"{name} supports FP16, BF16 and FP32 tensors, got {x.dtype}")
    raise ValueError(f"{name} expects a nonempty tensor of {ndim} dimensions, got shape {tuple(x.shape)}")


def check_like(name, what, t, shape, dtype, device):
    """``t`` has exactly this shape, dtype and device."""
    if isinstance(t, torch.Tensor) and t.shape == shape and t.dtype == dtype and t.device == device:
        return
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != tuple(shape):
        got = tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"{name}: {what} must have shape {tuple(shape)}, got {got}")
    if t.dtype != dtype:
        raise TypeError(f"{name}: {what} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: {what} must be on {device}, got {t.device}")


def check_param(name, what, t, shape, device):
    """A floating-point parameter of this shape on this device."""
    if isinstance(t, torch.Tensor) and t.shape == shape and t.is_floating_point() and t.device == device:
        return
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != tuple(shape):
        got = tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"{name}: {what} must have shape {tuple(shape)}, got {got}")
    if not t.is_floating_point():
        raise TypeError(f"{name}: {what} must be floating point, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: {what} must be on {device}, got {t.device}")


def line_lengths(name, lengths, batch, device):
    """Sequence lengths as int32 ``[B]`` on the device, or None."""
    if lengths is None:
        return None
    if not isinstance(lengths, torch.Tensor) or tuple(lengths.shape) != (batch,):
        raise ValueError(f"{name}: lengths must be a tensor of shape ({batch},)")
    if lengths.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: lengths must be int32 or int64, got {lengths.dtype}")
    if lengths.device != device:
        raise ValueError(f"{name}: lengths must be on {device}, got {lengths.device}")
    if lengths.dtype == torch.int64:   # clamped first: the kernels clamp what int32 holds
        lengths = lengths.clamp(0, 2**31 - 1).to(torch.int32)
    return lengths.contiguous()


def dense_channels(t):
    """``t`` with its last dimension dense; the strides of the others are the kernels' arguments."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def fp32_param(t):
    """A parameter as the kernels read it: FP32, dense."""
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.detach().float().contiguous()


def address(t):
    """A native pointer argument (an int: cheaper to pass than a ctypes object), or None."""
    return None if t is None else t.data_ptr()


def rows_of(t):
    """Native arguments of a token tensor: address and element strides of sequence and token."""
    return (None, 0, 0) if t is None else (t.data_ptr(), t.stride(0), t.stride(1))


def differentiated(*tensors):
    """Whether a call goes through its autograd Function: gradients are recorded for one of the
    tensors, or a forward-mode level is open (the Function then refuses tangents, which no
    kernel carries)."""
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


_LEAF_NODE = "torch::autograd::AccumulateGrad"
_DEFAULT_STREAM_GRAPHS = WeakValueDictionary()   # living nodes of Functions, by id


def note_stream(ctx, stream):
    """Called by a Function's forward: keeps in mind, for as long as its graph lives, that it was
    recorded on the default stream.  The nodes that accumulate its leaves' gradients keep that
    stream as long."""
    if stream == 0:
        _DEFAULT_STREAM_GRAPHS[id(ctx)] = ctx


def _leaf_nodes(roots, among=lambda node: True):
    """The nodes that accumulate leaves' gradients behind these ones: their own inputs', and those
    behind any operations between."""
    leaves, seen, stack = set(), set(roots), list(roots)
    while stack:
        for node, _ in stack.pop().next_functions:
            if node is None or node in seen or not among(node):
                continue
            seen.add(node)
            (leaves.add if node.name() == _LEAF_NODE else stack.append)(node)
    return leaves


def _runs(node):
    """Whether the backward pass under way goes to a node (asked about a leaf whose gradient is
    returned and not accumulated, which it does go to, autograd raises)."""
    try:
        return torch._C._will_engine_execute_node(node)
    except RuntimeError:
        return True


def refuse_held_leaves(name, ctx, capturing):
    """Called by a Function's backward: a captured backward must not reach a node of the default
    stream, which cannot take part in a capture (the process would end there)."""
    if not capturing:
        return
    held = [other for other in (ref() for ref in _DEFAULT_STREAM_GRAPHS.valuerefs()) if other is not None]
    if held and not _leaf_nodes([ctx], _runs).isdisjoint(_leaf_nodes(held)):
        raise RuntimeError(f"{name}: cannot capture this backward pass: an autograd graph that was recorded over "
                           "the same leaves on the default stream is still alive; drop its outputs before the "
                           "capture")


class _GuardFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, out, name):
        ctx.name = name
        return out.view_as(out)

    @staticmethod
    def backward(ctx, dy):
        refuse_held_leaves(ctx.name, ctx, torch.cuda.is_current_stream_capturing())
        return dy, None


@on_tensor_device
def guarded(name, out):
    """Called by a module on its output: in a capture its backward refuses held leaves here, before
    the pass comes to those of the module's operations behind the last operator."""
    if out.requires_grad and torch.cuda.is_current_stream_capturing():
        return _GuardFunction.apply(out, name)
    return out


def moved_on(state):
    """Marks a state that a kernel wrote as changed, so that a graph that saved it refuses to use
    what stands there now (inference tensors keep no such mark)."""
    if not state.is_inference():
        increment_version(state)


def refuse_gradients(name, *tensors):
    """Single-token calls write states in place and record no derivatives of either mode."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} is for inference; call it under torch.no_grad() or on detached tensors")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name} has no forward-mode derivative")

"""The short causal convolution on the GPU against the float64 oracle: prompts, gradients,
single tokens, states, lengths, strides, streams and graphs."""

import pytest
import torch

from oracle.oracle_torch import causal_conv_torch
from tests.helpers import randn
from tests.token_lines import DTYPES, compare, gradients, half_step, tolerance

pytestmark = pytest.mark.gpu


def _inputs(batch, length, channels, taps, dtype, seed=0):
    x = randn(batch, length, channels, seed=seed + 1).to(dtype)
    weight = randn(channels, taps, seed=seed + 2) * 0.5
    bias = randn(channels, seed=seed + 3) * 0.5
    state = randn(batch, taps - 1, channels, seed=seed + 4).to(dtype)
    return x, weight, bias, state


def _check(device, x, weight, bias, state, lengths, silu, what, terms=None):
    from visionhope_amd.utils.causal_conv import visionhope_causal_conv

    dtype, taps = x.dtype, weight.shape[-1]
    dy, dstate = randn(*x.shape, seed=91).to(dtype), randn(x.shape[0], taps - 1, x.shape[2], seed=92).to(dtype)
    want, grads = gradients(lambda *a: causal_conv_torch(a[0], a[1], a[2], silu, a[3], lengths),
                            (x, weight, bias, state), (dy, dstate))
    leaves = [None if t is None else t.to(device).requires_grad_() for t in (x, weight, bias, state)]
    y, new_state = visionhope_causal_conv(leaves[0], leaves[1], leaves[2], silu=silu, state=leaves[3],
                                          lengths=None if lengths is None else lengths.to(device), return_state=True)
    assert y.dtype == dtype and new_state.dtype == dtype
    tol = tolerance(dtype, taps)
    compare(y, want[0], tol, f"{what} y")
    assert torch.equal(new_state.double().cpu(), want[1]), f"{what}: new state"
    torch.autograd.backward((y, new_state), (dy.to(device), dstate.to(device)))
    rows = x.shape[0] * x.shape[1]
    for name, leaf, grad in zip(("x", "weight", "bias", "state"), leaves, grads):
        if leaf is None:
            continue
        tol = tolerance(torch.float32, rows) if name in ("weight", "bias") else tolerance(dtype, 2 * taps)
        compare(leaf.grad, grad, tol, f"{what} d{name}")
        assert leaf.grad.dtype == leaf.dtype


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("shape", [(1, 1, 1, 4), (2, 2, 8, 4), (3, 17, 12, 3), (2, 33, 30, 2), (1, 300, 7, 5),
                                   (2, 70, 64, 7), (5, 41, 96, 8), (2, 129, 192, 4), (1, 5, 4, 6)])
def test_prompt_and_gradients(device, dtype, silu, shape):
    x, weight, bias, state = _inputs(*shape, dtype)
    _check(device, x, weight, bias, state, None, silu, f"{shape} {dtype}")
    _check(device, x, weight, None, None, None, silu, f"{shape} {dtype} bare")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels", [64, 13])
def test_lengths(device, dtype, channels):
    x, weight, bias, state = _inputs(6, 45, channels, 4, dtype, seed=10)
    lengths = torch.tensor([45, 0, 1, 2, 32, 17], dtype=torch.int64)
    _check(device, x, weight, bias, state, lengths, True, f"lengths {dtype} {channels}")
    _check(device, x, weight, bias, None, lengths.to(torch.int32), False, f"lengths {dtype} {channels} int32")


def test_what_stands_behind_the_end_has_no_part(device):
    from visionhope_amd.utils.causal_conv import visionhope_causal_conv

    x, weight, bias, _ = (t.to(device) for t in _inputs(3, 40, 24, 4, torch.bfloat16, seed=20))
    lengths = torch.tensor([11, 0, 40], dtype=torch.int32, device=device)
    dy = randn(3, 40, 24, seed=21).to(device, torch.bfloat16)
    results = []
    for fill in (0.0, float("nan"), float("inf")):
        xf, dyf = x.clone(), dy.clone()
        for i, n in enumerate(lengths.tolist()):
            xf[i, n:] = fill
            dyf[i, n:] = fill
        leaves = [t.clone().requires_grad_() for t in (xf, weight, bias)]
        y, state = visionhope_causal_conv(*leaves, silu=True, lengths=lengths, return_state=True)
        results.append([y, state, *torch.autograd.grad(y, leaves, dyf)])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)
    # lengths outside 0 .. N are clamped
    wild = torch.tensor([11, -5, 2**40], dtype=torch.int64, device=device)
    assert torch.equal(visionhope_causal_conv(x, weight, bias, silu=True, lengths=wild), results[0][0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_slices_and_odd_addresses(device, dtype):
    from visionhope_amd.utils.causal_conv import visionhope_causal_conv

    x, weight, bias, state = (t.to(device) for t in _inputs(3, 37, 48, 4, dtype, seed=30))
    want = visionhope_causal_conv(x, weight, bias, silu=True, state=state)
    dy = randn(3, 37, 48, seed=31).to(device, dtype)

    def grad(xv, dyv):
        leaf = xv.detach().requires_grad_()
        return torch.autograd.grad(visionhope_causal_conv(leaf, weight, bias, silu=True, state=state), leaf, dyv)[0]

    want_dx = grad(x, dy)
    wide = torch.empty(3, 37, 96, device=device, dtype=dtype)
    wide[..., 48:] = x
    odd = torch.empty(3 * 37 * 48 + 1, device=device, dtype=dtype)[1:].view(3, 37, 48)
    odd.copy_(x)
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)
    planes = x.transpose(1, 2).contiguous().transpose(1, 2)
    for name, view in (("slice", wide[..., 48:]), ("odd", odd), ("tokens first", turned), ("channel planes", planes)):
        assert torch.equal(visionhope_causal_conv(view, weight, bias, silu=True, state=state), want), name
        assert torch.equal(grad(view, dy), want_dx), name
    # a broadcast cotangent, as y.sum() gives
    ones = torch.ones((), device=device, dtype=dtype).expand(3, 37, 48)
    assert torch.equal(grad(x, ones), grad(x, ones.contiguous()))
    # weight as a depthwise Conv1d keeps it, and in another floating type
    assert torch.equal(visionhope_causal_conv(x, weight[:, None], bias, silu=True, state=state), want)
    low = weight.to(torch.bfloat16)
    leaf = low.clone().requires_grad_()
    y = visionhope_causal_conv(x, leaf, bias)
    assert torch.equal(y, visionhope_causal_conv(x, low.float(), bias))
    y.sum().backward()
    assert leaf.grad.dtype == torch.bfloat16


def test_rows_past_32_bits(device):
    """A batch stride of 2^31 elements (4 GiB apart)."""
    from visionhope_amd.utils.causal_conv import visionhope_causal_conv

    base = torch.empty(2**31 + 64 * 32, device=device, dtype=torch.bfloat16)
    far = base.as_strided((2, 64, 32), (2**31, 32, 1))
    x = randn(2, 64, 32, seed=41).to(device, torch.bfloat16)
    far.copy_(x)
    weight = randn(32, 4, seed=42).to(device)
    assert torch.equal(visionhope_causal_conv(far, weight), visionhope_causal_conv(x, weight))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 4), (3, 30, 2), (64, 256, 4), (5, 97, 8)])
def test_tokens_one_by_one_continue_a_prompt(device, dtype, shape):
    from visionhope_amd.utils.causal_conv import visionhope_causal_conv, visionhope_causal_conv_step

    batch, channels, taps = shape
    x, weight, bias, first = (t.to(device) for t in _inputs(batch, 12, channels, taps, dtype, seed=50))
    whole, last = visionhope_causal_conv(x, weight, bias, silu=True, state=first, return_state=True)
    y, state = visionhope_causal_conv(x[:, :5], weight, bias, silu=True, state=first, return_state=True)
    rows = [y]
    for t in range(5, 12):
        if t % 2:
            rows.append(visionhope_causal_conv_step(x[:, t], state, weight, bias, silu=True)[:, None])
        else:
            before, after = state.clone(), torch.empty_like(state)
            rows.append(visionhope_causal_conv_step(x[:, t], state, weight, bias, silu=True, new_state=after)[:, None])
            assert torch.equal(state, before)
            state = after
    assert torch.equal(state, last)
    # the same sum in the same order, FP32
    compare(torch.cat(rows, 1), whole.double().cpu(), half_step(dtype) * 2, "steps")


def test_repeats_bit_by_bit_on_any_stream_and_in_a_graph(device):
    from visionhope_amd.utils.causal_conv import visionhope_causal_conv, visionhope_causal_conv_step

    x, weight, bias, state = (t.to(device) for t in _inputs(4, 200, 96, 4, torch.bfloat16, seed=60))
    dy = randn(4, 200, 96, seed=61).to(device, torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (x, weight, bias)]

    def step():
        y, new = visionhope_causal_conv(*leaves, silu=True, state=state, return_state=True)
        return [y.detach(), new.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = step()
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream(device).wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(want, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    live, token = state.clone(), x[:, 0].contiguous()
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        out = visionhope_causal_conv_step(token, live, weight, bias)
    for round_ in range(3):
        with torch.no_grad():
            leaves[0].copy_(x * (round_ + 1))
        want = step()
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, captured):
            assert torch.equal(a, b), f"replay {round_}"
        eager = live.clone()
        want_token = visionhope_causal_conv_step(token, eager, weight, bias)
        graph2.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want_token) and torch.equal(live, eager)


def test_gradients_only_where_asked(device):
    from visionhope_amd.utils.causal_conv import visionhope_causal_conv

    x, weight, bias, state = (t.to(device) for t in _inputs(2, 9, 8, 4, torch.float32, seed=70))
    weight.requires_grad_()
    y, new = visionhope_causal_conv(x, weight, bias, state=state, return_state=True)
    y.sum().backward()
    assert weight.grad is not None
    # only the returned state is used: it depends on x alone
    leaf = x.clone().requires_grad_()
    _, new = visionhope_causal_conv(leaf, weight.detach(), bias, return_state=True)
    grad, = torch.autograd.grad(new.sum(), leaf)
    assert torch.equal(grad[:, -3:], torch.ones_like(grad[:, -3:])) and not grad[:, :-3].any()
    with torch.no_grad():
        assert not visionhope_causal_conv(leaf, weight).requires_grad


def test_step_marks_the_state_as_changed(device):
    """A graph that saved the state refuses to run its backward with the moved-on one."""
    from visionhope_amd.utils.causal_conv import visionhope_causal_conv, visionhope_causal_conv_step

    x, weight, bias, state = (t.to(device) for t in _inputs(2, 9, 8, 4, torch.float32, seed=75))
    y = visionhope_causal_conv(x, weight.clone().requires_grad_(), state=state)
    visionhope_causal_conv_step(x[:, 0], state, weight)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals(device):
    from visionhope_amd.utils.causal_conv import visionhope_causal_conv, visionhope_causal_conv_step

    x, weight, bias, state = (t.to(device) for t in _inputs(2, 9, 8, 4, torch.float32, seed=80))
    bad = [
        (ValueError, "CUDA", lambda: visionhope_causal_conv(x.cpu(), weight)),
        (TypeError, "FP16, BF16 and FP32", lambda: visionhope_causal_conv(x.double(), weight)),
        (ValueError, "3 dimensions", lambda: visionhope_causal_conv(x[0], weight)),
        (ValueError, "nonempty", lambda: visionhope_causal_conv(x[:, :0], weight)),
        (ValueError, "taps", lambda: visionhope_causal_conv(x, weight[:, :1])),
        (ValueError, "taps", lambda: visionhope_causal_conv(x, torch.zeros(8, 9, device=device))),
        (ValueError, "weight must", lambda: visionhope_causal_conv(x, weight[0])),
        (ValueError, "weight must have shape", lambda: visionhope_causal_conv(x, weight[:7])),
        (ValueError, "bias", lambda: visionhope_causal_conv(x, weight, bias[:3])),
        (ValueError, "on cuda", lambda: visionhope_causal_conv(x, weight.cpu())),
        (ValueError, "state", lambda: visionhope_causal_conv(x, weight, state=state[:, :2])),
        (TypeError, "state", lambda: visionhope_causal_conv(x, weight, state=state.half())),
        (ValueError, "lengths", lambda: visionhope_causal_conv(x, weight, lengths=torch.ones(3, dtype=torch.int32, device=device))),
        (TypeError, "lengths", lambda: visionhope_causal_conv(x, weight, lengths=torch.ones(2, device=device))),
        (ValueError, "lengths", lambda: visionhope_causal_conv(x, weight, lengths=torch.ones(2, dtype=torch.int32))),
        (ValueError, "contiguous", lambda: visionhope_causal_conv_step(x[:, 0], state.transpose(0, 1).contiguous().transpose(0, 1), weight)),
        (RuntimeError, "inference", lambda: visionhope_causal_conv_step(x[:, 0], state, weight.clone().requires_grad_())),
    ]
    for error, match, call in bad:
        with pytest.raises(error, match=match):
            call()
    leaf = x.clone().requires_grad_()
    grad, = torch.autograd.grad(visionhope_causal_conv(leaf, weight).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_forward_mode_is_refused_and_saved_tensors_may_change_strides(device):
    from torch.autograd import forward_ad

    from visionhope_amd.utils.causal_conv import visionhope_causal_conv

    leaves = [t.to(device).requires_grad_() for t in _inputs(2, 30, 8, 4, torch.float32, seed=95)]
    dy = randn(2, 30, 8, seed=96).to(device)

    def call(x, weight, bias, state):
        return visionhope_causal_conv(x, weight, bias, silu=True, state=state)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            with pytest.raises(NotImplementedError):
                call(forward_ad.make_dual(leaves[0].detach(), torch.ones_like(leaves[0])), *leaves[1:])
    want = torch.autograd.grad(call(*leaves), leaves, dy)

    def spread(t):   # the same values, every other element of a wider tensor
        wide = torch.zeros(*t.shape, 2, device=t.device, dtype=t.dtype)
        wide[..., 0] = t
        return wide[..., 0]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread):
        got = torch.autograd.grad(call(*leaves), leaves, dy)
    for a, b in zip(got, want):
        assert torch.equal(a, b)

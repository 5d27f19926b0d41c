"""Linear attention where lines are cut into several segments of several chunks each, as large calls are:
outputs, states and gradients of single heads against the float64 oracle."""

import pytest
import torch

from oracle.oracle_torch import linear_attention_torch
from tests.helpers import randn
from tests.token_lines import DTYPES, compare, gradients, tolerance

pytestmark = pytest.mark.gpu

SHAPES = [(32, 785, 3, 64, 64), (8, 785, 8, 128, 128), (16, 1500, 6, 32, 32), (12, 1600, 8, 24, 64)]


def _segment(shape, dtype):
    """Tokens of a segment and of a chunk; asserts that there are several of both."""
    from visionhope_amd.utils import hip

    batch, length, heads, key_dim, value_dim = shape
    padded = next(d for d in (32, 64, 128) if max(key_dim, value_dim) <= d)
    nbytes = hip.load_library().vh_linear_attention_workspace_bytes(*shape, hip.dtype_code(dtype))
    segments = nbytes // (batch * heads * padded * padded * 4) + 1
    chunk = 64 if dtype == torch.bfloat16 else 32
    chunks = -(-length // chunk)
    each = -(-chunks // segments)
    assert segments > 1 and each > 1, (segments, each)
    assert -(-chunks // each) == segments
    return each * chunk, chunk


def _run(device, shape, dtype, lengths, states, fill):
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention

    batch, length, heads, key_dim, value_dim = shape
    rungs = 2 + 8 * torch.arange(heads) / (heads - 1)   # states that outlive a segment
    log_decay = torch.log1p(-torch.exp2(-rungs))
    lines = [randn(batch, length, heads, d, seed=seed).to(dtype)
             for seed, d in ((1, key_dim), (2, key_dim), (3, value_dim), (4, value_dim))]
    state, dstate = (randn(batch, heads, key_dim, value_dim, seed=seed) if states else None for seed in (5, 6))
    given = [t.clone() for t in lines]
    if lengths is not None:
        for t in given:
            for b, n in enumerate(lengths):
                t[b, n:] = fill
    leaves = [t.to(device).requires_grad_() for t in given[:3]]
    start = None if state is None else state.to(device).requires_grad_()
    o, last = visionhope_linear_attention(*leaves, log_decay.to(device), state=start, return_state=True,
                                          lengths=None if lengths is None else torch.tensor(lengths, device=device))
    outs, cotangents = [o], [given[3].to(device)]
    if states:
        outs.append(last)
        cotangents.append(dstate.to(device))
    wanted = leaves + ([start] if states else [])
    grads = torch.autograd.grad(outs, wanted, cotangents)
    return (*lines, log_decay, state, dstate), o.detach().cpu(), last.detach().cpu(), [g.cpu() for g in grads]


def _compare(device, shape, dtype, lengths, states, batches, head, fill=0.0):
    """Compares one head of some sequences."""
    (q, k, v, do, log_decay, state, dstate), o, last, grads = _run(device, shape, dtype, lengths, states, fill)
    length, key_dim, value_dim = shape[1], *shape[3:]

    def lines(t):
        return t[batches][:, :, head:head + 1]

    def of_states(t):
        return None if t is None else t[batches][:, head:head + 1]

    ends = None if lengths is None else torch.tensor(lengths)[batches]
    decay = log_decay[head:head + 1].double()
    want, wanted = gradients(lambda q, k, v, s: linear_attention_torch(q, k, v, decay, None, s, ends),
                             [*(lines(t) for t in (q, k, v)), of_states(state)], (lines(do), of_states(dstate)))
    terms = length + max(key_dim, value_dim)
    for i, b in enumerate(batches):
        what = f"{shape} {dtype} sequence {b} of {'all' if lengths is None else lengths[b]} head {head}"
        compare(lines(o)[i], want[0][i], tolerance(dtype, terms), f"{what} o")
        compare(of_states(last)[i], want[1][i], tolerance(torch.float32, length), f"{what} state")
        for name, grad, other in zip(("dq", "dk", "dv"), grads, wanted):
            compare(lines(grad)[i], other[i], tolerance(dtype, terms), f"{what} {name}")
        if states:
            compare(of_states(grads[3])[i], wanted[3][i], tolerance(torch.float32, terms), f"{what} dstate")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_whole_lines(device, dtype, states, shape):
    _segment(shape, dtype)
    batch, heads = shape[0], shape[2]
    _compare(device, shape, dtype, None, states, [0, batch // 2, batch - 1], heads - 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_lines_that_end_before_inside_and_at_segments(device, dtype, states, shape):
    segment, chunk = _segment(shape, dtype)
    length, heads = shape[1], shape[2]
    ends = [segment, segment + 1, segment - 1, 2 * segment - chunk, segment + chunk + 5, length - 1, 0, 1]
    lengths = [min(length, ends[b % len(ends)]) for b in range(shape[0])]
    _compare(device, shape, dtype, lengths, states, list(range(len(ends))), heads // 2, fill=float("nan"))

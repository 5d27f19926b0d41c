"""The selective state space scan on the GPU where it can go wrong beside the ordinary sizes:
state counts that leave lanes of a channel without a state, and what stands around its buffers."""

import pytest
import torch

from oracle.oracle_torch import state_space_scan_torch
from tests.helpers import randn
from tests.test_gpu_state_space import NAMES, _inputs
from tests.token_lines import DTYPES, compare, gradients, half_step, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("states", [1, 3, 4, 6, 8, 12, 13, 16, 20, 24, 28, 30, 32])
def test_step_writes_its_own_states_only(device, dtype, in_place, states):
    """Every state count, with the states inside a wider buffer whose rest keeps its values: a
    channel's lanes behind its last state (12, 20, 24 and 28 states) have no part."""
    from visionhope_amd.utils.state_space import visionhope_state_space_step

    batch, channels, guard = 3, 10, 64
    t = {k: v.to(device) for k, v in _inputs(batch, 1, channels, states, 2, dtype, seed=200).items()}
    count = batch * channels * states

    def guarded():
        buffer = torch.full((guard + count + guard,), 7.0, device=device)
        return buffer, buffer[guard:guard + count].view(batch, channels, states)

    buffer, state = guarded()
    state.copy_(t["state"])
    other, new_state = guarded()
    y = visionhope_state_space_step(
        t["x"][:, 0], t["dt"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0], state, t["D"], gate=t["gate"][:, 0],
        dt_bias=t["dt_bias"], new_state=None if in_place else new_state)
    args = {k: v.double().cpu() for k, v in t.items()}
    want, last = state_space_scan_torch(*(args[n] for n in ("x", "dt", "A", "B", "C", "D", "gate", "dt_bias")),
                                        True, args["state"])
    compare(y, want[:, 0], tolerance(dtype, 1), "y")
    compare(state if in_place else new_state, last, tolerance(torch.float32, 1), "state")
    for b in (buffer, other):
        assert (b[:guard] == 7.0).all() and (b[guard + count:] == 7.0).all()
    if not in_place:
        assert torch.equal(state, t["state"])


@pytest.mark.parametrize("states", [12, 20, 24, 28])
def test_tokens_one_by_one_continue_a_prompt(device, states):
    from visionhope_amd.utils.state_space import visionhope_state_space_scan, visionhope_state_space_step

    t = {k: v.to(device) for k, v in _inputs(5, 9, 33, states, 3, torch.bfloat16, seed=210).items()}

    def operands(rows):
        return ([t[n][:, rows] for n in ("x", "dt")] + [t["A"]] + [t[n][:, rows] for n in ("B", "C")],
                dict(gate=t["gate"][:, rows], dt_bias=t["dt_bias"]))

    args, kw = operands(slice(None))
    whole, last = visionhope_state_space_scan(*args, t["D"], state=t["state"], return_state=True, **kw)
    state, rows = t["state"].clone(), []
    for i in range(9):
        args, kw = operands(i)
        rows.append(visionhope_state_space_step(*args, state, t["D"], **kw))
    tol = tolerance(torch.float32, 9)
    compare(state, last.double().cpu(), tol, "state")
    compare(torch.stack(rows, 1), whole.double().cpu(), tol + 2 * half_step(torch.bfloat16), "steps")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 40, 24, 16, 1), (3, 300, 70, 16, 1), (2, 2100, 33, 6, 3), (5, 150, 64, 32, 2)])
def test_rates_of_minus_infinity(device, dtype, shape):
    """A state whose rate is -inf (an exponential that overflowed) forgets at every token, as one of
    rate -1e30 does: whole lines, lines in chunks, sequences that end early, outputs and gradients.
    (The oracle takes -1e30, since 0 x inf of its masked tokens has no value.)"""
    from visionhope_amd.utils.state_space import visionhope_state_space_scan

    batch, length, channels = shape[:3]
    inputs = _inputs(*shape, dtype, seed=220)
    lengths = torch.tensor([length, length // 3, 0, 1, length - 1][:batch])
    dy, dstate = randn(*inputs["x"].shape, seed=221).to(dtype), randn(*inputs["state"].shape, seed=222)
    rates = inputs["A"].clone()
    inputs["A"][::2, 1] = inputs["A"][::4, 2] = -1e30
    rates[::2, 1] = -torch.inf
    rates[::4, 2] = -3e38   # finite, but not as a power of two's exponent
    want, grads = gradients(lambda *a: state_space_scan_torch(*a[:8], True, a[8], lengths),
                            [inputs[n] for n in NAMES], (dy, dstate))
    leaves = [t.to(device).requires_grad_() for t in (rates if n == "A" else inputs[n] for n in NAMES)]
    x, dt, A, B, C, D, gate, dt_bias, state = leaves
    y, last = visionhope_state_space_scan(x, dt, A, B, C, D, gate=gate, dt_bias=dt_bias, state=state,
                                          lengths=lengths.to(device), return_state=True)
    compare(y, want[0], tolerance(dtype, length), "y")
    compare(last, want[1], tolerance(torch.float32, length), "state")
    torch.autograd.backward((y, last), (dy.to(device), dstate.to(device)))
    for name, leaf, grad in zip(NAMES, leaves, grads):
        terms = batch * length if name in ("A", "D", "dt_bias") else length + channels
        compare(leaf.grad, grad, tolerance(leaf.dtype, terms), f"d{name}")


def test_step_with_rates_of_minus_infinity(device):
    """Also where a step is zero: such a token leaves every state as it is."""
    from visionhope_amd.utils.state_space import visionhope_state_space_step

    t = {k: v.to(device) for k, v in _inputs(2, 1, 24, 16, 1, torch.float32, seed=230).items()}
    t["dt"][:, :, ::3] = -200.0
    results = []
    for rate in (-1e30, -torch.inf):
        t["A"][::2, 1] = rate
        state = t["state"].clone()
        y = visionhope_state_space_step(t["x"][:, 0], t["dt"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0], state, t["D"])
        results.append((y, state))
    for a, b in zip(*results):
        assert torch.isfinite(a).all() and torch.equal(a, b)

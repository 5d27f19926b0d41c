"""The selective state space scan on the GPU against the float64 oracle: prompts, gradients,
single tokens, states, lengths, groups, strides, streams and graphs."""

import pytest
import torch

from oracle.oracle_torch import state_space_scan_torch
from tests.helpers import randn
from tests.token_lines import DTYPES, compare, gradients, half_step, tolerance

pytestmark = pytest.mark.gpu

NAMES = ("x", "dt", "A", "B", "C", "D", "gate", "dt_bias", "state")


def _inputs(batch, length, channels, states, groups, dtype, seed=0):
    """Rates 0.2 .. S of both slow and fast states, steps about 0.02 .. 1."""
    lead = (batch, length)
    rates = torch.arange(1, states + 1).float().expand(channels, states)
    return dict(
        x=randn(*lead, channels, seed=seed + 1).to(dtype), dt=(randn(*lead, channels, seed=seed + 2)).to(dtype),
        A=-rates * torch.exp(0.5 * randn(channels, states, seed=seed + 3)),
        B=randn(*lead, groups, states, seed=seed + 4).to(dtype), C=randn(*lead, groups, states, seed=seed + 5).to(dtype),
        D=randn(channels, seed=seed + 6), gate=randn(*lead, channels, seed=seed + 7).to(dtype),
        dt_bias=randn(channels, seed=seed + 8) - 2, state=randn(batch, channels, states, seed=seed + 9))


def _oracle(softplus, lengths):
    def run(x, dt, A, B, C, D, gate, dt_bias, state):
        return state_space_scan_torch(x, dt, A, B, C, D, gate, dt_bias, softplus, state, lengths)
    return run


def _own(leaves, softplus, lengths):
    from visionhope_amd.utils.state_space import visionhope_state_space_scan

    x, dt, A, B, C, D, gate, dt_bias, state = leaves
    return visionhope_state_space_scan(x, dt, A, B, C, D, gate=gate, dt_bias=dt_bias, softplus=softplus, state=state,
                                       lengths=lengths, return_state=True)


def _check(device, inputs, what, softplus=True, lengths=None, with_state_grad=True):
    tensors = [inputs.get(name) for name in NAMES]
    x, A = tensors[0], tensors[2]
    dtype = x.dtype
    dy = randn(*x.shape, seed=91).to(dtype)
    dstate = randn(x.shape[0], *A.shape, seed=92) if with_state_grad else None
    want, grads = gradients(_oracle(softplus, lengths), tensors, (dy, dstate))
    leaves = [None if t is None else t.to(device).requires_grad_() for t in tensors]
    y, state = _own(leaves, softplus, None if lengths is None else lengths.to(device))
    assert y.dtype == dtype and state.dtype == torch.float32
    rows = x.shape[0] * x.shape[1]
    compare(y, want[0], tolerance(dtype, x.shape[1]), f"{what} y")
    compare(state, want[1], tolerance(torch.float32, x.shape[1]), f"{what} state")
    outs, cot = ((y, state), (dy.to(device), dstate.to(device))) if with_state_grad else ((y,), (dy.to(device),))
    torch.autograd.backward(outs, cot)
    for name, leaf, grad in zip(NAMES, leaves, grads):
        if leaf is None:
            continue
        terms = rows if name in ("A", "D", "dt_bias") else x.shape[1] + x.shape[2]
        assert leaf.grad.dtype == leaf.dtype
        compare(leaf.grad, grad, tolerance(leaf.dtype, terms), f"{what} d{name}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (2, 2, 3, 4, 1), (1, 33, 64, 16, 1), (2, 65, 70, 16, 1),
                                   (3, 40, 24, 8, 2), (1, 130, 96, 6, 3), (2, 50, 130, 32, 1), (1, 31, 20, 20, 4),
                                   (1, 700, 40, 16, 1), (2, 97, 6, 3, 6)])
def test_prompt_and_gradients(device, dtype, shape):
    _check(device, _inputs(*shape, dtype), f"{shape} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("missing", [("D", "gate", "dt_bias", "state"), ("gate",), ("D",), ("dt_bias", "state")])
def test_optional_operands(device, dtype, missing):
    inputs = _inputs(2, 70, 72, 16, 1, dtype, seed=20)
    for name in missing:
        inputs[name] = None
    _check(device, inputs, f"without {missing}", with_state_grad=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_given_steps(device, dtype):
    """softplus=False: dt + dt_bias is the step itself (positive here)."""
    inputs = _inputs(2, 45, 40, 16, 1, dtype, seed=30)
    inputs["dt"] = (inputs["dt"].float().abs() * 0.1 + 0.01).to(dtype)
    inputs["dt_bias"] = inputs["dt_bias"].abs() * 0.1
    _check(device, inputs, "given steps", softplus=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("states", [16, 5, 32])
def test_lengths(device, dtype, states):
    inputs = _inputs(7, 150, 72, states, 2, dtype, seed=40)
    lengths = torch.tensor([150, 0, 1, 2, 96, 97, 31])
    _check(device, inputs, f"lengths {states}", lengths=lengths)


def test_what_stands_behind_the_end_has_no_part(device):
    inputs = _inputs(3, 140, 64, 16, 1, torch.bfloat16, seed=50)
    lengths = torch.tensor([33, 0, 140], dtype=torch.int32, device=device)
    dy = randn(3, 140, 64, seed=51).to(device, torch.bfloat16)
    results = []
    for fill in (0.0, float("nan"), float("inf")):
        leaves = []
        for name in NAMES:
            t = inputs[name].to(device)
            if name in ("x", "dt", "B", "C", "gate"):
                for i, n in enumerate(lengths.tolist()):
                    t[i, n:] = fill
            leaves.append(t.clone().requires_grad_())
        dyf = dy.clone()
        for i, n in enumerate(lengths.tolist()):
            dyf[i, n:] = fill
        y, state = _own(leaves, True, lengths)
        results.append([y, state, *torch.autograd.grad(y, leaves, dyf)])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_slices_and_odd_addresses(device, dtype):
    inputs = {k: v.to(device) for k, v in _inputs(2, 75, 48, 16, 2, dtype, seed=60).items()}
    dy = randn(2, 75, 48, seed=61).to(device, dtype)

    def both(view):
        leaves = [(view(inputs[n]) if inputs[n].ndim >= 3 and n != "state" else inputs[n]).detach().requires_grad_()
                  for n in NAMES]
        y, state = _own(leaves, True, None)
        return [y.detach(), state.detach(), *torch.autograd.grad(y, leaves, view(dy))]

    def wide(t):
        w = torch.zeros(*t.shape[:2], 3, *t.shape[2:], device=device, dtype=t.dtype)
        w[:, :, 1] = t
        return w[:, :, 1]

    def odd(t):
        return torch.empty(t.numel() + 1, device=device, dtype=t.dtype)[1:].view(t.shape).copy_(t)

    def turned(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    def last_first(t):
        return t.transpose(1, -1).contiguous().transpose(1, -1)

    want = both(lambda t: t)
    for view in (wide, odd, turned, last_first):
        for name, a, b in zip(("y", "state", *NAMES), both(view), want):
            assert torch.equal(a, b), (view.__name__, name)


def test_shared_maps_and_broadcast_inputs(device):
    """B and C without a group axis equal one group; a step shared by all channels and a map
    shared by all sequences (stride 0) get the sum of the gradients."""
    from visionhope_amd.utils.state_space import visionhope_state_space_scan

    t = {k: v.to(device) for k, v in _inputs(3, 40, 24, 16, 1, torch.float32, seed=70).items()}
    flat = visionhope_state_space_scan(t["x"], t["dt"], t["A"], t["B"][:, :, 0], t["C"][:, :, 0], t["D"])
    assert torch.equal(flat, visionhope_state_space_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], t["D"]))
    step, shared = t["dt"][..., :1].clone().requires_grad_(), t["B"][:1, :, 0].clone().requires_grad_()
    y = visionhope_state_space_scan(t["x"], step.expand(3, 40, 24), t["A"], shared.expand(3, 40, 16), t["C"][:, :, 0])
    y.sum().backward()
    full = [step.detach().expand(3, 40, 24).contiguous().requires_grad_(),
            shared.detach().expand(3, 40, 16).contiguous().requires_grad_()]
    y2 = visionhope_state_space_scan(t["x"], full[0], t["A"], full[1], t["C"][:, :, 0])
    assert torch.equal(y, y2)
    y2.sum().backward()
    compare(step.grad, full[0].grad.sum(-1, keepdim=True).double().cpu(), tolerance(torch.float32, 24), "shared step")
    compare(shared.grad, full[1].grad.sum(0, keepdim=True).double().cpu(), tolerance(torch.float32, 3), "shared map")


def test_rows_past_32_bits(device):
    """A batch stride of 2^31 elements (4 GiB apart)."""
    from visionhope_amd.utils.state_space import visionhope_state_space_scan

    t = {k: v.to(device) for k, v in _inputs(2, 40, 32, 16, 1, torch.bfloat16, seed=75).items()}
    base = torch.empty(2**31 + 40 * 32, device=device, dtype=torch.bfloat16)
    far = base.as_strided((2, 40, 32), (2**31, 32, 1))
    far.copy_(t["x"])
    args = (t["dt"], t["A"], t["B"], t["C"])
    assert torch.equal(visionhope_state_space_scan(far, *args), visionhope_state_space_scan(t["x"], *args))


@pytest.mark.parametrize("shape", [(2, 3000, 64, 16, 1), (1, 5000, 200, 8, 2)])
def test_long_lines_match_their_pieces(device, shape):
    """A line that is cut into chunks against the same line in pieces that continue each other."""
    t = {k: v.to(device) for k, v in _inputs(*shape, torch.float32, seed=80).items()}
    leaves = [t[n] for n in NAMES]
    y, state = _own(leaves, True, None)
    rows, s, at = [], t["state"], 0
    for n in (1, 7, 500, 32, 64, shape[1] - 604):
        piece = [v[:, at:at + n] if name not in ("A", "D", "dt_bias", "state") else v for name, v in zip(NAMES, leaves)]
        piece[-1] = s
        out, s = _own(piece, True, None)
        rows.append(out)
        at += n
    tol = 2 * tolerance(torch.float32, shape[1])
    compare(torch.cat(rows, 1), y.double().cpu(), tol, "pieces")
    compare(s, state.double().cpu(), tol, "pieces' state")


def test_extreme_steps(device):
    """Steps of 0 (dt far below), steps of 90 (all state forgotten), rates of 0 (nothing
    forgotten) and of -1e30, and growing states (A > 0) that stay in range."""
    inputs = _inputs(1, 70, 64, 16, 1, torch.float32, seed=85)
    inputs["dt"][:, 10:20] = -120.0
    inputs["dt"][:, 30:33] = 90.0
    inputs["A"][:, 0] = 0.0
    inputs["A"][:, 1] = -1e30
    inputs["A"][:, 2] = 1e-3
    inputs["dt_bias"] = None
    _check(device, inputs, "extreme steps")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (3, 70, 16, 2), (64, 96, 8, 1), (5, 33, 3, 3), (2, 40, 32, 4),
                                   (2, 10, 13, 1)])
def test_tokens_one_by_one_continue_a_prompt(device, dtype, shape):
    from visionhope_amd.utils.state_space import visionhope_state_space_step

    batch, channels, states, groups = shape
    t = {k: v.to(device) for k, v in _inputs(batch, 12, channels, states, groups, dtype, seed=100).items()}
    whole, last = _own([t[n] for n in NAMES], True, None)
    head = [t[n][:, :5] if n not in ("A", "D", "dt_bias", "state") else t[n] for n in NAMES]
    y, state = _own(head, True, None)
    rows = [y]
    for i in range(5, 12):
        args = (t["x"][:, i], t["dt"][:, i], t["A"], t["B"][:, i], t["C"][:, i])
        kw = dict(gate=t["gate"][:, i], dt_bias=t["dt_bias"])
        if i % 2:
            rows.append(visionhope_state_space_step(*args, state, t["D"], **kw)[:, None])
        else:
            before, after = state.clone(), torch.empty_like(state)
            rows.append(visionhope_state_space_step(*args, state, t["D"], new_state=after, **kw)[:, None])
            assert torch.equal(state, before)
            state = after
    tol = tolerance(torch.float32, 12)
    compare(state, last.double().cpu(), tol, "steps' state")
    compare(torch.cat(rows, 1), whole.double().cpu(), tol + (2 * half_step(dtype) if dtype != torch.float32 else 0),
            "steps")
    # without the optional operands
    y = visionhope_state_space_step(t["x"][:, 0], t["dt"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0], t["state"].clone())
    want, _ = state_space_scan_torch(*(t[n].double().cpu() if n in ("A",) else t[n][:, :1].double().cpu()
                                       for n in ("x", "dt", "A", "B", "C")), state=t["state"].double().cpu())
    compare(y, want[:, 0], tolerance(dtype, 1), "bare step")


def test_repeats_bit_by_bit_on_any_stream_and_in_a_graph(device):
    from visionhope_amd.utils.state_space import visionhope_state_space_step

    t = {k: v.to(device) for k, v in _inputs(2, 300, 96, 16, 1, torch.bfloat16, seed=110).items()}
    dy = randn(2, 300, 96, seed=111).to(device, torch.bfloat16)
    leaves = [t[n].clone().requires_grad_() for n in NAMES]

    def step():
        y, state = _own(leaves, True, None)
        return [y.detach(), state.detach(), *torch.autograd.grad(y, leaves, dy)]

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
    graph_b = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph_b):
        captured_b = step()
    live = t["state"].clone()
    tokens = [t[n][:, 0].contiguous() for n in ("x", "dt", "B", "C", "gate")]
    graph_step = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph_step):
        out = visionhope_state_space_step(*tokens[:2], t["A"], *tokens[2:4], live, t["D"], gate=tokens[4])
    for round_ in range(3):
        with torch.no_grad():
            leaves[0].copy_(t["x"] * (round_ + 1))
        want = step()
        for c in captured + captured_b:
            c.zero_()
        graph.replay()
        graph_b.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(want, captured, captured_b):
            assert torch.equal(a, b) and torch.equal(a, c), f"replay {round_}"
        eager = live.clone()
        want_out = visionhope_state_space_step(*tokens[:2], t["A"], *tokens[2:4], eager, t["D"], gate=tokens[4])
        graph_step.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want_out) and torch.equal(live, eager)


def test_gradients_only_where_asked(device):
    from visionhope_amd.utils.state_space import visionhope_state_space_scan

    t = {k: v.to(device) for k, v in _inputs(2, 20, 24, 16, 1, torch.float32, seed=120).items()}
    A = t["A"].clone().requires_grad_()
    y = visionhope_state_space_scan(t["x"], t["dt"], A, t["B"], t["C"])
    y.sum().backward()
    assert A.grad.shape == A.shape
    x = t["x"].clone().requires_grad_()
    _, state = visionhope_state_space_scan(x, t["dt"], t["A"], t["B"], t["C"], return_state=True)
    grad, = torch.autograd.grad(state.sum(), x)
    assert grad.abs().sum() > 0
    half = t["A"].to(torch.bfloat16).requires_grad_()
    visionhope_state_space_scan(t["x"], t["dt"], half, t["B"], t["C"]).sum().backward()
    assert half.grad.dtype == torch.bfloat16


def test_step_marks_the_state_as_changed(device):
    from visionhope_amd.utils.state_space import visionhope_state_space_step

    t = {k: v.to(device) for k, v in _inputs(2, 3, 24, 5, 1, torch.float32, seed=125).items()}
    before = t["state"]._version
    visionhope_state_space_step(t["x"][:, 0], t["dt"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0], t["state"])
    assert t["state"]._version == before + 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_streams_at_once(device, dtype):
    """Two training steps that overlap on two streams give what they give alone."""
    runs = []
    for seed in (150, 160):
        inputs = _inputs(2, 600, 96, 16, 1, dtype, seed=seed)
        leaves = [inputs[n].to(device).requires_grad_() for n in NAMES]
        dy = randn(2, 600, 96, seed=seed + 10).to(device, dtype)

        def step(leaves=leaves, dy=dy):
            y, state = _own(leaves, True, None)
            return [y.detach(), state.detach(), *torch.autograd.grad(y, leaves, dy)]

        runs.append((step, step(), torch.cuda.Stream(device)))
    torch.cuda.synchronize()
    results = []
    for _ in range(4):
        for step, _, stream in runs:
            with torch.cuda.stream(stream):
                results.append(step())
    torch.cuda.synchronize()
    for i, got in enumerate(results):
        for a, b in zip(got, runs[i % 2][1]):
            assert torch.equal(a, b)


def test_refusals(device):
    from visionhope_amd.utils.state_space import visionhope_state_space_scan, visionhope_state_space_step

    t = {k: v.to(device) for k, v in _inputs(2, 9, 24, 16, 2, torch.float32, seed=130).items()}

    def scan(**kw):
        a = {**t, **kw}
        return visionhope_state_space_scan(a["x"], a["dt"], a["A"], a["B"], a["C"], a["D"], gate=a["gate"],
                                           dt_bias=a["dt_bias"], state=a["state"], lengths=a.get("lengths"))

    bad = [
        (ValueError, "CUDA", dict(x=t["x"].cpu())), (TypeError, "FP16, BF16 and FP32", dict(x=t["x"].double())),
        (ValueError, "3 dimensions", dict(x=t["x"][0])), (ValueError, "nonempty", dict(x=t["x"][:, :0])),
        (ValueError, "dt", dict(dt=t["dt"][:, :4])), (TypeError, "dt", dict(dt=t["dt"].half())),
        (ValueError, "A must", dict(A=t["A"][0])), (ValueError, "states", dict(A=torch.zeros(24, 33, device=device))),
        (ValueError, "A must have", dict(A=t["A"][:20])), (ValueError, "B must", dict(B=t["B"][0, 0])),
        (ValueError, "B must", dict(B=t["B"][..., :8])), (ValueError, "C must", dict(C=t["C"][:, :, 0])),
        (ValueError, "groups", dict(B=torch.zeros(2, 9, 5, 16, device=device))),
        (TypeError, "B must", dict(B=t["B"].half())), (ValueError, "D must", dict(D=t["D"][:2])),
        (ValueError, "gate", dict(gate=t["gate"][:1])), (ValueError, "dt_bias", dict(dt_bias=t["dt_bias"].cpu())),
        (ValueError, "state", dict(state=t["state"][:1])), (TypeError, "state", dict(state=t["state"].half())),
        (TypeError, "lengths", dict(lengths=torch.ones(2, device=device))),
    ]
    for error, match, kw in bad:
        with pytest.raises(error, match=match):
            scan(**kw)
    tokens = (t["x"][:, 0], t["dt"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0])
    with pytest.raises(RuntimeError, match="inference"):
        visionhope_state_space_step(*tokens[:2], t["A"].clone().requires_grad_(), *tokens[3:], t["state"])
    with pytest.raises(ValueError, match="contiguous"):
        visionhope_state_space_step(*tokens, t["state"].transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(TypeError, match="state"):
        visionhope_state_space_step(*tokens, t["state"].half())


def test_forward_mode_is_refused_and_saved_tensors_may_change_strides(device):
    from torch.autograd import forward_ad

    inputs = _inputs(2, 40, 24, 16, 2, torch.float32, seed=140)
    leaves = [inputs[n].to(device).requires_grad_() for n in NAMES]
    dy = randn(2, 40, 24, seed=141).to(device)

    def call(*tensors):
        return _own(tensors, True, None)[0]
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

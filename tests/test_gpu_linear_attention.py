"""Linear attention with a decay for each head on the GPU against the float64 oracle: prompts,
gradients, single tokens, states, lengths, strides, shared heads, streams and graphs."""

import pytest
import torch

from oracle.oracle_torch import linear_attention_torch
from tests.helpers import randn
from tests.token_lines import DTYPES, compare, gradients, half_step, tolerance

pytestmark = pytest.mark.gpu

NAMES = ("q", "k", "v", "log_decay", "state")


def _inputs(batch, length, heads, key_dim, value_dim, dtype, seed=0):
    """Decays from a half a token to one part in 500."""
    rungs = 1 + 8 * torch.arange(heads) / max(1, heads - 1)
    return dict(
        q=randn(batch, length, heads, key_dim, seed=seed + 1).to(dtype),
        k=randn(batch, length, heads, key_dim, seed=seed + 2).to(dtype),
        v=randn(batch, length, heads, value_dim, seed=seed + 3).to(dtype),
        log_decay=torch.log1p(-torch.exp2(-rungs)), state=randn(batch, heads, key_dim, value_dim, seed=seed + 4))


def _own(leaves, lengths, scale=None):
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention

    q, k, v, log_decay, state = leaves
    return visionhope_linear_attention(q, k, v, log_decay, scale=scale, state=state, lengths=lengths, return_state=True)


def _check(device, inputs, what, lengths=None, with_state_grad=True, scale=None, learned=True):
    tensors = [inputs.get(name) for name in NAMES]
    q, v = tensors[0], tensors[2]
    dtype, (batch, length, heads, key_dim) = q.dtype, q.shape
    do = randn(*v.shape, seed=91).to(dtype)
    dstate = randn(batch, heads, key_dim, v.shape[-1], seed=92) if with_state_grad else None
    want, grads = gradients(lambda *a: linear_attention_torch(*a[:4], scale, a[4], lengths), tensors, (do, dstate))
    leaves = [None if t is None else t.to(device).requires_grad_(learned or name != "log_decay")
              for name, t in zip(NAMES, tensors)]
    o, state = _own(leaves, None if lengths is None else lengths.to(device), scale)
    assert o.dtype == dtype and state.dtype == torch.float32 and o.is_contiguous()
    terms = length + max(key_dim, v.shape[-1])
    compare(o, want[0], tolerance(dtype, terms), f"{what} o")
    compare(state, want[1], tolerance(torch.float32, length), f"{what} state")
    outs, cot = ((o, state), (do.to(device), dstate.to(device))) if with_state_grad else ((o,), (do.to(device),))
    torch.autograd.backward(outs, cot)
    for name, leaf, grad in zip(NAMES, leaves, grads):
        if leaf is None or not leaf.requires_grad:
            continue
        assert leaf.grad.dtype == leaf.dtype
        # a decay's gradient adds a product of two sums for every pair of tokens up to 64 apart
        many = batch * length * (64 + terms) if name == "log_decay" else terms
        compare(leaf.grad, grad, tolerance(leaf.dtype, many), f"{what} d{name}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (2, 2, 3, 4, 5), (1, 31, 2, 16, 16), (2, 64, 2, 32, 32),
                                   (1, 65, 3, 20, 33), (2, 129, 2, 64, 64), (1, 200, 1, 7, 128), (2, 97, 2, 128, 24),
                                   (1, 70, 2, 128, 128), (3, 33, 1, 65, 3), (1, 500, 2, 48, 64)])
def test_prompt_and_gradients(device, dtype, shape):
    _check(device, _inputs(*shape, dtype), f"{shape} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dims", [(16, 16), (64, 48), (128, 128)])
def test_fixed_decays_without_states(device, dtype, dims):
    inputs = _inputs(2, 300, 2, *dims, dtype, seed=20)
    inputs["state"] = None
    _check(device, inputs, f"fixed {dims}", with_state_grad=False, learned=False, scale=0.3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("learned", [True, False])
def test_lengths(device, dtype, learned):
    inputs = _inputs(8, 150, 2, 40, 24, dtype, seed=40)
    lengths = torch.tensor([150, 0, 1, 2, 64, 65, 128, 31])
    _check(device, inputs, f"lengths {learned}", lengths=lengths, learned=learned)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_out_of_range_are_clamped(device, dtype):
    inputs = {k: v.to(device) for k, v in _inputs(3, 20, 1, 8, 8, dtype, seed=45).items()}
    tensors = [inputs[name] for name in NAMES]
    want = _own(tensors, torch.tensor([20, 0, 7], device=device))
    for lengths in (torch.tensor([2 ** 40, -5, 7], device=device), torch.tensor([21, -1, 7], device=device, dtype=torch.int32)):
        for a, b in zip(_own(tensors, lengths), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rate", [0.0, -1e-4, -3.0, -40.0, -3e38, float("-inf")])
def test_decays_from_none_to_all(device, rate):
    inputs = _inputs(1, 260, 2, 24, 24, torch.float32, seed=47)
    inputs["log_decay"] = torch.tensor([rate, -0.1])
    if rate < -1e5:   # the oracle's exp(rate) is zero, and so is its gradient
        _check(device, inputs, f"decay {rate}", learned=False)
    else:
        _check(device, inputs, f"decay {rate}")


def test_what_stands_behind_the_end_has_no_part(device):
    inputs = _inputs(3, 140, 2, 64, 32, torch.bfloat16, seed=50)
    lengths = torch.tensor([33, 0, 140], dtype=torch.int32, device=device)
    do = randn(3, 140, 2, 32, seed=51).to(device, torch.bfloat16)
    results = []
    for fill in (0.0, float("nan"), float("inf")):
        leaves = []
        for name in NAMES:
            t = inputs[name].to(device)
            if name in ("q", "k", "v"):
                for i, n in enumerate(lengths.tolist()):
                    t[i, n:] = fill
            leaves.append(t.clone().requires_grad_())
        filled = do.clone()
        for i, n in enumerate(lengths.tolist()):
            filled[i, n:] = fill
        o, state = _own(leaves, lengths)
        results.append([o, state, *torch.autograd.grad(o, leaves, filled)])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_slices_and_odd_addresses(device, dtype):
    inputs = {k: v.to(device) for k, v in _inputs(2, 75, 3, 32, 16, dtype, seed=60).items()}
    do = randn(2, 75, 3, 16, seed=61).to(device, dtype)

    def both(view):
        leaves = [(view(inputs[n]) if n in ("q", "k", "v") else inputs[n]).detach().requires_grad_() for n in NAMES]
        o, state = _own(leaves, None)
        return [o.detach(), state.detach(), *torch.autograd.grad(o, leaves, view(do))]

    def wide(t):
        w = torch.full((*t.shape[:2], 3, *t.shape[2:]), float("nan"), device=device, dtype=t.dtype)
        w[:, :, 1] = t
        return w[:, :, 1]

    def odd(t):
        return torch.empty(t.numel() + 1, device=device, dtype=t.dtype)[1:].view(t.shape).copy_(t)

    def heads_first(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def last_first(t):
        return t.transpose(1, -1).contiguous().transpose(1, -1)

    def reversed_rows(t):   # rows of an odd stride
        w = torch.zeros(*t.shape[:3], t.shape[3] + 3, device=device, dtype=t.dtype)
        w[..., 1:-2] = t
        return w[..., 1:-2]

    want = both(lambda t: t)
    for view in (wide, odd, heads_first, last_first, reversed_rows):
        for name, a, b in zip(("o", "state", *NAMES), both(view), want):
            assert torch.equal(a, b), (view.__name__, name)


@pytest.mark.parametrize("dtype", DTYPES)
def test_keys_and_values_that_heads_share(device, dtype):
    inputs = _inputs(2, 90, 4, 16, 32, dtype, seed=70)
    shared_k, shared_v = inputs["k"][:, :, :1].contiguous(), inputs["v"][:, :, :1].contiguous()
    inputs.update(k=shared_k.expand(-1, -1, 4, -1), v=shared_v.expand(-1, -1, 4, -1))
    do = randn(2, 90, 4, 32, seed=71).to(dtype)
    want, grads = gradients(lambda q, k, v, a, s: linear_attention_torch(q, k.expand(-1, -1, 4, -1), v.expand(-1, -1, 4, -1), a,
                                                                         None, s),
                            [inputs["q"], shared_k, shared_v, inputs["log_decay"], inputs["state"]], (do, None))
    q, k, v, a, s = (t.to(device).requires_grad_() for t in (inputs["q"], shared_k, shared_v, inputs["log_decay"], inputs["state"]))
    o, state = _own((q, k.expand(-1, -1, 4, -1), v.expand(-1, -1, 4, -1), a, s), None)
    compare(o, want[0], tolerance(dtype, 122), "shared o")
    compare(state, want[1], tolerance(torch.float32, 90), "shared state")
    got = torch.autograd.grad(o, (k, v), do.to(device))
    for name, a, b in zip("kv", got, grads[1:3]):
        # four rounded gradients are added in dtype: four roundings of the terms, three of the sums
        compare(a, b, tolerance(dtype, 122) + 7 * half_step(dtype), f"shared d{name}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_after_a_prompt(device, dtype):
    """A prompt, its state, a second prompt and single tokens give what one prompt gives."""
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention_step

    inputs = _inputs(3, 90, 2, 48, 40, dtype, seed=80)
    want, last = linear_attention_torch(*(inputs[n].double() for n in NAMES[:4]), None, inputs["state"].double())
    q, k, v, a, s = (inputs[n].to(device) for n in NAMES)
    o1, s = _own((q[:, :70], k[:, :70], v[:, :70], a, s), None)
    o2, s = _own((q[:, 70:81], k[:, 70:81], v[:, 70:81], a, s), None)
    outs = [o1, o2]
    for t in range(81, 90):
        if t % 2:
            moved = torch.empty_like(s)
            kept = s.clone()
            outs.append(visionhope_linear_attention_step(q[:, t], k[:, t], v[:, t], a, s, new_state=moved)[:, None])
            assert torch.equal(s, kept)
            s = moved
        else:
            outs.append(visionhope_linear_attention_step(q[:, t], k[:, t], v[:, t], a, s)[:, None])
    compare(torch.cat(outs, 1), want, tolerance(dtype, 138), "pieces")
    compare(s, last, tolerance(torch.float32, 90), "state of pieces")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (3, 2, 5, 7), (2, 3, 64, 64), (1, 2, 128, 128), (2, 1, 33, 100), (5, 4, 16, 20),
                                   (1, 1, 128, 1), (1, 1, 1, 127)])
def test_single_tokens(device, dtype, shape):
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention_step

    batch, heads, key_dim, value_dim = shape
    inputs = _inputs(batch, 1, heads, key_dim, value_dim, dtype, seed=85)
    want, last = linear_attention_torch(*(inputs[n].double() for n in NAMES[:4]), 0.7, inputs["state"].double())
    wide = torch.cat([inputs[n].flatten(2)[:, 0] for n in "qkv"], -1).to(device)
    q, k, v = wide.split((heads * key_dim, heads * key_dim, heads * value_dim), -1)
    q, k, v = q.unflatten(-1, (heads, key_dim)), k.unflatten(-1, (heads, key_dim)), v.unflatten(-1, (heads, value_dim))
    # a state at an odd address as well
    for state in (inputs["state"].to(device), torch.zeros(inputs["state"].numel() + 1, device=device)[1:].view(last.shape)):
        state.copy_(inputs["state"])
        o = visionhope_linear_attention_step(q, k, v, inputs["log_decay"].to(device), state, scale=0.7)
        assert o.shape == (batch, heads, value_dim) and o.dtype == dtype
        compare(o, want[:, 0], tolerance(dtype, key_dim), "step o")
        compare(state, last, tolerance(torch.float32, 2), "step state")


@pytest.mark.parametrize("dtype", DTYPES)
def test_cut_lines_and_whole_ones(device, dtype):
    """Many sequences run uncut, few are cut into segments: the same values to FP32 rounding."""
    heads, length = 1, 640
    inputs = {k: v.to(device) for k, v in _inputs(1, length, heads, 16, 16, dtype, seed=88).items()}
    inputs["log_decay"] = torch.tensor([-0.01], device=device)
    do = randn(1, length, heads, 16, seed=89).to(device, dtype)
    found = []
    for copies in (1, 1600):
        tensors = [inputs[n].expand(copies, *inputs[n].shape[1:]).contiguous() if n != "log_decay" else inputs[n] for n in NAMES]
        leaves = [t.clone().requires_grad_() for t in tensors]
        o, state = _own(leaves, None)
        grads = torch.autograd.grad(o, leaves[:3], do.expand(copies, -1, -1, -1).contiguous())
        for t in (o, state, *grads):
            assert torch.equal(t[0], t[-1])
        found.append([t[:1].detach() for t in (o, state, *grads)])
    for name, a, b in zip(("o", "state", "dq", "dk", "dv"), *found):
        # both round once, at the same values but for FP32's
        compare(a, b.double().cpu(), tolerance(a.dtype, length) + half_step(a.dtype), name)


def test_gradients_against_differences(device):
    """Of a sum of the outputs and the last state, by central differences of float32 outputs summed in float64."""
    inputs = _inputs(2, 70, 2, 12, 8, torch.float32, seed=100)
    lengths = torch.tensor([70, 41], device=device)
    do, dstate = randn(2, 70, 2, 8, seed=101).to(device), randn(2, 2, 12, 8, seed=102).to(device)
    leaves = [inputs[n].to(device).requires_grad_() for n in NAMES]

    def total(tensors):
        o, state = _own(tensors, lengths)
        return (o.double() * do).sum() + (state.double() * dstate).sum()

    grads = torch.autograd.grad(total(leaves), leaves)
    with torch.no_grad():
        for name, leaf, grad in zip(NAMES, leaves, grads):
            step = 2.0 ** -6 if name != "log_decay" else 2.0 ** -9
            direction = randn(*leaf.shape, seed=103).to(device).sign()
            other = [t for t in leaves]
            at = NAMES.index(name)
            values = []
            for sign in (1, -1):
                other[at] = leaf + sign * step * direction
                values.append(total(other))
            slope = ((values[0] - values[1]) / (2 * step)).item()
            expected = (grad.double() * direction).sum().item()
            # linear in every tensor but the decays; a decay's third derivative is below 70^2 of its
            # first and the step's square 2^-18: 2 %.  FP32 outputs: 2^-24 of their sum of magnitudes
            # over the step, about 1e-3 of a slope.
            room = 0.02 if name == "log_decay" else 2e-3
            assert abs(slope - expected) <= room * max(abs(expected), grad.double().abs().sum().item() ** 0.5), name


def test_repeats_bit_by_bit_on_any_stream_and_in_a_graph(device):
    inputs = {k: v.to(device) for k, v in _inputs(2, 1000, 3, 64, 64, torch.bfloat16, seed=110).items()}
    leaves = [inputs[n].clone().requires_grad_() for n in NAMES]
    do = randn(2, 1000, 3, 64, seed=111).to(device, torch.bfloat16)

    def step():
        o, state = _own(leaves, None)
        return [o.detach(), state.detach(), *torch.autograd.grad(o, leaves, do)]

    want = step()
    for _ in range(3):
        for a, b in zip(want, step()):
            assert torch.equal(a, b)
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
    for round_ in range(3):
        with torch.no_grad():
            leaves[0].copy_(inputs["q"] * (round_ + 1))
            leaves[2].copy_(inputs["v"] + round_)
        want = step()
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, captured):
            assert torch.equal(a, b), f"replay {round_}"


def test_captured_single_tokens(device):
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention_step

    inputs = {k: v.to(device) for k, v in _inputs(4, 6, 2, 32, 32, torch.bfloat16, seed=120).items()}
    q, k, v = (inputs[n][:, 0].contiguous() for n in "qkv")
    state, a = inputs["state"].clone(), inputs["log_decay"]
    visionhope_linear_attention_step(q, k, v, a, state.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = visionhope_linear_attention_step(q, k, v, a, state)
    eager = inputs["state"].clone()
    state.copy_(inputs["state"])
    for t in range(6):
        for name, buffer in zip("qkv", (q, k, v)):
            buffer.copy_(inputs[name][:, t])
        graph.replay()
        want = visionhope_linear_attention_step(*(inputs[n][:, t] for n in "qkv"), a, eager)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(state, eager), t


def test_refusals(device):
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention, visionhope_linear_attention_step

    q, k, v, a, s = (_inputs(2, 5, 3, 8, 4, torch.float32, seed=130)[n].to(device) for n in NAMES)
    attend, step = visionhope_linear_attention, visionhope_linear_attention_step
    wide = torch.zeros(1, 2, 1, 129, device=device)
    one = torch.zeros(1, device=device)
    token = (q[:, 0], k[:, 0], v[:, 0], a)
    leaf, memory = q[:, 0].clone().requires_grad_(), torch.zeros(s.numel() + 4, device=device)
    bad = [
        (ValueError, "CUDA", lambda: attend(q.cpu(), k, v, a)),
        (TypeError, "FP16, BF16 and FP32", lambda: attend(q.double(), k, v, a)),
        (ValueError, "nonempty", lambda: attend(q[:, :0], k[:, :0], v[:, :0], a)),
        (ValueError, "4 dimensions", lambda: attend(q[0], k[0], v[0], a)),
        (ValueError, "k must have shape", lambda: attend(q, k[..., :4], v, a)),
        (TypeError, "k must be", lambda: attend(q, k.half(), v, a)),
        (ValueError, "v must", lambda: attend(q, k, v[:, :4], a)),
        (ValueError, "v must", lambda: attend(q, k, v[..., :0], a)),
        (ValueError, "128", lambda: attend(wide, wide, wide[..., :4], one)),
        (ValueError, "128", lambda: attend(wide[..., :4], wide[..., :4], wide, one)),
        (ValueError, "log_decay", lambda: attend(q, k, v, a[:2])),
        (TypeError, "log_decay", lambda: attend(q, k, v, a.int())),
        (ValueError, "state", lambda: attend(q, k, v, a, state=s[:1])),
        (TypeError, "state", lambda: attend(q, k, v, a, state=s.half())),
        (ValueError, "lengths", lambda: attend(q, k, v, a, lengths=torch.ones(3, device=device, dtype=torch.int32))),
        (TypeError, "lengths", lambda: attend(q, k, v, a, lengths=torch.ones(2, device=device))),
        (ValueError, "state must have", lambda: step(*token, s[:, :2])),
        (ValueError, "contiguous", lambda: step(*token, s.transpose(2, 3).contiguous().transpose(2, 3))),
        (ValueError, "new_state", lambda: step(*token, s, new_state=s[:1])),
        (RuntimeError, "same memory or not overlap", lambda: step(*token, memory[:-4].view(s.shape),
                                                                  new_state=memory[4:].view(s.shape))),
        (RuntimeError, "inference", lambda: step(leaf, *token[1:], s)),
    ]
    for error, match, call in bad:
        with pytest.raises(error, match=match):
            call()


def test_forward_mode_is_refused_and_saved_tensors_may_change_strides(device):
    from torch.autograd import forward_ad

    leaves = [_inputs(2, 70, 2, 16, 16, torch.float32, seed=140)[n].to(device).requires_grad_() for n in NAMES]
    do = randn(2, 70, 2, 16, seed=141).to(device)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            with pytest.raises(NotImplementedError):
                _own([forward_ad.make_dual(leaves[0].detach(), torch.ones_like(leaves[0])), *leaves[1:]], None)
    want = torch.autograd.grad(_own(leaves, None)[0], leaves, do)

    def spread(t):   # the same values, every other element of a wider tensor
        wide = torch.zeros(*t.shape, 2, device=t.device, dtype=t.dtype)
        wide[..., 0] = t
        return wide[..., 0]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread):
        got = torch.autograd.grad(_own(leaves, None)[0], leaves, do)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_only_the_state_has_a_gradient(device):
    """Gradients that come through the last state alone, and inputs that want none."""
    inputs = _inputs(2, 50, 2, 16, 16, torch.float32, seed=150)
    dstate = randn(2, 2, 16, 16, seed=151)
    want, grads = gradients(lambda *a: linear_attention_torch(*a[:4], None, a[4]), [inputs[n] for n in NAMES], (None, dstate))
    leaves = [inputs[n].to(device).requires_grad_() for n in NAMES]
    got = torch.autograd.grad(_own(leaves, None)[1], leaves, dstate.to(device), allow_unused=True)
    assert got[0].abs().max() == 0 and grads[0] is None   # the oracle's last state does not read q
    for name, a, b in list(zip(NAMES, got, grads))[1:]:
        compare(a, b, tolerance(torch.float32, 2 * 50 * 130 if name == "log_decay" else 66), f"d{name}")


@pytest.mark.parametrize("learned", [False, True])
def test_a_graph_that_is_kept_gives_the_same_gradients_again(device, learned):
    """The backward starts from the states that the forward left, and leaves them as they were."""
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention

    shape = (1, 4096, 2, 32)   # cut into segments
    q, k, v = (randn(*shape, seed=s).to(device).requires_grad_() for s in (1, 2, 3))
    decay = torch.full((2,), -0.01, device=device, requires_grad=learned)
    o = visionhope_linear_attention(q, k, v, decay)
    do = randn(*shape, seed=4).to(device)
    leaves = [q, k, v] + ([decay] if learned else [])
    first = torch.autograd.grad(o, leaves, do, retain_graph=True)
    again = torch.autograd.grad(o, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(first, again))

"""The refusal of captured backward passes over leaves that a living graph of the default stream
holds, where other operations stand between the leaves and the operator.  The capture itself is
played on the CPU: the Function's two calls get the stream and the state."""

import pytest
import torch

from visionhope_amd.utils.token_lines import note_stream, refuse_held_leaves


class Double(torch.autograd.Function):
    stream, capturing = 0, False

    @staticmethod
    def forward(ctx, x, weight):
        note_stream(ctx, Double.stream)
        return x * weight

    @staticmethod
    def backward(ctx, dy):
        refuse_held_leaves("double", ctx, Double.capturing)
        return dy, dy


def _forward(stream, capturing, x, weight):
    Double.stream, Double.capturing = stream, capturing
    return Double.apply(x, weight)


BETWEEN = {
    "unsqueeze": lambda t: t.unsqueeze(1).squeeze(1),          # B and C without a group axis
    "contiguous": lambda t: t[:, ::2].contiguous(),            # operands that are copied first
    "exp": lambda t: -torch.exp(t.float()),                    # a mixer's rates
    "cast": lambda t: t.to(torch.bfloat16).float(),
    "linear": lambda t: torch.ones(4, 4) @ t,
    "function": lambda t: Double.apply(t * 2, torch.ones(()))
}


@pytest.mark.parametrize("held, captured", [(a, b) for a in BETWEEN for b in ("none", "unsqueeze", "exp")] +
                         [("none", b) for b in BETWEEN])
def test_leaves_behind_other_operations(held, captured):
    between = {**BETWEEN, "none": lambda t: t}
    leaf = torch.ones(4, 4, requires_grad=True)

    def run(stream, capturing, kind):
        Double.stream, Double.capturing = stream, capturing
        x = between[kind](leaf)
        y = _forward(stream, capturing, x, torch.ones(x.shape))
        y.sum().backward()
        return y

    alive = run(0, False, held)
    with pytest.raises(RuntimeError, match="still alive"):
        run(7, True, captured)
    run(7, False, captured)          # not a capture
    del alive
    run(7, True, captured)           # the graph is gone


def test_leaves_that_the_pass_does_not_reach_do_not_matter():
    """Gradients of an intermediate tensor stop there: the leaf behind it is not touched."""
    leaf = torch.ones(4, requires_grad=True)
    alive = _forward(0, False, leaf.exp(), torch.ones(4))
    middle = leaf.exp()
    y = _forward(7, True, middle * 2, torch.ones(4))
    grad, = torch.autograd.grad(y.sum(), middle, retain_graph=True)
    assert torch.equal(grad, torch.full((4,), 2.0))
    for inputs in ([leaf], [middle, leaf]):
        with pytest.raises(RuntimeError, match="still alive"):
            torch.autograd.grad(y.sum(), inputs, retain_graph=True)
    with pytest.raises(RuntimeError, match="still alive"):
        y.sum().backward()
    assert alive.requires_grad

"""Gradients of the token-line operators for operands whose rows lie far apart: batch strides past 32
bits, and token strides of B and C up to and past what the kernels read in place (2^24 elements)."""

import pytest
import torch

from tests.helpers import randn
from tests.test_gpu_state_space import NAMES, _inputs

pytestmark = pytest.mark.gpu

FAR = 2 ** 31   # elements; 4 GiB of a 16-bit type


def _far(base, at, t):
    """``t`` [2, N, C] inside `base` from element `at` on, its two sequences FAR elements apart."""
    return base.as_strided(t.shape, (FAR, t.shape[2], 1), at).copy_(t)


@pytest.mark.parametrize("states", [16, 8])
def test_scan_gradients_of_rows_past_32_bits(device, states):
    """Three blocks of tokens in whole lines, and lines in chunks."""
    from visionhope_amd.utils.state_space import visionhope_state_space_scan

    for length in (40, 200):
        t = {k: v.to(device) for k, v in _inputs(2, length, 32, states, 1, torch.bfloat16, seed=400).items()}
        dy = randn(2, length, 32, seed=401).to(device, torch.bfloat16)
        base = torch.empty(FAR + 6 * length * 32, device=device, dtype=torch.bfloat16)

        def run(place):
            tensors = {**t, **{n: place(i, t[n]) for i, n in enumerate(("x", "dt", "gate"))}}
            tensors.update({n: place(3 + i, t[n][:, :, 0])[:, :, None] for i, n in enumerate(("B", "C"))})
            cotangent = place(5, dy)
            leaves = [tensors[n].detach().requires_grad_() for n in NAMES]
            x, dt, A, B, C, D, gate, dt_bias, state = leaves
            y = visionhope_state_space_scan(x, dt, A, B, C, D, gate=gate, dt_bias=dt_bias, state=state)
            return [y.detach(), *torch.autograd.grad(y, leaves, cotangent)]

        for name, a, b in zip(("y", *NAMES), run(lambda i, v: _far(base, i * length * 32, v)), run(lambda i, v: v)):
            assert torch.equal(a, b), name


def test_conv_gradients_of_rows_past_32_bits(device):
    from visionhope_amd.utils.causal_conv import visionhope_causal_conv

    x, dy = (randn(2, 64, 32, seed=410 + i).to(device, torch.bfloat16) for i in range(2))
    weight, bias = randn(32, 4, seed=412).to(device), randn(32, seed=413).to(device)
    base = torch.empty(FAR + 2 * 64 * 32, device=device, dtype=torch.bfloat16)

    def run(place):
        x_at, dy_at = place(0, x), place(1, dy)
        leaves = [x_at.detach().requires_grad_(), weight.clone().requires_grad_(), bias.clone().requires_grad_()]
        y = visionhope_causal_conv(*leaves, silu=True)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy_at)]

    for a, b in zip(run(lambda i, v: _far(base, i * 64 * 32, v)), run(lambda i, v: v)):
        assert torch.equal(a, b)


def test_norm_gradients_of_rows_past_32_bits(device):
    from visionhope_amd.utils.gated_norm import visionhope_gated_layernorm

    x, gate, dy = (randn(2, 1, 64, seed=420 + i).to(device, torch.bfloat16) for i in range(3))
    weight, bias = randn(64, seed=423).to(device), randn(64, seed=424).to(device)
    base = torch.empty(FAR + 3 * 64, device=device, dtype=torch.bfloat16)

    def run(place):
        x_at, gate_at, dy_at = (place(i, v) for i, v in enumerate((x, gate, dy)))
        leaves = [x_at.detach().requires_grad_(), weight.clone().requires_grad_(), bias.clone().requires_grad_(),
                  gate_at.detach().requires_grad_()]
        y = visionhope_gated_layernorm(*leaves[:3], gate=leaves[3])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy_at)]

    for a, b in zip(run(lambda i, v: _far(base, i * 64, v)), run(lambda i, v: v)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("stride", [2 ** 24 - 2, 2 ** 24, 2 ** 24 + 2])
@pytest.mark.parametrize("states", [16, 32])
def test_tokens_of_the_maps_far_apart(device, states, stride):
    """B and C of 35 tokens over 1.2 GB: read in place below 2^24 elements, packed from there."""
    from visionhope_amd.utils.state_space import visionhope_state_space_scan

    length = 35
    t = {k: v.to(device) for k, v in _inputs(1, length, 40, states, 1, torch.bfloat16, seed=430).items()}
    dy = randn(1, length, 40, seed=431).to(device, torch.bfloat16)
    base = torch.empty((length - 1) * stride + 2 * states, device=device, dtype=torch.bfloat16)

    def run(apart):
        tensors = dict(t)
        if apart:
            for i, n in enumerate(("B", "C")):
                view = base.as_strided((1, length, 1, states), (length * stride, stride, states, 1), i * states)
                tensors[n] = view.copy_(t[n])
        leaves = [tensors[n].detach().requires_grad_() for n in NAMES]
        x, dt, A, B, C, D, gate, dt_bias, state = leaves
        y, last = visionhope_state_space_scan(x, dt, A, B, C, D, gate=gate, dt_bias=dt_bias, state=state,
                                              return_state=True)
        return [y.detach(), last.detach(), *torch.autograd.grad(y, leaves, dy)]

    for name, a, b in zip(("y", "state", *NAMES), run(True), run(False)):
        assert torch.equal(a, b), name

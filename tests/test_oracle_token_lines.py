"""The token-line operators' oracle against element-by-element restatements and finite
differences (CPU, float64)."""

import math

import pytest
import torch

from oracle.oracle_torch import causal_conv_torch, gated_layernorm_torch, state_space_scan_torch
from tests.helpers import randn


def _silu(v):
    return v / (1 + math.exp(-v))


@pytest.mark.parametrize("silu", [False, True])
def test_causal_conv_element_by_element(silu):
    x, w, b, s = (randn(*shape, seed=i).double() for i, shape in enumerate(((2, 6, 3), (3, 4), (3,), (2, 3, 3))))
    lengths = torch.tensor([6, 2])
    y, state = causal_conv_torch(x, w, b, silu, s, lengths)
    for i, n in enumerate(lengths.tolist()):
        line = torch.cat((s[i], x[i, :n]))
        for t in range(6):
            for c in range(3):
                pre = b[c].item() + sum(w[c, k].item() * line[t + k, c].item() for k in range(4)) if t < n else 0.0
                want = (_silu(pre) if silu else pre) if t < n else 0.0
                assert y[i, t, c].item() == pytest.approx(want, rel=1e-12, abs=1e-15)
        assert torch.equal(state[i], line[-3:])


def test_scan_element_by_element():
    groups, width, states, length = 2, 2, 3, 5
    x, dt, gate = (randn(2, length, 4, seed=i).double() for i in (1, 2, 3))
    A, B, C = -randn(4, states, seed=4).double().abs(), *(randn(2, length, groups, states, seed=i).double() for i in (5, 6))
    D, bias, s = randn(4, seed=7).double(), randn(4, seed=8).double(), randn(2, 4, states, seed=9).double()
    lengths = torch.tensor([3, 5])
    y, last = state_space_scan_torch(x, dt, A, B, C, D, gate, bias, True, s, lengths)
    for i, n in enumerate(lengths.tolist()):
        for c in range(4):
            h = s[i, c].tolist()
            for t in range(length):
                if t >= n:
                    assert y[i, t, c] == 0
                    continue
                step = math.log1p(math.exp(dt[i, t, c].item() + bias[c].item()))
                h = [math.exp(step * A[c, k].item()) * h[k] + step * x[i, t, c].item() * B[i, t, c // width, k].item()
                     for k in range(states)]
                v = sum(C[i, t, c // width, k].item() * h[k] for k in range(states)) + D[c].item() * x[i, t, c].item()
                assert y[i, t, c].item() == pytest.approx(v * _silu(gate[i, t, c].item()), rel=1e-12)
            assert last[i, c].tolist() == pytest.approx(h, rel=1e-12)


def test_gated_layernorm_element_by_element():
    x, w, b, gate = (randn(*shape, seed=i).double() for i, shape in enumerate(((3, 5), (5,), (5,), (3, 5))))
    y = gated_layernorm_torch(x, w, b, 1e-3, gate)
    for r in range(3):
        row = x[r].tolist()
        mean = sum(row) / 5
        var = sum((v - mean) ** 2 for v in row) / 5
        for c in range(5):
            want = ((row[c] - mean) / math.sqrt(var + 1e-3) * w[c].item() + b[c].item()) * _silu(gate[r, c].item())
            assert y[r, c].item() == pytest.approx(want, rel=1e-12)


def test_gradients_by_differences():
    def leaves(*shapes):
        return [randn(*s, seed=20 + i).double().requires_grad_() for i, s in enumerate(shapes)]

    assert torch.autograd.gradcheck(lambda x, w, b, s: causal_conv_torch(x, w, b, True, s, torch.tensor([4, 2])),
                                    leaves((2, 4, 2), (2, 3), (2,), (2, 2, 2)))
    assert torch.autograd.gradcheck(
        lambda x, dt, A, B, C, D, g, b, s: state_space_scan_torch(x, dt, A, B, C, D, g, b, True, s, torch.tensor([3, 2])),
        leaves((2, 3, 2), (2, 3, 2), (2, 2), (2, 3, 1, 2), (2, 3, 1, 2), (2,), (2, 3, 2), (2,), (2, 2, 2)))
    assert torch.autograd.gradcheck(lambda x, w, b, g: gated_layernorm_torch(x, w, b, 1e-3, g),
                                    leaves((2, 4), (4,), (4,), (2, 4)))

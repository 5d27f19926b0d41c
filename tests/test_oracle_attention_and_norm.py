"""The linear attention's and the group norm's oracle against other forms of the same and finite
differences (CPU, float64)."""

import math

import pytest
import torch
from torch.nn import functional as F

from oracle.oracle_torch import group_norm_torch, linear_attention_torch
from tests.helpers import randn


def test_attention_pair_by_pair():
    """o[t] as a sum over the tokens up to t, the state's share beside."""
    q, k, v = (randn(2, 7, 3, d, seed=i).double() for i, d in enumerate((4, 4, 5)))
    a, s = -randn(3, seed=4).double().abs(), randn(2, 3, 4, 5, seed=5).double()
    lengths = torch.tensor([7, 3])
    o, last = linear_attention_torch(q, k, v, a, 0.3, s, lengths)
    for b, n in enumerate(lengths.tolist()):
        for h in range(3):
            g = math.exp(a[h].item())
            for t in range(7):
                if t >= n:
                    assert not o[b, t, h].any()
                    continue
                want = g ** (t + 1) * (q[b, t, h] @ s[b, h])
                for j in range(t + 1):
                    want = want + g ** (t - j) * (q[b, t, h] @ k[b, j, h]) * v[b, j, h]
                assert torch.allclose(o[b, t, h], 0.3 * want, rtol=1e-12, atol=1e-14)
            state = g ** n * s[b, h] + sum(g ** (n - 1 - j) * torch.outer(k[b, j, h], v[b, j, h]) for j in range(n))
            assert torch.allclose(last[b, h], state, rtol=1e-12, atol=1e-14)


@pytest.mark.parametrize("activation", [None, "silu", "gelu"])
def test_group_norm_against_the_library(activation):
    x, w, b = randn(2, 12, 4, 3, seed=1).double(), randn(12, seed=2).double(), randn(12, seed=3).double()
    want = F.group_norm(x, 3, w, b, 1e-3)
    want = {None: want, "silu": F.silu(want), "gelu": F.gelu(want)}[activation]
    assert torch.allclose(group_norm_torch(x, 3, w, b, 1e-3, activation), want, rtol=1e-12, atol=1e-13)


def test_gradients_by_differences():
    def leaves(*shapes):
        return [randn(*s, seed=20 + i).double().requires_grad_() for i, s in enumerate(shapes)]

    assert torch.autograd.gradcheck(lambda q, k, v, a, s: linear_attention_torch(q, k, v, a, None, s, torch.tensor([4, 2])),
                                    leaves((2, 4, 2, 3), (2, 4, 2, 3), (2, 4, 2, 2), (2,), (2, 2, 3, 2)))
    for activation in (None, "silu", "gelu"):
        assert torch.autograd.gradcheck(lambda x, w, b: group_norm_torch(x, 2, w, b, 1e-3, activation),
                                        leaves((2, 4, 2, 3), (4,), (4,)))

"""The gated LayerNorm's forward and gradients on rows that lie far from zero beside their spread,
where the rounding of a row's mean is a visible part of the normalised values."""

import pytest
import torch

from oracle.oracle_torch import gated_layernorm_torch
from tests.helpers import randn
from tests.token_lines import compare, gradients, tolerance

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("offset, spread", [(1000.0, 0.01), (1000.0, 0.1), (-200.0, 1.0), (0.0, 1.0)])
@pytest.mark.parametrize("channels", [96, 450, 1001, 1024, 2048, 4100, 6000, 8191])
def test_gradients_of_rows_far_from_zero(device, channels, offset, spread, gated):
    """FP32 rows.  With a mean that is rounded to FP32 the centred values are exact differences of
    neighbours in magnitude, and their own mean (up to 2^-24 of the offset) is taken off again, so
    the result is as exact as that of rows around zero: the tolerance is theirs."""
    from visionhope_amd.utils.gated_norm import visionhope_gated_layernorm

    rows = 37
    x = offset + spread * randn(rows, channels, seed=1)
    weight, bias = 1 + 0.2 * randn(channels, seed=2), 0.2 * randn(channels, seed=3)
    gate = randn(rows, channels, seed=4) if gated else None
    dy = randn(rows, channels, seed=5)
    want, grads = gradients(lambda *a: gated_layernorm_torch(a[0], a[1], a[2], EPS, a[3]), (x, weight, bias, gate), (dy,))
    leaves = [None if t is None else t.to(device).requires_grad_() for t in (x, weight, bias, gate)]
    y = visionhope_gated_layernorm(*leaves[:3], EPS, gate=leaves[3])
    compare(y, want[0], tolerance(torch.float32, channels), "y")
    y.backward(dy.to(device))
    for name, leaf, grad in zip(("x", "weight", "bias", "gate"), leaves, grads):
        if leaf is not None:
            terms = rows + channels if name in ("weight", "bias") else channels
            compare(leaf.grad, grad, tolerance(torch.float32, terms), f"d{name}")

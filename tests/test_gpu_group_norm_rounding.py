"""The group norm's 16-bit outputs are those of FP32 arithmetic, rounded once, with every activation."""

import pytest
import torch

from oracle.oracle_torch import group_norm_torch
from tests.helpers import randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", [None, "silu", "gelu"])
@pytest.mark.parametrize("shape, groups", [((8, 64, 9, 9), 4), ((4, 96, 60, 50), 6)])   # registers, slabs
def test_few_outputs_are_not_the_nearest(device, dtype, activation, shape, groups):
    """The share of outputs that are not the exact value rounded to the type.

    An error e turns a rounding with the probability |e| / u, u the distance of neighbours at the
    output, at least 2^-8 (bf16; FP16 2^-11) of it.  rstd, the centred value, its weight and the
    activation's exponential, reciprocal and fit each leave 2^-24 to 2^-23: together 2^-22 of the
    outputs' spread.  Of values spread normally, small ones among them, six times that over u turn, three
    quarters of it for the larger u within a binade: 4.5 * 2^(8 - 22).
    """
    from visionhope_amd.utils.group_norm import visionhope_group_norm

    channels = shape[1]
    x = (randn(*shape, seed=1) * torch.exp(0.3 * randn(1, channels, 1, 1, seed=2)) + randn(1, channels, 1, 1, seed=3)).to(dtype)
    weight, bias = 1 + 0.2 * randn(channels, seed=4), 0.2 * randn(channels, seed=5)
    want = group_norm_torch(x.double(), groups, weight.double(), bias.double(), 1e-5, activation)
    got = visionhope_group_norm(x.to(device).contiguous(memory_format=torch.channels_last), groups, weight.to(device),
                                bias.to(device), 1e-5, activation=activation)
    share = (got.cpu() != want.to(dtype)).double().mean().item()
    assert share <= 4.5 * 2.0 ** ((8 if dtype == torch.bfloat16 else 11) - 22), share

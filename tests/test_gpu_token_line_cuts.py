"""Token-line operators at sizes whose work is cut as that of large maps and long prompts: chunks of
several blocks, adjoint chunks that are parts of them, joins with many slots, workgroups that
walk many rows, parameter sums in two launches.  Outputs and gradients against the float64 oracle;
what a size reaches is asserted first."""

import pytest
import torch

from oracle.oracle_torch import causal_conv_torch, gated_layernorm_torch
from tests import token_line_cuts as cuts
from tests.helpers import randn
from tests.test_gpu_state_space import _check as check_scan
from tests.test_gpu_state_space import _inputs as scan_inputs
from tests.token_lines import DTYPES, compare, gradients, tolerance

pytestmark = pytest.mark.gpu

# (batch, length, channels, states, groups): tokens of a forward chunk, of a backward chunk and of
# an adjoint chunk.  Many small groups cut a line as many channels would.
CUTS = [
    ((8, 400, 32, 16, 32), 32, 112, 28),
    ((8, 330, 48, 16, 16), 16, 48, 24),
    ((8, 330, 560, 8, 8), 16, 32, 16),     # 70 channels a group: one workgroup of the gradients' pass, two tiles
    ((8, 520, 32, 32, 16), 16, 144, 18),
    ((4, 300, 96, 5, 32), 16, 64, 16),
    ((3, 260, 384, 12, 64), 32, 64, 16),
    ((16, 410, 32, 16, 32), 48, 208, 52),
    ((24, 150, 64, 16, 64), 160, 160, 160),   # whole lines of more than four blocks
]


def _lengths(batch, length, chunk, fine):
    ends = [length, 0, chunk + 1, fine + 5, length - 1, chunk - 1, 2 * chunk, 3 * fine - 1, 1, fine]
    return torch.tensor([min(n, length) for n in (ends * (batch // len(ends) + 1))[:batch]])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("shape, chunk, back, fine", CUTS, ids=[str(c[0]) for c in CUTS])
def test_scan_in_chunks_of_several_blocks(device, shape, chunk, back, fine, ragged, dtype):
    batch, length, channels, states, groups = shape
    cut = cuts.backward_cut(*shape)
    assert (min(cuts.forward_chunk(batch, length, channels, groups), cuts.ceil(length, 16) * 16), cut.chunk, cut.fine) == \
        (chunk, back, fine)
    lengths = _lengths(batch, length, back, fine) if ragged else None
    check_scan(device, scan_inputs(*shape, dtype, seed=300), f"{shape}", lengths=lengths)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("shape", [(1, 2200, 64, 16, 1), (1, 2500, 40, 6, 1), (1, 2300, 20, 32, 2)])
def test_scan_with_many_chunks(device, shape, ragged, dtype):
    """More than 128 slots of a join: its waves walk ranges that their registers do not hold."""
    batch, length, channels, states, groups = shape
    assert cuts.backward_cut(*shape).fine_chunks - 1 > 128
    assert cuts.ceil(length, cuts.forward_chunk(batch, length, channels, groups)) - 1 > 128
    lengths = torch.tensor([length - 37]) if ragged else None
    check_scan(device, scan_inputs(*shape, dtype, seed=310), f"{shape}", lengths=lengths)


def test_scan_parameter_sums_in_two_launches(device):
    shape = (520, 5, 10, 4, 1)
    cut = cuts.backward_cut(*shape)
    assert cuts.sum_splits(shape[0] * cut.chunks, (cuts.padded(4) + 2) * 64) > 1
    check_scan(device, scan_inputs(*shape, torch.float32, seed=320), f"{shape}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels, taps", [(8, 4), (13, 3), (200, 7)])
def test_conv_parameter_sums_in_two_launches(device, dtype, channels, taps):
    from visionhope_amd.utils.causal_conv import visionhope_causal_conv

    batch, length = 530, 9   # a strip of partial sums a sequence at least
    assert cuts.sum_splits(batch, (taps + 1) * channels) > 1
    x, dy = randn(batch, length, channels, seed=330).to(dtype), randn(batch, length, channels, seed=331).to(dtype)
    weight, bias = randn(channels, taps, seed=332) * 0.5, randn(channels, seed=333) * 0.5
    want, grads = gradients(lambda *a: causal_conv_torch(a[0], a[1], a[2], True, None, None)[0], (x, weight, bias), (dy,))
    leaves = [t.to(device).requires_grad_() for t in (x, weight, bias)]
    y = visionhope_causal_conv(*leaves, silu=True)
    compare(y, want[0], tolerance(dtype, taps), "y")
    y.backward(dy.to(device))
    for name, leaf, grad in zip(("x", "weight", "bias"), leaves, grads):
        tol = tolerance(dtype, 2 * taps) if name == "x" else tolerance(torch.float32, batch * length)
        compare(leaf.grad, grad, tol, f"d{name}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("channels", [40, 96, 450, 1024, 2500, 6000])
def test_norm_workgroups_walk_many_rows(device, channels, gated, dtype):
    """A lane takes 32 elements at most and a row four lanes at least, so a workgroup of 256 lanes
    takes no more rows a step than 8192 / channels or 64: more steps than the forward's 2048
    workgroups, and enough in the backward for sums in two launches."""
    from visionhope_amd.utils.gated_norm import visionhope_gated_layernorm

    rows = 2060 * max(1, min(8192 // channels, 64)) + 1
    assert cuts.sum_splits(512, 2 * channels) > 1
    x, gate, dy = ((randn(rows, channels, seed=340 + i)).to(dtype) for i in range(3))
    weight, bias = 1 + 0.2 * randn(channels, seed=344), 0.2 * randn(channels, seed=345)
    gate = gate if gated else None
    want, grads = gradients(lambda *a: gated_layernorm_torch(a[0], a[1], a[2], 1e-6, a[3]), (x, weight, bias, gate), (dy,))
    leaves = [None if t is None else t.to(device).requires_grad_() for t in (x, weight, bias, gate)]
    y = visionhope_gated_layernorm(*leaves[:3], 1e-6, gate=leaves[3])
    compare(y, want[0], tolerance(dtype, channels), "y")
    y.backward(dy.to(device))
    for name, leaf, grad in zip(("x", "weight", "bias", "gate"), leaves, grads):
        if leaf is not None:
            compare(leaf.grad, grad, tolerance(leaf.dtype, rows + channels if name in ("weight", "bias") else channels),
                    f"d{name}")

"""Group norm where its plans change: the largest maps in registers, bundles of groups that the last one does
not fill, several bundles of a large map, one slab an image."""

import pytest
import torch

from oracle.oracle_torch import group_norm_torch
from tests.helpers import randn
from tests.token_lines import compare, gradients, tolerance

pytestmark = pytest.mark.gpu

HALVES = (torch.bfloat16, torch.float16)
EPS = 1e-5


def _run(device, x, weight, bias, dy, groups, activation):
    from visionhope_amd.utils.group_norm import visionhope_group_norm

    leaves = [t.to(device).requires_grad_() for t in (x, weight, bias)]
    y = visionhope_group_norm(leaves[0], groups, *leaves[1:], EPS, activation=activation)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy.to(device))]


def _inputs(shape, dtype):
    channels = shape[1]
    x = randn(*shape, seed=1) * torch.exp(0.3 * randn(1, channels, 1, 1, seed=2)) + randn(1, channels, 1, 1, seed=3)
    x, dy = (t.to(dtype).contiguous(memory_format=torch.channels_last) for t in (x, randn(*shape, seed=4)))
    return x, 1 + 0.2 * randn(channels, seed=5), 0.2 * randn(channels, seed=6), dy


def _check(device, shape, groups, dtype, activation):
    x, weight, bias, dy = _inputs(shape, dtype)
    got = _run(device, x, weight, bias, dy, groups, activation)
    want, grads = gradients(lambda *a: group_norm_torch(a[0], groups, a[1], a[2], EPS, activation), (x, weight, bias), (dy,))
    values, rows = x.numel() // (shape[0] * groups), x.numel() // shape[1]
    for name, a, b, tol in zip(("y", "dx", "dweight", "dbias"), got, (want[0], *grads),
                               [tolerance(dtype, values)] * 2 + [tolerance(torch.float32, rows + values)] * 2):
        compare(a, b, tol, f"{shape} {groups} {dtype} {activation} {name}")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("activation", [None, "silu", "gelu"])
@pytest.mark.parametrize("shape, groups", [
    ((2, 320, 20, 20), 20),    # eight vectors of eight a thread, in registers
    ((2, 80, 9, 9), 5),        # four groups in a bundle, and one in the last
    ((3, 176, 14, 14), 11),    # the same, more vectors a thread
    ((2, 72, 11, 7), 9),       # vectors of eight, one group each: eight groups and one
    ((1, 2096, 29, 31), 131),  # slabs: bundles of 66 groups and of 65
    ((1, 2304, 40, 30), 3),    # slabs: bundles of two groups and of one
])
def test_bundles_of_16_bits(device, dtype, activation, shape, groups):
    _check(device, shape, groups, dtype, activation)


@pytest.mark.parametrize("activation", [None, "silu", "gelu"])
@pytest.mark.parametrize("shape, groups", [
    ((2, 160, 20, 20), 10),    # eight vectors of four a thread, in registers
    ((2, 48, 9, 9), 3),        # two groups in a bundle, and one in the last
    ((3, 28, 10, 10), 7),      # vectors of four, one group each
    ((2, 1040, 25, 31), 65),   # slabs: bundles of 33 groups and of 32
    ((1, 1161, 24, 40), 9),    # slabs: groups of 129 values, one by one
])
def test_bundles_of_fp32(device, activation, shape, groups):
    _check(device, shape, groups, torch.float32, activation)


@pytest.mark.parametrize("dtype", (torch.float32, *HALVES))
@pytest.mark.parametrize("shape, groups", [((2100, 32, 37, 31), 2), ((1100, 2096, 13, 40), 131)])   # one bundle, and two or three
def test_one_slab_an_image(device, dtype, shape, groups):
    """More images than workgroups wanted: each image (of each bundle) is one slab.  y and dx of some images
    against the oracle, the parameters' gradients against those of the images in two parts."""
    from visionhope_amd.utils import hip

    batch, channels, height, width = shape
    gen = torch.Generator(device=device).manual_seed(7)
    x, dy = (torch.randn(batch, height, width, channels, generator=gen, device=device).to(dtype).permute(0, 3, 1, 2) for _ in range(2))
    weight, bias = 1 + 0.2 * randn(channels, seed=5), 0.2 * randn(channels, seed=6)
    assert 0 < hip.load_library().vh_group_norm_workspace_bytes(batch, height * width, channels, groups, hip.dtype_code(dtype))
    got = _run(device, x, weight, bias, dy, groups, "silu")
    some = [0, batch // 2, batch - 1]
    part = [t[some].cpu() for t in (x, dy)]
    want, grads = gradients(lambda *a: group_norm_torch(a[0], groups, a[1], a[2], EPS, "silu"), (part[0], weight, bias), (part[1],))
    values = height * width * channels // groups
    compare(got[0][some], want[0], tolerance(dtype, values), f"{shape} y")
    compare(got[1][some], grads[0], tolerance(dtype, values), f"{shape} dx")
    half = batch // 2
    parts = [_run(device, a, weight, bias, b, groups, "silu") for a, b in ((x[:half], dy[:half]), (x[half:], dy[half:]))]
    for at, name in ((2, "dweight"), (3, "dbias")):
        total = parts[0][at].double() + parts[1][at].double()
        compare(got[at], total.cpu(), 2 * tolerance(torch.float32, batch * height * width), f"{shape} {name}")

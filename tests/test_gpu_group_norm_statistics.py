"""Statistics of maps that are cut into slabs: long runs of a thread, values far from the others."""

import pytest
import torch

from tests.helpers import randn

pytestmark = pytest.mark.gpu

EPS = 1e-5
# Relative error of y and dx where they are not near zero: rstd's is half the variance's, which sums 32
# values in a row, each sum off by 2^-24 at most (2^-20 for the variance with its division and root); the
# centred value, its products and the mean's rest add four roundings of 2^-24.
BOUND = 2.0 ** -20
# dx also takes xhat times the mean of dy xhat, whose FP32 sum passes through some 256 additions (a run of a
# thread, the threads, the slabs) that round by 2^-25 of the running value: four standard deviations of
# 2^4 * 2^-25.  It counts at a value far from the others, where that product is nearly all of dy.
SUM = 2.0 ** -19


def _takes_slabs(batch, pixels, channels, groups):
    from visionhope_amd.utils import hip

    return hip.load_library().vh_group_norm_workspace_bytes(batch, pixels, channels, groups, hip.VH_DTYPE_F32) > 0


def _check(x, dy, groups, images, what):
    from visionhope_amd.utils.group_norm import visionhope_group_norm

    batch, channels, height, width = x.shape
    assert _takes_slabs(batch, height * width, channels, groups)
    leaf = x.requires_grad_()
    y = visionhope_group_norm(leaf, groups, torch.ones(channels, device=x.device), torch.zeros(channels, device=x.device), EPS)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    for image in images:
        rows = x.detach()[image].double().reshape(groups, -1)
        grads = dy[image].double().reshape(groups, -1)
        centred = rows - rows.mean(1, keepdim=True)
        rstd = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
        xhat = centred * rstd
        along = xhat * (grads * xhat).mean(1, keepdim=True)
        slope = rstd * (grads - grads.mean(1, keepdim=True) - along)
        for name, got, want, rest in (("y", y, xhat, None), ("dx", dx, slope, SUM * rstd * along.abs())):
            got = got.detach()[image].double().reshape(groups, -1)
            counted = want.abs() > 0.5 * torch.minimum(want.std(1, keepdim=True), rstd)
            wrong = (got - want).abs() if rest is None else (got - want).abs() - rest
            worst = (wrong / want.abs())[counted].max().item()
            assert worst <= BOUND, f"{what} image {image} {name}: {worst:.2e}"


@pytest.mark.parametrize("where", [0, 77, -1])
@pytest.mark.parametrize("channels, groups", [(16, 1), (24, 3), (7, 1)])   # vectors of four, and of one
def test_one_value_far_from_the_others_of_a_large_map(device, where, channels, groups):
    """10^4 beside a spread of one; at 0 it is the first of its thread's and its slab's values."""
    x = randn(1, 512, 512, channels, seed=1)
    x.view(-1, channels)[where] = 1e4
    dy = randn(1, 512, 512, channels, seed=2).to(device).permute(0, 3, 1, 2)
    _check(x.to(device).permute(0, 3, 1, 2), dy, groups, (0,), f"{channels} {groups} {where}")


def test_a_border_far_from_the_rest(device):
    """The first rows of a map stand 1000 spreads away, as a padded image's do."""
    x = randn(1, 512, 512, 16, seed=3)
    x[:, :3] += 1000.0
    dy = randn(1, 512, 512, 16, seed=4).to(device).permute(0, 3, 1, 2)
    _check(x.to(device).permute(0, 3, 1, 2), dy, 1, (0,), "border")


def test_one_slab_an_image(device):
    """As many images as there are workgroups wanted: a thread sums a 36th of a map by itself."""
    batch = 2048
    gen = torch.Generator(device=device).manual_seed(5)
    x, dy = (torch.randn(batch, 96, 96, 16, generator=gen, device=device) for _ in range(2))
    x[:, 0, 0] = 1e4
    _check(x.permute(0, 3, 1, 2), dy.permute(0, 3, 1, 2), 1, (0, 1000, batch - 1), "one slab")


def test_a_large_offset_of_a_large_map(device):
    """4096 beside a spread of one: what the input's rounding leaves is normalised as around zero."""
    x = randn(1, 512, 512, 16, seed=6) + 4096.0
    dy = randn(1, 512, 512, 16, seed=7).to(device).permute(0, 3, 1, 2)
    _check(x.to(device).permute(0, 3, 1, 2), dy, 1, (0,), "offset")

"""GroupNorm2d's arguments are checked when the module is built."""

import pytest
import torch

from visionhope_amd.models import HierarchicalVisionHOPE
from visionhope_amd.models.layers import GroupNorm2d, build_norm
from visionhope_amd.utils.group_norm import MAX_GROUP_CHANNELS


@pytest.mark.parametrize("build", [lambda: GroupNorm2d(MAX_GROUP_CHANNELS + 6), lambda: GroupNorm2d(2048, groups=1),
                                   lambda: build_norm(MAX_GROUP_CHANNELS + 6, "groupnorm2d"),
                                   lambda: HierarchicalVisionHOPE(conv_norm="group", projection_dim=1030)])
def test_groups_beyond_the_kernels_are_refused(build):
    with pytest.raises(ValueError, match=f"at most {MAX_GROUP_CHANNELS} channels"):
        build()


def test_groups_that_the_kernels_take_are_built():
    for dim, groups, want in ((1030, 2, 2), (1024, 1, 1), (1023, None, 1), (2048, None, 128), (40, None, 1)):
        norm = GroupNorm2d(dim, groups)
        assert norm.groups == want
        assert norm(torch.ones(1, dim, 2, 2)).shape == (1, dim, 2, 2)


@pytest.mark.parametrize("dim, groups", [(0, None), (16, 0), (16, 3), (16, -2)])
def test_groups_that_do_not_divide_are_refused(dim, groups):
    with pytest.raises(ValueError, match="divide"):
        GroupNorm2d(dim, groups)

"""Arguments that StateSpaceMixer refuses when it is built (CPU)."""

import pytest

from visionhope_amd.models import StateSpaceMixer


@pytest.mark.parametrize("taps", [-1, 0, 1, 9])
def test_taps_that_the_convolution_does_not_take(taps):
    with pytest.raises(ValueError, match="conv_taps must be 2 to 8"):
        StateSpaceMixer(16, conv_taps=taps)


@pytest.mark.parametrize("taps", [2, 8])
def test_taps_that_it_takes(taps):
    conv, scan = StateSpaceMixer(16, conv_taps=taps).allocate_state(3)
    assert conv.shape == (3, taps - 1, 32) and scan.shape == (3, 32, 16)

"""A single-token call writes its new state in place, so that tensor may not record gradients."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["conv", "scan"])
def test_new_state_that_records_gradients_is_refused(device, which):
    from visionhope_amd.utils.causal_conv import visionhope_causal_conv_step
    from visionhope_amd.utils.state_space import visionhope_state_space_step

    x, maps = torch.ones(2, 8, device=device), torch.ones(2, 16, device=device)
    shape = (2, 3, 8) if which == "conv" else (2, 8, 16)
    state, new_state = torch.zeros(shape, device=device), torch.full(shape, 5.0, device=device)

    def call(target):
        if which == "conv":
            return visionhope_causal_conv_step(x, state, torch.ones(8, 4, device=device), new_state=target)
        return visionhope_state_space_step(x, x, -torch.ones(8, 16, device=device), maps, maps, state, new_state=target)

    leaf = new_state.clone().requires_grad_()
    for target in (leaf, leaf * 1.0):
        before = target.detach().clone()
        with pytest.raises(RuntimeError, match="inference"):
            call(target)
        assert torch.equal(target.detach(), before)
    with torch.no_grad():
        y = call(leaf)
    assert torch.equal(call(new_state), y) and torch.equal(leaf.detach(), new_state)

"""What stands behind the ends of a padded batch has no part in a mixer's outputs and gradients."""

import pytest
import torch

from tests.helpers import randn
from tests.test_gpu_state_space_mixer import _mixer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_what_stands_behind_the_end_has_no_part(device, norm, index):
    mixer = _mixer(norm).to(device)
    lengths = torch.tensor([40, 0, 17, 1], dtype=index, device=device)
    x, dout = randn(4, 40, 48, seed=1).to(device), randn(4, 40, 48, seed=2).to(device)
    behind = (torch.arange(40, device=device) >= lengths[:, None])[..., None]
    results = []
    for fill in (0.0, float("nan"), float("inf")):
        leaf = torch.where(behind, fill, x).requires_grad_()
        out, (conv, scan) = mixer(leaf, lengths=lengths, return_state=True)
        grads = torch.autograd.grad(out, [leaf, *mixer.parameters()], torch.where(behind, fill, dout))
        with torch.no_grad():
            assert torch.equal(mixer(leaf, lengths=lengths), out)
        results.append([out.detach(), conv.detach(), scan.detach(), *grads])
    names = ["out", "conv state", "scan state", "x", *(n for n, _ in mixer.named_parameters())]
    for other in results[1:]:
        for name, a, b in zip(names, results[0], other):
            assert torch.isfinite(b).all(), name
            assert torch.equal(a, b), name
    assert not results[0][0][behind.expand_as(x)].any() and not results[0][3][behind.expand_as(x)].any()


def test_lengths_are_checked(device):
    mixer = _mixer(True).to(device)
    x = torch.zeros(2, 5, 48, device=device)
    with pytest.raises(TypeError, match="lengths"):
        mixer(x, lengths=torch.ones(2, device=device))
    for lengths in (torch.ones(3, dtype=torch.int32, device=device), torch.ones(2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="lengths"):
            mixer(x, lengths=lengths)

"""What stands behind the ends of a padded batch has no part in a mixer's outputs and gradients."""

import pytest
import torch

from tests.helpers import randn
from tests.test_gpu_state_space_mixer import _mixer
from tests.token_lines import compare, tolerance

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


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("ragged", [False, True])
def test_captured_training_step(device, norm, ragged):
    """Forward and backward of the whole module in one graph, replayed with new inputs."""
    mixer = _mixer(norm).to(device)
    lengths = torch.tensor([40, 0, 17, 1], dtype=torch.int32, device=device) if ragged else None
    x, dout = randn(4, 40, 48, seed=5).to(device), randn(4, 40, 48, seed=6).to(device)
    live = x.clone().requires_grad_()

    def step():
        out = mixer(live, lengths=lengths)
        return [out.detach(), *torch.autograd.grad(out, [live, *mixer.parameters()], dout)]

    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        step()   # the library's products choose their kernels outside the capture
    torch.cuda.current_stream(device).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for replay in range(3):
        with torch.no_grad():
            live.copy_(x * (replay + 1))
        want = step()
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for name, a, b in zip(("out", "x", *(n for n, _ in mixer.named_parameters())), captured, want):
            compare(a, b.double().cpu(), tolerance(torch.float32, 4 * 40 + 96), f"replay {replay} {name}")

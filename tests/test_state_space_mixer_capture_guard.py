"""A mixer whose captured backward must be refused is refused before its own output projection's
leaf is reached.  The operators run as their oracle on the CPU and the capture is played."""

import pytest
import torch

from oracle.oracle_torch import causal_conv_torch, gated_layernorm_torch, state_space_scan_torch
from visionhope_amd.models import StateSpaceMixer
from visionhope_amd.models import state_space as module
from visionhope_amd.utils.token_lines import note_stream, refuse_held_leaves


class Played(torch.autograd.Function):
    """Stands where an operator's Function does: notes the stream, and refuses in a capture."""
    stream = 0

    @staticmethod
    def forward(ctx, x):
        note_stream(ctx, Played.stream)
        return x.clone()

    @staticmethod
    def backward(ctx, dy):
        refuse_held_leaves("operator", ctx, torch.cuda.is_current_stream_capturing())
        return dy


@pytest.fixture
def mixer(monkeypatch):
    monkeypatch.setattr(module, "visionhope_causal_conv", lambda x, w, b, *, silu, state, lengths, return_state:
                        causal_conv_torch(Played.apply(x), w, b, silu, state, lengths)[0])
    monkeypatch.setattr(module, "visionhope_state_space_scan", lambda x, dt, A, B, C, D, *, gate, dt_bias, state, lengths,
                        return_state: state_space_scan_torch(Played.apply(x), dt, A, B[:, :, None], C[:, :, None], D, gate,
                                                             dt_bias, True, state, lengths)[0])
    monkeypatch.setattr(module, "visionhope_gated_layernorm", lambda y, w, b, eps, *, gate:
                        gated_layernorm_torch(Played.apply(y), w, b, eps, gate))
    return StateSpaceMixer(16, state_dim=3)


@pytest.mark.parametrize("ragged", [False, True])
def test_refused_before_the_output_projection(monkeypatch, mixer, ragged):
    lengths = torch.tensor([5, 2]) if ragged else None

    def run(stream, capturing):
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
        Played.stream = stream
        out = mixer(torch.ones(2, 5, 16), lengths=lengths)
        out.sum().backward()
        return out

    alive = run(0, False)
    want = mixer.out_proj.weight.grad.clone()
    mixer.zero_grad()
    with pytest.raises(RuntimeError, match="still alive"):
        run(7, True)
    assert all(p.grad is None for p in mixer.parameters())
    del alive
    run(7, True)
    assert torch.equal(mixer.out_proj.weight.grad, want)

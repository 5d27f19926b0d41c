"""A linear attention mixer whose captured backward must be refused is refused before its own output
projection's leaf is reached.  The operators run as their oracle on the CPU and the capture is played."""

import pytest
import torch

from oracle.oracle_torch import gated_layernorm_torch, linear_attention_torch
from tests.test_state_space_mixer_capture_guard import Played
from visionhope_amd.models import LinearAttentionMixer
from visionhope_amd.models import linear_attention as module


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("learn_decay", [False, True])
def test_refused_before_the_output_projection(monkeypatch, ragged, learn_decay):
    monkeypatch.setattr(module, "visionhope_linear_attention", lambda q, k, v, a, *, state, lengths, return_state:
                        linear_attention_torch(Played.apply(q), k, v, a, None, state, lengths)[0])
    monkeypatch.setattr(module, "visionhope_gated_layernorm", lambda y, w, b, eps, *, gate:
                        gated_layernorm_torch(Played.apply(y), w, b, eps, gate))
    mixer = LinearAttentionMixer(16, heads=2, learn_decay=learn_decay)
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

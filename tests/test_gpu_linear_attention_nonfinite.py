"""How far a value that is not finite reaches in linear attention."""

import pytest
import torch

from tests.helpers import randn
from tests.token_lines import DTYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["q", "k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_value_that_is_not_finite_stays_in_its_head_from_its_chunk_on(device, dtype, which, value):
    """Other heads and sequences, and tokens before its chunk of 64, are those of finite inputs bit by bit; a
    query reaches its own token alone."""
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention

    lines = {name: randn(3, 2000, 2, 48, seed=seed).to(device, dtype) for seed, name in enumerate("qkv")}
    log_decay = torch.tensor([-0.01, -0.2], device=device)

    def run():
        return visionhope_linear_attention(*lines.values(), log_decay, return_state=True)

    want, want_state = run()
    token = 1000
    lines[which][1, token, 0, 7] = value
    got, state = run()
    first = token // 64 * 64
    assert torch.equal(got[[0, 2]], want[[0, 2]]) and torch.equal(got[1, :, 1], want[1, :, 1])
    assert torch.equal(got[1, :first, 0], want[1, :first, 0])
    assert not torch.isfinite(got[1, token, 0]).all()
    assert torch.equal(state[[0, 2]], want_state[[0, 2]]) and torch.equal(state[1, 1], want_state[1, 1])
    if which == "q":
        assert torch.equal(got[1, :token, 0], want[1, :token, 0]) and torch.equal(got[1, token + 1:, 0], want[1, token + 1:, 0])
        assert torch.equal(state, want_state)
    else:
        assert not torch.isfinite(got[1, -1, 0]).all() and not torch.isfinite(state[1, 0]).all()

"""The gated LayerNorm of token rows on the GPU against the float64 oracle."""

import pytest
import torch

from oracle.oracle_torch import gated_layernorm_torch
from tests.helpers import randn
from tests.token_lines import DTYPES, compare, gradients, tolerance

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _inputs(shape, dtype, seed=0):
    channels = shape[-1]
    x = (randn(*shape, seed=seed + 1) * 1.5 + 0.3).to(dtype)
    return x, 1 + 0.2 * randn(channels, seed=seed + 2), 0.2 * randn(channels, seed=seed + 3), randn(*shape, seed=seed + 4).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("shape", [(1, 2), (5, 7), (3, 8), (33, 96), (2, 9, 192), (70, 450), (9, 1001), (4, 1024),
                                   (600, 64), (3, 2050), (2, 4097), (5, 6000), (2, 8191), (3, 8192), (1, 1, 1, 40)])
def test_rows_and_gradients(device, dtype, gated, shape):
    from visionhope_amd.utils.gated_norm import visionhope_gated_layernorm

    x, weight, bias, gate = _inputs(shape, dtype)
    gate = gate if gated else None
    dy = randn(*shape, seed=5).to(dtype)
    want, grads = gradients(lambda *a: gated_layernorm_torch(a[0], a[1], a[2], EPS, a[3]), (x, weight, bias, gate), (dy,))
    leaves = [None if t is None else t.to(device).requires_grad_() for t in (x, weight, bias, gate)]
    y = visionhope_gated_layernorm(*leaves[:3], EPS, gate=leaves[3])
    assert y.dtype == dtype and y.is_contiguous()
    channels, rows = shape[-1], x.numel() // shape[-1]
    compare(y, want[0], tolerance(dtype, channels), f"{shape} y")
    y.backward(dy.to(device))
    for name, leaf, grad in zip(("x", "weight", "bias", "gate"), leaves, grads):
        if leaf is None:
            continue
        # two channels: x's gradient is what is left of terms that cancel to (eps / var) of them
        if channels == 2 and name == "x":
            assert (leaf.grad.double().cpu() - grad).abs().max() <= 2.0 ** -20 * dy.abs().max()
            continue
        terms = rows + channels if name in ("weight", "bias") else channels
        compare(leaf.grad, grad, tolerance(leaf.dtype, terms), f"{shape} {dtype} d{name}")
    with torch.no_grad():
        assert torch.equal(visionhope_gated_layernorm(*leaves[:3], EPS, gate=leaves[3]), y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_constant_and_offset_rows(device, dtype):
    """Rows without variance (x - mean is zero), and rows far from zero beside their spread."""
    from visionhope_amd.utils.gated_norm import visionhope_gated_layernorm

    x = torch.full((4, 48), 3.0)
    x[1] = 0.0
    x[2] = 100.0 + (torch.arange(48) % 4)
    x[3] = -200.0 + (torch.arange(48) % 2) * 2
    x = x.to(dtype)
    weight, bias = randn(48, seed=11), randn(48, seed=12)
    want = gated_layernorm_torch(x.double(), weight.double(), bias.double(), EPS)
    got = visionhope_gated_layernorm(x.to(device), weight.to(device), bias.to(device), EPS)
    # the mean of 48 values near 200 is off by at most 200 * 2^-23, the spread is 1
    compare(got, want, tolerance(dtype, 48) + 200 * 2.0 ** -23, "offset rows")


@pytest.mark.parametrize("dtype", DTYPES)
def test_slices_and_odd_addresses(device, dtype):
    from visionhope_amd.utils.gated_norm import visionhope_gated_layernorm

    x, weight, bias, gate = (t.to(device) for t in _inputs((3, 21, 64), dtype, seed=20))
    dy = randn(3, 21, 64, seed=25).to(device, dtype)

    def both(xv, gv, dyv):
        leaves = [t.detach().requires_grad_() for t in (xv, gv)]
        y = visionhope_gated_layernorm(leaves[0], weight, bias, EPS, gate=leaves[1])
        return [y.detach(), *torch.autograd.grad(y, leaves, dyv)]

    def wide(t):
        w = torch.zeros(3, 21, 130, device=device, dtype=dtype)
        w[..., 66:] = t
        return w[..., 66:]

    def odd(t):
        o = torch.empty(t.numel() + 1, device=device, dtype=dtype)[1:].view(t.shape)
        return o.copy_(t)

    def turned(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    want = both(x, gate, dy)
    for view in (wide, odd, turned, lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
        got = both(view(x), view(gate), view(dy))
        for a, b in zip(got, want):
            # another vector width sums a row in another order
            compare(a, b.double().cpu(), 2 * tolerance(dtype, 64), "view")
    ones = torch.ones((), device=device, dtype=dtype).expand(3, 21, 64)
    for a, b in zip(both(x, gate, ones), both(x, gate, ones.contiguous())):
        assert torch.equal(a, b)


def test_repeats_bit_by_bit_on_any_stream_and_in_a_graph(device):
    from visionhope_amd.utils.gated_norm import visionhope_gated_layernorm

    x, weight, bias, gate = (t.to(device) for t in _inputs((5000, 96), torch.bfloat16, seed=30))
    dy = randn(5000, 96, seed=35).to(device, torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (x, weight, bias, gate)]

    def step():
        y = visionhope_gated_layernorm(*leaves[:3], EPS, gate=leaves[3])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = step()
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream(device).wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(want, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for round_ in range(3):
        with torch.no_grad():
            leaves[0].copy_(x * (round_ + 1) + round_)
        want = step()
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, captured):
            assert torch.equal(a, b), f"replay {round_}"


def test_refusals(device):
    from visionhope_amd.utils.gated_norm import visionhope_gated_layernorm

    x, weight, bias, gate = (t.to(device) for t in _inputs((3, 16), torch.float32, seed=40))
    bad = [
        (ValueError, "CUDA", lambda: visionhope_gated_layernorm(x.cpu(), weight, bias)),
        (TypeError, "FP16, BF16 and FP32", lambda: visionhope_gated_layernorm(x.double(), weight, bias)),
        (ValueError, "nonempty", lambda: visionhope_gated_layernorm(x[:0], weight, bias)),
        (ValueError, "8192", lambda: visionhope_gated_layernorm(torch.zeros(1, 8193, device=device), weight, bias)),
        (ValueError, "weight", lambda: visionhope_gated_layernorm(x, weight[:4], bias)),
        (ValueError, "bias", lambda: visionhope_gated_layernorm(x, weight, None)),
        (ValueError, "gate", lambda: visionhope_gated_layernorm(x, weight, bias, gate=gate[:2])),
        (TypeError, "gate", lambda: visionhope_gated_layernorm(x, weight, bias, gate=gate.half())),
    ]
    for error, match, call in bad:
        with pytest.raises(error, match=match):
            call()


def test_forward_mode_is_refused_and_saved_tensors_may_change_strides(device):
    from torch.autograd import forward_ad

    from visionhope_amd.utils.gated_norm import visionhope_gated_layernorm

    leaves = [t.to(device).requires_grad_() for t in _inputs((9, 48), torch.float32, seed=95)]
    dy = randn(9, 48, seed=96).to(device)

    def call(x, weight, bias, gate):
        return visionhope_gated_layernorm(x, weight, bias, EPS, gate=gate)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            with pytest.raises(NotImplementedError):
                call(forward_ad.make_dual(leaves[0].detach(), torch.ones_like(leaves[0])), *leaves[1:])
    want = torch.autograd.grad(call(*leaves), leaves, dy)

    def spread(t):   # the same values, every other element of a wider tensor
        wide = torch.zeros(*t.shape, 2, device=t.device, dtype=t.dtype)
        wide[..., 0] = t
        return wide[..., 0]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread):
        got = torch.autograd.grad(call(*leaves), leaves, dy)
    for a, b in zip(got, want):
        assert torch.equal(a, b)

"""Linear attention's 16-bit results are those of FP32 products, rounded once, whatever else a call returns."""

import pytest
import torch

from oracle.oracle_torch import linear_attention_torch
from tests.helpers import randn
from tests.token_lines import gradients

pytestmark = pytest.mark.gpu

HALVES = (torch.bfloat16, torch.float16)


def _inputs(dim, dtype, batch=2, length=300, heads=4):
    rungs = 1 + 8 * torch.arange(heads) / (heads - 1)
    q, k, v, do = (randn(batch, length, heads, dim, seed=s).to(dtype) for s in (1, 2, 3, 4))
    return q, k, v, torch.log1p(-torch.exp2(-rungs)), do


def _own(device, q, k, v, log_decay, do, return_state, state_gradient=False):
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention

    leaves = [t.to(device).requires_grad_() for t in (q, k, v)]
    start = torch.zeros(*q.shape[:1], q.shape[2], q.shape[3], v.shape[3], device=device, requires_grad=state_gradient)
    out = visionhope_linear_attention(*leaves, log_decay.to(device), state=start, return_state=return_state)
    o = out[0] if return_state else out
    return [o.detach(), *torch.autograd.grad(o, leaves + [start] * state_gradient, do.to(device))[:3]]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim", [16, 64, 128])
def test_results_do_not_depend_on_what_else_is_returned(device, dtype, dim):
    args = (device, *_inputs(dim, dtype))
    want = _own(*args, False)
    for more in ((True,), (False, True), (True, True)):
        for name, a, b in zip(("o", "dq", "dk", "dv"), _own(*args, *more), want):
            assert torch.equal(a, b), (more, name)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim", [16, 64, 128])
def test_few_results_are_not_the_nearest(device, dtype, dim):
    """The share of results that are not the exact value rounded to the type.

    An error e turns a rounding with the probability |e| / u, u the distance of neighbours at the
    result, at least half a step's double 2^-8 (bf16; FP16 2^-11) of it.  The errors are those of FP32
    sums: each of 64 to 128 additions of a product, and of as many of the sum over tokens, leaves 2^-25 of
    the running value, and a power of the decay 2^-22: together 2^-20.5 of the results' spread s.  For
    values spread normally the mean of min(1, e / (u / |x| |x|)) is 0.8 ln(1 / p) p with p = e s / u, six
    at these sizes, three quarters of it for the larger u within a binade: 4.5 * 2^(8 - 20.5).
    Operands of 16 bits err by 2^-17 of a term: ten times that.
    """
    q, k, v, log_decay, do = _inputs(dim, dtype)
    want, grads = gradients(lambda *a: linear_attention_torch(*a, log_decay.double()), (q, k, v), (do, None))
    got = _own(device, q, k, v, log_decay, do, False)
    bits = 8 if dtype == torch.bfloat16 else 11
    for name, a, b in zip(("o", "dq", "dk", "dv"), got, (want[0], *grads)):
        share = (a.cpu() != b.to(dtype)).double().mean().item()
        assert share <= 4.5 * 2.0 ** (bits - 20.5), (name, share)

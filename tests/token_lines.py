"""Inputs and tolerances of the token-line operators' tests."""

import math

import torch

DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def half_step(dtype):
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def tolerance(dtype, terms):
    """Relative error (normwise, and of the largest element) of a result that was formed in FP32
    from ``terms`` values in a row and rounded once to ``dtype``.

    About four roundings a term, each of at most 2^-24 of the running value and independent of
    the others, grow as the square root of their number; the constant part (64 roundings)
    stands for exponentials, softplus and the sum over states.  The factor 16 covers the
    cancellation between the terms (a sum is smaller than its terms by their spread) and the
    largest of some thousand elements (4 standard deviations).
    """
    own = half_step(dtype) if dtype != torch.float32 else 0.0
    return own + 16 * math.sqrt(4 * terms + 64) * 2.0 ** -24


def gradients(fn, inputs, cotangents):
    """Outputs of ``fn`` in float64 on the CPU and the gradients of sum(out * cotangent) in the
    inputs that are given (None stays None)."""
    leaves = [None if t is None else t.detach().double().cpu().requires_grad_() for t in inputs]
    outs = fn(*leaves)
    outs = outs if isinstance(outs, tuple) else (outs,)
    total = sum((o * c.double().cpu()).sum() for o, c in zip(outs, cotangents) if c is not None)
    grads = torch.autograd.grad(total, [t for t in leaves if t is not None], allow_unused=True)
    it = iter(grads)
    return [o.detach() for o in outs], [None if t is None else next(it) for t in leaves]


def compare(got, want, tol, what):
    """``got`` against the float64 ``want``: error of every element at most ``tol`` of the largest
    value, and normwise at most ``tol``."""
    assert tuple(got.shape) == tuple(want.shape), f"{what}: shape {tuple(got.shape)} vs {tuple(want.shape)}"
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    diff = got - want
    scale, norm = want.abs().max().item(), want.norm().item()
    if scale == 0.0:
        assert diff.abs().max().item() == 0.0, f"{what}: expected zeros, got up to {got.abs().max():.3e}"
        return
    worst, rel = diff.abs().max().item() / scale, diff.norm().item() / norm
    assert worst <= tol and rel <= tol, f"{what}: elementwise {worst:.3e}, normwise {rel:.3e} > {tol:.3e}"

"""The state space mixer: convolution, scan and gated norm together, as a model runs them,
against the same module in float64 from the oracle's operators."""

import pytest
import torch
from torch.nn import functional as F

from oracle.oracle_torch import causal_conv_torch, gated_layernorm_torch, state_space_scan_torch
from tests.helpers import randn
from tests.token_lines import compare, half_step, tolerance

pytestmark = pytest.mark.gpu


def _mixer(norm, seed=0, dim=48, **kw):
    from visionhope_amd.models import StateSpaceMixer

    torch.manual_seed(seed)
    mixer = StateSpaceMixer(dim, norm=norm, **kw)
    with torch.no_grad():
        for p in mixer.parameters():
            p.add_(torch.randn(p.shape) * 0.1)
    return mixer


def _reference(mixer, x, lengths=None):
    """The module's formula in float64 on the CPU; returns the output and the parameters used."""
    p = {k: v.detach().double().cpu().requires_grad_() for k, v in mixer.named_parameters()}
    h, gate = F.linear(x, p["in_proj.weight"]).chunk(2, -1)
    h, _ = causal_conv_torch(h, p["conv.weight"], p["conv.bias"], True, None, lengths)
    dt, B, C = F.linear(h, p["x_proj.weight"]).split((mixer.dt_rank, mixer.state_dim, mixer.state_dim), -1)
    dt = F.linear(dt, p["dt_proj.weight"])
    norm = "norm_weight" in p
    y, _ = state_space_scan_torch(h, dt, -p["A_log"].exp(), B[:, :, None], C[:, :, None], p["D"], None if norm else gate,
                                  p["dt_proj.bias"], True, None, lengths)
    if norm:
        y = gated_layernorm_torch(y, p["norm_weight"], p["norm_bias"], mixer.eps, gate)
    out = F.linear(y, p["out_proj.weight"])
    if lengths is not None:
        out = torch.where((torch.arange(x.shape[1])[None] < lengths[:, None])[..., None], out, 0.0)
    return out, p


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("ragged", [False, True])
def test_training_step(device, norm, ragged):
    mixer = _mixer(norm).to(device)
    lengths = torch.tensor([90, 17, 1]) if ragged else None
    x, dout = randn(3, 90, 48, seed=1), randn(3, 90, 48, seed=2)
    xr = x.double().requires_grad_()
    want, params = _reference(mixer, xr, lengths)
    (want * dout.double()).sum().backward()
    xg = x.to(device).requires_grad_()
    out = mixer(xg, lengths=None if lengths is None else lengths.to(device))
    # the library's FP32 products of up to 96 terms before and after
    tol = tolerance(torch.float32, 90 + 4 * 96)
    compare(out, want.detach(), tol, "output")
    (out * dout.to(device)).sum().backward()
    compare(xg.grad, xr.grad, tol, "dx")
    tol = tolerance(torch.float32, 3 * 90 * 4 + 4 * 96)
    for name, p in mixer.named_parameters():
        compare(p.grad, params[name].grad, tol, f"d{name}")


@pytest.mark.parametrize("norm", [True, False])
def test_checkpointed_step_has_the_same_gradients(device, norm):
    from torch.utils.checkpoint import checkpoint

    mixer = _mixer(norm, state_dim=5, conv_taps=3).to(device)
    x = randn(2, 40, 48, seed=3).to(device)
    grads = []
    for run in (mixer, lambda t: checkpoint(mixer, t, use_reentrant=False)):
        mixer.zero_grad()
        leaf = x.clone().requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out = run(leaf)
        assert out.dtype == torch.bfloat16
        out.float().square().sum().backward()
        grads.append([leaf.grad, *(p.grad for p in mixer.parameters())])
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norm", [True, False])
def test_serving_prompt_then_tokens(device, dtype, norm):
    """A padded batch of prompts, then tokens one by one in a captured graph, against the whole
    sequences at once."""
    mixer = _mixer(norm).to(device, dtype).eval()
    lengths = torch.tensor([20, 7, 0], device=device)
    x = randn(3, 26, 48, seed=4).to(device, dtype)
    with torch.no_grad():
        out, state = mixer(x[:, :20], lengths=lengths, return_state=True)
        token = torch.empty(3, 48, device=device, dtype=dtype)
        warm = tuple(t.clone() for t in state)
        token.copy_(x[:, 20])
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            mixer.step(token, warm)   # the library's products choose their kernels outside the capture
        torch.cuda.current_stream(device).wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = mixer.step(token, state)
        steps = []
        for t in range(20, 26):
            token.copy_(x[:, t])
            graph.replay()
            steps.append(captured.clone())
        torch.cuda.synchronize()
        steps = torch.stack(steps, 1)
        for i, n in enumerate(lengths.tolist()):
            whole = mixer(torch.cat((x[i:i + 1, :n], x[i:i + 1, 20:]), 1))
            # the library's product of one row sums in another order: in bf16 each activation of
            # the chain (five of them) may round to its neighbour
            tol = 2 * tolerance(torch.float32, 26 + 4 * 96) if dtype == torch.float32 else 5 * 4 * half_step(dtype)
            compare(steps[i], whole[0, n:].double().cpu(), tol, f"tokens behind {n}")
            if n:
                compare(out[i, :n], whole[0, :n].double().cpu(), tol, f"prompt of {n}")
            assert not out[i, n:].any()


def test_inference_mode(device):
    mixer = _mixer(True).to(device).eval()
    x = randn(2, 9, 48, seed=6).to(device)
    with torch.no_grad():
        want = mixer(x)
    with torch.inference_mode():
        out, state = mixer(x[:, :8], return_state=True)
        last = mixer.step(x[:, 8], state)
    tol = 2 * tolerance(torch.float32, 9 + 4 * 96)
    compare(torch.cat((out, last[:, None]), 1), want.double().cpu(), tol, "inference mode")


def test_module_surface(device):
    from visionhope_amd.models import StateSpaceMixer

    mixer = StateSpaceMixer(16, state_dim=4).to(device)
    conv, scan = mixer.allocate_state(3, torch.bfloat16)
    assert conv.shape == (3, 3, 32) and conv.dtype == torch.bfloat16
    assert scan.shape == (3, 32, 4) and scan.dtype == torch.float32
    with pytest.raises(ValueError, match="expects"):
        mixer(torch.zeros(2, 16, device=device))
    with pytest.raises(ValueError, match="state_dim"):
        StateSpaceMixer(16, state_dim=33)
    with pytest.raises(RuntimeError, match="inference"):
        mixer.step(torch.zeros(3, 16, device=device), mixer.allocate_state(3))
    with pytest.raises(ValueError, match="CUDA"):
        StateSpaceMixer(16)(torch.zeros(1, 4, 16))

"""The linear attention mixer and its block on maps: projection, attention, gated norm and group norm
together, as a model runs them, against the same modules in float64 from the oracle's operators."""

import pytest
import torch
from torch.nn import functional as F

from oracle.oracle_torch import gated_layernorm_torch, group_norm_torch, linear_attention_torch
from tests.helpers import randn
from tests.token_lines import compare, half_step, tolerance

pytestmark = pytest.mark.gpu

DIM = 48


def _mixer(learn_decay=False, seed=0, **kw):
    from visionhope_amd.models import LinearAttentionMixer

    torch.manual_seed(seed)
    mixer = LinearAttentionMixer(DIM, heads=3, learn_decay=learn_decay, **kw)
    with torch.no_grad():
        mixer.log_rate.copy_(torch.tensor([-3.0, -1.0, 0.5]))
        for p in mixer.parameters():
            p.add_(torch.randn(p.shape) * 0.1)
    return mixer


def _reference(mixer, x, lengths=None, params=None):
    """The module's formula in float64 on the CPU; returns the output and the parameters used."""
    p = params or {k: v.detach().double().cpu().requires_grad_() for k, v in mixer.named_parameters()}
    rate = p["log_rate"] if "log_rate" in p else mixer.log_rate.double().cpu()
    widths = [mixer.heads * w for w in (mixer.key_dim, mixer.key_dim, mixer.value_dim, mixer.value_dim)]
    q, k, v, gate = (t.unflatten(-1, (mixer.heads, -1)) for t in F.linear(x, p["in_proj.weight"]).split(widths, -1))
    o, _ = linear_attention_torch(q, k, v, -rate.exp(), None, None, lengths)
    y = gated_layernorm_torch(o, p["norm_weight"], p["norm_bias"], mixer.eps, gate)
    out = F.linear(y.flatten(-2), p["out_proj.weight"])
    if lengths is not None:
        out = torch.where((torch.arange(x.shape[1])[None] < lengths[:, None])[..., None], out, 0.0)
    return out, p


@pytest.mark.parametrize("learn_decay", [True, False])
@pytest.mark.parametrize("ragged", [False, True])
def test_training_step(device, learn_decay, ragged):
    mixer = _mixer(learn_decay, key_dim=20, value_dim=24).to(device)
    lengths = torch.tensor([90, 17, 1]) if ragged else None
    x, dout = randn(3, 90, DIM, seed=1), randn(3, 90, DIM, seed=2)
    xr = x.double().requires_grad_()
    want, params = _reference(mixer, xr, lengths)
    (want * dout.double()).sum().backward()
    xg = x.to(device).requires_grad_()
    out = mixer(xg, lengths=None if lengths is None else lengths.to(device))
    # The library's FP32 products of up to 264 terms before and after.  The norm divides a head's
    # outputs by their spread, and what it divides has the errors of sums that may be larger than they
    # are: four times the room of the sums alone.
    tol = 4 * tolerance(torch.float32, 90 + 4 * 264)
    compare(out, want.detach(), tol, "output")
    (out * dout.to(device)).sum().backward()
    compare(xg.grad, xr.grad, tol, "dx")
    tol = 4 * tolerance(torch.float32, 3 * 90 * 64 + 4 * 264)
    for name, p in mixer.named_parameters():
        compare(p.grad, params[name].grad, tol, f"d{name}")


@pytest.mark.parametrize("learn_decay", [True, False])
def test_checkpointed_step_has_the_same_gradients(device, learn_decay):
    from torch.utils.checkpoint import checkpoint

    mixer = _mixer(learn_decay).to(device)
    x = randn(2, 40, DIM, seed=3).to(device)
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
def test_serving_prompt_then_tokens(device, dtype):
    """A padded batch of prompts, then tokens one by one in a captured graph, against the whole
    sequences at once."""
    mixer = _mixer().to(device, dtype).eval()
    lengths = torch.tensor([70, 7, 0], device=device)
    x = randn(3, 76, DIM, seed=4).to(device, dtype)
    with torch.no_grad():
        out, state = mixer(x[:, :70], lengths=lengths, return_state=True)
        token = torch.empty(3, DIM, device=device, dtype=dtype)
        warm = state.clone()
        token.copy_(x[:, 70])
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
        for t in range(70, 76):
            token.copy_(x[:, t])
            graph.replay()
            steps.append(captured.clone())
        torch.cuda.synchronize()
        steps = torch.stack(steps, 1)
        for i, n in enumerate(lengths.tolist()):
            whole = mixer(torch.cat((x[i:i + 1, :n], x[i:i + 1, 70:]), 1))
            # in bf16 each activation of the chain (four of them) may round to its neighbour where a
            # product of one row sums in another order
            tol = 8 * tolerance(torch.float32, 76 + 4 * 96) if dtype == torch.float32 else 4 * 4 * half_step(dtype)
            compare(steps[i], whole[0, n:].double().cpu(), tol, f"tokens behind {n}")
            if n:
                compare(out[i, :n], whole[0, :n].double().cpu(), tol, f"prompt of {n}")
            assert not out[i, n:].any()


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_what_stands_behind_the_end_has_no_part(device, index):
    mixer = _mixer(True).to(device)
    lengths = torch.tensor([40, 0, 17, 1], dtype=index, device=device)
    x, dout = randn(4, 40, DIM, seed=5).to(device), randn(4, 40, DIM, seed=6).to(device)
    behind = (torch.arange(40, device=device) >= lengths[:, None])[..., None]
    results = []
    for fill in (0.0, float("nan"), float("inf")):
        leaf = torch.where(behind, fill, x).requires_grad_()
        out, state = mixer(leaf, lengths=lengths, return_state=True)
        grads = torch.autograd.grad(out, [leaf, *mixer.parameters()], torch.where(behind, fill, dout))
        with torch.no_grad():
            assert torch.equal(mixer(leaf, lengths=lengths), out)
        results.append([out.detach(), state.detach(), *grads])
    names = ["out", "state", "x", *(n for n, _ in mixer.named_parameters())]
    for other in results[1:]:
        for name, a, b in zip(names, results[0], other):
            assert torch.isfinite(b).all(), name
            assert torch.equal(a, b), name
    assert not results[0][0][behind.expand_as(x)].any() and not results[0][2][behind.expand_as(x)].any()


@pytest.mark.parametrize("learn_decay", [True, False])
def test_captured_training_step(device, learn_decay):
    """Forward and backward of the whole module in one graph, replayed with new inputs; a graph of the
    same leaves that still lives on the default stream is refused first."""
    mixer = _mixer(learn_decay).to(device)
    lengths = torch.tensor([70, 0, 17, 1], dtype=torch.int32, device=device)
    x, dout = randn(4, 70, DIM, seed=7).to(device), randn(4, 70, DIM, seed=8).to(device)
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
            compare(a, b.double().cpu(), tolerance(torch.float32, 4 * 70 + 96), f"replay {replay} {name}")


def _block_reference(block, x):
    p = {k: v.detach().double().cpu().requires_grad_() for k, v in block.named_parameters()}
    mixed = {k[6:]: v for k, v in p.items() if k.startswith("mixer.")}
    tokens = group_norm_torch(x, block.norm.groups, p["norm.weight"], p["norm.bias"], block.norm.eps).flatten(2).transpose(1, 2)
    if block.reverse:
        tokens = tokens.flip(1)
    tokens, _ = _reference(block.mixer, tokens, params=mixed)
    if block.reverse:
        tokens = tokens.flip(1)
    return x + tokens.transpose(1, 2).reshape(x.shape), p


@pytest.mark.parametrize("reverse", [False, True])
def test_block_on_maps(device, reverse):
    """Group norm, attention over the pixels and gated norm in a run, forward and backward."""
    from visionhope_amd.models import LinearAttentionBlock

    torch.manual_seed(3)
    block = LinearAttentionBlock(DIM, heads=3, reverse=reverse, learn_decay=True)
    with torch.no_grad():
        for p in block.parameters():
            p.add_(torch.randn(p.shape) * 0.1)
    block = block.to(device)
    x, dout = randn(2, DIM, 11, 9, seed=9), randn(2, DIM, 11, 9, seed=10)
    xr = x.double().requires_grad_()
    want, params = _block_reference(block, xr)
    (want * dout.double()).sum().backward()
    xg = x.to(device).contiguous(memory_format=torch.channels_last).requires_grad_()
    out = block(xg)
    tol = 4 * tolerance(torch.float32, 99 + 4 * 192)
    compare(out, want.detach(), tol, "output")
    (out * dout.to(device)).sum().backward()
    compare(xg.grad, xr.grad, tol, "dx")
    tol = 4 * tolerance(torch.float32, 2 * 99 * 64 + 4 * 192)
    for name, p in block.named_parameters():
        compare(p.grad, params[name].grad, tol, f"d{name}")
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        half = block(xg.to(torch.bfloat16))
    assert half.dtype == torch.bfloat16
    # seven roundings to bf16 on the way, of values and weights
    compare(half, want.detach(), 7 * 4 * half_step(torch.bfloat16), "autocast")


def test_module_surface(device):
    from visionhope_amd.models import LinearAttentionMixer

    mixer = LinearAttentionMixer(32, heads=2).to(device)
    assert mixer.allocate_state(3).shape == (3, 2, 16, 16)
    assert "log_rate" in mixer.state_dict() and "log_rate" not in dict(mixer.named_parameters())
    with pytest.raises(ValueError, match="expects"):
        mixer(torch.zeros(2, 32, device=device))
    with pytest.raises(ValueError, match="divide"):
        LinearAttentionMixer(32, heads=3)
    with pytest.raises(ValueError, match="key_dim"):
        LinearAttentionMixer(512, heads=2)
    with pytest.raises(RuntimeError, match="inference"):
        mixer.step(torch.zeros(3, 32, device=device), mixer.allocate_state(3))
    with pytest.raises(ValueError, match="CUDA"):
        LinearAttentionMixer(32)(torch.zeros(1, 4, 32))

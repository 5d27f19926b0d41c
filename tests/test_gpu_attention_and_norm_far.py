"""Linear attention and group norm on tensors beyond 32-bit offsets, far-apart rows, other devices' streams
and calls that overlap."""

import pytest
import torch

from oracle.oracle_torch import group_norm_torch, linear_attention_torch
from tests.helpers import randn
from tests.token_lines import compare, gradients, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("token", [(1 << 23) + 8, (1 << 24) + 8])
@pytest.mark.parametrize("dims", [(16, 16), (5, 7)])
def test_tokens_far_apart(device, token, dims):
    """Rows 2^23 elements apart are read in place (300 of them: offsets beyond 2^32 bytes), rows beyond
    2^24 are copied first."""
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention

    length = 300 if token < 1 << 24 else 70
    made = [randn(1, length, 2, d, seed=i).bfloat16() for i, d in enumerate((dims[0], dims[0], dims[1], dims[1]))]
    a = torch.tensor([-0.7, -0.01])
    want, grads = gradients(lambda q, k, v: linear_attention_torch(q, k, v, a.double())[0], made[:3], (made[3],))
    memory = torch.empty(length * token, device=device, dtype=torch.bfloat16)
    views = []
    for i, t in enumerate(made):
        view = memory.as_strided(t.shape, (length * token, token, t.shape[3], 1), 512 * i)
        views.append(view.copy_(t))
    leaves = [t.detach().requires_grad_() for t in views[:3]]
    o = visionhope_linear_attention(*leaves, a.to(device))
    got = torch.autograd.grad(o, leaves, views[3])
    compare(o, want[0], tolerance(torch.bfloat16, length + 16), "o")
    for name, x, y in zip("qkv", got, grads):
        compare(x, y, tolerance(torch.bfloat16, length + 16), f"d{name}")


def test_maps_beyond_31_bits(device):
    """A map of more than 2^31 values made of one small map's rows again and again: the statistics are the
    small map's, and so is every repetition of it."""
    from visionhope_amd.utils.group_norm import visionhope_group_norm

    small, repeats = randn(1, 32, 8, 256, seed=1).bfloat16(), 32800
    weight, bias = 1 + 0.1 * randn(32, seed=2), 0.1 * randn(32, seed=3)
    dy = randn(1, 32, 8, 256, seed=4).bfloat16()
    want, grads = gradients(lambda x, w, b: group_norm_torch(x, 2, w, b, 1e-5, "silu"), (small, weight, bias), (dy,))

    def tall(t):
        return t.to(device).permute(0, 2, 3, 1).repeat(1, repeats, 1, 1).permute(0, 3, 1, 2)

    x, dy = tall(small).requires_grad_(), tall(dy)
    assert x.numel() > 1 << 31
    w, b = weight.to(device).requires_grad_(), bias.to(device).requires_grad_()
    y = visionhope_group_norm(x, 2, w, b, 1e-5, activation="silu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    for name, got, one in (("y", y.detach(), want[0]), ("dx", dx, grads[0])):
        parts = got.permute(0, 2, 3, 1).view(repeats, 8, 256, 32)
        assert torch.equal(parts, parts[:1].expand_as(parts)), name
        compare(parts[0].permute(2, 0, 1)[None], one, tolerance(torch.bfloat16, 8 * 256 * 16), name)
    for name, got, one in (("dweight", dw, grads[1]), ("dbias", db, grads[2])):
        compare(got / repeats, one, tolerance(torch.float32, 8 * 256 * 128), name)


def test_two_streams_at_once_and_two_graphs(device):
    """Calls that overlap on two streams, and replays of two graphs in turn, do not share workspaces."""
    from visionhope_amd.utils.group_norm import visionhope_group_norm
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention

    def inputs(seed):
        q, k, v = (randn(2, 1500, 4, 64, seed=seed + i).to(device, torch.bfloat16).requires_grad_() for i in range(3))
        x = randn(4, 64, 60, 60, seed=seed + 3).to(device, torch.bfloat16).contiguous(memory_format=torch.channels_last)
        return q, k, v, x.requires_grad_()

    a = torch.tensor([-0.5, -0.1, -0.01, -0.002], device=device)
    weight, bias = torch.ones(64, device=device), torch.zeros(64, device=device)

    def work(made):
        q, k, v, x = made
        o, state = visionhope_linear_attention(q, k, v, a, return_state=True)
        y = visionhope_group_norm(x, 4, weight, bias, activation="gelu")
        grads = torch.autograd.grad((o, y), made, (torch.ones_like(o), x.detach()))
        return [o.detach(), state.detach(), y.detach(), *grads]

    sets = [inputs(10), inputs(20)]
    want = [work(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    for _ in range(3):
        got = []
        for s, stream in zip(sets, streams):
            stream.wait_stream(torch.cuda.current_stream(device))
            with torch.cuda.stream(stream):
                got.append(work(s))
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            for p, q in zip(x, y):
                assert torch.equal(p, q)
    got = None
    graphs, captured = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured.append(work(s))
        graphs.append(graph)
    for _ in range(3):
        for t in captured[0] + captured[1]:
            t.zero_()
        for graph in graphs:
            graph.replay()
        again = work(sets[0])
        torch.cuda.synchronize()
        for x, y in zip([*captured, again], [*want, want[0]]):
            for p, q in zip(x, y):
                assert torch.equal(p, q)


def test_the_same_tensor_three_times(device):
    """q, k and v of one tensor: its gradient is the three gradients' sum."""
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention

    x, do = randn(2, 100, 2, 32, seed=31), randn(2, 100, 2, 32, seed=32)
    a = torch.tensor([-0.3, -0.02])
    want, (grad,) = gradients(lambda t: linear_attention_torch(t, t, t, a.double(), 0.05)[0], (x,), (do,))
    leaf = x.to(device).requires_grad_()
    o = visionhope_linear_attention(leaf, leaf, leaf, a.to(device), scale=0.05)
    compare(o, want[0], tolerance(torch.float32, 132), "o")
    (got,) = torch.autograd.grad(o, leaf, do.to(device))
    compare(got, grad, tolerance(torch.float32, 3 * 132), "d")


def test_prompts_of_one_token_and_a_long_line(device):
    """One token beside the step form, and 70,000 tokens of one head (many segments) whose slow decay
    keeps the first of them, against the float64 recurrence by chunks."""
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention, visionhope_linear_attention_step

    q, k, v = (randn(3, 1, 2, 32, seed=i).to(device, torch.bfloat16) for i in (41, 42, 43))
    a, s = torch.tensor([-0.4, -0.01], device=device), randn(3, 2, 32, 32, seed=44).to(device)
    o, last = visionhope_linear_attention(q, k, v, a, state=s, return_state=True)
    moved = torch.empty_like(s)
    step = visionhope_linear_attention_step(q[:, 0], k[:, 0], v[:, 0], a, s, new_state=moved)
    compare(o[:, 0], step.double().cpu(), 2 * tolerance(torch.bfloat16, 64), "o")
    compare(last, moved.double().cpu(), tolerance(torch.float32, 2), "state")

    length, rate = 70_001, -2e-5
    q, k, v = (randn(1, length, 1, 16, seed=i).to(device) for i in (45, 46, 47))
    a = torch.tensor([rate], device=device)
    o, last = visionhope_linear_attention(q, k, v, a, return_state=True)
    age = torch.arange(length - 1, -1, -1, device=device).double()
    want = ((k[0, :, 0].double() * torch.exp(a.double() * age)[:, None]).t() @ v[0, :, 0].double())
    compare(last[0, 0], want.cpu(), tolerance(torch.float32, length), "last state")
    for t in (0, 1, 31, 32, 63, 64, 35_000, length - 1):
        weight = torch.exp(a.double() * torch.arange(t, -1, -1, device=device).double())
        row = ((k[0, :t + 1, 0].double() @ q[0, t, 0].double()) * weight) @ v[0, :t + 1, 0].double() * 0.25
        compare(o[0, t, 0], row.cpu(), tolerance(torch.float32, t + 33), f"token {t}")

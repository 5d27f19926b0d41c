"""Argument checks of the token-line entry points: every call below is refused on the host,
before any GPU work, with a status code and a message."""

import ctypes

import pytest

from visionhope_amd.utils import hip

P = 0x1000   # never dereferenced: validation fails first
F32 = hip.VH_DTYPE_F32


@pytest.fixture(scope="module")
def lib():
    return hip.load_library()


def _call(lib, name, defaults, **kw):
    assert not set(kw) - set(defaults), kw
    args = {**defaults, **kw}
    return getattr(lib, name)(*args.values())


CONV = dict(x=P, xb=80, xt=8, io=F32, weight=P, bias=None, silu=0, state=None, lengths=None, y=P, new_state=None,
            B=2, N=10, C=8, taps=4, stream=None)
CONV_BACK = dict(dy=P, dyb=80, dyt=8, x=P, xb=80, xt=8, io=F32, weight=P, bias=None, silu=0, state=None, lengths=None,
                 dnew=None, dx=P, dweight=P, dbias=P, dstate=None, B=2, N=10, C=8, taps=4, ws=P, wsn=1 << 30,
                 stream=None)
CONV_STEP = dict(x=P, xb=8, io=F32, weight=P, bias=None, silu=0, state=P, new_state=P, y=P, B=2, C=8, taps=4, stream=None)
SCAN = dict(x=P, xb=80, xt=8, dt=P, dtb=80, dtt=8, gate=None, gb=0, gt=0, io=F32, b=P, bb=160, bt=16, c=P, cb=160,
            ct=16, A=P, D=None, bias=None, softplus=1, state=None, lengths=None, y=P, new_state=None, kept=None,
            B=2, N=10, C=8, groups=1, states=16, ws=P, wsn=1 << 30, stream=None)
SCAN_BACK = dict(dy=P, dyb=80, dyt=8, x=P, xb=80, xt=8, dt=P, dtb=80, dtt=8, gate=None, gb=0, gt=0, io=F32, b=P,
                 bb=160, bt=16, c=P, cb=160, ct=16, A=P, D=None, bias=None, softplus=1, lengths=None, kept=P,
                 dnew=None, dx=P, ddt=P, dgate=None, db=P, dc=P, dA=P, dD=None, dbias=None, dstate=None, B=2, N=10,
                 C=8, groups=1, states=16, ws=P, wsn=1 << 30, stream=None)
SCAN_STEP = dict(x=P, xb=8, dt=P, dtb=8, gate=None, gb=0, io=F32, b=P, bb=16, c=P, cb=16, A=P, D=None, bias=None,
                 softplus=1, state=P, new_state=P, y=P, B=2, C=8, groups=1, states=16, stream=None)
NORM = dict(x=P, xr=8, gate=None, gr=0, io=F32, weight=P, bias=P, y=P, mean=None, rstd=None, rows=3, C=8, eps=1e-6,
            stream=None)
NORM_BACK = dict(dy=P, dyr=8, x=P, xr=8, gate=None, gr=0, io=F32, weight=P, bias=P, mean=P, rstd=P, dx=P, dgate=None,
                 dweight=P, dbias=P, rows=3, C=8, ws=P, wsn=1 << 30, stream=None)

REFUSED = [
    ("vh_causal_conv_forward", CONV, dict(io=7), hip.VH_ERR_DTYPE, "io_dtype"),
    ("vh_causal_conv_forward", CONV, dict(N=0), hip.VH_ERR_SHAPE, "nonempty"),
    ("vh_causal_conv_forward", CONV, dict(taps=1), hip.VH_ERR_SHAPE, "taps"),
    ("vh_causal_conv_forward", CONV, dict(taps=9), hip.VH_ERR_SHAPE, "taps"),
    ("vh_causal_conv_forward", CONV, dict(x=None), hip.VH_ERR_ARG, "null"),
    ("vh_causal_conv_forward", CONV, dict(N=1 << 31), hip.VH_ERR_SHAPE, "range"),
    ("vh_causal_conv_forward", CONV, dict(B=1 << 23, N=1 << 20, C=1 << 12), hip.VH_ERR_SHAPE, "one launch"),
    ("vh_causal_conv_backward", CONV_BACK, dict(wsn=16), hip.VH_ERR_WORKSPACE, "workspace"),
    ("vh_causal_conv_backward", CONV_BACK, dict(dx=None), hip.VH_ERR_ARG, "null"),
    ("vh_causal_conv_step", CONV_STEP, dict(state=None), hip.VH_ERR_ARG, "null"),
    ("vh_causal_conv_forward", CONV, dict(state=P, new_state=P), hip.VH_ERR_ARG, "overlap"),
    ("vh_causal_conv_step", CONV_STEP, dict(new_state=P + 2 * 3 * 8 * 4 - 4), hip.VH_ERR_ARG, "overlap"),
    ("vh_causal_conv_step", CONV_STEP, dict(state=P + 4), hip.VH_ERR_ARG, "overlap"),
    ("vh_causal_conv_step", CONV_STEP, dict(taps=0), hip.VH_ERR_SHAPE, "taps"),
    ("vh_state_space_forward", SCAN, dict(io=-1), hip.VH_ERR_DTYPE, "io_dtype"),
    ("vh_state_space_forward", SCAN, dict(states=0), hip.VH_ERR_SHAPE, "states"),
    ("vh_state_space_forward", SCAN, dict(states=33), hip.VH_ERR_SHAPE, "states"),
    ("vh_state_space_forward", SCAN, dict(groups=3), hip.VH_ERR_SHAPE, "groups"),
    ("vh_state_space_forward", SCAN, dict(C=1 << 16, groups=1 << 16), hip.VH_ERR_SHAPE, "groups"),
    ("vh_state_space_forward", SCAN, dict(b=None), hip.VH_ERR_ARG, "null"),
    ("vh_state_space_forward", SCAN, dict(A=None), hip.VH_ERR_ARG, "null"),
    ("vh_state_space_forward", SCAN, dict(N=4096, wsn=16), hip.VH_ERR_WORKSPACE, "workspace"),
    ("vh_state_space_forward", SCAN, dict(B=1 << 23, C=1 << 20), hip.VH_ERR_SHAPE, "one launch"),
    ("vh_state_space_backward", SCAN_BACK, dict(kept=None), hip.VH_ERR_ARG, "kept"),
    ("vh_state_space_backward", SCAN_BACK, dict(gate=P), hip.VH_ERR_ARG, "dgate"),
    ("vh_state_space_backward", SCAN_BACK, dict(ws=P + 4), hip.VH_ERR_WORKSPACE, "aligned"),
    ("vh_state_space_backward", SCAN_BACK, dict(wsn=16), hip.VH_ERR_WORKSPACE, "workspace"),
    ("vh_state_space_forward", SCAN, dict(state=P, new_state=P + 16), hip.VH_ERR_ARG, "overlap"),
    ("vh_state_space_step", SCAN_STEP, dict(new_state=P + 2 * 8 * 16 * 4 - 4), hip.VH_ERR_ARG, "overlap"),
    ("vh_state_space_step", SCAN_STEP, dict(states=33), hip.VH_ERR_SHAPE, "states"),
    ("vh_state_space_step", SCAN_STEP, dict(B=0), hip.VH_ERR_SHAPE, "nonempty"),
    ("vh_state_space_step", SCAN_STEP, dict(state=None), hip.VH_ERR_ARG, "null"),
    ("vh_gated_layernorm_forward", NORM, dict(C=8193), hip.VH_ERR_SHAPE, "8192"),
    ("vh_gated_layernorm_forward", NORM, dict(rows=0), hip.VH_ERR_SHAPE, "nonempty"),
    ("vh_gated_layernorm_forward", NORM, dict(mean=P), hip.VH_ERR_ARG, "together"),
    ("vh_gated_layernorm_backward", NORM_BACK, dict(gate=P), hip.VH_ERR_ARG, "dgate"),
    ("vh_gated_layernorm_backward", NORM_BACK, dict(wsn=16), hip.VH_ERR_WORKSPACE, "workspace"),
]


@pytest.mark.parametrize("name, defaults, change, status, message", REFUSED,
                         ids=[f"{r[0]}-{next(iter(r[2]))}-{i}" for i, r in enumerate(REFUSED)])
def test_refused_before_any_launch(lib, name, defaults, change, status, message):
    assert _call(lib, name, defaults, **change) == status
    assert message in lib.vh_last_error().decode()


def test_workspace_sizes(lib):
    assert lib.vh_state_space_kept_bytes(2, 33, 70, 1, 16) == 2 * 3 * 16 * 128 * 4
    assert lib.vh_state_space_kept_bytes(2, 33, 70, 2, 8) == 2 * 3 * 8 * 128 * 4
    assert lib.vh_state_space_workspace_bytes(1, 1, 64, 1, 12) == 2 * 16 * 4   # packed B and C, one chunk
    assert lib.vh_state_space_workspace_bytes(0, 5, 64, 1, 16) == 0
    for name, args in (("vh_causal_conv_backward_workspace_bytes", (2, 10, 8, 4)),
                       ("vh_state_space_backward_workspace_bytes", (2, 10, 8, 1, 16)),
                       ("vh_gated_layernorm_backward_workspace_bytes", (3, 8))):
        assert 0 < getattr(lib, name)(*args) < 1 << 20


def test_cpu_tensors_are_refused():
    import torch

    from visionhope_amd.utils.causal_conv import visionhope_causal_conv, visionhope_causal_conv_step
    from visionhope_amd.utils.gated_norm import visionhope_gated_layernorm
    from visionhope_amd.utils.state_space import visionhope_state_space_scan, visionhope_state_space_step

    x, m = torch.zeros(1, 4, 8), torch.zeros(1, 4, 16)
    for call in (lambda: visionhope_causal_conv(x, torch.zeros(8, 4)),
                 lambda: visionhope_causal_conv_step(x[:, 0], torch.zeros(1, 3, 8), torch.zeros(8, 4)),
                 lambda: visionhope_state_space_scan(x, x, torch.zeros(8, 16), m, m),
                 lambda: visionhope_state_space_step(x[:, 0], x[:, 0], torch.zeros(8, 16), m[:, 0], m[:, 0],
                                                     torch.zeros(1, 8, 16)),
                 lambda: visionhope_gated_layernorm(x, torch.ones(8), torch.zeros(8))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_captured_backward_refuses_leaves_of_a_living_default_stream_graph():
    """The capture itself is played: the Function's two calls get the stream and the state."""
    import torch

    from visionhope_amd.utils.token_lines import note_stream, refuse_held_leaves

    class Double(torch.autograd.Function):
        stream, capturing = 0, False

        @staticmethod
        def forward(ctx, x, weight):
            note_stream(ctx, Double.stream)
            return x * weight

        @staticmethod
        def backward(ctx, dy):
            refuse_held_leaves("double", ctx, Double.capturing)
            return dy, dy

    x, weight = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)

    def run(stream, capturing, inputs):
        Double.stream, Double.capturing = stream, capturing
        y = Double.apply(*inputs)
        y.sum().backward()
        return y

    alive = run(0, False, (x, weight))
    for inputs in ((x, weight), (x * 2, weight), (x, weight.detach())):
        with pytest.raises(RuntimeError, match="still alive"):
            run(7, True, inputs)
    run(7, False, (x, weight))               # not a capture
    run(7, True, (x.detach() * 2, weight.clone().detach().requires_grad_()))
    del alive
    alive = run(7, True, (x, weight))        # the graph is gone; one of another stream may live
    run(8, True, (x, weight))

"""Argument checks of the linear attention and group norm entry points: every call below is refused on
the host, before any GPU work, with a status code and a message."""

import pytest

from visionhope_amd.utils import hip

P = 0x1000   # never dereferenced: validation fails first
F32 = hip.VH_DTYPE_F32


@pytest.fixture(scope="module")
def lib():
    return hip.load_library()


def _call(lib, name, defaults, **kw):
    assert not set(kw) - set(defaults), kw
    return getattr(lib, name)(*{**defaults, **kw}.values())


def _lines(*names):
    return {f"{n}{part}": value for n in names for part, value in (("", P), ("b", 320), ("t", 32), ("h", 8))}


SIZES = dict(B=2, N=10, H=4, K=8, V=8)
WS = dict(ws=P, wsn=1 << 30, stream=None)
ATTEND = dict(**_lines("q", "k", "v"), io=F32, decay=P, scale=1.0, state=None, lengths=None, out=P, new_state=None, **SIZES, **WS)
BACK = dict(**_lines("do", "q", "k", "v"), io=F32, decay=P, scale=1.0, state=None, lengths=None, kept=None, dnew=None, dq=P,
            dk=P, dv=P, dstate=None, ddecay=None, **SIZES, **WS)
STEP = dict(q=P, qb=32, qh=8, k=P, kb=32, kh=8, v=P, vb=32, vh=8, io=F32, decay=P, scale=1.0, state=P, new_state=P, out=P, B=2,
            H=4, K=8, V=8, stream=None)
NORM = dict(x=P, io=F32, weight=P, bias=P, act=0, y=P, stats=None, B=2, pixels=10, C=16, G=2, eps=1e-5, **WS)
NORM_BACK = dict(dy=P, x=P, io=F32, weight=P, bias=P, act=0, stats=P, dx=P, dweight=P, dbias=P, B=2, pixels=10, C=16, G=2, **WS)
STATE = 2 * 4 * 8 * 8 * 4   # bytes of a state

REFUSED = [
    ("vh_linear_attention_forward", ATTEND, dict(io=7), hip.VH_ERR_DTYPE, "io_dtype"),
    ("vh_linear_attention_forward", ATTEND, dict(N=0), hip.VH_ERR_SHAPE, "nonempty"),
    ("vh_linear_attention_forward", ATTEND, dict(K=129), hip.VH_ERR_SHAPE, "128"),
    ("vh_linear_attention_forward", ATTEND, dict(V=129), hip.VH_ERR_SHAPE, "128"),
    ("vh_linear_attention_forward", ATTEND, dict(V=0), hip.VH_ERR_SHAPE, "nonempty"),
    ("vh_linear_attention_forward", ATTEND, dict(q=None), hip.VH_ERR_ARG, "null"),
    ("vh_linear_attention_forward", ATTEND, dict(decay=None), hip.VH_ERR_ARG, "null"),
    ("vh_linear_attention_forward", ATTEND, dict(N=1 << 30), hip.VH_ERR_SHAPE, "range"),
    ("vh_linear_attention_forward", ATTEND, dict(B=1 << 20), hip.VH_ERR_SHAPE, "range"),
    ("vh_linear_attention_forward", ATTEND, dict(B=1, H=1 << 21), hip.VH_ERR_SHAPE, "range"),
    ("vh_linear_attention_forward", ATTEND, dict(kt=1 << 24), hip.VH_ERR_SHAPE, "stride"),
    ("vh_linear_attention_forward", ATTEND, dict(vt=-1), hip.VH_ERR_SHAPE, "stride"),
    ("vh_linear_attention_forward", ATTEND, dict(N=4096, wsn=16), hip.VH_ERR_WORKSPACE, "workspace"),
    ("vh_linear_attention_forward", ATTEND, dict(N=4096, ws=P + 4), hip.VH_ERR_WORKSPACE, "workspace"),
    ("vh_linear_attention_forward", ATTEND, dict(state=P, new_state=P + STATE - 4), hip.VH_ERR_ARG, "overlap"),
    ("vh_linear_attention_backward", BACK, dict(dq=None), hip.VH_ERR_ARG, "null"),
    ("vh_linear_attention_backward", BACK, dict(dot=1 << 24), hip.VH_ERR_SHAPE, "stride"),
    ("vh_linear_attention_backward", BACK, dict(N=4096), hip.VH_ERR_ARG, "forward left"),
    ("vh_linear_attention_backward", BACK, dict(N=4096, kept=P, wsn=16), hip.VH_ERR_WORKSPACE, "workspace"),
    ("vh_linear_attention_backward", BACK, dict(ddecay=P, wsn=0), hip.VH_ERR_WORKSPACE, "workspace"),
    ("vh_linear_attention_backward", BACK, dict(ddecay=P, N=1 << 28), hip.VH_ERR_SHAPE, "range"),
    ("vh_linear_attention_backward", BACK, dict(dstate=P, dnew=P + 16), hip.VH_ERR_ARG, "overlap"),
    ("vh_linear_attention_step", STEP, dict(state=None), hip.VH_ERR_ARG, "null"),
    ("vh_linear_attention_step", STEP, dict(new_state=P + STATE - 4), hip.VH_ERR_ARG, "overlap"),
    ("vh_linear_attention_step", STEP, dict(B=0), hip.VH_ERR_SHAPE, "nonempty"),
    ("vh_linear_attention_step", STEP, dict(V=200), hip.VH_ERR_SHAPE, "128"),
    ("vh_group_norm_forward", NORM, dict(io=3), hip.VH_ERR_DTYPE, "io_dtype"),
    ("vh_group_norm_forward", NORM, dict(pixels=0), hip.VH_ERR_SHAPE, "nonempty"),
    ("vh_group_norm_forward", NORM, dict(G=3), hip.VH_ERR_SHAPE, "groups"),
    ("vh_group_norm_forward", NORM, dict(G=0), hip.VH_ERR_SHAPE, "groups"),
    ("vh_group_norm_forward", NORM, dict(C=2050, G=2), hip.VH_ERR_SHAPE, "1024"),
    ("vh_group_norm_forward", NORM, dict(B=1 << 21), hip.VH_ERR_SHAPE, "range"),
    ("vh_group_norm_forward", NORM, dict(act=3), hip.VH_ERR_ARG, "activation"),
    ("vh_group_norm_forward", NORM, dict(y=None), hip.VH_ERR_ARG, "null"),
    ("vh_group_norm_forward", NORM, dict(pixels=100000, wsn=16), hip.VH_ERR_WORKSPACE, "workspace"),
    ("vh_group_norm_backward", NORM_BACK, dict(stats=None), hip.VH_ERR_ARG, "null"),
    ("vh_group_norm_backward", NORM_BACK, dict(wsn=16), hip.VH_ERR_WORKSPACE, "workspace"),
    ("vh_group_norm_backward", NORM_BACK, dict(ws=None), hip.VH_ERR_WORKSPACE, "workspace"),
]


@pytest.mark.parametrize("name, defaults, change, status, message", REFUSED,
                         ids=[f"{r[0]}-{next(iter(r[2]))}-{i}" for i, r in enumerate(REFUSED)])
def test_refused_before_any_launch(lib, name, defaults, change, status, message):
    assert _call(lib, name, defaults, **change) == status
    assert message in lib.vh_last_error().decode()


def test_workspace_sizes(lib):
    attend, back = lib.vh_linear_attention_workspace_bytes, lib.vh_linear_attention_backward_workspace_bytes
    assert attend(1, 1, 1, 64, 64, F32) == 0 and back(1, 1, 1, 64, 64, F32, 0) == 0   # one segment: no states between
    assert attend(0, 5, 1, 64, 64, F32) == 0 and attend(1, 5, 1, 129, 64, F32) == 0
    states = attend(1, 4096, 4, 20, 33, F32)   # heads padded to 64
    assert states > 0 and states % (4 * 64 * 64 * 4) == 0 and back(1, 4096, 4, 20, 33, F32, 0) == states
    chunks = 4096 // 32                        # a decay's gradient takes the states of every chunk, both ways
    assert back(1, 4096, 4, 20, 33, F32, 1) == 2 * 4 * (chunks - 1) * 64 * 64 * 4 + 4 * chunks * 4
    norm, norm_back = lib.vh_group_norm_workspace_bytes, lib.vh_group_norm_backward_workspace_bytes
    assert norm(2, 100, 16, 3, F32) == 0 and norm(2, 0, 16, 2, F32) == 0
    assert 0 < norm(2, 100000, 16, 2, F32) < 1 << 20 and 0 < norm_back(2, 100000, 16, 2, F32) < 1 << 20


def test_cpu_tensors_are_refused():
    import torch

    from visionhope_amd.utils.group_norm import visionhope_group_norm
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention, visionhope_linear_attention_step

    q, a = torch.zeros(1, 4, 2, 8), torch.zeros(2)
    for call in (lambda: visionhope_linear_attention(q, q, q, a),
                 lambda: visionhope_linear_attention_step(q[:, 0], q[:, 0], q[:, 0], a, torch.zeros(1, 2, 8, 8)),
                 lambda: visionhope_group_norm(torch.zeros(1, 8, 2, 2), 2, torch.ones(8), torch.zeros(8))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("change", [dict(B=1 << 15, H=32, N=65, K=128, V=128),   # 2^20 heads of 128 x 128 / 4 threads
                                    dict(B=1 << 17, H=16, N=257, K=128, V=8),
                                    dict(B=1 << 10, H=16, N=1 << 14, K=128, V=8)])   # 2^14 heads in 2^9 segments of 512 threads
def test_launches_of_too_many_threads_are_refused(lib, change):
    """A trained decay takes the states of every chunk: their passes may exceed the 2^32 threads of a launch."""
    strides = {f"{n}{part}": 0 for n in ("do", "q", "k", "v") for part in "bth"}
    assert _call(lib, "vh_linear_attention_backward", BACK, ddecay=P, ws=None, wsn=0, **strides, **change) == hip.VH_ERR_SHAPE
    assert "range" in lib.vh_last_error().decode()

"""Performance cases of the linear attention with a decay for each head and of the group norm of
channels-last maps.

A case is a dict with a ``kind``, the sizes, the activation type and the options of one call:

* ``attn``: linear attention of a prompt, outputs and the states that single tokens continue
  from; ``attn_train``: forward and backward (with ``learned`` the decays are trained too);
  ``attn_step``: one token of every sequence;
* ``norm``: group norm of maps with an activation; ``norm_train``: forward and backward.

Sequence lengths and maps are those of the backbones' stages (224 and 512 pixel images), widths
are the registered backbones' widths and twice them, and odd ones beside.
"""

import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_EPS = 1e-5
_CHUNK = 64


# ---- the cases ------------------------------------------------------------------------

def listed():
    return [
        # Serving: one new token for each of 64 sequences of a 1024-wide mixer.
        dict(name="attn_step_b64", kind="attn_step", dtype="bf16", batch=64, heads=16, key_dim=64, value_dim=64),
        # Serving a wide model: large states, many sequences.
        dict(name="attn_step_wide", kind="attn_step", dtype="fp16", batch=200, heads=8, key_dim=128, value_dim=128),
        # Serving: a padded batch of prompts of different lengths that continue sequences.
        dict(name="attn_prompt_ragged", kind="attn", dtype="fp16", batch=7, length=785, heads=7, key_dim=64,
             value_dim=64, ragged=True, state=True),
        # One long prompt: the tokens of a 512-pixel image's first stage in one line.
        dict(name="attn_prompt_long", kind="attn", dtype="bf16", batch=1, length=16384, heads=16, key_dim=64,
             value_dim=64, ragged=False, state=False),
        # A short full-precision model's training step, odd head widths, trained decays.
        dict(name="attn_train_small", kind="attn_train", dtype="fp32", batch=2, length=197, heads=3, key_dim=24,
             value_dim=40, learned=True),
        # Classifier training, 28 x 28 maps, wide heads.
        dict(name="attn_train_28_wide", kind="attn_train", dtype="bf16", batch=8, length=784, heads=8, key_dim=128,
             value_dim=128, learned=False),
        # Classifier training, first-stage maps (56 x 56 tokens, Base width twice).
        dict(name="attn_train_56_b32", kind="attn_train", dtype="bf16", batch=32, length=3136, heads=3, key_dim=64,
             value_dim=64, learned=False),
        # A last-stage map of two images (latency).
        dict(name="norm_7_b2", kind="norm", dtype="bf16", batch=2, height=7, width=7, channels=640, groups=40,
             activation="silu"),
        # Dense prediction, serving: first stage of eight 512-pixel images.
        dict(name="norm_128_b8", kind="norm", dtype="bf16", batch=8, height=128, width=128, channels=96, groups=6,
             activation="gelu"),
        # Full-precision training on odd maps and widths.
        dict(name="norm_train_fp32", kind="norm_train", dtype="fp32", batch=3, height=29, width=37, channels=90,
             groups=5, activation="silu"),
        # Training, third-stage maps.
        dict(name="norm_train_14_b32", kind="norm_train", dtype="bf16", batch=32, height=14, width=14, channels=448,
             groups=28, activation="none"),
        # Training, first-stage maps at the elementwise benchmark's size.
        dict(name="norm_train_56_b128", kind="norm_train", dtype="bf16", batch=128, height=56, width=56, channels=96,
             groups=6, activation="gelu"),
    ]


def _log_int(rng, low, high):
    """An integer spread evenly over the logarithm of [low, high]."""
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn_train", "attn_train", "attn_step", "norm", "norm_train"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    case = dict(kind=kind, dtype=dtype)
    if kind.startswith("norm"):
        per_group = rng.choice((16, 16, 8, 32, rng.randint(3, 48)))
        groups = max(1, _log_int(rng, 16, 1024) // per_group)
        channels, batch = per_group * groups, _log_int(rng, 1, 128)
        height, width = _log_int(rng, 2, 128), _log_int(rng, 2, 128)
        while batch * height * width * channels > 38_000_000 * 2 // _BYTES[dtype]:
            batch, height = (batch // 2, height) if batch > 1 else (batch, height // 2)
        return dict(case, batch=batch, height=height, width=width, channels=channels, groups=groups,
                    activation=rng.choice(("none", "silu", "gelu")))
    heads = _log_int(rng, 1, 16)
    dims = (16, 32, 64, 64, 64, 128, rng.randint(1, 128))
    key_dim = rng.choice(dims)
    value_dim = key_dim if rng.random() < 0.6 else rng.choice(dims)
    case.update(heads=heads, key_dim=key_dim, value_dim=value_dim)
    if kind == "attn_step":
        batch = _log_int(rng, 1, 256)
        while batch > 1 and batch * heads * key_dim * value_dim > 26_000_000:
            batch //= 2
        return dict(case, batch=batch)
    length, batch = _log_int(rng, 1, 16384), _log_int(rng, 1, 32)
    while batch * length * heads * max(key_dim, value_dim, 16) > 19_000_000 * 2 // _BYTES[dtype]:
        batch, length = (batch // 2, length) if batch > 1 else (batch, length // 2)
    case.update(batch=batch, length=length)
    if kind == "attn_train":
        case.update(learned=rng.random() < 0.25)
    else:
        case.update(ragged=rng.random() < 0.5, state=rng.random() < 0.5)
    return case


def work(case):
    e, kind = _BYTES[case["dtype"]], case["kind"]
    train = kind.endswith("train")
    if kind.startswith("norm"):
        n = case["batch"] * case["height"] * case["width"] * case["channels"]
        # forward: x -> y; backward besides: x, dy -> dx
        return {"bytes": n * e * (5 if train else 2) + case["channels"] * 4 * (4 if train else 2),
                "flops": n * (32 if train else 12)}
    dk, dv, heads = case["key_dim"], case["value_dim"], case["heads"]
    states = case["batch"] * heads * dk * dv
    if kind == "attn_step":
        return {"bytes": states * 8 + case["batch"] * heads * 2 * (dk + dv) * e, "flops": 5 * states}
    rows = case["batch"] * case["length"] * heads
    if train:
        # forward: q, k, v -> o; backward: q, k, v, do -> dq, dk, dv.  Operations of the token by
        # token form: two products of the state forward, the states again and four more backward
        return {"bytes": rows * e * (2 * dk + 2 * dv + 4 * dk + 3 * dv), "flops": rows * dk * dv * 16}
    kept = states * 4 * (2 if case["state"] else 1)
    return {"bytes": rows * e * 2 * (dk + dv) + kept, "flops": rows * dk * dv * 5}


# ---- inputs ---------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, kind = _DTYPES[case["dtype"]], case["kind"]

    def randn(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device=dev) * scale

    st = {"case": case, "kind": kind}
    batch = case["batch"]
    train = kind.endswith("train")
    if kind.startswith("norm"):
        shape = (batch, case["height"], case["width"], case["channels"])

        def channels_last(t):
            return t.to(dtype).permute(0, 3, 1, 2)

        # a convolution's outputs: every channel with its own offset and spread
        offset, spread = randn(case["channels"], scale=0.5), torch.exp(randn(case["channels"], scale=0.3))
        st["x"] = channels_last(randn(*shape) * spread + offset)
        st["weight"], st["bias"] = 1.0 + randn(case["channels"], scale=0.1), randn(case["channels"], scale=0.1)
        if train:
            st["dy"] = channels_last(randn(*shape))
            st["leaves"] = ("x", "weight", "bias")
    else:
        heads, dk, dv = case["heads"], case["key_dim"], case["value_dim"]
        # decays from a half a token to one part in a thousand, a fixed ladder with some spread
        rungs = 1.0 + 9.0 * torch.arange(heads, device=dev) / max(1, heads - 1)
        st["log_decay"] = torch.log1p(-torch.exp2(-rungs)) * torch.exp(randn(heads, scale=0.1))
        if kind == "attn_step":
            st["q"], st["k"] = (randn(batch, heads, dk).to(dtype) for _ in range(2))
            st["v"] = randn(batch, heads, dv).to(dtype)
            st["state"] = randn(batch, heads, dk, dv)
            st["new_state"] = torch.empty_like(st["state"])
        else:
            # q, k and v as slices of one projection of the tokens
            wide = randn(batch, case["length"], heads * (2 * dk + dv)).to(dtype)
            q, k, v = wide.split((heads * dk, heads * dk, heads * dv), dim=-1)
            st["q"], st["k"], st["v"] = q.unflatten(-1, (heads, dk)), k.unflatten(-1, (heads, dk)), v.unflatten(-1, (heads, dv))
            if train:
                st["do"] = randn(batch, case["length"], heads, dv).to(dtype)
                st["leaves"] = ("q", "k", "v", "log_decay") if case["learned"] else ("q", "k", "v")
            else:
                st["state"] = randn(batch, heads, dk, dv) if case["state"] else None
    st["lengths"] = None
    if case.get("ragged"):
        lengths = torch.randint(1, case["length"] + 1, (batch,), generator=gen, device=dev)
        st["lengths"] = lengths.to(torch.int32)
    for name in st.get("leaves", ()):
        st[name] = st[name].detach().requires_grad_()
    return st


# ---- one pass -------------------------------------------------------------------------

def run(st):
    if own:
        return _run_own(st)
    kind = st["kind"]
    if kind == "norm":
        return _norm_plain(st)
    if kind == "attn":
        return _attn_plain(st)
    if kind == "attn_step":
        return _step_plain(st)
    y = _norm_plain(st) if kind == "norm_train" else _attn_plain(st)[0]
    grad = st["dy"] if kind == "norm_train" else st["do"]
    return [y.detach(), *torch.autograd.grad(y, [st[name] for name in st["leaves"]], grad)]


def _run_own(st):
    from visionhope_amd.utils.group_norm import visionhope_group_norm
    from visionhope_amd.utils.linear_attention import visionhope_linear_attention, visionhope_linear_attention_step

    kind = st["kind"]
    if kind.startswith("norm"):
        activation = st["case"]["activation"]
        y = visionhope_group_norm(st["x"], st["case"]["groups"], st["weight"], st["bias"], _EPS,
                                  activation=None if activation == "none" else activation)
        if kind == "norm":
            return y
        return [y.detach(), *torch.autograd.grad(y, [st[name] for name in st["leaves"]], st["dy"])]
    if kind == "attn":
        return visionhope_linear_attention(st["q"], st["k"], st["v"], st["log_decay"], state=st["state"],
                                           lengths=st["lengths"], return_state=True)
    if kind == "attn_step":
        o = visionhope_linear_attention_step(st["q"], st["k"], st["v"], st["log_decay"], st["state"],
                                             new_state=st["new_state"])
        return o, st["new_state"]
    o = visionhope_linear_attention(st["q"], st["k"], st["v"], st["log_decay"])
    return [o.detach(), *torch.autograd.grad(o, [st[name] for name in st["leaves"]], st["do"])]


# ---- the plain forms ------------------------------------------------------------------

def _norm_plain(st):
    x, groups, activation = st["x"], st["case"]["groups"], st["case"]["activation"]
    batch, channels, height, width = x.shape
    rows = x.permute(0, 2, 3, 1).reshape(batch, height * width, groups, channels // groups).float()
    centred = rows - rows.mean(dim=(1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=(1, 3), keepdim=True) + _EPS)
    y = (centred * rstd).reshape(batch, height, width, channels) * st["weight"] + st["bias"]
    if activation == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif activation == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    return y.to(x.dtype).permute(0, 3, 1, 2)


def _step_plain(st):
    decay = torch.exp(st["log_decay"])[:, None, None]
    state = decay * st["state"] + st["k"].float()[..., None] * st["v"].float()[..., None, :]
    o = (st["q"].float()[..., None] * state).sum(dim=-2) * st["case"]["key_dim"] ** -0.5
    return o.to(st["q"].dtype), state


def _attn_plain(st):
    """o[t] = scale q[t] S[t], S[t] = exp(log_decay) S[t-1] + k[t] v[t]^T, in chunks of 64 tokens:
    products within the chunks, the chunks' own states, the states at the chunks' starts as sums of
    those before them, and the outputs that come from there; and the last state of every sequence."""
    dtype, a = st["q"].dtype, st["log_decay"]
    batch, length, heads, dk = st["q"].shape
    dv, dev = st["v"].shape[-1], st["q"].device
    scale = dk ** -0.5
    q, k, v = (st[name].float() for name in ("q", "k", "v"))
    token = torch.arange(length, device=dev)
    ends = torch.full((batch,), length, device=dev) if st["lengths"] is None else st["lengths"].long()
    live = token[None, :] < ends[:, None]
    if st["lengths"] is not None:
        q, k, v = (torch.where(live[..., None, None], t, 0.0) for t in (q, k, v))
    chunks = -(-length // _CHUNK)

    def cut(t):   # [B, N, H, D] -> [B, H, chunks, 64, D]
        tail = t.new_zeros(batch, chunks * _CHUNK - length, heads, t.shape[-1])
        return torch.cat((t, tail), dim=1).reshape(batch, chunks, _CHUNK, heads, -1).permute(0, 3, 1, 2, 4)

    def powers(steps):   # exp(log_decay * steps) where steps >= 0, zero elsewhere, for each head
        factor = torch.exp(a.reshape(-1, *(1,) * steps.ndim) * steps.clamp(min=0))
        return torch.where(steps >= 0, factor, 0.0)

    i = torch.arange(_CHUNK, device=dev)
    c = torch.arange(chunks, device=dev)
    cq, ck, cv = cut(q), cut(k), cut(v)
    scores = torch.matmul(cq, ck.transpose(-1, -2)) * powers(i[:, None] - i)[:, None]
    local = torch.matmul((ck * powers(_CHUNK - 1 - i)[:, None, :, None]).transpose(-1, -2), cv)
    starts = torch.matmul(powers((c[:, None] - 1 - c) * _CHUNK), local.reshape(batch, heads, chunks, dk * dv))
    state = st.get("state")
    if state is not None:
        starts = starts + powers(c * _CHUNK)[:, :, None] * state.reshape(batch, heads, 1, dk * dv)
    starts = starts.reshape(batch, heads, chunks, dk, dv)
    o = torch.matmul(scores, cv) + torch.matmul(cq, starts) * powers(i + 1)[:, None, :, None]
    o = (o * scale).permute(0, 2, 3, 1, 4).reshape(batch, chunks * _CHUNK, heads, dv)[:, :length]
    if st["lengths"] is not None:
        o = torch.where(live[..., None, None], o, 0.0)
    if st["kind"] == "attn_train":
        return o.to(dtype), None
    weight = powers(ends[:, None] - 1 - token).permute(1, 2, 0)
    last = torch.matmul((k * weight[..., None]).permute(0, 2, 3, 1), v.permute(0, 2, 1, 3))
    if state is not None:
        last = last + powers(ends).t()[..., None, None] * state
    return o.to(dtype), last


# ---- the definitions in 64 bits -------------------------------------------------------

def exact(case, seed):
    st = {k: v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v
          for k, v in prepare(case, seed).items()}
    with torch.no_grad():
        return _norm_exact(st, case) if case["kind"].startswith("norm") else _attn_exact(st, case)


def _norm_exact(st, case):
    x, groups = st["x"], case["groups"]
    per = x.shape[1] // groups
    w, b = st["weight"][:, None, None], st["bias"][:, None, None]

    def spread(t):   # [B, groups] -> [B, C, 1, 1]
        return t.repeat_interleave(per, dim=1)[..., None, None]

    var, mean = torch.var_mean(x.unflatten(1, (groups, per)), dim=(2, 3, 4), unbiased=False)
    rstd = spread(torch.rsqrt(var + _EPS))
    xhat = (x - spread(mean)) * rstd
    z = xhat * w + b
    if case["activation"] == "silu":
        gate = torch.sigmoid(z)
        y, slope = z * gate, gate + z * gate * (1 - gate)
    elif case["activation"] == "gelu":
        gate = torch.special.ndtr(z)
        y, slope = z * gate, gate + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    else:
        y, slope = z, torch.ones_like(z)
    if case["kind"] == "norm":
        return y
    dz = st["dy"] * slope
    dw, db = (dz * xhat).sum((0, 2, 3)), dz.sum((0, 2, 3))
    g = dz * w
    mean_g = spread(g.unflatten(1, (groups, per)).mean((2, 3, 4)))
    mean_gx = spread((g * xhat).unflatten(1, (groups, per)).mean((2, 3, 4)))
    return [y, rstd * (g - mean_g - xhat * mean_gx), dw, db]


def _attn_exact(st, case):
    q, k, v = st["q"], st["k"], st["v"]
    scale = case["key_dim"] ** -0.5
    decay = torch.exp(st["log_decay"])[:, None, None]
    if case["kind"] == "attn_step":
        state = decay * st["state"] + torch.einsum("bhk,bhv->bhkv", k, v)
        return torch.einsum("bhk,bhkv->bhv", q, state) * scale, state
    batch, length, heads, dk = q.shape
    dv = v.shape[-1]
    q, k, v = (t.permute(1, 0, 2, 3).contiguous() for t in (q, k, v))
    state = st.get("state")
    state = q.new_zeros(batch, heads, dk, dv) if state is None else state.clone()
    o = torch.empty_like(v)
    if case["kind"] == "attn":
        ends = [length] * batch if st["lengths"] is None else st["lengths"].tolist()
        last = state.clone()
        for t in range(length):
            state = decay * state + k[t][..., :, None] * v[t][..., None, :]
            o[t] = torch.matmul(q[t][..., None, :], state)[..., 0, :] * scale
            for b in (b for b, n in enumerate(ends) if n == t + 1):
                last[b] = state[b]
        for b, n in enumerate(ends):
            o[n:, b] = 0.0
        return o.permute(1, 0, 2, 3), last
    do = st["do"].permute(1, 0, 2, 3).contiguous()
    dq, dk_, dv_ = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    slope, dlog = torch.zeros_like(state), torch.zeros_like(st["log_decay"])   # slope: d state / d log_decay
    for t in range(length):
        if case["learned"]:
            slope = decay * (slope + state)
            dlog += scale * (q[t] * torch.matmul(slope, do[t][..., None])[..., 0]).sum((0, 2))
        state = decay * state + k[t][..., :, None] * v[t][..., None, :]
        o[t] = torch.matmul(q[t][..., None, :], state)[..., 0, :] * scale
        dq[t] = torch.matmul(state, do[t][..., None])[..., 0] * scale
    adjoint = torch.zeros_like(state)
    for t in range(length - 1, -1, -1):
        adjoint = decay * adjoint + scale * q[t][..., :, None] * do[t][..., None, :]
        dk_[t] = torch.matmul(adjoint, v[t][..., None])[..., 0]
        dv_[t] = torch.matmul(k[t][..., None, :], adjoint)[..., 0, :]
    found = [t.permute(1, 0, 2, 3) for t in (o, dq, dk_, dv_)]
    return found + [dlog] if case["learned"] else found

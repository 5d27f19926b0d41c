"""Linear attention mixer of token lines and its block on maps: the modules around the native operators.

``LinearAttentionMixer`` mixes ``[B, N, dim]`` sequences as ``StateSpaceMixer`` does, by linear
attention with a decay for each head (``utils/linear_attention.py``): one projection to queries,
keys, values and gates, the attention, a gated LayerNorm of each head's output and an output
projection.  Prompts run through ``forward``, single tokens through ``step`` on the state that
the prompt returned.  ``LinearAttentionBlock`` runs it over the pixels of a map behind a group norm.
"""

import torch
from torch import nn
from torch.nn.init import trunc_normal_

from ..utils.gated_norm import visionhope_gated_layernorm
from ..utils.linear_attention import MAX_HEAD_DIM, visionhope_linear_attention, visionhope_linear_attention_step
from ..utils.token_lines import guarded, line_lengths
from .layers import GroupNorm2d


class LinearAttentionMixer(nn.Module):
    """Linear attention over ``dim`` channels in ``heads`` heads (module docstring).

    ``key_dim`` and ``value_dim`` are a head's widths (default ``dim // heads``, at most 128).  The
    heads' decays stand on a ladder from 1 - 2^-5 to 1 - 2^-12 a token; ``learn_decay`` trains them
    from there, as ``exp(-exp(log_rate))``.  ``norm_weight`` and ``norm_bias`` are shared by the heads.
    """

    def __init__(self, dim, heads=4, key_dim=None, value_dim=None, learn_decay=False, eps=1e-6):
        super().__init__()
        if dim <= 0 or heads <= 0:
            raise ValueError("dim and heads must be positive")
        if (key_dim is None or value_dim is None) and dim % heads:
            raise ValueError(f"{dim} channels do not divide into {heads} heads; give key_dim and value_dim")
        self.dim, self.heads, self.eps = int(dim), int(heads), eps
        self.key_dim = self.dim // self.heads if key_dim is None else int(key_dim)
        self.value_dim = self.dim // self.heads if value_dim is None else int(value_dim)
        if not (1 <= self.key_dim <= MAX_HEAD_DIM and 1 <= self.value_dim <= MAX_HEAD_DIM):
            raise ValueError(f"key_dim and value_dim must be 1 to {MAX_HEAD_DIM}")
        self.in_proj = nn.Linear(self.dim, 2 * self.heads * (self.key_dim + self.value_dim), bias=False)
        if learn_decay:
            self.log_rate = nn.Parameter(torch.empty(self.heads))
        else:
            self.register_buffer("log_rate", torch.empty(self.heads))
        self.norm_weight = nn.Parameter(torch.empty(self.value_dim))
        self.norm_bias = nn.Parameter(torch.empty(self.value_dim))
        self.out_proj = nn.Linear(self.heads * self.value_dim, self.dim, bias=False)
        self.reset_parameters()

    def reset_parameters(self):
        """The ladder of decays, unit norms, projections truncated normal of std 0.02."""
        for linear in (self.in_proj, self.out_proj):
            trunc_normal_(linear.weight, std=0.02)
        with torch.no_grad():
            rungs = torch.linspace(5.0, 12.0, self.heads)
            self.log_rate.copy_(torch.log(-torch.log1p(-torch.exp2(-rungs))))
            self.norm_weight.fill_(1.0)
            self.norm_bias.zero_()

    def allocate_state(self, batch):
        """The FP32 state before a first token."""
        return torch.zeros(batch, self.heads, self.key_dim, self.value_dim, device=self.log_rate.device)

    def _log_decay(self):
        return -torch.exp(self.log_rate.float())

    def _projected(self, x):
        """Queries, keys, values and gates of tokens, each ``[..., heads, width]``."""
        widths = (self.key_dim, self.key_dim, self.value_dim, self.value_dim)
        parts = self.in_proj(x).split([self.heads * w for w in widths], dim=-1)
        return [part.unflatten(-1, (self.heads, w)) for part, w in zip(parts, widths)]

    def _output(self, o, gate):
        o = visionhope_gated_layernorm(o, self.norm_weight, self.norm_bias, self.eps, gate=gate)
        return self.out_proj(o.flatten(-2))

    def forward(self, x, *, state=None, lengths=None, return_state=False):
        """``[B, N, dim]`` -> ``[B, N, dim]``, or ``(output, state)`` with ``return_state``.
        ``state`` continues earlier tokens; ``lengths`` ``[B]`` ends sequences of a padded batch
        early: their outputs and gradients behind the end are zero, whatever stands there."""
        if x.ndim != 3 or x.shape[-1] != self.dim:
            raise ValueError(f"LinearAttentionMixer expects [B, N, {self.dim}]")
        live = None
        if lengths is not None:
            lengths = line_lengths("LinearAttentionMixer", lengths, x.shape[0], x.device)
            live = (torch.arange(x.shape[1], device=x.device) < lengths[:, None])[..., None]
            if torch.is_grad_enabled():   # the projection's weight gradient takes all rows
                x = torch.where(live, x, 0.0)
        q, k, v, gate = self._projected(x)
        o = visionhope_linear_attention(q, k, v, self._log_decay(), state=state, lengths=lengths, return_state=return_state)
        if return_state:
            o, state = o
        out = self._output(o, gate)
        if live is not None:
            # the norm does not leave rows of zeros zero, and out's gradient may be anything there
            out = torch.where(live, out, 0.0)
        out = guarded("LinearAttentionMixer", out)
        return (out, state) if return_state else out

    def step(self, x, state):
        """One token of every sequence, ``[B, dim]`` -> ``[B, dim]``; moves ``state`` on in place.
        Inference only."""
        if x.ndim != 2 or x.shape[-1] != self.dim:
            raise ValueError(f"LinearAttentionMixer.step expects [B, {self.dim}]")
        q, k, v, gate = self._projected(x)
        return self._output(visionhope_linear_attention_step(q, k, v, self._log_decay(), state), gate)

    def extra_repr(self):
        return f"dim={self.dim}, heads={self.heads}, key_dim={self.key_dim}, value_dim={self.value_dim}"


class LinearAttentionBlock(nn.Module):
    """Pre-norm residual block on NCHW maps: ``x + mixer(norm(x))`` with a ``GroupNorm2d`` and the mixer
    over the pixels in row order, or from the last pixel to the first with ``reverse``.  Runs on
    channels-last storage, whose pixels are a token line as they stand."""

    def __init__(self, dim, heads=4, groups=None, reverse=False, **mixer):
        super().__init__()
        self.norm = GroupNorm2d(dim, groups)
        self.mixer = LinearAttentionMixer(dim, heads, **mixer)
        self.reverse = bool(reverse)

    def forward(self, x):
        height, width = x.shape[2:]
        tokens = self.norm(x).flatten(2).transpose(1, 2)
        tokens = self.mixer(tokens.flip(1)).flip(1) if self.reverse else self.mixer(tokens)
        return x + tokens.transpose(1, 2).unflatten(2, (height, width))

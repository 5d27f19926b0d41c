"""Selective state space mixer of token lines: the module around the native scan.

``StateSpaceMixer`` mixes ``[B, N, dim]`` sequences as ``SRNL`` does, by the framework's other
recurrence: an input projection, a short causal convolution with SiLU, the selective scan
(``utils/state_space.py``) and an output projection, with a gate from the input projection on
the LayerNorm of the scan's output (``norm=True``) or on the output itself.  Prompts run
through ``forward``, single tokens through ``step`` on the state that the prompt returned.
"""

import math

import torch
from torch import nn
from torch.nn import functional as F
from torch.nn.init import trunc_normal_

from ..utils.causal_conv import MAX_TAPS, visionhope_causal_conv, visionhope_causal_conv_step
from ..utils.gated_norm import visionhope_gated_layernorm
from ..utils.state_space import MAX_STATES, visionhope_state_space_scan, visionhope_state_space_step
from ..utils.token_lines import guarded, line_lengths


class StateSpaceMixer(nn.Module):
    """Selective state space mixer over ``dim`` channels (module docstring).

    ``expand`` widens the recurrence to ``expand * dim`` channels of ``state_dim`` FP32 states
    each; ``conv_taps`` is the length of the causal convolution, ``dt_rank`` the width of the
    projection that the step sizes come from (default ``ceil(dim / 16)``).
    """

    def __init__(self, dim, state_dim=16, expand=2, conv_taps=4, dt_rank=None, norm=True, eps=1e-6):
        super().__init__()
        if dim <= 0 or int(dim * expand) <= 0:
            raise ValueError("dim and expand must be positive")
        if not 1 <= state_dim <= MAX_STATES:
            raise ValueError(f"state_dim must be 1 to {MAX_STATES}")
        if not 2 <= conv_taps <= MAX_TAPS:
            raise ValueError(f"conv_taps must be 2 to {MAX_TAPS}")
        self.dim, self.inner, self.state_dim, self.eps = int(dim), int(dim * expand), int(state_dim), eps
        self.dt_rank = math.ceil(dim / 16) if dt_rank is None else int(dt_rank)
        self.in_proj = nn.Linear(self.dim, 2 * self.inner, bias=False)
        self.conv = nn.Conv1d(self.inner, self.inner, conv_taps, groups=self.inner)   # its parameters; run natively
        self.x_proj = nn.Linear(self.inner, self.dt_rank + 2 * self.state_dim, bias=False)
        self.dt_proj = nn.Linear(self.dt_rank, self.inner)                            # its bias enters the scan
        self.A_log = nn.Parameter(torch.empty(self.inner, self.state_dim))
        self.D = nn.Parameter(torch.empty(self.inner))
        self.norm_weight = nn.Parameter(torch.empty(self.inner)) if norm else None
        self.norm_bias = nn.Parameter(torch.empty(self.inner)) if norm else None
        self.out_proj = nn.Linear(self.inner, self.dim, bias=False)
        self.reset_parameters()

    def reset_parameters(self):
        """Decay rates 1 .. state_dim, steps log-uniform in [0.001, 0.1], unit skip and norm,
        projections truncated normal of std 0.02."""
        for linear in (self.in_proj, self.x_proj, self.dt_proj, self.out_proj):
            trunc_normal_(linear.weight, std=0.02)
        self.conv.reset_parameters()
        with torch.no_grad():
            self.A_log.copy_(torch.arange(1, self.state_dim + 1).float().log().expand_as(self.A_log))
            step = torch.exp(torch.rand(self.inner) * math.log(100.0) + math.log(0.001))
            self.dt_proj.bias.copy_(step + torch.log(-torch.expm1(-step)))   # softplus of it is the step
            self.D.fill_(1.0)
            if self.norm_weight is not None:
                self.norm_weight.fill_(1.0)
                self.norm_bias.zero_()

    def allocate_state(self, batch, dtype=torch.float32):
        """The state before a first token: the convolution's last inputs (``dtype``, that of the
        activations) and the FP32 states of the scan."""
        device = self.A_log.device
        return (torch.zeros(batch, self.conv.kernel_size[0] - 1, self.inner, device=device, dtype=dtype),
                torch.zeros(batch, self.inner, self.state_dim, device=device))

    def _rates(self):
        return -torch.exp(self.A_log.float())

    def _selected(self, x):
        """Step sizes (without their bias), B and C of convolved tokens."""
        dt, B, C = self.x_proj(x).split((self.dt_rank, self.state_dim, self.state_dim), dim=-1)
        return F.linear(dt, self.dt_proj.weight), B, C

    def _output(self, y, gate):
        if self.norm_weight is not None:
            y = visionhope_gated_layernorm(y, self.norm_weight, self.norm_bias, self.eps, gate=gate)
        return self.out_proj(y)

    def forward(self, x, *, state=None, lengths=None, return_state=False):
        """``[B, N, dim]`` -> ``[B, N, dim]``, or ``(output, state)`` with ``return_state``.
        ``state`` continues earlier tokens; ``lengths`` ``[B]`` ends sequences of a padded batch
        early: their outputs and gradients behind the end are zero, whatever stands there."""
        if x.ndim != 3 or x.shape[-1] != self.dim:
            raise ValueError(f"StateSpaceMixer expects [B, N, {self.dim}]")
        conv_state, scan_state = (None, None) if state is None else state
        live = None
        if lengths is not None:
            lengths = line_lengths("StateSpaceMixer", lengths, x.shape[0], x.device)
            live = (torch.arange(x.shape[1], device=x.device) < lengths[:, None])[..., None]
            if torch.is_grad_enabled():   # the projections' weight gradients take all rows
                x = torch.where(live, x, 0.0)
        x, gate = self.in_proj(x).chunk(2, dim=-1)
        x = visionhope_causal_conv(x, self.conv.weight, self.conv.bias, silu=True, state=conv_state, lengths=lengths,
                                   return_state=return_state)
        if return_state:
            x, conv_state = x
        dt, B, C = self._selected(x)
        y = visionhope_state_space_scan(x, dt, self._rates(), B, C, self.D, dt_bias=self.dt_proj.bias,
                                        gate=gate if self.norm_weight is None else None, state=scan_state,
                                        lengths=lengths, return_state=return_state)
        if return_state:
            y, scan_state = y
        out = self._output(y, gate)
        if live is not None and (self.norm_weight is not None or torch.is_grad_enabled()):
            # the norm does not leave rows of zeros zero, and out's gradient may be anything there
            out = torch.where(live, out, 0.0)
        out = guarded("StateSpaceMixer", out)
        return (out, (conv_state, scan_state)) if return_state else out

    def step(self, x, state):
        """One token of every sequence, ``[B, dim]`` -> ``[B, dim]``; moves ``state`` on in place.
        Inference only."""
        if x.ndim != 2 or x.shape[-1] != self.dim:
            raise ValueError(f"StateSpaceMixer.step expects [B, {self.dim}]")
        conv_state, scan_state = state
        x, gate = self.in_proj(x).chunk(2, dim=-1)
        x = visionhope_causal_conv_step(x, conv_state, self.conv.weight, self.conv.bias, silu=True)
        dt, B, C = self._selected(x)
        y = visionhope_state_space_step(x, dt, self._rates(), B, C, scan_state, self.D, dt_bias=self.dt_proj.bias,
                                        gate=gate if self.norm_weight is None else None)
        return self._output(y, gate)

    def extra_repr(self):
        return f"dim={self.dim}, state_dim={self.state_dim}, inner={self.inner}, norm={self.norm_weight is not None}"

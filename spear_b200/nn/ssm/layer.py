"""Selective state space layer on the sm_100a kernels: the long-memory partner of the Phalanx window layer.

    x, z = in_proj(u)                                    [B, L, inner] each
    x = silu(causal_conv(x))
    delta_low, B, C = x_proj(x)                          [B, L, rank], [B, L, N], [B, L, N]
    y = selective_scan(x, dt_proj(delta_low), -exp(A_log), B, C, D, z, delta_bias)
    out = out_proj(y)

Token-major throughout: the convolution and the scan read their inputs as column slices of the projections' outputs, nothing
is copied or transposed.  ``forward`` trains, ``prefill`` takes prompts (of different lengths in one padded batch) and hands
on the state, ``step`` takes one token.  CUDA only, no fallback.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn

from ...ops.ssm import causal_conv, causal_conv_step, selective_scan, selective_scan_step


@dataclass
class SSMState:
    """Streaming state of one layer."""

    conv: torch.Tensor  # (B, width - 1, inner) the convolution's last inputs, oldest first
    ssm: torch.Tensor   # (B, inner, N) float32 state of the scan

    def clone_detached(self) -> "SSMState":
        return SSMState(conv=self.conv.detach().clone(), ssm=self.ssm.detach().clone())


class SelectiveSSM(nn.Module):
    """Selective state space mixer, [B, L, dim] -> [B, L, dim].

    Args:
        dim: width of the input and output.
        state_size: states per channel (1 ... 64).
        width: taps of the short convolution (2, 3 or 4).
        expand: inner channels per input channel.
        rank: width of the step size's low-rank projection, default ceil(dim / 16).
        dtype: of the projections, the convolution and the activations; A, D and the step bias stay float32.
        dt_min, dt_max: range of the step sizes that the step bias starts with.
    """

    def __init__(self, dim: int, state_size: int = 16, width: int = 4, expand: int = 2, rank: int | None = None,
                 dtype: torch.dtype = torch.float32, dt_min: float = 1e-3, dt_max: float = 1e-1):
        super().__init__()
        if dim < 1 or expand < 1:
            raise ValueError(f"dim and expand must be positive (got {dim}, {expand})")
        if not 1 <= state_size <= 64:
            raise ValueError(f"state_size must be in 1 ... 64 (got {state_size})")
        if width not in (2, 3, 4):
            raise ValueError(f"width must be 2, 3 or 4 (got {width})")
        if not 0.0 < dt_min <= dt_max:
            raise ValueError(f"need 0 < dt_min <= dt_max (got {dt_min}, {dt_max})")
        self.dim, self.state_size, self.width, self.inner = dim, state_size, width, expand * dim
        self.rank = -(-dim // 16) if rank is None else rank
        self.in_proj = nn.Linear(dim, 2 * self.inner, bias=False, dtype=dtype)
        self.conv_weight = nn.Parameter(torch.empty(self.inner, width, dtype=dtype).uniform_(-1, 1) / math.sqrt(width))
        self.conv_bias = nn.Parameter(torch.zeros(self.inner, dtype=dtype))
        self.x_proj = nn.Linear(self.inner, self.rank + 2 * state_size, bias=False, dtype=dtype)
        self.dt_proj = nn.Linear(self.rank, self.inner, bias=False, dtype=dtype)
        size = torch.exp(torch.empty(self.inner).uniform_(math.log(dt_min), math.log(dt_max)))
        self.dt_bias = nn.Parameter(size + torch.log(-torch.expm1(-size)))  # softplus(dt_bias) = size
        self.A_log = nn.Parameter(torch.arange(1, state_size + 1, dtype=torch.float32).log().repeat(self.inner, 1))
        self.D = nn.Parameter(torch.ones(self.inner))
        self.out_proj = nn.Linear(self.inner, dim, bias=False, dtype=dtype)

    @property
    def dtype(self) -> torch.dtype:
        """Type of the projections as they are now: `.to()` may have cast the module."""
        return self.in_proj.weight.dtype

    def _parameters_of_scan(self):
        """Rates, input weight and step bias in float32, also where `.to()` has cast the module."""
        return -torch.exp(self.A_log.float()), self.D.float(), self.dt_bias.float()

    def _split(self, x: torch.Tensor):
        """(delta, B, C) from the convolution's output; B and C are column slices of one product."""
        low, B, C = self.x_proj(x).split([self.rank, self.state_size, self.state_size], dim=-1)
        return self.dt_proj(low), B, C

    def _run(self, u, state, lengths, return_state):
        if u.dim() != 3 or u.shape[2] != self.dim:
            raise ValueError(f"SelectiveSSM takes [B, L, {self.dim}], got {tuple(u.shape)}")
        if lengths is not None and torch.is_grad_enabled():
            # in_proj's weight gradient sums over all tokens: behind a sequence's end zero times whatever the padding holds, NaN for NaN
            u = u.masked_fill((torch.arange(u.shape[1], device=u.device) >= lengths[:, None])[..., None], 0.0)
        x, z = self.in_proj(u.to(self.dtype)).split(self.inner, dim=-1)
        conv = causal_conv(x, self.conv_weight, self.conv_bias, activation="silu", initial_state=None if state is None else state.conv,
                           lengths=lengths, return_state=return_state)
        x, conv_state = conv if return_state else (conv, None)
        delta, B, C = self._split(x)
        A, D, dt_bias = self._parameters_of_scan()
        out = selective_scan(x, delta, A, B, C, D, z, delta_bias=dt_bias, delta_softplus=True,
                             initial_state=None if state is None else state.ssm, lengths=lengths, return_state=return_state)
        y, ssm_state = out if return_state else (out, None)
        return self.out_proj(y), None if not return_state else SSMState(conv=conv_state, ssm=ssm_state)

    def forward(self, u: torch.Tensor, lengths: torch.Tensor | None = None) -> torch.Tensor:
        """[B, L, dim] -> [B, L, dim]; outputs from lengths[b] (int32) on are 0."""
        return self._run(u, None, lengths, False)[0]

    @torch.no_grad()
    def prefill(self, u: torch.Tensor, state: SSMState | None = None, lengths: torch.Tensor | None = None):
        """A prompt, or the next part of one: returns (out [B, L, dim], SSMState after each sequence's last token)."""
        return self._run(u, state, lengths, True)

    @torch.no_grad()
    def step(self, u_t: torch.Tensor, state: SSMState, *, in_place: bool = False):
        """One token [B, dim]: returns (out_t [B, dim], SSMState).

        The given state stays valid and the new one is fresh, unless `in_place` (the form for a captured graph).
        """
        if u_t.dim() != 2 or u_t.shape[1] != self.dim:
            raise ValueError(f"SelectiveSSM.step takes [B, {self.dim}], got {tuple(u_t.shape)}")
        x, z = self.in_proj(u_t.to(self.dtype)).split(self.inner, dim=-1)
        x, conv = causal_conv_step(x, state.conv, self.conv_weight, self.conv_bias, activation="silu",
                                   state_out=state.conv if in_place else None)
        delta, B, C = self._split(x)
        A, D, dt_bias = self._parameters_of_scan()
        y, ssm = selective_scan_step(x, delta, A, B, C, state.ssm, D, z, delta_bias=dt_bias, delta_softplus=True,
                                     state_out=state.ssm if in_place else None)
        return self.out_proj(y), state if in_place else SSMState(conv=conv, ssm=ssm)

    def empty_state(self, batch: int) -> SSMState:
        """The state before the first token."""
        dev = self.A_log.device
        return SSMState(conv=torch.zeros(batch, self.width - 1, self.inner, device=dev, dtype=self.dtype),
                        ssm=torch.zeros(batch, self.inner, self.state_size, device=dev, dtype=torch.float32))

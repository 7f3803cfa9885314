"""Pre-norm residual block around a mixer (Phalanx, SelectiveSSM): the residual's addition and the norm are one kernel.

    h = x + residual          out = mixer(rms_norm(h))          returns (out, h)

The block hands its mixer's output and the residual stream on separately; the next block adds them while it normalises, so the
stream is read and written once per layer.  The stream may be float32 next to 16-bit activations.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from ..ops.norm import rms_norm


class MixerBlock(nn.Module):
    """``out, h = block(x, residual)`` with ``residual=None`` for the first block.

    Args:
        mixer: a module [B, L, dim] -> [B, L, dim] (Phalanx or SelectiveSSM).  ``prefill`` and ``step`` need one that has them
            (SelectiveSSM).
        dim: width of the residual stream.
        eps: of the norm.
        dtype: of the norm's weight.
        residual_dtype: of the residual stream, or None for the input's dtype.
    """

    def __init__(self, mixer: nn.Module, dim: int, eps: float = 1e-6, dtype: torch.dtype = torch.float32,
                 residual_dtype: torch.dtype | None = torch.float32):
        super().__init__()
        self.mixer = mixer
        self.dim, self.eps, self.residual_dtype = dim, eps, residual_dtype
        self.norm_weight = nn.Parameter(torch.ones(dim, dtype=dtype))

    def _norm(self, x: torch.Tensor, residual: torch.Tensor | None):
        if x.shape[-1] != self.dim:
            raise ValueError(f"MixerBlock takes [..., {self.dim}], got {tuple(x.shape)}")
        if residual is None:
            return rms_norm(x, self.norm_weight, eps=self.eps), x if self.residual_dtype is None else x.to(self.residual_dtype)
        return rms_norm(x, self.norm_weight, residual, eps=self.eps)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, **kwargs):
        y, h = self._norm(x, residual)
        return self.mixer(y, **kwargs), h

    def _streams(self, name: str):
        if not hasattr(self.mixer, name):
            raise TypeError(f"MixerBlock.{name}: {type(self.mixer).__name__} has no {name}")
        return getattr(self.mixer, name)

    @torch.no_grad()
    def prefill(self, x: torch.Tensor, residual: torch.Tensor | None = None, state=None, lengths: torch.Tensor | None = None):
        """A prompt through a mixer that has ``prefill``: returns (out, h, state)."""
        prefill = self._streams("prefill")
        y, h = self._norm(x, residual)
        out, state = prefill(y, state, lengths)
        return out, h, state

    @torch.no_grad()
    def step(self, x_t: torch.Tensor, residual: torch.Tensor | None, state, *, in_place: bool = False):
        """One token through a mixer that has ``step``: returns (out_t, h, state)."""
        step = self._streams("step")
        y, h = self._norm(x_t, residual)
        out, state = step(y, state, in_place=in_place)
        return out, h, state

"""Root-mean-square norm with the residual's addition, in the activations' type or in 8 bits with scales."""

from .interface import rms_norm, rms_norm_8bit

__all__ = ["rms_norm", "rms_norm_8bit"]

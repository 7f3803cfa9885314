"""Selective state space operators: the short causal convolution and the selective scan, for prompts and single tokens."""

from .conv import causal_conv, causal_conv_step
from .scan import selective_scan, selective_scan_step

__all__ = ["causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step"]

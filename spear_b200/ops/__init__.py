from .btp import btp
from .norm import rms_norm, rms_norm_8bit
from .ssm import causal_conv, causal_conv_step, selective_scan, selective_scan_step

__all__ = ["btp", "rms_norm", "rms_norm_8bit", "causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step"]

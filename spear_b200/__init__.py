"""spear_b200: the block two-pass (BTP) hot path of SPEAR, hand-written for NVIDIA B200 (sm_100a).

    from spear_b200.ops.btp import btp          # same signature as spear.ops.btp.btp
    from spear_b200.nn.phalanx import Phalanx   # same constructor / state_dict as spear.nn.phalanx.Phalanx
    from spear_b200.ops.ssm import causal_conv, selective_scan    # selective state space operators, and their token forms
    from spear_b200.ops.norm import rms_norm, rms_norm_8bit       # norm with the residual's addition
    from spear_b200.nn.ssm import SelectiveSSM                    # the layer of these operators
    from spear_b200.nn.block import MixerBlock                    # pre-norm residual block around either layer

The native library is loaded on first use; there is no CPU or PyTorch fallback.
"""

__version__ = "0.1.0"

__all__ = ["btp", "Phalanx", "SigmoidA", "SelectiveSSM", "MixerBlock", "install_as_spear_backend"]


def install_as_spear_backend():
    """Makes an UNMODIFIED installation of the reference package `spear` run on these kernels.

    Registers `spear_b200._btp` as the compiled extension module `spear._btp` that the reference imports
    (spear/ops/btp/interface.py:16) and calls (interface.py:63,87).  Call it before or after `import spear`.
    Returns the imported `spear` package.
    """
    import importlib
    import sys

    from . import _btp as native

    sys.modules["spear._btp"] = native
    spear = importlib.import_module("spear")
    spear._btp = native  # `spear._btp.forward(...)` is looked up as an attribute at call time
    return spear


def __getattr__(name):  # lazy: importing the package must not require torch ops to be registered
    if name == "btp":
        from .ops.btp import btp

        return btp
    if name in ("Phalanx", "SigmoidA"):
        from .nn import phalanx

        return getattr(phalanx, name)
    if name == "SelectiveSSM":
        from .nn.ssm import SelectiveSSM

        return SelectiveSSM
    if name == "MixerBlock":
        from .nn.block import MixerBlock

        return MixerBlock
    raise AttributeError(name)

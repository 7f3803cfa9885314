"""Refusals of the root-mean-square norm: every one names its argument, on a machine without a GPU too."""

from __future__ import annotations

import ctypes

import pytest
import torch

from spear_b200.ops.norm import rms_norm, rms_norm_8bit


@pytest.mark.parametrize("fn", [rms_norm, rms_norm_8bit])
@pytest.mark.parametrize("args,kw,err,text", [
    ((torch.zeros(()),), {}, ValueError, "x must be"),
    ((torch.zeros(4, 0),), {}, ValueError, "x must be"),
    ((torch.zeros(1, 16385),), {}, ValueError, "x must be"),
    ((torch.zeros(4, 8, dtype=torch.float64),), {}, RuntimeError, "x must be bfloat16"),
    ((torch.zeros(4, 8), torch.ones(4)), {}, ValueError, "weight must be"),
    ((torch.zeros(4, 8), torch.ones(8).half()), {}, RuntimeError, "weight must have"),
    ((torch.zeros(4, 8), None, torch.zeros(4, 9)), {}, ValueError, "residual must have"),
    ((torch.zeros(4, 8), None, torch.zeros(1, 8)), {}, ValueError, "residual must have"),
    ((torch.zeros(4, 8).bfloat16(), None, torch.zeros(4, 8).half()), {}, RuntimeError, "residual must have"),
    ((torch.zeros(4, 8),), {"eps": -1.0}, ValueError, "eps"),
    ((torch.zeros(4, 8),), {"eps": float("nan")}, ValueError, "eps"),
    ((torch.zeros(4, 8),), {}, RuntimeError, "no CPU path"),
])
def test_refusals(fn, args, kw, err, text):
    with pytest.raises(err, match=text):
        fn(*args, **kw)


def test_block_is_none_or_128():
    with pytest.raises(ValueError, match="block"):
        rms_norm_8bit(torch.zeros(4, 8), block=64)


def test_entry_refuses_bad_arguments_before_any_launch():
    from spear_b200 import _lib

    lib = _lib.load()
    p = ctypes.c_void_p(16)

    def fwd(x=p, res=None, w=None, y=p, h=None, rows=1, dim=8, ld=8, eps=1e-6, dt=0, rt=0, wt=0, mode=0, scale=None):
        return lib.btp_sm100_rms_norm_forward(x, res, w, y, h, None, scale, rows, dim, ld, ld, eps, dt, rt, wt, mode, None)

    assert fwd(rows=0) == -2 and fwd(dim=0) == -2 and fwd(dim=16385) == -2 and fwd(rows=1 << 31) == -2
    assert fwd(ld=7) == -2 and fwd(eps=-1.0) == -2
    assert fwd(dt=2) == -4 and fwd(res=p, h=p, rt=3) == -4 and fwd(w=p, wt=3) == -4
    assert fwd(mode=3) == -3
    assert fwd(x=None) == -1 and fwd(y=None) == -1 and fwd(res=p) == -1 and fwd(mode=1) == -1
    bwd = lib.btp_sm100_rms_norm_backward
    assert bwd(None, None, p, None, p, p, None, None, None, 1, 8, 8, 0, 0, 0, None) == -1
    assert bwd(p, p, p, None, p, p, None, p, None, 1, 8, 8, 0, 0, 0, None) == -1  # dweight without its scratch
    assert bwd(p, p, p, None, p, p, None, None, None, 1, 8, 7, 0, 0, 0, None) == -2

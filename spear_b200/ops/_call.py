"""What the token-major operators (norm, convolution, scan) share: argument checks and the call into the library.

Checks of shapes and types come before the check for CUDA, so that a refusal names the argument that is wrong on any
machine.  Like the other operators here these have no CPU path and no fallback.
"""

from __future__ import annotations

import torch

from .. import _btp as _native
from .. import _lib

TAG = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


def activation(t: torch.Tensor, what: str) -> None:
    if t.dtype not in TAG:
        raise RuntimeError(f"{what} must be bfloat16, float16 or float32 (got {t.dtype})")


def on_gpu(what: str, *tensors) -> int:
    """All tensors (None is skipped) on one CUDA device; returns its index."""
    index = -1
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{what} needs CUDA tensors: this package has no CPU path and no fallback")
        if index < 0:
            index = t.device.index
        elif t.device.index != index:
            raise RuntimeError(f"{what}: all tensors must be on one device (got cuda:{index} and {t.device})")
    return index


def ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def call(name: str, index: int, *args) -> None:
    """Enqueues a launch on the current stream of device `index`; the stream is the entry's last argument."""
    fn = getattr(_lib._lib or _lib.load(), name)
    if index == _native._current_device():
        rc = fn(*args, _native._raw_stream(index))
    else:
        with _native._OnDevice(index) as stream:
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc, name)


def query(name: str, index: int, *args) -> int:
    """A size that depends on the device's launch shape."""
    fn = getattr(_lib._lib or _lib.load(), name)
    if index == _native._current_device():
        n = fn(*args)
    else:
        with _native._OnDevice(index):
            n = fn(*args)
    if n < 0:
        _lib.check(int(n), name)
    return int(n)

"""What the token-major operators (norm, convolution, scan) share: argument checks and the call into the library.

Checks of shapes and types come before the check for CUDA, so that a refusal names the argument that is wrong on any
machine.  Like the other operators here these have no CPU path and no fallback.
"""

from __future__ import annotations

import torch

from .. import _btp as _native
from .. import _lib

TAG = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


_current_device, _raw_stream = _native._current_device, _native._raw_stream
_fns: dict = {}  # the library's functions by name, looked up once


def _entry(name: str):
    _fns[name] = fn = getattr(_lib.load(), name)
    return fn


def activation(t: torch.Tensor, what: str) -> None:
    if t.dtype not in TAG:
        raise RuntimeError(f"{what} must be bfloat16, float16 or float32 (got {t.dtype})")


def on_gpu(what: str, first: torch.Tensor, *others) -> int:
    """All tensors (None is skipped) on one CUDA device; returns its index."""
    index = first.get_device()
    if index < 0:
        raise RuntimeError(f"{what} needs CUDA tensors: this package has no CPU path and no fallback")
    for t in others:
        if t is not None and t.get_device() != index:
            if t.get_device() < 0:
                raise RuntimeError(f"{what} needs CUDA tensors: this package has no CPU path and no fallback")
            raise RuntimeError(f"{what}: all tensors must be on one device (got cuda:{index} and {t.device})")
    return index


def ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def call(name: str, index: int, *args) -> None:
    """Enqueues a launch on the current stream of device `index`; the stream is the entry's last argument."""
    fn = _fns.get(name) or _entry(name)
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with _native._OnDevice(index) as stream:
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc, name)


def query(name: str, index: int, *args) -> int:
    """A size that depends on the device's launch shape."""
    fn = _fns.get(name) or _entry(name)
    if index == _current_device():
        n = fn(*args)
    else:
        with _native._OnDevice(index):
            n = fn(*args)
    if n < 0:
        _lib.check(int(n), name)
    return int(n)


def traceable(name: str, direct):
    """The registered op `spear_btp::name` while torch.compile traces, the function behind it otherwise (the dispatcher takes
    longer than a small launch)."""
    op = getattr(torch.ops.spear_btp, name)
    compiling = torch.compiler.is_compiling

    def run(*args):
        if compiling():
            op(*args)
        else:
            direct(*args)

    return run

"""What the token-major operators (norm, convolution, scan) share: argument checks and the call into the library.

Checks of shapes and types come before the check for CUDA, so that a refusal names the argument that is wrong on any
machine.  Like the other operators here these have no CPU path and no fallback.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from .. import _btp as _native
from .. import _lib

TAG = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}

# a call has CUDA tensors, so CUDA is initialised and the plain lookup will do
_current_device, _raw_stream = getattr(torch._C, "_cuda_getDevice", _native._current_device), _native._raw_stream
_fns: dict = {}  # the library's functions by name, looked up once


def _entry(name: str):
    _fns[name] = fn = getattr(_lib.load(), name)
    return fn


def activation(what: str, name: str, t: torch.Tensor) -> None:
    """A type that the kernels read, and sizes that fit: the C entries take 32 bits, and ctypes would cut a larger one off without a word."""
    if t.dtype not in TAG:
        raise RuntimeError(f"{what}: {name} must be bfloat16, float16 or float32 (got {t.dtype})")
    if t.numel() > 0x7FFFFFFF and max(t.shape) > 0x7FFFFFFF:
        raise ValueError(f"{what}: every size must be below 2^31, got {tuple(t.shape)}")


def on_gpu(what: str, first: torch.Tensor, *others) -> int:
    """All tensors (None is skipped) on one CUDA device and without tangents; returns the device's index."""
    if forward_ad._current_level >= 0:  # a dual tensor does not require grad: nothing else would notice it, and its tangent would be lost
        for t in (first, *others):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what} has no forward-mode derivative")
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


def dense(t: torch.Tensor | None) -> torch.Tensor | None:
    return t if t is None or t.is_contiguous() else t.contiguous()


def dense_last(t: torch.Tensor | None) -> torch.Tensor | None:
    return t if t is None or t.is_contiguous() or t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def buffers(what: str, index: int, *wanted) -> None:
    """Refuses buffers of a registered op, each (tensor or None, name, elements, dtype), that a launch would reach past."""
    for t, name, n, dtype in wanted:
        if t is not None and (t.numel() != n or t.dtype != dtype or not t.is_contiguous() or t.get_device() != index):
            raise ValueError(f"{what}: {name} must hold {n} contiguous {dtype} on cuda:{index}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def pass_on(into: torch.Tensor | None, given: torch.Tensor | None) -> None:
    """No tokens: a state (or its gradient) goes through as it came, zeros where none came."""
    if into is not None:
        into.zero_() if given is None else into.copy_(given)


_modes, _tracing = torch._C._len_torch_dispatch_stack, torch._C._is_tracing
_compiling = torch.compiler.is_compiling
_PLAIN = frozenset((torch.Tensor, torch.nn.Parameter, type(None)))


def recorded(*tensors) -> bool:
    """Whether somebody records or interprets a call with these arguments (torch.compile, make_fx and other dispatch modes,
    torch.jit.trace, a tensor subclass): it then goes through the registered ops `spear_btp::...`.

    A recorded op is replayed on tensors that no public function has looked at, so the ops check their arguments themselves."""
    return _compiling() or _modes() > 0 or _tracing() or not _PLAIN.issuperset(map(type, tensors))


def training(*tensors) -> bool:
    """Whether the call takes an autograd node (always while torch.compile traces: it may add gradients later)."""
    return _compiling() or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors))


def no_gradient(lib: torch.library.Library, name: str) -> None:
    """The op is no step of autograd's: it runs as it is under any gradient mode, and what it writes does not require grad."""
    lib.impl(name, torch.library.fallthrough_kernel, "Autograd")


native = _lib.native

"""``selective_scan`` and ``selective_scan_step``: a state space recurrence whose step size, input and output depend on the token.

    Delta_t = softplus(delta_t + delta_bias)                       step size per channel
    h_t[d, n] = exp(Delta_t[d] A[d, n]) h_{t-1}[d, n] + Delta_t[d] x_t[d] B_t[n]
    y_t[d] = sum_n C_t[n] h_t[d, n] + D[d] x_t[d],   times silu(z_t) where there is a gate

Token-major, [batch, length, channels]; the state is float32.  Where the BTP recurrence looks back over one block, this
one's state reaches over the whole prompt.  CUDA only, no fallback.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ..btp import interface as _iface
from .. import _call
from .._call import dense, dense_last
from .conv import check_lengths, check_state_out, row, strides, written

__all__ = ["selective_scan", "selective_scan_step", "MAX_STATES"]

MAX_STATES = 64
_CHECKPOINT = 16  # tokens between the states that the forward keeps for the backward


def _aligned(t: torch.Tensor | None) -> torch.Tensor | None:
    """16-byte aligned: a dense view that starts elsewhere gets copied."""
    return t if t is None or t.data_ptr() % 16 == 0 else t.clone()


def _check_params(what, dim, A, D, delta_bias) -> int:
    shape = A.shape
    if len(shape) != 2 or shape[0] != dim or not 1 <= shape[1] <= MAX_STATES:
        raise ValueError(f"{what}: A must be [{dim}, N] with 1 <= N <= {MAX_STATES}, got {tuple(shape)}")
    if A.dtype != torch.float32:
        raise RuntimeError(f"{what}: A must be float32 (got {A.dtype})")
    for t, name in ((D, "D"), (delta_bias, "delta_bias")):
        if t is None:
            continue
        if t.shape != (dim,):
            raise ValueError(f"{what}: {name} must be [{dim}], got {tuple(t.shape)}")
        if t.dtype != torch.float32:
            raise RuntimeError(f"{what}: {name} must be float32 (got {t.dtype})")
    return shape[1]


def _check_tokens(what, x, delta, z, B, C, states, at="") -> None:
    dtype, shape = x.dtype, x.shape
    if (delta.shape == shape and B.shape == states and C.shape == states and delta.dtype == dtype and B.dtype == dtype and C.dtype == dtype
            and (z is None or (z.shape == shape and z.dtype == dtype))):
        return
    for t, name, shape in ((delta, "delta" + at, shape), (z, "z" + at, shape), (B, "B" + at, states), (C, "C" + at, states)):
        if t is None:
            continue
        if t.shape != shape:
            raise ValueError(f"{what}: {name} must be {tuple(shape)}, got {tuple(t.shape)}")
        if t.dtype != dtype:
            raise RuntimeError(f"{what}: {name} must have x's dtype ({dtype}), got {t.dtype}")


def _check(what, x, delta, A, B, C, D, z, delta_bias, initial, lengths) -> tuple[int, int]:
    """(states, device) of a scan over [B, L, D]."""
    if x.dim() != 3 or x.shape[2] < 1:
        raise ValueError(f"{what}: x must be [B, L, D], got {tuple(x.shape)}")
    Bsz, L, dim = x.shape
    _call.activation(what, "x", x)
    N = _check_params(what, dim, A, D, delta_bias)
    _check_tokens(what, x, delta, z, B, C, (Bsz, L, N))
    if initial is not None and (tuple(initial.shape) != (Bsz, dim, N) or initial.dtype != torch.float32):
        raise ValueError(f"{what}: initial_state must be float32 {(Bsz, dim, N)}, got {initial.dtype} {tuple(initial.shape)}")
    check_lengths(what, lengths, Bsz)
    return N, _call.on_gpu(what, x, delta, A, B, C, D, z, delta_bias, initial, lengths)


def _check_step(what, x_t, delta_t, A, B_t, C_t, state, D, z_t, delta_bias) -> int:
    """The device of a single token's scan."""
    if x_t.dim() != 2 or x_t.shape[1] < 1:
        raise ValueError(f"{what}: x_t must be [B, D], got {tuple(x_t.shape)}")
    Bsz, dim = x_t.shape
    _call.activation(what, "x_t", x_t)
    N = _check_params(what, dim, A, D, delta_bias)
    _check_tokens(what, x_t, delta_t, z_t, B_t, C_t, (Bsz, N), "_t")
    if state.shape != (Bsz, dim, N) or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"{what}: state must be contiguous float32 {(Bsz, dim, N)}, got {state.dtype} {tuple(state.shape)}")
    return _call.on_gpu(what, x_t, delta_t, A, B_t, C_t, state, D, z_t, delta_bias)


def _shape_args(x, delta, A, B, C, z):
    zb, zt = (0, 0) if z is None else strides(z)
    return (x.shape[0], x.shape[1], x.shape[2], A.shape[1], *strides(x), *strides(delta), *strides(B), *strides(C), zb, zt)


def _launch_forward(x, delta, A, B, C, D, z, delta_bias, initial, lengths, y, state, checkpoints, softplus) -> None:
    index = x.device.index
    A, initial = _aligned(A), _aligned(initial)
    shape = _shape_args(x, delta, A, B, C, z)
    n = _call.query("btp_sm100_scan_carry_floats", index, *shape[:4])
    carry = torch.empty(n, device=x.device, dtype=torch.float32) if n else None
    p = _call.ptr
    _call.call("btp_sm100_scan_forward", index, x.data_ptr(), delta.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), p(D), p(z),
               p(delta_bias), p(initial), p(lengths), y.data_ptr(), p(state), p(checkpoints), p(carry), *shape, int(softplus),
               _call.TAG[x.dtype])


def _op_forward(x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: Optional[torch.Tensor],
                z: Optional[torch.Tensor], delta_bias: Optional[torch.Tensor], initial: Optional[torch.Tensor],
                lengths: Optional[torch.Tensor], y: torch.Tensor, state: Optional[torch.Tensor], checkpoints: Optional[torch.Tensor],
                softplus: bool) -> None:
    what = "spear_btp::scan_forward"
    N, index = _check(what, x, delta, A, B, C, D, z, delta_bias, initial, lengths)
    Bsz, L, dim = x.shape
    _call.buffers(what, index, (y, "y", x.numel(), x.dtype), (state, "state", Bsz * dim * N, torch.float32),
                  (checkpoints, "checkpoints", Bsz * -(-L // _CHECKPOINT) * dim * N, torch.float32))
    if x.numel():
        _launch_forward(dense_last(x), dense_last(delta), dense(A), dense_last(B), dense_last(C), dense(D), dense_last(z),
                        dense(delta_bias), dense(initial), dense(lengths), y, state, checkpoints, softplus)
    else:
        _call.pass_on(state, initial)


def _op_backward(x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: Optional[torch.Tensor],
                 z: Optional[torch.Tensor], delta_bias: Optional[torch.Tensor], lengths: Optional[torch.Tensor],
                 checkpoints: torch.Tensor, dy: torch.Tensor, dstate: Optional[torch.Tensor], dx: torch.Tensor, ddelta: torch.Tensor,
                 dparams: torch.Tensor, dB: torch.Tensor, dC: torch.Tensor, dz: Optional[torch.Tensor],
                 dinitial: Optional[torch.Tensor], softplus: bool) -> None:
    what = "spear_btp::scan_backward"
    N, index = _check(what, x, delta, A, B, C, D, z, delta_bias, None, lengths)
    Bsz, L, dim = x.shape
    n, m, f32 = x.numel(), Bsz * dim * N, torch.float32
    if z is not None and dz is None:
        raise ValueError(f"{what}: z comes with dz")
    _call.buffers(what, index, (checkpoints, "checkpoints", Bsz * -(-L // _CHECKPOINT) * dim * N, f32), (dy, "dy", n, x.dtype),
                  (dstate, "dstate", m, f32), (dx, "dx", n, x.dtype), (ddelta, "ddelta", n, x.dtype),
                  (dparams, "dparams", _parameter_floats(dim, N), f32), (dB, "dB", B.numel(), x.dtype), (dC, "dC", C.numel(), x.dtype),
                  (dz, "dz", n, x.dtype), (dinitial, "dinitial", m, f32))
    if n:
        _launch_backward(dense_last(x), dense_last(delta), dense(A), dense_last(B), dense_last(C), dense(D), dense_last(z),
                         dense(delta_bias), dense(lengths), checkpoints, dy, dstate, dx, ddelta, dparams, dB, dC, dz, dinitial, softplus)
    else:
        _call.pass_on(dinitial, dstate), _call.pass_on(dparams, None)


def _parameter_floats(dim: int, N: int) -> int:
    """Elements of dA, dD and dbias, one after the other, up to a whole 16 bytes."""
    return -(-dim * (N + 2) // 4) * 4


def _launch_backward(x, delta, A, B, C, D, z, delta_bias, lengths, checkpoints, dy, dstate, dx, ddelta, dparams, dB, dC, dz, dinitial,
                     softplus) -> None:
    index = x.device.index
    A, dstate = _aligned(A), _aligned(dstate)
    shape = _shape_args(x, delta, A, B, C, z)
    buffer = torch.empty(_call.query("btp_sm100_scan_backward_floats", index, *shape[:4]), device=x.device, dtype=torch.float32)
    p = _call.ptr
    _call.call("btp_sm100_scan_backward", index, x.data_ptr(), delta.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), p(D), p(z),
               p(delta_bias), p(lengths), checkpoints.data_ptr(), dy.data_ptr(), p(dstate), dx.data_ptr(), ddelta.data_ptr(),
               dparams.data_ptr(), dB.data_ptr(), dC.data_ptr(), p(dz), p(dinitial), buffer.data_ptr(), *shape, int(softplus),
               _call.TAG[x.dtype])


def _launch_step(x_t, delta_t, A, B_t, C_t, state, D, z_t, delta_bias, y, state_out, softplus) -> None:
    Bsz, dim = x_t.shape
    if (state.data_ptr() | state_out.data_ptr()) % 16:
        raise ValueError("selective_scan_step: state and state_out must be 16-byte aligned")
    (x_t, px), (delta_t, pd), (B_t, pB), (C_t, pC), (z_t, pz) = row(x_t), row(delta_t), row(B_t), row(C_t), row(z_t)
    A, D, delta_bias = _aligned(dense(A)), dense(D), dense(delta_bias)
    p = _call.ptr
    _call.call("btp_sm100_scan_step", x_t.get_device(), x_t.data_ptr(), delta_t.data_ptr(), A.data_ptr(), B_t.data_ptr(), C_t.data_ptr(),
               p(D), p(z_t), p(delta_bias), state.data_ptr(), y.data_ptr(), state_out.data_ptr(), Bsz, dim, A.shape[1], px, pd, pB, pC, pz,
               1 if softplus else 0, _call.TAG[x_t.dtype])


def _op_step(x_t: torch.Tensor, delta_t: torch.Tensor, A: torch.Tensor, B_t: torch.Tensor, C_t: torch.Tensor, state: torch.Tensor,
             D: Optional[torch.Tensor], z_t: Optional[torch.Tensor], delta_bias: Optional[torch.Tensor], y: torch.Tensor,
             state_out: torch.Tensor, softplus: bool) -> None:
    what = "spear_btp::scan_step"
    index = _check_step(what, x_t, delta_t, A, B_t, C_t, state, D, z_t, delta_bias)
    check_state_out(what, state, state_out)
    _call.buffers(what, index, (y, "y", x_t.numel(), x_t.dtype))
    if x_t.numel():
        _launch_step(x_t, delta_t, A, B_t, C_t, state, D, z_t, delta_bias, y, state_out, softplus)


def _fake(*args) -> None:
    return None


_iface._register(_iface._LIB, "spear_btp", "scan_forward", _op_forward, _fake, ["y", "state", "checkpoints"])
_iface._register(_iface._LIB, "spear_btp", "scan_backward", _op_backward, _fake, ["dx", "ddelta", "dparams", "dB", "dC", "dz", "dinitial"])
_iface._register(_iface._LIB, "spear_btp", "scan_step", _op_step, _fake, ["y", "state_out"])
_call.no_gradient(_iface._LIB, "scan_step")
_op, _backward_op, _token_op = torch.ops.spear_btp.scan_forward, torch.ops.spear_btp.scan_backward, torch.ops.spear_btp.scan_step


class _SelectiveScan(torch.autograd.Function):
    """The training pass where it is recorded; otherwise the same steps run in C++ (csrc/btp_torch.cpp)."""

    @staticmethod
    def forward(ctx, x, delta, A, B, C, D, z, delta_bias, initial, lengths, softplus, want_state):
        Bsz, L, dim = x.shape
        N = A.shape[1]
        y = x.new_empty((Bsz, L, dim))
        state = x.new_empty((Bsz, dim, N), dtype=torch.float32) if want_state else None
        checkpoints = x.new_empty((Bsz, -(-L // _CHECKPOINT), dim, N), dtype=torch.float32)
        _op(x, delta, A, B, C, D, z, delta_bias, initial, lengths, y, state, checkpoints, softplus)
        ctx.save_for_backward(x, delta, A, B, C, D, z, delta_bias, lengths, checkpoints)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return (y, state) if want_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate=None):
        x, delta, A, B, C, D, z, delta_bias, lengths, checkpoints = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dy is None and dstate is None:
            return (None,) * 12
        Bsz, L, dim = x.shape
        N = A.shape[1]
        dy = x.new_zeros(x.shape) if dy is None else dy.contiguous()
        dstate = dense(dstate)
        dx, ddelta = (x.new_empty(x.shape) for _ in range(2))
        dz = None if z is None else x.new_empty(x.shape)
        dB, dC = (x.new_empty(B.shape) for _ in range(2))
        dparams = x.new_empty(_parameter_floats(dim, N), dtype=torch.float32)
        dinitial = x.new_empty((Bsz, dim, N), dtype=torch.float32) if need[8] else None
        _backward_op(x, delta, A, B, C, D, z, delta_bias, lengths, checkpoints, dy, dstate, dx, ddelta, dparams, dB, dC, dz, dinitial,
                     ctx.softplus)
        dA, dD, dbias = dparams[:dim * N].view(dim, N), dparams[dim * N:dim * (N + 1)], dparams[dim * (N + 1):dim * (N + 2)]
        grads = (dx, ddelta, dA, dB, dC, None if D is None else dD, dz, None if delta_bias is None else dbias, dinitial)
        return (*(g if n else None for g, n in zip(grads, need)), None, None, None)


def selective_scan(x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: torch.Tensor | None = None, z: torch.Tensor | None = None, *, delta_bias: torch.Tensor | None = None,
                   delta_softplus: bool = False, initial_state: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                   return_state: bool = False):
    """Selective state space scan over tokens.

    Args:
        x: [B, L, D] inputs, bfloat16, float16 or float32 (views with dense channels are read in place, here and below).
        delta: [B, L, D] step sizes before bias and softplus, in x's dtype.
        A: [D, N] float32 rates (negative for a decaying state), 1 <= N <= 64.
        B, C: [B, L, N] input and output weights of the states, in x's dtype; all channels share them.
        D: [D] float32 weight of the input itself, or None.
        z: [B, L, D] gate in x's dtype, or None: y is multiplied by silu(z).
        delta_bias: [D] float32 added to delta, or None.
        delta_softplus: whether the step size is softplus(delta + delta_bias).
        initial_state: [B, D, N] float32 state before token 0, None for zeros.
        lengths: int32 [B] on the GPU: tokens from lengths[b] on (a padded batch) are not read and give 0; values are
            held to 0 ... L.
        return_state: also return the state after each sequence's last token, the ``state`` of ``selective_scan_step``.
    Returns:
        y [B, L, D], or (y, state [B, D, N] float32).  Gradients for every floating-point argument; the backward pass
        keeps one state per 16 tokens from the forward.
    """
    N, _ = _check("selective_scan", x, delta, A, B, C, D, z, delta_bias, initial_state, lengths)
    Bsz, L, dim = x.shape
    if Bsz == 0 or L == 0:  # nothing to compute; the state passes through
        y = x * 1
        if not return_state:
            return y
        return y, (x.new_zeros((Bsz, dim, N), dtype=torch.float32) if initial_state is None else initial_state.clone())
    x, delta, B, C, z = dense_last(x), dense_last(delta), dense_last(B), dense_last(C), dense_last(z)
    A, D, delta_bias, initial_state, lengths = dense(A), dense(D), dense(delta_bias), dense(initial_state), dense(lengths)
    tensors = (x, delta, A, B, C, D, z, delta_bias, initial_state)
    if not _call.recorded(*tensors, lengths):
        y, state = _call.native().selective_scan(*tensors, lengths, bool(delta_softplus), bool(return_state))
        return (y, state) if return_state else y
    if _call.training(*tensors):
        return _SelectiveScan.apply(*tensors, lengths, bool(delta_softplus), bool(return_state))
    y = x.new_empty((Bsz, L, dim))
    state = x.new_empty((Bsz, dim, N), dtype=torch.float32) if return_state else None
    _op(x, delta, A, B, C, D, z, delta_bias, initial_state, lengths, y, state, None, bool(delta_softplus))
    return (y, state) if return_state else y


def selective_scan_step(x_t: torch.Tensor, delta_t: torch.Tensor, A: torch.Tensor, B_t: torch.Tensor, C_t: torch.Tensor,
                        state: torch.Tensor, D: torch.Tensor | None = None, z_t: torch.Tensor | None = None, *,
                        delta_bias: torch.Tensor | None = None, delta_softplus: bool = False, state_out: torch.Tensor | None = None):
    """One token of ``selective_scan``: returns (y_t [B, D], new state [B, D, N] float32).

    x_t, delta_t, z_t [B, D] and B_t, C_t [B, N] as there, without the token dimension.  One kernel launch, no gradient:
    neither result requires grad, whatever the inputs do.  ``state`` stays valid and the new state is a fresh tensor,
    unless ``state_out`` says where to write it: passing the state itself updates it in place (the form for a captured
    graph).
    """
    what = "selective_scan_step"
    _check_step(what, x_t, delta_t, A, B_t, C_t, state, D, z_t, delta_bias)
    if state_out is not None:
        check_state_out(what, state, state_out)
    tensors = (x_t, delta_t, A, B_t, C_t, state, D, z_t, delta_bias)
    if not _call.recorded(*tensors, state_out):
        y, out = _call.native().selective_scan_step(*tensors, state_out, bool(delta_softplus))
    else:
        out = check_state_out(what, state, state_out)
        y = torch.empty_like(x_t, memory_format=torch.contiguous_format)
        _token_op(*tensors, y, out, bool(delta_softplus))
    if state_out is None:
        return y, out
    written(state_out)
    return y, state_out

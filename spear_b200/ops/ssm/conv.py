"""``causal_conv`` and ``causal_conv_step``: a short convolution over tokens, one filter per channel.

    pre[b, t, d] = bias[d] + sum_w weight[d, w] * x[b, t - (W - 1) + w, d]        y = pre, or silu(pre)

Token-major, [batch, length, channels], as a projection leaves its output (a column slice of a wider one is read in
place).  CUDA only, no fallback.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ..btp import interface as _iface
from .. import _call
from .._call import dense, dense_last

__all__ = ["causal_conv", "causal_conv_step"]

WIDTHS = (2, 3, 4)


def _check_filter(what, dim, dtype, weight, bias, activation) -> int:
    shape = weight.shape
    if len(shape) != 2 or shape[0] != dim or shape[1] not in WIDTHS:
        raise ValueError(f"{what}: weight must be [{dim}, W] with W in {WIDTHS}, got {tuple(weight.shape)}")
    if weight.dtype != dtype and weight.dtype != torch.float32:
        raise RuntimeError(f"{what}: weight must have x's dtype ({dtype}) or be float32 (got {weight.dtype})")
    if bias is not None:
        if bias.shape != (dim,):
            raise ValueError(f"{what}: bias must be [{dim}], got {tuple(bias.shape)}")
        if bias.dtype != weight.dtype:
            raise RuntimeError(f"{what}: bias must have the weight's dtype ({weight.dtype}), got {bias.dtype}")
    if activation not in (None, "silu"):
        raise ValueError(f"{what}: activation must be None or 'silu' (got {activation!r})")
    return shape[1]


def check_lengths(what, lengths, batch) -> None:
    if lengths is None:
        return
    if tuple(lengths.shape) != (batch,) or lengths.dtype != torch.int32:
        raise ValueError(f"{what}: lengths must be int32 [{batch}], got {lengths.dtype} {tuple(lengths.shape)}")


def _check(what, x, weight, bias, activation, initial, lengths) -> tuple[int, int]:
    """(taps, device) of a convolution over [B, L, D]."""
    if x.dim() != 3 or x.shape[2] < 1:
        raise ValueError(f"{what}: x must be [B, L, D], got {tuple(x.shape)}")
    B, L, D = x.shape
    _call.activation(what, "x", x)
    W = _check_filter(what, D, x.dtype, weight, bias, activation)
    if initial is not None:
        if tuple(initial.shape) != (B, W - 1, D):
            raise ValueError(f"{what}: initial_state must be {(B, W - 1, D)}, got {tuple(initial.shape)}")
        if initial.dtype != x.dtype:
            raise RuntimeError(f"{what}: initial_state must have x's dtype ({x.dtype}), got {initial.dtype}")
    check_lengths(what, lengths, B)
    return W, _call.on_gpu(what, x, weight, bias, initial, lengths)


def _check_step(what, x_t, state, weight, bias, activation) -> int:
    """The device of a single token's convolution."""
    if x_t.dim() != 2 or x_t.shape[1] < 1:
        raise ValueError(f"{what}: x_t must be [B, D], got {tuple(x_t.shape)}")
    B, D = x_t.shape
    _call.activation(what, "x_t", x_t)
    W = _check_filter(what, D, x_t.dtype, weight, bias, activation)
    if state.shape != (B, W - 1, D) or state.dtype != x_t.dtype or not state.is_contiguous():
        raise ValueError(f"{what}: state must be contiguous {(B, W - 1, D)} of x_t's dtype, got {state.dtype} {tuple(state.shape)}")
    return _call.on_gpu(what, x_t, state, weight, bias)


def row(t: torch.Tensor | None):
    """[B, D] with dense rows, and its pitch."""
    if t is None:
        return None, 0
    if t.is_contiguous():
        return t, t.shape[1]
    t = dense_last(t)
    return t, t.stride(0)


def strides(t: torch.Tensor) -> tuple[int, int]:
    """Batch and token strides of [B, L, D]; a dimension of one element has none of its own."""
    st = t.stride(1) if t.shape[1] > 1 else t.shape[2]
    return (t.stride(0) if t.shape[0] > 1 else t.shape[1] * st), st


def _launch_forward(x, weight, bias, initial, lengths, y, state, silu) -> None:
    B, L, D = x.shape
    sb, st = strides(x)
    _call.call("btp_sm100_causal_conv_forward", x.device.index, x.data_ptr(), weight.data_ptr(), _call.ptr(bias), _call.ptr(initial),
               _call.ptr(lengths), y.data_ptr(), _call.ptr(state), B, L, D, weight.shape[1], sb, st, int(silu), _call.TAG[x.dtype],
               _call.TAG[weight.dtype])


def _op_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], initial: Optional[torch.Tensor],
                lengths: Optional[torch.Tensor], y: torch.Tensor, state: Optional[torch.Tensor], silu: bool) -> None:
    what = "spear_btp::causal_conv_forward"
    W, index = _check(what, x, weight, bias, None, initial, lengths)
    B, L, D = x.shape
    _call.buffers(what, index, (y, "y", B * L * D, x.dtype), (state, "state", B * (W - 1) * D, x.dtype))
    if x.numel():
        _launch_forward(dense_last(x), dense(weight), dense(bias), dense(initial), dense(lengths), y, state, silu)
    else:
        _call.pass_on(state, initial)


def _op_backward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], initial: Optional[torch.Tensor],
                 lengths: Optional[torch.Tensor], dy: torch.Tensor, dstate: Optional[torch.Tensor], dx: torch.Tensor,
                 dweight: Optional[torch.Tensor], dbias: Optional[torch.Tensor], dinitial: Optional[torch.Tensor], silu: bool) -> None:
    what = "spear_btp::causal_conv_backward"
    W, index = _check(what, x, weight, bias, None, initial, lengths)
    B, L, D = x.shape
    n, m = B * L * D, B * (W - 1) * D
    _call.buffers(what, index, (dy, "dy", n, x.dtype), (dstate, "dstate", m, x.dtype), (dx, "dx", n, x.dtype),
                  (dweight, "dweight", D * W, weight.dtype), (dbias, "dbias", D, weight.dtype), (dinitial, "dinitial", m, x.dtype))
    if n:
        _launch_backward(dense_last(x), dense(weight), dense(bias), dense(initial), dense(lengths), dy, dstate, dx, dweight, dbias,
                         dinitial, silu)
    else:
        _call.pass_on(dinitial, dstate), _call.pass_on(dweight, None), _call.pass_on(dbias, None)


def _launch_backward(x, weight, bias, initial, lengths, dy, dstate, dx, dweight, dbias, dinitial, silu) -> None:
    B, L, D = x.shape
    W = weight.shape[1]
    index = x.device.index
    sb, st = strides(x)
    partial = None
    if dweight is not None or dbias is not None:
        rows = _call.query("btp_sm100_causal_conv_partial_rows", index, B, L, D)
        partial = torch.empty(rows, W + 1, D, device=x.device, dtype=torch.float32)
    _call.call("btp_sm100_causal_conv_backward", index, x.data_ptr(), weight.data_ptr(), _call.ptr(bias), _call.ptr(initial),
               _call.ptr(lengths), dy.data_ptr(), _call.ptr(dstate), dx.data_ptr(), _call.ptr(dweight), _call.ptr(dbias),
               _call.ptr(dinitial), _call.ptr(partial), B, L, D, W, sb, st, int(silu), _call.TAG[x.dtype], _call.TAG[weight.dtype])


def _launch_step(x_t, state, weight, bias, y, state_out, silu) -> None:
    B, D = x_t.shape
    (x_t, pitch), weight, bias = row(x_t), dense(weight), dense(bias)
    _call.call("btp_sm100_causal_conv_step", x_t.get_device(), x_t.data_ptr(), state.data_ptr(), weight.data_ptr(), _call.ptr(bias),
               y.data_ptr(), state_out.data_ptr(), B, D, weight.shape[1], pitch, int(silu), _call.TAG[x_t.dtype],
               _call.TAG[weight.dtype])


def _op_step(x_t: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], y: torch.Tensor,
             state_out: torch.Tensor, silu: bool) -> None:
    what = "spear_btp::causal_conv_step"
    index = _check_step(what, x_t, state, weight, bias, None)
    check_state_out(what, state, state_out)
    _call.buffers(what, index, (y, "y", x_t.numel(), x_t.dtype))
    if x_t.numel():
        _launch_step(x_t, state, weight, bias, y, state_out, silu)


def _fake(*args) -> None:
    return None


_iface._register(_iface._LIB, "spear_btp", "causal_conv_forward", _op_forward, _fake, ["y", "state"])
_iface._register(_iface._LIB, "spear_btp", "causal_conv_backward", _op_backward, _fake, ["dx", "dweight", "dbias", "dinitial"])
_iface._register(_iface._LIB, "spear_btp", "causal_conv_step", _op_step, _fake, ["y", "state_out"])
_call.no_gradient(_iface._LIB, "causal_conv_step")
_op, _backward_op, _token_op = (torch.ops.spear_btp.causal_conv_forward, torch.ops.spear_btp.causal_conv_backward,
                                torch.ops.spear_btp.causal_conv_step)


class _CausalConv(torch.autograd.Function):
    """The training pass where it is recorded; otherwise the same steps run in C++ (csrc/btp_torch.cpp)."""

    @staticmethod
    def forward(ctx, x, weight, bias, initial, lengths, silu, want_state):
        B, L, D = x.shape
        y = x.new_empty((B, L, D))
        state = x.new_empty((B, weight.shape[1] - 1, D)) if want_state else None
        _op(x, weight, bias, initial, lengths, y, state, silu)
        ctx.save_for_backward(x, weight, bias, initial, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return (y, state) if want_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate=None):
        x, weight, bias, initial, lengths = ctx.saved_tensors
        need_x, need_w, need_b, need_i = ctx.needs_input_grad[:4]
        if dy is None and dstate is None:
            return (None,) * 7
        dy = x.new_zeros(x.shape) if dy is None else dy.contiguous()
        dstate = None if dstate is None else dstate.contiguous()
        dx = x.new_empty(x.shape)
        dw = weight.new_empty(weight.shape) if need_w else None
        db = bias.new_empty(bias.shape) if need_b and bias is not None else None
        di = x.new_empty(initial.shape) if need_i and initial is not None else None
        _backward_op(x, weight, bias, initial, lengths, dy, dstate, dx, dw, db, di, ctx.silu)
        return dx if need_x else None, dw, db, di, None, None, None


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None,
                initial_state: torch.Tensor | None = None, lengths: torch.Tensor | None = None, return_state: bool = False):
    """Short causal convolution over tokens, one filter per channel.

    Args:
        x: [B, L, D] bfloat16, float16 or float32 (a view with dense channels is read in place).
        weight: [D, W], W = 2, 3 or 4, the last tap on the token itself; x's dtype or float32.
        bias: [D] in the weight's dtype, or None.
        activation: None or "silu".
        initial_state: [B, W-1, D] in x's dtype, the inputs before token 0, oldest first; None for zeros.
        lengths: int32 [B] on the GPU: tokens from lengths[b] on (a padded batch) are not read and give 0; values are
            held to 0 ... L.
        return_state: also return the last W-1 inputs of each sequence, the ``state`` of ``causal_conv_step``.
    Returns:
        y [B, L, D], or (y, state [B, W-1, D]).  Gradients for x, weight, bias and initial_state.
    """
    W, _ = _check("causal_conv", x, weight, bias, activation, initial_state, lengths)
    B, L, D = x.shape
    if B == 0 or L == 0:  # nothing to compute; the state passes through
        y = x * 1
        if not return_state:
            return y
        return y, (x.new_zeros(B, W - 1, D) if initial_state is None else initial_state.clone())
    x, weight, bias = dense_last(x), dense(weight), dense(bias)
    initial_state, lengths = dense(initial_state), dense(lengths)
    silu = activation == "silu"
    if not _call.recorded(x, weight, bias, initial_state, lengths):
        y, state = _call.native().causal_conv(x, weight, bias, initial_state, lengths, silu, bool(return_state))
        return (y, state) if return_state else y
    if _call.training(x, weight, bias, initial_state):
        return _CausalConv.apply(x, weight, bias, initial_state, lengths, silu, bool(return_state))
    y = x.new_empty((B, L, D))
    state = x.new_empty((B, W - 1, D)) if return_state else None
    _op(x, weight, bias, initial_state, lengths, y, state, silu)
    return (y, state) if return_state else y


def check_state_out(what, state, state_out) -> torch.Tensor:
    """Where the new state goes: fresh memory, or the caller's tensor, which may be the old state itself."""
    if state_out is None:
        return torch.empty_like(state)  # contiguous, as the state is
    if state_out.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: state_out requires grad, and a token has no gradient: detach it, or call under torch.no_grad()")
    if state_out is state:
        return state_out
    if state_out.shape != state.shape or state_out.dtype != state.dtype or state_out.device != state.device or not state_out.is_contiguous():
        raise ValueError(f"{what}: state_out must be contiguous and have the state's shape, dtype and device")
    a, b, n = state.data_ptr(), state_out.data_ptr(), state.numel() * state.element_size()
    if a != b and a < b + n and b < a + n:
        raise ValueError(f"{what}: state_out overlaps the state without being the same memory")
    return state_out


def written(state_out: torch.Tensor) -> None:
    """Tells autograd that the caller's tensor has changed, so that a backward pass that needs its old values fails."""
    if not torch.compiler.is_compiling() and not state_out.is_inference():
        torch.autograd.graph.increment_version(state_out)


def causal_conv_step(x_t: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                     activation: str | None = None, state_out: torch.Tensor | None = None):
    """One token of ``causal_conv``: returns (y_t [B, D], new state [B, W-1, D]).

    One kernel launch, no gradient: neither result requires grad, whatever the inputs do.  ``state`` stays valid and the
    new state is a fresh tensor, unless ``state_out`` says where to write it: passing the state itself updates it in
    place (the form for a captured graph).
    """
    what = "causal_conv_step"
    _check_step(what, x_t, state, weight, bias, activation)
    if state_out is not None:
        check_state_out(what, state, state_out)
    if not _call.recorded(x_t, state, weight, bias, state_out):
        y, out = _call.native().causal_conv_step(x_t, state, weight, bias, state_out, activation is not None)
    else:
        out = check_state_out(what, state, state_out)
        y = torch.empty_like(x_t, memory_format=torch.contiguous_format)
        _token_op(x_t, state, weight, bias, y, out, activation is not None)
    if state_out is None:
        return y, out
    written(state_out)
    return y, state_out

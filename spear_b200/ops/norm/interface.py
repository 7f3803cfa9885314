"""``rms_norm`` and ``rms_norm_8bit`` on the sm_100a kernels.

    h = x + residual            y = h * rsqrt(mean(h^2) + eps) * weight

One pass over the row: the sum, its norm and the output (in 8 bits: with its scale) come from registers.  The
residual stream may be float32 next to 16-bit activations.  CUDA only, no fallback.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ..btp import interface as _iface
from .. import _call

__all__ = ["rms_norm", "rms_norm_8bit", "F8_MAX", "SCALE_BLOCK", "MAX_DIM"]

F8_MAX = 448.0     # largest e4m3 magnitude
SCALE_BLOCK = 128  # columns that share a scale in the blockwise form
MAX_DIM = 16384


def _check(what, x, weight, residual, eps) -> int:
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_DIM:
        raise ValueError(f"{what}: x must be [..., D] with 1 <= D <= {MAX_DIM}, got {tuple(x.shape)}")
    _call.activation(what, "x", x)
    if weight is not None:
        if weight.shape != x.shape[-1:]:
            raise ValueError(f"{what}: weight must be [{x.shape[-1]}], got {tuple(weight.shape)}")
        if weight.dtype != x.dtype and weight.dtype != torch.float32:
            raise RuntimeError(f"{what}: weight must have x's dtype ({x.dtype}) or be float32 (got {weight.dtype})")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"{what}: residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
        if residual.dtype != x.dtype and residual.dtype != torch.float32:
            raise RuntimeError(f"{what}: residual must have x's dtype ({x.dtype}) or be float32 (got {residual.dtype})")
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps must not be negative (got {eps})")
    return _call.on_gpu(what, x, weight, residual)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as [rows, D] with dense rows at one pitch; copied only where its strides allow no such view."""
    d = t.shape[-1]
    if t.dim() == 2 and t.is_contiguous():
        return t
    r = t.reshape(-1, d)
    if (d > 1 and r.stride(1) != 1) or (r.shape[0] > 1 and r.stride(0) < d):
        r = r.contiguous()
    return r


def _pitch(r: torch.Tensor) -> int:
    return r.stride(0) if r.shape[0] > 1 else r.shape[1]


def _launch_forward(x, residual, weight, y, h, rstd, eps, scale=None, out_mode=0) -> None:
    rows, dim = x.shape
    if rows == 0:
        return
    _call.call("btp_sm100_rms_norm_forward", x.get_device(), x.data_ptr(), _call.ptr(residual), _call.ptr(weight), y.data_ptr(),
               _call.ptr(h), _call.ptr(rstd), _call.ptr(scale), rows, dim, _pitch(x), dim if residual is None else _pitch(residual),
               eps, _call.TAG[x.dtype], 0 if residual is None else _call.TAG[residual.dtype],
               0 if weight is None else _call.TAG[weight.dtype], out_mode)


def _op_forward(x: torch.Tensor, residual: Optional[torch.Tensor], weight: Optional[torch.Tensor], y: torch.Tensor,
                h: Optional[torch.Tensor], rstd: Optional[torch.Tensor], eps: float) -> None:
    what = "spear_btp::rms_norm_forward"
    index = _check(what, x, weight, residual, eps)
    n = x.numel()
    _check_h(what, residual, h)
    _call.buffers(what, index, (y, "y", n, x.dtype), (rstd, "rstd", n // x.shape[-1], torch.float32),
                  (h, "h", n, x.dtype if residual is None else residual.dtype))
    _launch_forward(_rows(x), None if residual is None else _rows(residual), _call.dense(weight), y, h, rstd, eps)


def _op_8bit(x: torch.Tensor, residual: Optional[torch.Tensor], weight: Optional[torch.Tensor], q: torch.Tensor,
             h: Optional[torch.Tensor], scale: torch.Tensor, eps: float, blocks: bool) -> None:
    what = "spear_btp::rms_norm_8bit"
    index = _check(what, x, weight, residual, eps)
    n, dim = x.numel(), x.shape[-1]
    _check_h(what, residual, h)
    _call.buffers(what, index, (q, "q", n, torch.float8_e4m3fn), (scale, "scale", n // dim * (-(-dim // SCALE_BLOCK) if blocks else 1), torch.float32),
                  (h, "h", n, x.dtype if residual is None else residual.dtype))
    _launch_8bit(_rows(x), None if residual is None else _rows(residual), _call.dense(weight), q, h, scale, eps, blocks)


def _check_h(what, residual, h) -> None:
    if residual is not None and h is None:
        raise ValueError(f"{what}: a residual comes with h")


def _launch_8bit(x, residual, weight, q, h, scale, eps, blocks) -> None:
    _launch_forward(x, residual, weight, q, h, None, eps, scale, 2 if blocks else 1)


def _op_backward(h: torch.Tensor, weight: Optional[torch.Tensor], dy: torch.Tensor, dh: Optional[torch.Tensor], rstd: torch.Tensor,
                 dx: Optional[torch.Tensor], dresidual: Optional[torch.Tensor], dweight: Optional[torch.Tensor]) -> None:
    what = "spear_btp::rms_norm_backward"
    index = _check(what, _rows(dy), weight, _rows(h), 0.0)
    n, dim = dy.numel(), dy.shape[-1]
    if dweight is not None and weight is None:
        raise ValueError(f"{what}: dweight needs the weight")
    _call.buffers(what, index, (rstd, "rstd", n // dim, torch.float32), (dh, "dh", n, h.dtype), (dx, "dx", n, dy.dtype),
                  (dresidual, "dresidual", n, h.dtype), (dweight, "dweight", dim, None if weight is None else weight.dtype))
    _launch_backward(_rows(h), _call.dense(weight), dy.contiguous(), dh, rstd, dx, dresidual, dweight)


def _launch_backward(h: torch.Tensor, weight: Optional[torch.Tensor], dy: torch.Tensor, dh: Optional[torch.Tensor], rstd: torch.Tensor,
                     dx: Optional[torch.Tensor], dresidual: Optional[torch.Tensor], dweight: Optional[torch.Tensor]) -> None:
    rows, dim = h.shape
    if rows == 0:
        if dweight is not None:
            dweight.zero_()
        return
    index = h.device.index
    partial = None
    if dweight is not None:
        parts = _call.query("btp_sm100_rms_norm_partial_rows", index, rows, dim)
        partial = torch.empty(parts, dim, device=h.device, dtype=torch.float32)
    _call.call("btp_sm100_rms_norm_backward", index, h.data_ptr(), _call.ptr(weight), dy.data_ptr(), _call.ptr(dh), rstd.data_ptr(),
               _call.ptr(dx), _call.ptr(dresidual), _call.ptr(dweight), _call.ptr(partial), rows, dim, _pitch(h),
               _call.TAG[dy.dtype], _call.TAG[h.dtype], 0 if weight is None else _call.TAG[weight.dtype])


def _fake(*args) -> None:
    return None


_iface._register(_iface._LIB, "spear_btp", "rms_norm_forward", _op_forward, _fake, ["y", "h", "rstd"])
_iface._register(_iface._LIB, "spear_btp", "rms_norm_backward", _op_backward, _fake, ["dx", "dresidual", "dweight"])
_iface._register(_iface._LIB, "spear_btp", "rms_norm_8bit", _op_8bit, _fake, ["q", "h", "scale"])
_call.no_gradient(_iface._LIB, "rms_norm_8bit")
_op, _backward_op = torch.ops.spear_btp.rms_norm_forward, torch.ops.spear_btp.rms_norm_backward


class _RMSNorm(torch.autograd.Function):
    """The training pass where it is recorded; otherwise the same steps run in C++ (csrc/btp_torch.cpp)."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        x2 = _rows(x)
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
        h = None if residual is None else torch.empty_like(residual, memory_format=torch.contiguous_format)
        rstd = x.new_empty(x2.shape[0], dtype=torch.float32)
        _op(x2, None if residual is None else _rows(residual), weight, y, h, rstd, eps)
        ctx.save_for_backward(x2 if h is None else h, weight, rstd)
        ctx.dtype = x.dtype
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        if dy is None:  # y was not used: the sum passes its gradient on
            dx = dh.to(ctx.dtype) if dh is not None and need_x else None
            return dx, None, dh if need_r else None, None
        dy = dy.contiguous()
        dh = None if dh is None else dh.contiguous()
        one = h.dtype == ctx.dtype  # one tensor serves as the gradient of both terms of the sum
        dx = torch.empty_like(dy) if need_x or (one and need_r) else None
        dres = torch.empty_like(dy, dtype=h.dtype) if need_r and not one else None
        dw = torch.empty_like(weight) if need_w and weight is not None else None
        if dx is not None or dres is not None or dw is not None:
            _backward_op(_rows(h), weight, dy, dh, rstd, dx, dres, dw)
        return dx if need_x else None, dw, (dx if one else dres) if need_r else None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, *, eps: float = 1e-6):
    """Root-mean-square norm over the last dimension, with the residual's addition.

    Args:
        x: [..., D] bfloat16, float16 or float32, D <= 16384; the last dimension is copied to be dense if it is not.
        weight: [D] in x's dtype or float32, or None for ones.
        residual: [..., D] in x's dtype or float32 (a residual stream kept in 32 bits), or None.  Gradients are taken of
            the sum as it is stored, so a float16 stream must stay below 65504: a sum beyond that is stored as infinity,
            and its row's gradients and its column of the weight's are lost, though y is right.
        eps: added to the mean square.
    Returns:
        y [..., D] in x's dtype; with a residual (y, h) where h = x + residual in the residual's dtype.  y is the
        norm of the sum before that rounding.  Both outputs have gradients.
    """
    _check("rms_norm", x, weight, residual, eps)
    weight = _call.dense(weight)
    if not _call.recorded(x, weight, residual):
        y, h = _call.native().rms_norm(x, weight, residual, float(eps))
        return y if h is None else (y, h)
    if _call.training(x, weight, residual):
        return _RMSNorm.apply(x, weight, residual, float(eps))
    x2 = _rows(x)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    if residual is None:
        _op(x2, None, weight, y, None, None, float(eps))
        return y
    h = torch.empty_like(residual, memory_format=torch.contiguous_format)
    _op(x2, _rows(residual), weight, y, h, None, float(eps))
    return y, h


def rms_norm_8bit(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, *,
                  eps: float = 1e-6, block: int | None = None):
    """rms_norm whose output is e4m3 with float32 scales, the operand of an 8-bit product.  No gradient.

    Args:
        x, weight, residual, eps: as for ``rms_norm``.
        block: None for one scale per row, 128 for one scale per 128 columns (the last may hold fewer).
    Returns:
        (q, scale) or, with a residual, (q, scale, h): q [..., D] float8_e4m3fn, scale [...] or
        [..., ceil(D / 128)] with y = q * scale; scale = max|y| / 448, or 1 where that is NaN or below 1e-37
        (a row of zeros).
    """
    if block not in (None, SCALE_BLOCK):
        raise ValueError(f"rms_norm_8bit: block must be None or {SCALE_BLOCK} (got {block})")
    _check("rms_norm_8bit", x, weight, residual, eps)
    weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    x2 = _rows(x)  # no output below is computed from a tensor that autograd follows
    q = torch.empty_like(x, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
    scale = x.new_empty(x.shape[:-1] if block is None else (*x.shape[:-1], -(-x.shape[-1] // SCALE_BLOCK)), dtype=torch.float32)
    h = None if residual is None else torch.empty_like(residual, memory_format=torch.contiguous_format)
    launch = torch.ops.spear_btp.rms_norm_8bit if _call.recorded(x, weight, residual) else _launch_8bit
    launch(x2, None if residual is None else _rows(residual), weight, q, h, scale, float(eps), block is not None)
    return (q, scale) if h is None else (q, scale, h)

"""The residual's addition and the RMS norm in front of the MoE layer (no
reference counterpart), differentiable, and with an int8 output.

    h = x + residual
    y = h / sqrt(mean(h^2) + eps) * weight

``rms_norm`` gives y (and h, the residual stream of the next block) in x's
type.  ``rms_norm_quant_int8`` gives y as int8 with one scale per token, the
``a`` / ``a_row_scale`` of ``ops.int8_grouped_mm_scaled``, and on request y as
well, for the router.  Sums, norms and scales are fp32; y and the int8 values
come from the unrounded h.

x is [..., K] in bf16, fp16 or fp32 on a CUDA device, of any K and alignment;
rows may have any stride (a last dimension that is not contiguous is copied).
``weight`` is [K] in x's type or fp32; ``residual`` has x's shape and type.
Outputs are new contiguous tensors; nothing synchronises with the host.  Both
passes can be captured into a CUDA graph; as for every autograd graph, drop
eager graphs that hold the same leaves before capturing a backward pass.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import BF16, FP16, FP32, launch

_DT = {torch.bfloat16: BF16, torch.float16: FP16, torch.float32: FP32}


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as [rows, K]: a view where its strides allow one, else a copy."""
    if t.dim() != 2:
        t = t.reshape(-1, t.size(-1))
    return t if t.stride(1) == 1 or t.size(1) == 1 else t.contiguous()


def _check_args(what: str, x, weight, eps, residual) -> None:
    _check(x.is_cuda, f"{what}: x must be a CUDA tensor")
    _check(x.dtype in _DT, f"{what}: x must be bfloat16, float16 or float32")
    _check(x.dim() >= 1 and x.size(-1) >= 1, f"{what}: x must have shape [..., K] with K >= 1")
    _check(weight.device == x.device, f"{what}: weight must be on x's device")
    _check(weight.dtype in (x.dtype, torch.float32),
           f"{what}: weight must have x's dtype or float32")
    _check(weight.dim() == 1 and weight.size(0) == x.size(-1), f"{what}: weight must have shape [K]")
    _check(0.0 <= eps < 3e38, f"{what}: eps must be finite and not negative")
    if residual is not None:
        _check(residual.device == x.device, f"{what}: residual must be on x's device")
        _check(residual.dtype == x.dtype, f"{what}: residual must have x's dtype")
        _check(residual.shape == x.shape, f"{what}: residual must have x's shape")


def _forward(x, weight, eps, residual, y, rstd, q=None, scale=None):
    """Launches the norm; returns the residual stream (None without one)."""
    xr = _rows(x)
    rr = _rows(residual) if residual is not None else None
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else None
    w = weight.contiguous()
    launch("i8moe_rms_norm", x.device, xr.data_ptr(), xr.stride(0),
           rr.data_ptr() if rr is not None else None, rr.stride(0) if rr is not None else 0,
           _DT[x.dtype], w.data_ptr(), _DT[w.dtype], xr.size(0), xr.size(1), eps,
           h.data_ptr() if h is not None else None, y.data_ptr() if y is not None else None,
           rstd.data_ptr() if rstd is not None else None,
           q.data_ptr() if q is not None else None,
           scale.data_ptr() if scale is not None else None)
    return h


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        rstd = torch.empty(x.numel() // x.size(-1), dtype=torch.float32, device=x.device)
        h = _forward(x, weight, eps, residual, y, rstd)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        need_x, need_w, _, need_r = ctx.needs_input_grad
        if dy is None:  # y was not used: only the residual stream's gradient passes
            return (dh if need_x else None), None, None, (dh if need_r else None)
        h, weight, rstd = ctx.saved_tensors
        dx, dw = rms_norm_backward(dy, h, weight, rstd, dh, weight_grad=need_w)
        return (dx if need_x else None), dw, None, (dx if need_r else None)


def rms_norm_backward(dy, h, weight, rstd, residual_grad=None, weight_grad: bool = True):
    """Gradients of ``rms_norm``: (gradient of x and residual, gradient of
    weight or None).  ``h`` is the residual stream (x without a residual),
    ``rstd`` fp32 [rows] = 1 / sqrt(mean(h^2) + eps)."""
    _check_args("rms_norm_backward", h, weight, 0.0, residual_grad)
    _check(dy.shape == h.shape and dy.dtype == h.dtype and dy.device == h.device,
           "rms_norm_backward: dy must have h's shape, dtype and device")
    _check(rstd.dtype == torch.float32 and rstd.is_contiguous() and rstd.device == h.device
           and rstd.numel() == h.numel() // h.size(-1),
           "rms_norm_backward: rstd must be float32 [rows] on h's device")
    hr, gr = _rows(h), _rows(dy)
    rr = _rows(residual_grad) if residual_grad is not None else None
    dx = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    w = weight.contiguous()
    dw = ws = None
    nbytes = 0
    if weight_grad:
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=h.device)
        nbytes = _lib.LIB.i8moe_rms_norm_backward_workspace_size(hr.size(0), hr.size(1))
        ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=h.device)
    launch("i8moe_rms_norm_backward", h.device, gr.data_ptr(), gr.stride(0),
           rr.data_ptr() if rr is not None else None, rr.stride(0) if rr is not None else 0,
           hr.data_ptr(), hr.stride(0), _DT[h.dtype], w.data_ptr(), _DT[w.dtype],
           rstd.data_ptr(), hr.size(0), hr.size(1), dx.data_ptr(),
           dw.data_ptr() if dw is not None else None, ws.data_ptr() if ws is not None else None,
           nbytes)
    return dx, dw


def rms_norm(x, weight, eps: float = 1e-6, residual=None):
    """y, or (y, h) with a residual.  Differentiable in x, weight and
    residual (once); the gradient of weight is summed in a fixed order."""
    _check_args("rms_norm", x, weight, eps, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        return _RMSNorm.apply(x, weight, eps, residual)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = _forward(x, weight, eps, residual, y, None)
    return y if h is None else (y, h)


def rms_norm_quant_int8(x, weight, eps: float = 1e-6, residual=None, return_norm: bool = False):
    """(q int8 [..., K], scale fp32 [...], y or None, h or None): per token
    scale = max(max|y|, 1e-10) / 127 and q = rint(y / scale); y with
    ``return_norm``, h with a residual.  No gradients."""
    _check_args("rms_norm_quant_int8", x, weight, eps, residual)
    _check(not (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (
        residual is not None and residual.requires_grad))),
        "rms_norm_quant_int8 has no gradient: call it under torch.no_grad()")
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if return_norm else None
    h = _forward(x, weight, eps, residual, y, None, q, scale)
    return q, scale, y, h

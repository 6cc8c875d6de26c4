"""The residual's addition and the RMS norm in front of the MoE layer (no
reference counterpart), differentiable, and with an int8 output.

    h = x + residual
    y = h / sqrt(mean(h^2) + eps) * weight

``rms_norm`` gives y (and h, the residual stream of the next block) in x's
type.  ``rms_norm_quant_int8`` gives y as int8 with one scale per token, and on
request y as well, for the router.  Sorted by expert (``q[src]``, ``scale[src]``
with src = permuted_idx // topk) they are the ``a`` and ``a_row_scale`` of
``ops.int8_grouped_mm_scaled``.  Sums, norms and scales are fp32; y and the int8 values
come from the unrounded h, and so do the gradients (x and residual are kept for
them).

x is [..., K] in bf16, fp16 or fp32 on a CUDA device, of any K and alignment;
rows may have any stride (a last dimension that is not contiguous is copied).
``weight`` is [K] in x's type or fp32; ``residual`` has x's shape and type.
Outputs are new contiguous tensors; nothing synchronises with the host.  Both
passes can be captured into a CUDA graph; drop eager graphs that hold the same
leaves before capturing a backward pass (a call on such a leaf is refused
during capture).

Arguments are checked in the compiled binding, which raises RuntimeError, also
for tensors with a forward-mode tangent: there are no such derivatives.
"""

from __future__ import annotations

from ._lib import TORCH_OPS


def rms_norm(x, weight, eps: float = 1e-6, residual=None):
    """y, or (y, h) with a residual.  Differentiable in x, weight and
    residual (once); the gradient of weight is summed in a fixed order.  Sums
    of squares are fp32: where one overflows (values of 1e18 and more) y is 0."""
    return TORCH_OPS.rms_norm(x, weight, eps, residual)


def rms_norm_quant_int8(x, weight, eps: float = 1e-6, residual=None, return_norm: bool = False):
    """(q int8 [..., K], scale fp32 [...], y or None, h or None): per token
    scale = max(max|y|, 1e-10) / 127 and q = rint(y / scale); y with
    ``return_norm``, h with a residual.  The quotient is fp32, off by a few of
    its last bits, so that one next to a half may round to either side.  A token
    whose norm is not finite (or whose squares leave fp32) gets scale NaN and q
    0.  No gradients."""
    return TORCH_OPS.rms_norm_quant_int8(x, weight, eps, residual, return_norm)


def rms_norm_backward(dy, x, weight, rstd, residual=None, residual_grad=None,
                      weight_grad: bool = True):
    """Gradients of ``rms_norm``: (gradient of x and residual, gradient of
    weight or None).  ``rstd`` is fp32 [rows] = 1 / sqrt(mean(h^2) + eps) of
    h = x + residual, ``residual_grad`` the gradient of h as an output."""
    return TORCH_OPS.rms_norm_backward(dy, x, weight, rstd, residual, residual_grad, weight_grad)

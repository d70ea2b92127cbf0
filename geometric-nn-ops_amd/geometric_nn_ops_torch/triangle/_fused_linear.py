"""``fused_linear``: a linear layer with bias, activation and residual in one pass over its output, as the
transitions and the projections around a pairformer's updates need it.

The reference has no such entry point; its linear layers are ``F.linear`` and separate elementwise ops
(geometric_nn_ops_torch/triangle/_reference/trimul.py:86-97, _reference/attention_pair_bias.py:86-89).
Dispatch: bf16, fp16 and fp32 tensors on a HIP device run the gfx950 kernels, forward (through the
``gnn_amd::fused_linear_fwd`` operator where no backward can follow) and backward; CPU tensors, fp64,
widths above 2^20 and forward-mode differentiation take the differentiable torch path. Without the HIP
library a GPU call raises.
"""

import torch
from torch.autograd.function import once_differentiable

from .. import _ops, _precision
from ._kernels import fused_linear as _hip
from ._reference.fused_linear import ACTIVATIONS, fused_linear_torch

__all__ = ["fused_linear"]

_KERNEL_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


class _FusedLinearHip(torch.autograd.Function):
    """HIP forward and backward; the backward forms the activation's input again from x and the weight (which are
    kept as the kernels read them: themselves, or their padded copies) with the precision that the forward resolved,
    and records no graph: a second derivative raises."""

    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual):
        ctx.precision = _precision.matmul_precision(fp32_operands=x.dtype == torch.float32)
        ctx.activation = activation
        ctx.shape = x.shape
        out, x, weight = _hip.fused_linear_hip(x, weight, bias, activation, residual, precision=ctx.precision, keep=True)
        ctx.save_for_backward(x, weight, bias)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        need_x, need_w, need_b, _, need_r = ctx.needs_input_grad
        dx = dw = db = None
        if need_x or need_w or need_b:
            dx, dw, db = _hip.fused_linear_bwd_hip(ctx.shape, x, weight, bias, ctx.activation, dy,
                                                   precision=ctx.precision, need_x=need_x, need_w=need_w, need_b=need_b)
        return dx, dw, db, None, dy if need_r else None


def _check(x, weight, bias, activation, residual) -> None:
    if x.dim() < 1 or not x.is_floating_point():
        raise ValueError(f"x must be a floating-point tensor of at least one dimension, got {x.dtype} {tuple(x.shape)}")
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or not weight.numel():
        raise ValueError(f"weight must have shape [outputs, {x.shape[-1]}], got {tuple(weight.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    outputs = weight.shape[0]
    for name, t, shape in (("weight", weight, None), ("bias", bias, (outputs,)),
                           ("residual", residual, (*x.shape[:-1], outputs))):
        if t is None:
            continue
        if shape is not None and tuple(t.shape) != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
        if t.dtype != x.dtype:
            raise ValueError(f"{name} must be {x.dtype} like x, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")


def fused_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``.

    Args:
        x: ``[..., I]``, from one row (a decoded token) to the pixels of a pair tensor.
        weight: ``[O, I]`` (nn.Linear layout); bias: ``[O]`` or ``None``.
        activation: ``None``, ``"relu"``, ``"gelu"`` (the exact form), ``"silu"`` or ``"sigmoid"``.
        residual: ``[..., O]`` or ``None``, added after the activation.

    All in one dtype. Products and epilogue run in fp32 and the result rounds once; fp32 products follow
    ``torch.backends.cuda.matmul.fp32_precision`` (the weight's gradient is full precision). In the backward the
    gradient at the activation's input is rounded to x's dtype once, as the operand of x's, the weight's and the
    bias's gradients, as stock torch's linear layers in that dtype have it.

    Returns:
        A fresh contiguous ``[..., O]`` tensor of x's dtype. Differentiable in x, weight, bias and residual;
        repeated calls give the same bits.
    """
    _check(x, weight, bias, activation, residual)
    if (not x.is_cuda or x.dtype not in _KERNEL_DTYPES or not _hip.supports(weight)
            or _ops.carries_tangent(x, weight, bias, residual)):
        return fused_linear_torch(x, weight, bias, activation, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _FusedLinearHip.apply(x, weight, bias, activation, residual)
    if _ops.eager_ok(x, weight, bias, residual):
        precision = _precision.matmul_precision(fp32_operands=x.dtype == torch.float32)
        return _hip.fused_linear_hip(x, weight, bias, activation, residual, precision=precision)
    return _ops.fused_linear_fwd(x, weight, bias, activation, residual)

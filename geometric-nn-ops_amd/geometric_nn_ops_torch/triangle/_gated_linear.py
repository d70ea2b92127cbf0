"""``gated_linear``: the gated layer of a transition, both projections, the activation and the product in one pass.

The reference has no such entry point. Dispatch: bf16, fp16 and fp32 tensors on a HIP device run the gfx950
kernels, forward (through the ``gnn_amd::gated_linear_fwd`` operator where no backward can follow) and
backward; CPU tensors, fp64, more than 2^20 inputs or 2^19 outputs and forward-mode differentiation take the
differentiable torch path. Without the HIP library a GPU call raises.
"""

import torch
from torch.autograd.function import once_differentiable

from .. import _ops, _precision
from ._kernels import gated_linear as _hip
from ._reference.fused_linear import ACTIVATIONS
from ._reference.gated_linear import gated_linear_torch

__all__ = ["gated_linear"]

_KERNEL_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


class _GatedLinearHip(torch.autograd.Function):
    """HIP forward and backward; the backward forms both products again from x and the weights (which are kept as
    the kernels read them) with the precision that the forward resolved, and records no graph: a second
    derivative raises."""

    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, gate_bias, up_bias, activation):
        ctx.precision = _precision.matmul_precision(fp32_operands=x.dtype == torch.float32)
        ctx.activation = activation
        ctx.shape = x.shape
        out, x, gate_weight, up_weight = _hip.gated_linear_hip(x, gate_weight, up_weight, gate_bias, up_bias, activation,
                                                               precision=ctx.precision, keep=True)
        ctx.save_for_backward(x, gate_weight, up_weight, gate_bias, up_bias)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        grads = _hip.gated_linear_bwd_hip(ctx.shape, *ctx.saved_tensors, ctx.activation, dy, precision=ctx.precision,
                                          need=ctx.needs_input_grad[:5])
        return (*grads, None)


def _check(x, gate_weight, up_weight, gate_bias, up_bias, activation) -> None:
    if x.dim() < 1 or not x.is_floating_point():
        raise ValueError(f"x must be a floating-point tensor of at least one dimension, got {x.dtype} {tuple(x.shape)}")
    if gate_weight.dim() != 2 or gate_weight.shape[1] != x.shape[-1] or not gate_weight.numel():
        raise ValueError(f"gate_weight must have shape [outputs, {x.shape[-1]}], got {tuple(gate_weight.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    outputs = gate_weight.shape[0]
    for name, t, shape in (("gate_weight", gate_weight, None), ("up_weight", up_weight, tuple(gate_weight.shape)),
                           ("gate_bias", gate_bias, (outputs,)), ("up_bias", up_bias, (outputs,))):
        if t is None:
            continue
        if shape is not None and tuple(t.shape) != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
        if t.dtype != x.dtype:
            raise ValueError(f"{name} must be {x.dtype} like x, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")


def gated_linear(
    x: torch.Tensor,
    gate_weight: torch.Tensor,
    up_weight: torch.Tensor,
    gate_bias: torch.Tensor | None = None,
    up_bias: torch.Tensor | None = None,
    activation: str | None = "silu",
) -> torch.Tensor:
    """``act(x @ gate_weight.T + gate_bias) * (x @ up_weight.T + up_bias)``.

    Args:
        x: ``[..., I]``, from one row (a decoded token) to the pixels of a pair tensor.
        gate_weight, up_weight: ``[O, I]`` (nn.Linear layout; halves of one stacked weight are read in place).
        gate_bias, up_bias: ``[O]`` or ``None``.
        activation: of the gate: ``"silu"``, ``"gelu"`` (the exact form), ``"sigmoid"``, ``"relu"`` or ``None``.

    All in one dtype. Products and epilogue run in fp32 and the result rounds once; fp32 products follow
    ``torch.backends.cuda.matmul.fp32_precision`` (the weights' gradients are full precision). In the backward the
    gradients at both products are rounded to x's dtype once, as the operands of x's, the weights' and the biases'
    gradients, as stock torch's linear layers in that dtype have them.

    Returns:
        A fresh contiguous ``[..., O]`` tensor of x's dtype, for the transition's second layer
        (``fused_linear(..., residual=x)``). Differentiable in x, the weights and the biases; repeated calls give
        the same bits.
    """
    _check(x, gate_weight, up_weight, gate_bias, up_bias, activation)
    args = (x, gate_weight, up_weight, gate_bias, up_bias)
    if not x.is_cuda or x.dtype not in _KERNEL_DTYPES or not _hip.supports(gate_weight) or _ops.carries_tangent(*args):
        return gated_linear_torch(*args, activation)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        return _GatedLinearHip.apply(*args, activation)
    if _ops.eager_ok(*args):
        precision = _precision.matmul_precision(fp32_operands=x.dtype == torch.float32)
        return _hip.gated_linear_hip(*args, activation, precision=precision)
    return _ops.gated_linear_fwd(*args, activation)

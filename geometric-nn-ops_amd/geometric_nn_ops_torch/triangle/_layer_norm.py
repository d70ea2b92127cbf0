"""``layer_norm``: the LayerNorm in front of a pairformer's updates, of the pair and the single stream.

The reference has no such entry point; its LayerNorms are ``F.layer_norm`` inside the ops
(geometric_nn_ops_torch/triangle/_reference/trimul.py:85, 94). Dispatch: bf16, fp16 and fp32 tensors on
a HIP device with rows of up to 16384 elements run the gfx950 kernels, forward (through the
``gnn_amd::layer_norm_fwd`` operator where no backward can follow) and backward; CPU tensors, fp64, wider
rows and forward-mode differentiation take the differentiable torch path. Without the HIP library a GPU
call raises.
"""

import torch
from torch.autograd.function import once_differentiable

from .. import _ops
from ._kernels import layer_norm as _hip
from ._reference.layer_norm import layer_norm_torch

__all__ = ["layer_norm"]

_KERNEL_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


class _LayerNormHip(torch.autograd.Function):
    """HIP forward that keeps each row's mean and 1 / standard deviation in fp32, HIP backward. The
    backward records no graph: a second derivative raises."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _hip.layer_norm_hip(x, weight, bias, eps, stats=True)
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        dw = torch.empty(weight.shape, device=x.device, dtype=weight.dtype) if need_w else None
        db = torch.empty(x.shape[-1:], device=x.device, dtype=ctx.bias_dtype) if need_b else None
        dx = _hip.layer_norm_bwd_hip(x, weight, stats, dy, need_dx=need_x, dweight=dw, dbias=db)
        return dx, dw, db, None


def _check(x, weight, bias) -> None:
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x needs a last dimension of at least 1, got shape {tuple(x.shape)}")
    if not x.is_floating_point():
        raise ValueError(f"x must be a floating-point tensor, got {x.dtype}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"{name} must have shape {(x.shape[-1],)}, got {tuple(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name} must be {x.dtype} like x, or torch.float32, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must have one dtype, got {weight.dtype} and {bias.dtype}")


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    eps: float = 1e-5,
) -> torch.Tensor:
    """LayerNorm over the last dimension: ``(x - mean) / sqrt(var + eps) * weight + bias``.

    Args:
        x: ``[..., C]`` in any strides; views that two strides of rows describe (a column slice, a
            transposed pair tensor) are read in place.
        weight, bias: ``[C]`` in x's dtype or fp32, or ``None`` (ones / zeros).
        eps: added to the (biased) variance.

    Returns:
        A fresh contiguous tensor of x's shape and dtype. The statistics and the gradients' sums are
        held in fp32; results round once. Differentiable in x, weight and bias; repeated calls give the
        same bits.
    """
    _check(x, weight, bias)
    if (not x.is_cuda or x.dtype not in _KERNEL_DTYPES or not _hip.supports(x)
            or _ops.carries_tangent(x, weight, bias)):
        return layer_norm_torch(x, weight, bias, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNormHip.apply(x, weight, bias, eps)
    if _ops.eager_ok(x, weight, bias):
        return _hip.layer_norm_hip(x, weight, bias, eps)
    return _ops.layer_norm_fwd(x, weight, bias, eps)

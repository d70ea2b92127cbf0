"""``cross_attention``: queries of one sequence over the states of another, of any length, from one decoded query on,
with key heads that several query heads share and a learned bias such as ``relative_position_bias`` makes.

The reference has no such entry point: its triangle attention has one length and as many key heads as query heads
(geometric_nn_ops_torch/triangle/_triattn.py:23-106). Dispatch: bf16, fp16 and fp32 tensors on a HIP device with
head dims that are multiples of 8 up to 128 run the gfx950 kernels, forward (through the
``gnn_amd::cross_attention_fwd`` operator where no backward can follow) and backward; CPU tensors, fp64, other head
dims and forward-mode differentiation take the differentiable torch path. Without the HIP library a GPU call raises.
"""

import math

import torch
from torch.autograd.function import once_differentiable

from .. import _ops, _precision
from ._kernels import cross_attention as _hip
from ._reference.cross_attention import cross_attention_torch

__all__ = ["cross_attention"]

_KERNEL_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


class _CrossAttentionHip(torch.autograd.Function):
    """HIP forward that keeps its output, what the rounding left of it, and each row's sum, HIP backward that forms the probabilities again with the
    precision that the forward resolved. The backward records no graph: a second derivative raises."""

    @staticmethod
    def forward(ctx, q, k, v, bias, mask, scale):
        ctx.precision = _precision.matmul_precision(fp32_operands=q.dtype == torch.float32)
        ctx.scale = scale
        out, low, stats = _hip.cross_attention_hip(q, k, v, bias, mask, scale, precision=ctx.precision, keep=True)
        ctx.save_for_backward(q, k, v, bias, mask, out, low, stats)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        need = ctx.needs_input_grad
        dq, dk, dv, dbias = _hip.cross_attention_bwd_hip(*ctx.saved_tensors, dout, ctx.scale, precision=ctx.precision,
                                                         need_kv=need[1] or need[2], need_bias=need[3])
        return dq, dk, dv, dbias, None, None


def _check(q, k, v, bias, mask, scale) -> None:
    if q.dim() != 4 or not q.is_floating_point() or not q.shape[3]:
        raise ValueError(f"q must be a floating-point [batch, queries, heads, head_dim], got {q.dtype} {tuple(q.shape)}")
    if k.dim() != 4 or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3] or not k.shape[2] or q.shape[2] % k.shape[2]:
        raise ValueError(f"k must be [{q.shape[0]}, keys, key_heads, {q.shape[3]}] with key_heads that divide q's "
                         f"{q.shape[2]} heads, got {tuple(k.shape)}")
    if v.shape != k.shape:
        raise ValueError(f"v must have k's shape {tuple(k.shape)}, got {tuple(v.shape)}")
    (B, U, H), V, dtype, device = q.shape[:3], k.shape[1], q.dtype, q.device
    if bias is not None and bias.shape not in ((B, H, U, V), (1, H, U, V)):
        raise ValueError(f"bias must have shape {(B, H, U, V)} or {(1, H, U, V)}, got {tuple(bias.shape)}")
    for name, t in (("k", k), ("v", v), ("bias", bias)):
        if t is not None and (t.dtype is not dtype or t.device != device):
            raise ValueError(f"{name} must be {dtype} like q, got {t.dtype}" if t.dtype is not dtype else
                             f"{name} is on {t.device}, q on {device}")
    if mask is not None:
        if mask.dtype is not torch.bool:
            raise ValueError(f"mask must be bool, got {mask.dtype}")
        if mask.shape != (B, V):
            raise ValueError(f"mask must have shape {(B, V)}, got {tuple(mask.shape)}")
        if mask.device != device:
            raise ValueError(f"mask is on {mask.device}, q on {device}")
    if scale is not None and not 0 < scale < 3e38:
        raise ValueError(f"scale must be positive, got {scale}")


def cross_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    bias: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """``softmax(scale * q @ k.T + bias) @ v`` for each head, over the keys that the mask keeps.

    Args:
        q: ``[B, U, H, D]``; k, v: ``[B, V, Hk, D]`` in any strides (unit stride over D is read in place), with
            Hk key heads that divide the H query heads: head h reads key head ``h // (H // Hk)``.
        bias: ``[B, H, U, V]`` or ``[1, H, U, V]`` (one for all sequences), added to the logits, or ``None``. Unit
            stride over the keys is read in place, so a ``relative_position_bias`` needs no copy.
        mask: bool ``[B, V]``, True where a key counts (the padding of the states), or ``None``. What masked keys
            hold, in k, v or the bias, has no effect, and their gradients are zeros.
        scale: of the logits, positive; ``None`` -> ``D ** -0.5``.

    All floating tensors in one dtype. Logits, softmax and sums run in fp32 and results round once; probabilities and
    the logits' gradients are rounded to the inputs' dtype as operands of the products behind them (the output's
    probabilities in two parts, which lose nothing, of up to 64 keys or up to 32 queries and heads a key head). fp32
    products follow ``torch.backends.cuda.matmul.fp32_precision``.

    Returns:
        A fresh contiguous ``[B, U, H, D]`` tensor of q's dtype: zeros, with zero gradients, for queries to which the
        mask, or a bias of -inf, leaves no key (an output gradient of infinities or NaN there still reaches k and v
        where a bias took the keys away). Differentiable in q, k, v and bias (a shared bias's gradient is summed over the batch, in fp32);
        repeated calls give the same bits.
    """
    _check(q, k, v, bias, mask, scale)
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    tensors = (q, k, v, bias)
    if not q.is_cuda or q.dtype not in _KERNEL_DTYPES or not _hip.supports(q, k) or _ops.carries_tangent(*tensors):
        return cross_attention_torch(q, k, v, bias, mask, scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        return _CrossAttentionHip.apply(q, k, v, bias, mask, scale)
    if _ops.eager_ok(q, k, v, bias, mask):
        precision = _precision.matmul_precision(fp32_operands=q.dtype == torch.float32)
        return _hip.cross_attention_hip(q, k, v, bias, mask, scale, precision=precision)
    return _ops.cross_attention_fwd(q, k, v, bias, mask, scale)

"""``relative_position_bias``: a learned bias by buckets of the distance between residues (or tokens), in
the layout of an attention bias or of the pair stream.

The reference has no such entry point; its callers build the bias that they hand to ``triangle_attention``
or ``attention_pair_bias``, and the pair stream, with stock torch. Dispatch: bf16, fp16 and fp32 tables on a
HIP device run the gfx950 kernels, forward (through the ``gnn_amd::relative_position_bias_fwd`` operator
where no backward can follow) and backward; CPU tensors, fp64, tables of more than 4096 buckets or 256
logarithmic ones a side, and forward-mode differentiation take the differentiable torch path. Without the
HIP library a GPU call raises.
"""

import torch
from torch.autograd.function import once_differentiable

from .. import _ops
from ._kernels import relative_position as _hip
from ._reference.relative_position import SPACINGS, relative_position_bias_torch, side_buckets

__all__ = ["relative_position_bias"]

_KERNEL_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_POSITION_DTYPES = (torch.int32, torch.int64)


class _RelativePositionHip(torch.autograd.Function):
    """HIP lookup and the HIP reduction of the table's gradient, which records no graph: a second
    derivative raises."""

    @staticmethod
    def forward(ctx, weight, query_pos, key_pos, how):
        out, ctx.args, query_pos, key_pos = _hip.relative_position_bias_hip(weight, query_pos, key_pos, *how, keep=True)
        ctx.save_for_backward(query_pos, key_pos)
        ctx.shape = weight.shape
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        # what saved-tensor hooks and checkpoints hand back may lie elsewhere than what the forward read
        query_pos, key_pos = ctx.saved_tensors
        return _hip.relative_position_bias_bwd_hip(ctx.shape, ctx.args, query_pos, key_pos, dout), None, None, None


def _check(weight, query_pos, key_pos, max_distance, spacing, bidirectional) -> None:
    if weight.dim() != 2 or weight.shape[0] < 1 or not weight.is_floating_point():
        raise ValueError(f"weight must be a floating-point [num_buckets, heads], got {weight.dtype} "
                         f"{tuple(weight.shape)}")
    for name, t in (("query_pos", query_pos), ("key_pos", key_pos)):
        if t.dtype not in _POSITION_DTYPES:
            raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
        if t.dim() not in (1, 2):
            raise ValueError(f"{name} must have shape [length] or [batch, length], got {tuple(t.shape)}")
        if t.device != weight.device:
            raise ValueError(f"{name} is on {t.device}, weight on {weight.device}")
    if spacing not in SPACINGS:
        raise ValueError(f"spacing must be one of {SPACINGS}, got {spacing!r}")
    if max_distance < 1:
        raise ValueError(f"max_distance must be at least 1, got {max_distance}")
    buckets = weight.shape[0]
    if spacing == "clip":
        want = (2 if bidirectional else 1) * max_distance + 1
        if buckets != want:
            raise ValueError(f"weight needs {want} buckets for max_distance {max_distance}, got {buckets}")
        return
    n, near = side_buckets(buckets, bidirectional)
    if n < 2 or (bidirectional and buckets % 2):
        raise ValueError(f"weight needs {'an even number of buckets, at least 4' if bidirectional else '2 buckets'}, "
                         f"got {buckets}")
    if max_distance <= near:
        raise ValueError(f"max_distance must be above the {near} distances that have buckets of their own, got "
                         f"{max_distance}")


def relative_position_bias(
    weight: torch.Tensor,
    query_pos: torch.Tensor,
    key_pos: torch.Tensor | None = None,
    *,
    max_distance: int,
    spacing: str = "log",
    bidirectional: bool = True,
    channels_last: bool = False,
) -> torch.Tensor:
    """``out[b, h, i, j] = weight[bucket(key_pos[b, j] - query_pos[b, i]), h]``.

    Args:
        weight: ``[num_buckets, heads]`` table (bf16, fp16 or fp32; its dtype is the result's).
        query_pos, key_pos: positions, int32 or int64, ``[U]`` or ``[B, U]`` and ``[V]`` or ``[B, V]`` in any
            order (gaps, chain offsets, one decoded position); ``key_pos=None`` takes the queries'. A
            position without a batch goes with every batch.
        max_distance: distances from here on share the last bucket of their side.
        spacing: ``"clip"``: one bucket a distance, ``clamp(key - query, -max_distance, max_distance)``, so
            ``2 * max_distance + 1`` buckets (``max_distance + 1`` unless ``bidirectional``). ``"log"``: of the
            n buckets a side, ``n // 2`` for the nearest distances one by one, the others widening
            geometrically up to ``max_distance``; borders are exact.
        bidirectional: keys ahead of the query have buckets of their own (for ``"log"`` the table's second
            half); otherwise they count as distance 0.
        channels_last: ``[B, U, V, heads]``, the pair stream's layout, for ``[B, heads, U, V]``, an
            attention bias.

    Returns:
        The bias in ``weight``'s dtype; B is 1 for positions without a batch. ``[B, heads, U, V]`` is a view
        whose row pitch is V rounded up to 8, which ``triangle_attention`` and ``attention_pair_bias`` read
        without a copy. Differentiable in ``weight``; the gradient is summed in fp32 in a fixed order. It reads the
        output gradient once for every 256 buckets (128 with ``channels_last``), and without ``channels_last`` it
        is fastest where positions ascend or descend: neighbouring keys then share buckets.
    """
    if key_pos is None:
        key_pos = query_pos
    _check(weight, query_pos, key_pos, max_distance, spacing, bidirectional)
    if query_pos.dim() == 1:
        query_pos = query_pos[None]
    if key_pos.dim() == 1:
        key_pos = key_pos[None]
    if query_pos.shape[0] != key_pos.shape[0]:
        if 1 not in (query_pos.shape[0], key_pos.shape[0]):
            raise ValueError(f"query_pos and key_pos have batches {query_pos.shape[0]} and {key_pos.shape[0]}")
        batch = max(query_pos.shape[0], key_pos.shape[0]) if query_pos.shape[0] and key_pos.shape[0] else 0
        query_pos, key_pos = (t.expand(batch, -1) for t in (query_pos, key_pos))
    if query_pos.dtype != key_pos.dtype:
        query_pos, key_pos = query_pos.to(torch.int64), key_pos.to(torch.int64)
    how = (max_distance, spacing, bool(bidirectional), bool(channels_last))
    if (not weight.is_cuda or weight.dtype not in _KERNEL_DTYPES or not _hip.supports(weight, query_pos, key_pos, *how[:3])
            or _ops.carries_tangent(weight)):
        return relative_position_bias_torch(weight, query_pos, key_pos, *how)
    if torch.is_grad_enabled() and weight.requires_grad:
        return _RelativePositionHip.apply(weight, query_pos, key_pos, how)
    if _ops.eager_ok(weight, query_pos, key_pos):
        return _hip.relative_position_bias_hip(weight, query_pos, key_pos, *how)
    return _ops.relative_position_bias_fwd(weight, query_pos, key_pos, *how)

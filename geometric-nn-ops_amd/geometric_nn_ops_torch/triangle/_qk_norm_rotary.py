"""``qk_norm_rotary``: the norm of each head's queries and keys and their rotation by position, in one pass, as
attention over residues or tokens has it between its projections and its logits.

The reference has no such entry point. Dispatch: bf16, fp16 and fp32 tensors on a HIP device with head dims and
rotary dims that are multiples of 8, up to 256, run the gfx950 kernels, forward (through the
``gnn_amd::qk_norm_rotary_fwd`` operator where no backward can follow) and backward; CPU tensors, fp64, other
dims and forward-mode differentiation take the differentiable torch path. Without the HIP library a GPU call
raises.
"""

import functools
from collections.abc import Sequence

import torch
from torch.autograd.function import once_differentiable

from .. import _ops
from ._kernels import qk_norm_rotary as _hip
from ._reference.qk_norm_rotary import qk_norm_rotary_torch

__all__ = ["qk_norm_rotary"]

_KERNEL_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_POSITION_DTYPES = (torch.int32, torch.int64)


class _QkNormRotaryHip(torch.autograd.Function):
    """HIP forward that keeps its inputs alone, HIP backward that forms the norms again. The backward records no
    graph: a second derivative raises."""

    @staticmethod
    def forward(ctx, q, k, q_pos, k_pos, q_weight, k_weight, how):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, q_pos, k_pos, q_weight, k_weight)
        ctx.how = how
        return _hip.qk_norm_rotary_hip(q, k, q_pos, k_pos, q_weight, k_weight, *how)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, q_pos, k_pos, q_weight, k_weight = ctx.saved_tensors
        need = [ctx.needs_input_grad[i] for i in (0, 1, 4, 5)]
        gq, gk, gqw, gkw = _hip.qk_norm_rotary_bwd_hip(q, k, dq, dk, q_pos, k_pos, q_weight, k_weight, *ctx.how, need)
        return gq, gk, None, None, gqw, gkw, None


@functools.lru_cache(maxsize=256)
def _frequencies(base: float, rotary_dim: int) -> tuple[float, ...]:
    return tuple(float(base) ** (-2.0 * j / rotary_dim) for j in range(rotary_dim // 2))


def _check(q, k, q_pos, k_pos, q_weight, k_weight, eps) -> None:
    if q.dim() != 4 or k.dim() != 4 or not q.is_floating_point():
        raise ValueError(f"q and k must be floating-point [batch, tokens, heads, head_dim], got {q.dtype} "
                         f"{tuple(q.shape)} and {tuple(k.shape)}")
    if k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3] or not q.shape[3]:
        raise ValueError(f"k must have q's batch and head dim {(q.shape[0], q.shape[3])}, got {tuple(k.shape)}")
    dtype, device, d = q.dtype, q.device, q.shape[3]
    if k.dtype is not dtype or k.device != device:
        raise ValueError(f"k must be {dtype} on {device} like q, got {k.dtype} on {k.device}")
    for name, t, x in (("q_pos", q_pos, q), ("k_pos", k_pos, k)):
        if t is None or (t is q_pos and name == "k_pos" and k.shape[1] == q.shape[1]):
            continue
        if t.dtype not in _POSITION_DTYPES:
            raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
        b, n = x.shape[:2]
        if t.shape not in ((b, n), (n,), (1, n)):
            raise ValueError(f"{name} must have shape [{n}] or [{b}, {n}], got {tuple(t.shape)}")
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, q on {device}")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t is None:
            continue
        if eps is None:
            raise ValueError(f"{name} goes with a norm: eps must not be None")
        if t.shape != (d,):
            raise ValueError(f"{name} must have shape {(d,)}, got {tuple(t.shape)}")
        if t.dtype is not dtype and t.dtype is not torch.float32:
            raise ValueError(f"{name} must be {dtype} like q, or torch.float32, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, q on {device}")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError(f"q_weight and k_weight must have one dtype, got {q_weight.dtype} and {k_weight.dtype}")


def qk_norm_rotary(
    q: torch.Tensor,
    k: torch.Tensor,
    q_pos: torch.Tensor | None = None,
    k_pos: torch.Tensor | None = None,
    *,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float | None = 1e-6,
    base: float = 10000.0,
    frequencies: Sequence[float] | None = None,
    rotary_dim: int | None = None,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``n = x / sqrt(mean(x^2) + eps) * weight`` over each head, and ``n`` rotated by its token's position.

    Args:
        q: ``[B, U, H, D]``; k: ``[B, V, Hk, D]``, in any strides (unit stride over D is read in place: views of a
            stacked projection need no copy), from one decoded token on.
        q_pos, k_pos: positions, int32 or int64, ``[U]`` or ``[B, U]`` and ``[V]`` or ``[B, V]``. ``k_pos=None``
            takes the queries' (U must equal V then); without both nothing is rotated.
        q_weight, k_weight: ``[D]`` in q's dtype or fp32, or ``None`` (ones).
        eps: added to the mean square; ``None`` leaves the norms out.
        base: pair j of the rotated elements turns by ``position * base ** (-2 j / rotary_dim)``.
        frequencies: the pairs' angles a position instead, ``rotary_dim / 2`` numbers (for scaled positions).
        rotary_dim: the first elements of a head that are rotated, an even number; ``None``: twice the number of
            ``frequencies``, or all.
        interleaved: pairs are neighbours (2 j, 2 j + 1) instead of (j, j + rotary_dim / 2).

    Returns:
        ``(q', k')``: fresh contiguous tensors of q's and k's shapes and dtype. Angles are reduced in fp64, norms
        and rotation run in fp32, results round once. Differentiable in q, k and the weights (not in positions or
        frequencies); repeated calls give the same bits.
    """
    if k_pos is None and q_pos is not None:
        if k.dim() == 4 and q.dim() == 4 and k.shape[1] != q.shape[1]:
            raise ValueError(f"k_pos is required where q and k have {q.shape[1]} and {k.shape[1]} tokens")
        k_pos = q_pos
    _check(q, k, q_pos, k_pos, q_weight, k_weight, eps)
    d = q.shape[3]
    if q_pos is None and k_pos is None:
        how = ()
    elif frequencies is not None:
        how = tuple(float(f) for f in frequencies)
        if rotary_dim is not None and rotary_dim != 2 * len(how):
            raise ValueError(f"frequencies must hold {rotary_dim / 2} numbers for rotary_dim {rotary_dim}, got {len(how)}")
        if not how or 2 * len(how) > d:
            raise ValueError(f"frequencies must hold 1 to {d // 2} numbers, got {len(how)}")
    else:
        r = d if rotary_dim is None else rotary_dim
        if r % 2 or not 2 <= r <= d:
            raise ValueError(f"rotary_dim must be an even number from 2 to {d}, got {r}")
        if not base > 0:
            raise ValueError(f"base must be positive, got {base}")
        how = _frequencies(base, r)
    if q_pos is not None and q_pos.dim() == 1:
        q_pos = q_pos[None]
    if k_pos is not None and k_pos.dim() == 1:
        k_pos = k_pos[None]
    if q_pos is not None and k_pos is not None and q_pos.dtype != k_pos.dtype:
        q_pos, k_pos = q_pos.to(torch.int64), k_pos.to(torch.int64)
    args = (q, k, q_pos, k_pos, q_weight, k_weight)
    how = (None if eps is None else float(eps), how, bool(interleaved))
    tensors = (q, k, q_weight, k_weight)
    if (not q.is_cuda or q.dtype not in _KERNEL_DTYPES or not _hip.supports(q, k, 2 * len(how[1]))
            or _ops.carries_tangent(*tensors)):
        return qk_norm_rotary_torch(*args, *how)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad
                                    or any(t is not None and t.requires_grad for t in (q_weight, k_weight))):
        return _QkNormRotaryHip.apply(*args, how)
    if _ops.eager_ok(*args):
        return _hip.qk_norm_rotary_hip(*args, *how)
    return _ops.qk_norm_rotary_fwd(*args, how[0], list(how[1]), how[2])

"""Host side of the HIP LayerNorm: ``layer_norm_hip`` (forward, optionally keeping the rows'
statistics) and ``layer_norm_bwd_hip`` (gradients of the rows and the parameters)."""

import torch

from ... import _lib
from .rows import as_rows

MAX_WIDTH = 16384


def supports(x: torch.Tensor) -> bool:
    """Whether the HIP kernels cover rows of this width (dtype handled by the caller)."""
    return 1 <= x.shape[-1] <= MAX_WIDTH


def _param_code(x, weight, bias) -> int:
    p = weight if weight is not None else bias
    return _lib.DTYPE_CODE[x.dtype if p is None else p.dtype]


def layer_norm_hip(x, weight=None, bias=None, eps=1e-5, *, stats=False):
    """``y`` (fresh, contiguous, like x) or, with ``stats``, ``(y, stats)`` with the fp32 ``[2, rows]`` means
    and 1 / standard deviations."""
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    kept = None
    xr, rows, inner, outer, stride = as_rows(x)
    if stats:
        kept = torch.empty((2, rows), device=x.device, dtype=torch.float32)
    if rows:
        w, b = (None if t is None else t.contiguous() for t in (weight, bias))
        mean = 0 if kept is None else kept.data_ptr()
        a = _lib.LayerNormFwdArgs()
        _lib.pack_layer_norm_fwd(
            a, 0, xr.data_ptr(), 0 if w is None else w.data_ptr(), 0 if b is None else b.data_ptr(), y.data_ptr(),
            mean, mean and mean + 4 * rows, rows, x.shape[-1], inner, outer, stride, float(eps),
            _lib.DTYPE_CODE[x.dtype], _param_code(x, w, b), 0)
        _lib.call("gnn_layer_norm_fwd", a, x.device)
    return (y, kept) if stats else y


def layer_norm_bwd_hip(x, weight, stats, dy, *, need_dx=True, dweight=None, dbias=None):
    """``dx`` like x (None unless ``need_dx``). ``dweight`` / ``dbias``: tensors ``[K]`` that receive the
    parameters' gradients, in their own dtype."""
    K = x.shape[-1]
    dx = torch.empty(x.shape, device=x.device, dtype=x.dtype) if need_dx else None
    xr, rows, inner, outer, stride = as_rows(x)
    if not rows:
        for t in (dweight, dbias):
            if t is not None:
                t.zero_()
        return dx
    gr, _, ginner, gouter, gstride = as_rows(dy)
    dt = _lib.DTYPE_CODE[x.dtype]
    w = None if weight is None else weight.contiguous()
    stats = stats.contiguous()  # two rows, one behind the other, in whatever pitch saved-tensor hooks return them
    part = None
    parts = _lib.load().gnn_layer_norm_bwd_parts(rows, K, dt)
    if dweight is not None or dbias is not None:
        part = torch.empty((parts, 2, K), device=x.device, dtype=torch.float32)
    a = _lib.LayerNormBwdArgs()
    _lib.pack_layer_norm_bwd(
        a, 0, xr.data_ptr(), gr.data_ptr(), 0 if w is None else w.data_ptr(), stats.data_ptr(),
        stats.data_ptr() + 4 * rows, 0 if dx is None else dx.data_ptr(),
        0 if part is None else part.data_ptr(), parts, rows, K, inner, outer, stride, ginner, gouter, gstride, dt,
        _param_code(x, w, dbias), 0 if dweight is None else dweight.data_ptr(), 0 if dbias is None else dbias.data_ptr())
    _lib.call("gnn_layer_norm_bwd", a, x.device)
    return dx

"""Host side of the HIP LayerNorm: ``layer_norm_hip`` (forward, optionally keeping the rows'
statistics) and ``layer_norm_bwd_hip`` (gradients of the rows and the parameters)."""

import torch

from ... import _lib
from .rows import as_rows
from .trimul import reduce_parts_hip

MAX_WIDTH = 16384


def supports(x: torch.Tensor) -> bool:
    """Whether the HIP kernels cover rows of this width (dtype handled by the caller)."""
    return 1 <= x.shape[-1] <= MAX_WIDTH


def _param_code(x, weight, bias) -> int:
    p = weight if weight is not None else bias
    return _lib.DTYPE_CODE[x.dtype if p is None else p.dtype]


def layer_norm_hip(x, weight=None, bias=None, eps=1e-5, *, stats=False):
    """``y`` (fresh, contiguous, like x) or, with ``stats``, ``(y, mean, rstd)`` with the fp32 statistics
    of every row."""
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    mean = rstd = None
    xr, rows, inner, outer, stride = as_rows(x)
    if stats:
        mean, rstd = torch.empty((2, rows), device=x.device, dtype=torch.float32)
    if rows:
        w, b = (None if t is None else t.contiguous() for t in (weight, bias))
        a = _lib.LayerNormFwdArgs()
        _lib.pack_layer_norm_fwd(
            a, 0, xr.data_ptr(), 0 if w is None else w.data_ptr(), 0 if b is None else b.data_ptr(), y.data_ptr(),
            0 if mean is None else mean.data_ptr(), 0 if rstd is None else rstd.data_ptr(), rows, x.shape[-1], inner,
            outer, stride, float(eps), _lib.DTYPE_CODE[x.dtype], _param_code(x, w, b), 0)
        _lib.call("gnn_layer_norm_fwd", a, x.device)
    return (y, mean, rstd) if stats else y


def layer_norm_bwd_hip(x, weight, mean, rstd, dy, *, need_dx=True, dweight=None, dbias=None):
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
    part = None
    parts = _lib.load().gnn_layer_norm_bwd_parts(rows, K, dt)
    if dweight is not None or dbias is not None:
        part = torch.empty((parts, 2, K), device=x.device, dtype=torch.float32)
    a = _lib.LayerNormBwdArgs()
    _lib.pack_layer_norm_bwd(
        a, 0, xr.data_ptr(), gr.data_ptr(), 0 if w is None else w.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
        0 if dx is None else dx.data_ptr(), 0 if part is None else part.data_ptr(), parts, rows, K, inner, outer,
        stride, ginner, gouter, gstride, dt, _param_code(x, w, None))
    _lib.call("gnn_layer_norm_bwd", a, x.device)
    if part is not None:
        reduce_parts_hip([(part, i * K, K, t) for i, t in enumerate((dweight, dbias)) if t is not None], x.device)
    return dx

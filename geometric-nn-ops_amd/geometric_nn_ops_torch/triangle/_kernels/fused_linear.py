"""Host side of the HIP linear layer with its epilogue: ``fused_linear_hip`` and the gradients,
``fused_linear_bwd_hip``.

The kernels read x and the weight in 16-byte chunks of rows: rows of another alignment, and widths that are
no multiple of 8, are copied once into padded rows. Results, residuals and output gradients are read and
written in place at any alignment."""

import ctypes

import torch

from ... import _lib
from .trimul import reduce_parts_hip

ACTIVATION_CODE = {None: 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}
MAX_WIDTH = 1 << 20


def supports(weight: torch.Tensor) -> bool:
    """Whether the HIP kernels cover these widths (dtype handled by the caller)."""
    return 1 <= weight.shape[0] <= MAX_WIDTH and 1 <= weight.shape[1] <= MAX_WIDTH


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]  # one row's stride says nothing


def _chunked(t: torch.Tensor) -> torch.Tensor:
    """``[R, C]`` rows of 16-byte chunks: C padded with zeros to a multiple of 8."""
    c = t.shape[1]
    if c % 8 == 0 and t.stride(1) == 1 and t.data_ptr() % 16 == 0:
        pitch = _pitch(t)
        if pitch >= c and pitch * t.element_size() % 16 == 0:
            return t
    return _padded(t, t.shape[0], c, t.stride(0), t.stride(1))


def _padded(t, rows, cols, row_stride, col_stride):
    """t's elements at these strides as ``[rows, cols padded with zeros to a multiple of 8]``."""
    pitch = (cols + 7) // 8 * 8
    out = torch.empty((rows, pitch), device=t.device, dtype=t.dtype)
    a = _lib.PadRowsArgs()
    _lib.pack_pad_rows(a, 0, t.data_ptr(), out.data_ptr(), rows, cols, pitch, row_stride, col_stride,
                       _lib.DTYPE_CODE[t.dtype], 0)
    _lib.call("gnn_pad_rows", a, t.device)
    return out


def _unit(t: torch.Tensor) -> torch.Tensor:
    """``[R, C]`` with unit stride in a row, at any pitch and alignment."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _linear(x, w, bias, side, outputs, activation, precision, *, dz=False, pad=False, transposed=False,
            want_dx=False):
    """One kernel over chunked rows ``x [M, K]`` and ``w [>= outputs, K]`` (``transposed``: ``[<= K, >= outputs]``);
    ``[M, outputs]``, with ``pad`` in rows of a multiple of 8 columns, zeros behind. With ``dz`` ``(out, dx)``,
    dx None unless it is wanted and the kernel forms ``dx = out w`` in the same pass."""
    M, K = x.shape
    cols = (outputs + 7) // 8 * 8 if pad else outputs
    out = torch.empty((M, cols), device=x.device, dtype=x.dtype)
    a = _lib.LinearArgs()
    _lib.pack_linear(
        a, 0, x.data_ptr(), w.data_ptr(), 0 if bias is None else bias.data_ptr(), 0 if side is None else side.data_ptr(),
        out.data_ptr(), M, K, outputs, cols, _pitch(x), _pitch(w), 0 if side is None else _pitch(side), cols, 0, 0,
        ACTIVATION_CODE[activation], dz, transposed, _lib.DTYPE_CODE[x.dtype], _lib.PRECISION_CODE[precision], 0)
    # a weight of fewer rows than the padded columns of x has nothing to stand beside their zeros
    if transposed and (w.shape[0] < K or not _lib.load().gnn_linear_takes_transposed(ctypes.byref(a))):
        w = _padded(w, outputs, w.shape[0], 1, _pitch(w))
        a.w, a.w_ld, a.w_transposed = w.data_ptr(), w.shape[1], 0
    dx = None
    if want_dx:
        a.dx, a.dx_ld = a.out, K  # as aligned as what is allocated where the kernel takes it
        if _lib.load().gnn_linear_takes_dx(ctypes.byref(a)):
            dx = torch.empty((M, K), device=x.device, dtype=x.dtype)
            a.dx = dx.data_ptr()
        else:
            a.dx = None
    _lib.call("gnn_linear", a, x.device)
    return (out, dx) if dz else out


def fused_linear_hip(x, weight, bias=None, activation=None, residual=None, *, precision, keep=False):
    """``act(x weight^T + bias) + residual``, fresh and contiguous; with ``keep`` ``(out, rows of x, weight)``, as
    the kernels read them, for the backward."""
    O, I = weight.shape
    shape = (*x.shape[:-1], O)
    M = x.numel() // I
    if not M:
        out = torch.empty(shape, device=x.device, dtype=x.dtype)
        return (out, x.reshape(0, I), weight) if keep else out
    side = None if residual is None else _unit(residual.reshape(M, O))
    bias = None if bias is None else bias.contiguous()
    x, weight = _chunked(x if x.dim() == 2 else x.reshape(M, I)), _chunked(weight)
    out = _linear(x, weight, bias, side, O, activation, precision)
    if len(shape) != 2:
        out = out.view(shape)
    return (out, x, weight) if keep else out


def _parameter_grads(dz, x, outputs, want_b):
    """``(dw, db)`` from chunked rows ``dz [M, >= outputs]`` and ``x [M, I]``: ``[outputs, I]`` and, where wanted,
    ``[outputs]``."""
    (M, O), I, dt, device = dz.shape, x.shape[1], dz.dtype, dz.device
    dw = torch.empty((outputs, I), device=device, dtype=dt)
    db = torch.empty((outputs,), device=device, dtype=dt) if want_b else None
    a = _lib.LinearWgradArgs()
    _lib.pack_linear_wgrad(a, 0, dz.data_ptr(), x.data_ptr(), 0, dw.data_ptr(), 0 if db is None else db.data_ptr(), M, O, I,
                           outputs, _pitch(dz), _pitch(x), 0, _lib.DTYPE_CODE[dt], 0)
    a.slices = _lib.load().gnn_linear_wgrad_slices(ctypes.byref(a))
    part = torch.empty((a.slices, O * I + O), device=device, dtype=torch.float32)
    a.partial = part.data_ptr()
    _lib.call("gnn_linear_wgrad", a, device)
    return dw, db


def _column_sums(d, outputs):
    """fp32 partial sums ``[parts, outputs]`` over the rows of ``d``."""
    parts = _lib.load().gnn_column_sums_parts(d.shape[0], outputs)
    part = torch.empty((parts, outputs), device=d.device, dtype=torch.float32)
    a = _lib.ColumnSumsArgs()
    _lib.pack_column_sums(a, 0, d.data_ptr(), part.data_ptr(), d.shape[0], outputs, _pitch(d), parts,
                          _lib.DTYPE_CODE[d.dtype], 0)
    _lib.call("gnn_column_sums", a, d.device)
    return part


def fused_linear_bwd_hip(shape, x2, w2, bias, activation, dy, *, precision, need_x=True, need_w=True, need_b=True):
    """``(dx, dweight, dbias)``, None where not needed, for x of ``shape`` from what the forward kept. The
    activation's input is formed again from x and the weight (in fp32); its gradient dz is rounded to x's dtype
    once, as the operand of the products."""
    M, O, I = x2.shape[0], w2.shape[0], shape[-1]
    if not M:
        grads = (shape, (O, I), (O,))
        return tuple(torch.zeros(s, device=x2.device, dtype=x2.dtype) if need else None
                     for s, need in zip(grads, (need_x, need_w, need_b)))
    x2, w2 = _chunked(x2), _chunked(w2)  # as kept, but where saved-tensor hooks return them in another layout
    dx = dw = db = None
    dz = _unit(dy.reshape(M, O))
    if activation is not None:
        b = None if bias is None else bias.contiguous()
        dz, dx = _linear(x2, w2, b, dz, O, activation, precision, dz=True, pad=True, want_dx=need_x and I % 8 == 0)
    elif need_x or need_w:
        dz = _chunked(dz)
    if need_x:
        if dx is None:
            dx = _linear(dz, w2, None, None, I, None, precision, transposed=True)
        if len(shape) != 2:
            dx = dx.view(shape)
    if need_w:
        dw, db = _parameter_grads(dz, x2, O, need_b)
        if x2.shape[1] != I:
            dw = dw[:, :I].contiguous()
    elif need_b:
        db = torch.empty((O,), device=x2.device, dtype=x2.dtype)
        reduce_parts_hip([(_column_sums(dz, O), 0, O, db)], x2.device)
    return dx, dw, db

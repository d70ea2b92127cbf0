"""Host side of the HIP gated layer: ``gated_linear_hip`` and the gradients, ``gated_linear_bwd_hip``.

x and the weights are read in 16-byte chunks of rows: rows of another alignment, and widths that are no multiple
of 8, are copied once into padded rows. Results and output gradients are read and written in place at any
alignment."""

import ctypes

import torch

from ... import _lib
from .fused_linear import ACTIVATION_CODE, _chunked, _linear, _pitch, _unit

MAX_INPUTS, MAX_OUTPUTS = 1 << 20, 1 << 19  # both gradients side by side are rows of 2^20


def supports(gate_weight: torch.Tensor) -> bool:
    """Whether the HIP kernels cover these widths (dtype handled by the caller)."""
    return 1 <= gate_weight.shape[0] <= MAX_OUTPUTS and 1 <= gate_weight.shape[1] <= MAX_INPUTS


def _gated(x, wg, wu, bg, bu, dy, outputs, activation, precision):
    """``[M, outputs]`` from chunked rows, or with dy the two gradients side by side, ``[M, 2 * round_up(outputs, 8)]``
    with zeros behind each."""
    M, K = x.shape
    half = (outputs + 7) // 8 * 8
    cols = outputs if dy is None else 2 * half
    out = torch.empty((M, cols), device=x.device, dtype=x.dtype)
    a = _lib.GatedLinearArgs()
    _lib.pack_gated_linear(
        a, 0, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), 0 if bg is None else bg.data_ptr(),
        0 if bu is None else bu.data_ptr(), 0 if dy is None else dy.data_ptr(), out.data_ptr(), M, K, outputs, half,
        _pitch(x), _pitch(wg), _pitch(wu), 0 if dy is None else _pitch(dy), cols, ACTIVATION_CODE[activation],
        _lib.DTYPE_CODE[x.dtype], _lib.PRECISION_CODE[precision], 0)
    _lib.call("gnn_gated_linear", a, x.device)
    return out


def gated_linear_hip(x, gate_weight, up_weight, gate_bias, up_bias, activation, *, precision, keep=False):
    """``act(x gate_weight^T + gate_bias) * (x up_weight^T + up_bias)``, fresh and contiguous; with ``keep``
    ``(out, rows of x, gate_weight, up_weight)``, as the kernels read them, for the backward."""
    O, I = gate_weight.shape
    shape = (*x.shape[:-1], O)
    M = x.numel() // I
    if not M:
        out = torch.empty(shape, device=x.device, dtype=x.dtype)
        return (out, x.reshape(0, I), gate_weight, up_weight) if keep else out
    bg, bu = (None if t is None else t.contiguous() for t in (gate_bias, up_bias))
    x = _chunked(x if x.dim() == 2 else x.reshape(M, I))
    wg, wu = _chunked(gate_weight), _chunked(up_weight)
    out = _gated(x, wg, wu, bg, bu, None, O, activation, precision)
    if len(shape) != 2:
        out = out.view(shape)
    return (out, x, wg, wu) if keep else out


def _turned(wg, wu, half):
    """``[I, 2 * half]``: both weights ``[O, I]`` turned and side by side, zeros behind each."""
    O, I = wg.shape
    out = torch.empty((I, 2 * half), device=wg.device, dtype=wg.dtype)
    a = _lib.GatedTurnArgs()
    _lib.pack_gated_turn(a, 0, wg.data_ptr(), wu.data_ptr(), out.data_ptr(), I, O, half, _pitch(wg), _pitch(wu),
                         _lib.DTYPE_CODE[wg.dtype], 0)
    _lib.call("gnn_gated_turn", a, wg.device)
    return out


def _parameter_grads(dz, x, outputs, need):
    """``(dwg, dwu, dbg, dbu)`` where ``need`` says so: ``[outputs, I]`` and ``[outputs]``."""
    M, I, half, dt = dz.shape[0], x.shape[1], dz.shape[1] // 2, dz.dtype
    grads = [torch.empty((outputs, I) if k < 2 else (outputs,), device=dz.device, dtype=dt) if n else None
             for k, n in enumerate(need)]
    a = _lib.GatedLinearWgradArgs()
    _lib.pack_gated_linear_wgrad(a, 0, dz.data_ptr(), x.data_ptr(), 0, *(0 if t is None else t.data_ptr() for t in grads), M,
                                 half, I, outputs, _pitch(dz), _pitch(x), 0, _lib.DTYPE_CODE[dt], 0)
    a.slices = _lib.load().gnn_gated_linear_wgrad_slices(ctypes.byref(a))
    part = torch.empty((a.slices, 2 * half * (I + 1)), device=dz.device, dtype=torch.float32)
    a.partial = part.data_ptr()
    _lib.call("gnn_gated_linear_wgrad", a, dz.device)
    return grads


def gated_linear_bwd_hip(shape, x2, wg, wu, gate_bias, up_bias, activation, dy, *, precision, need):
    """``[dx, dgate_weight, dup_weight, dgate_bias, dup_bias]``, None where ``need`` says so, for x of ``shape`` from what
    the forward kept. Both products are formed again (in fp32); their gradients are rounded to x's dtype once, as
    the operands of the products behind them."""
    M, O, I = x2.shape[0], wg.shape[0], shape[-1]
    if not M:
        return [torch.zeros(s, device=x2.device, dtype=x2.dtype) if n else None
                for s, n in zip((shape, (O, I), (O, I), (O,), (O,)), need)]
    x2, wg, wu = _chunked(x2), _chunked(wg), _chunked(wu)  # as kept, but where saved-tensor hooks return another layout
    bg, bu = (None if t is None else t.contiguous() for t in (gate_bias, up_bias))
    dz = _gated(x2, wg, wu, bg, bu, _unit(dy.reshape(M, O)), O, activation, precision)
    dx, grads = None, [None] * 4
    if need[0]:
        dx = _linear(dz, _turned(wg, wu, dz.shape[1] // 2), None, None, I, None, precision)
        if len(shape) != 2:
            dx = dx.view(shape)
    if any(need[1:]):
        grads = _parameter_grads(dz, x2, O, need[1:])
        if x2.shape[1] != I:
            grads[:2] = [None if t is None else t[:, :I].contiguous() for t in grads[:2]]
    return [dx, *grads]

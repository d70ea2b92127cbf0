"""Host side of the HIP relative position bias: ``relative_position_bias_hip`` and the table's gradient,
``relative_position_bias_bwd_hip``. Positions come as ``[B, U]`` / ``[B, V]`` of one integer dtype."""

import ctypes
import functools

import torch

from ... import _lib
from .._reference.relative_position import log_borders, side_buckets

MAX_BUCKETS = 4096
MAX_BORDERS = 256  # logarithmic buckets of a side


def supports(weight, query_pos, key_pos, max_distance, spacing, bidirectional) -> bool:
    """Whether the HIP kernels cover the call (dtype handled by the caller)."""
    buckets, heads = weight.shape
    if buckets > MAX_BUCKETS or max_distance > 1 << 28:
        return False
    # rows, and 64-element pieces of rows, are numbered in 32 bits
    row, rows = key_pos.shape[1] * heads, query_pos.shape[0] * query_pos.shape[1]
    if row >= (1 << 31) - 4096 or rows * ((row + 63) // 64 + 1) >= 1 << 31:
        return False
    if spacing == "clip":
        return True
    n, near = side_buckets(buckets, bidirectional)
    return n - near <= MAX_BORDERS


@functools.lru_cache(maxsize=256)
def _borders(n: int, near: int, max_distance: int):
    found = log_borders(n, near, max_distance)
    return (ctypes.c_int32 * max(1, len(found)))(*found)


def _pos(t):
    """Unit stride along the positions; the batch may be expanded."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def relative_position_bias_hip(weight, query_pos, key_pos, max_distance, spacing, bidirectional, channels_last, *,
                               keep=False):
    """``[B, H, U, V]``, a view with a row pitch rounded up to 8 elements (what the attention kernels read
    without a copy), or the contiguous ``[B, U, V, H]``. With ``keep`` ``(out, args, query_pos, key_pos)``: the
    call's arguments (None for an empty result) and its positions, for the backward."""
    B, U = query_pos.shape
    V, (buckets, H) = key_pos.shape[1], weight.shape
    query_pos, key_pos, weight = _pos(query_pos), _pos(key_pos), weight.contiguous()
    device, dtype, pitch = weight.device, weight.dtype, (V + 7) // 8 * 8
    if channels_last:
        out = torch.empty((B, U, V, H), device=device, dtype=dtype)
        strides = (U * V * H, 0, V * H)
    else:
        out = torch.empty((B, H, U, pitch), device=device, dtype=dtype)
        strides = (H * U * pitch, U * pitch, pitch)
        if pitch != V:
            out = out[..., :V]
    a = None
    if B and U and V and H:
        log, borders = spacing == "log", 0
        a = _lib.RelposArgs()
        if log:
            n, near = side_buckets(buckets, bidirectional)
            a.kept = _borders(n, near, max_distance)  # the arguments may outlive the cache's entry
            borders = ctypes.addressof(a.kept)
        _lib.pack_relpos(
            a, 0, weight.data_ptr(), query_pos.data_ptr(), key_pos.data_ptr(), out.data_ptr(), 0, 0, borders, 0,
            query_pos.stride(0), key_pos.stride(0), *strides, B, U, V, H, buckets, max_distance, log, bidirectional,
            channels_last, query_pos.element_size(), _lib.DTYPE_CODE[dtype], 0, 0)
        _lib.call("gnn_relpos_fwd", a, device)
    return (out, a, query_pos, key_pos) if keep else out


def relative_position_bias_bwd_hip(shape, args, query_pos, key_pos, dout):
    """The table's gradient ``[buckets, H]`` in dout's dtype, from the forward's kept shape and buckets and its
    positions, wherever they lie now."""
    grad = torch.empty(shape, device=dout.device, dtype=dout.dtype)
    if args is None:
        return grad.zero_()
    s0, s1, s2, s3 = dout.stride()
    if args.channels_last:
        if (args.H > 1 and s3 != 1) or (args.V > 1 and s2 != args.H):
            dout = dout.contiguous()
            s0, s1 = dout.stride()[:2]
        strides = (s0, 0, s1)
    else:
        if args.V > 1 and s3 != 1:
            dout = dout.contiguous()
            s0, s1, s2 = dout.stride()[:3]
        strides = (s0, s1, s2)
    a = _lib.RelposArgs.from_buffer_copy(args)  # a graph that is kept may run its backward again, on any thread
    a.stride = strides
    query_pos, key_pos = _pos(query_pos), _pos(key_pos)
    a.query_pos, a.query_stride, a.key_pos, a.key_stride = (
        query_pos.data_ptr(), query_pos.stride(0), key_pos.data_ptr(), key_pos.stride(0))
    a.table = a.out = None  # the forward's
    parts = _lib.load().gnn_relpos_parts(ctypes.byref(a))
    part = torch.empty((parts, *shape), device=dout.device, dtype=torch.float32)
    a.dout, a.parts, a.partial, a.dtable = dout.data_ptr(), parts, part.data_ptr(), grad.data_ptr()
    _lib.call("gnn_relpos_bwd", a, dout.device)
    return grad

"""Tensors as rows for the kernels that work row by row."""

import torch


def as_rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int, int, int]:
    """``(t, rows, inner, outer_stride, stride)``: the last dimension as rows, row r at element
    ``(r / inner) * outer_stride + (r % inner) * stride``. A tensor whose leading dimensions need more
    than two strides, or whose last one has another stride than 1, is copied."""
    k = t.shape[-1]
    if t.is_contiguous():
        rows = t.numel() // k
        return t, rows, rows, 0, k
    if t.stride(-1) == 1 or k == 1:
        dims = []  # (size, stride) of the leading dimensions, neighbours merged
        for size, stride in zip(t.shape[:-1], t.stride()[:-1]):
            if size == 1:
                continue
            if dims and dims[-1][1] == size * stride:
                dims[-1] = (dims[-1][0] * size, stride)
            else:
                dims.append((size, stride))
        if not dims:
            return t, 1, 1, 0, k
        if len(dims) == 1:
            return t, dims[0][0], dims[0][0], 0, dims[0][1]
        if len(dims) == 2:
            return t, dims[0][0] * dims[1][0], dims[1][0], dims[0][1], dims[1][1]
    t = t.contiguous()
    rows = t.numel() // k
    return t, rows, rows, 0, k

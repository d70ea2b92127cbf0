"""Relative position buckets in whole numbers, and the differentiable bias lookup in stock torch."""

import functools

import torch

SPACINGS = ("log", "clip")


def side_buckets(num_buckets: int, bidirectional: bool) -> tuple[int, int]:
    """``(n, near)`` of the logarithmic spacing: buckets of a side, and of them with one distance each."""
    n = num_buckets // 2 if bidirectional else num_buckets
    return n, n // 2


@functools.lru_cache(maxsize=256)
def log_borders(n: int, near: int, max_distance: int) -> tuple[int, ...]:
    """The distances from which the buckets near + 1, ..., n - 1 on count: the least d with
    ``d >= near * (max_distance / near) ** (k / (n - near))``, k = 1, 2, ..., decided in exact integers
    (both sides to the power n - near), so that no rounding moves a border."""
    m = n - near
    found = []
    d = near
    for k in range(1, m):
        need = near ** (m - k) * max_distance**k
        lo, hi = d, max_distance  # max_distance ** m >= need
        while lo < hi:
            mid = (lo + hi) // 2
            if mid**m >= need:
                hi = mid
            else:
                lo = mid + 1
        d = lo
        found.append(d)
    return tuple(found)


def buckets_torch(query_pos, key_pos, num_buckets, max_distance, spacing, bidirectional):
    """``[B, U, V]`` bucket of every (query, key) for positions ``[B, U]`` and ``[B, V]``."""
    ahead = key_pos.to(torch.int64)[:, None, :] - query_pos.to(torch.int64)[:, :, None]
    ahead = ahead.clamp(-max_distance, max_distance)
    if spacing == "clip":
        return ahead + max_distance if bidirectional else (-ahead).clamp(min=0)
    n, near = side_buckets(num_buckets, bidirectional)
    d = ahead.abs() if bidirectional else (-ahead).clamp(min=0)
    borders = torch.tensor(log_borders(n, near, max_distance), dtype=torch.int64, device=d.device)
    side = torch.where(d < near, d, near + torch.bucketize(d, borders, right=True))
    return side + n * (ahead > 0) if bidirectional else side


def relative_position_bias_torch(weight, query_pos, key_pos, max_distance, spacing, bidirectional, channels_last):
    rows = buckets_torch(query_pos, key_pos, weight.shape[0], max_distance, spacing, bidirectional)
    out = weight[rows]
    return out if channels_last else out.permute(0, 3, 1, 2).contiguous()

"""Norm, rotation and append with explicit positions in 64 bits (oracle; see oracle/__init__.py): the same rounding points
as oracle/kv_append.py - the normalised halves and the result, to 16 bits -, the angle of every pair from the axis it
belongs to."""
from __future__ import annotations

import torch


def axis_of_pair(half: int, sections, interleaved: bool):
    """The axis that turns each of ``half`` pairs, as a list."""
    owner = []
    for i in range(half):
        if interleaved:
            a = i % len(sections)
            owner.append(a if i // len(sections) < sections[a] else 0)
        else:
            left, a = i, 0
            while left >= sections[a]:
                left -= sections[a]
                a += 1
            owner.append(a)
    return owner


def norm_rope(x, w, eps, cos, sin, positions, sections, interleaved):
    """x [B, T, H, D] 16-bit -> (result [B, T, H, D] float64 before the last rounding, pair [B, T, H, D]: |y0| + |y1| of the
    pair an element belongs to).  cos, sin [S, >= D/2] or [B, S, >= D/2] fp32; positions [A, B, T] int."""
    half = x.shape[-1] // 2
    xd = x.double()
    y = w.double() * (xd / torch.sqrt(xd.square().mean(-1, keepdim=True) + eps))
    y = y.to(x.dtype).double()
    y0, y1 = y[..., :half], y[..., half:]
    c, s = torch.empty(x.shape[:2] + (half,), dtype=torch.float64), torch.empty(x.shape[:2] + (half,), dtype=torch.float64)
    for i, a in enumerate(axis_of_pair(half, sections, interleaved)):
        at = positions[a].long().clamp(0, cos.shape[-2] - 1)
        for b in range(x.shape[0]):
            cb, sb = (cos, sin) if cos.dim() == 2 else (cos[b % cos.shape[0]], sin[b % sin.shape[0]])
            c[b, :, i], s[b, :, i] = cb[at[b], i].double(), sb[at[b], i].double()
    c, s = c[:, :, None], s[:, :, None]
    pair = y0.abs() + y1.abs()
    return torch.cat((y0 * c - y1 * s, y1 * c + y0 * s), -1), torch.cat((pair, pair), -1)

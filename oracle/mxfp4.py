"""MXFP4 rows in 64 bits, from the format's definition: a block of 32 values shares a scale 2^(byte - 127), a value is one
of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times that, with a sign; two values a byte, the first in the low four bits."""
from __future__ import annotations

import math

import torch

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MAX_EXP = {torch.bfloat16: 125, torch.float16: 13}


def dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """[..., D/2] uint8, [..., D/32] uint8 -> [..., D] float64."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), dtype=torch.float64)
    codes, scales = codes.cpu().view(torch.uint8), scales.cpu().view(torch.uint8)
    v = table[torch.stack((codes & 15, codes >> 4), -1).long()].flatten(-2)
    s = 2.0 ** (scales.double() - 127)
    s[scales == 255] = math.nan
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def quantize(x: torch.Tensor):
    """16-bit [..., D] -> codes [..., D/2], scales [..., D/32], both uint8: the scale by searching the powers of two, the
    code by searching the eight magnitudes for the nearest (of two as near, the even code)."""
    top = MAX_EXP[x.dtype]
    blocks = x.cpu().double().unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1)
    exps = torch.arange(-126, top + 1, dtype=torch.float64)
    fits = amax[..., None] <= 7.0 * 2.0 ** exps
    e = torch.where(fits.any(-1), exps[fits.int().argmax(-1)], torch.full_like(amax, float(top)))
    bad = ~torch.isfinite(blocks).all(-1)
    y = blocks / (2.0 ** e).unsqueeze(-1)
    dist = (y.abs()[..., None] - torch.tensor(MAGNITUDES, dtype=torch.float64)).abs()
    dist = dist + torch.tensor([0.0, 1.0] * 4, dtype=torch.float64) * 1e-9          # ties: far above 64-bit rounding, far
    code = dist.argmin(-1)                                                          # below the steps of a 16-bit value
    code = (code + 8 * torch.signbit(blocks)).to(torch.uint8).flatten(-2)
    scales = torch.where(bad, torch.full_like(e, 255.0), e + 127).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def decode(q, k, v, table, lens, sm_scale, soft_cap=0.0):
    """Attention of q [B, Hq, D] over 64-bit caches k, v [pages, P, Hkv, D(v)].  Returns (out, lse, spread): spread
    [B, Hq, Dv] = sum_n p_n |v_n|, the scale of what rounding the probabilities can move."""
    q = q.cpu().double()
    b, hq, _ = q.shape
    page, hkv, dv = k.shape[1], k.shape[2], v.shape[3]
    out = torch.zeros(b, hq, dv, dtype=torch.float64)
    spread = torch.zeros_like(out)
    lse = torch.full((b, hq), -math.inf, dtype=torch.float64)
    for i, n in enumerate(lens):
        if n <= 0:
            continue
        pos = torch.arange(n)
        pages = table[i].cpu().long()[pos // page]
        ki, vi = k[pages, pos % page], v[pages, pos % page]              # [n, Hkv, D]
        qi = q[i].unflatten(0, (hkv, -1))                                # [Hkv, G, D]
        s = torch.einsum("hgd,nhd->hgn", qi, ki) * sm_scale
        if soft_cap:
            s = soft_cap * torch.tanh(s / soft_cap)
        l = torch.logsumexp(s, -1)
        p = torch.exp(s - l[..., None])
        lse[i] = l.flatten()
        out[i] = torch.einsum("hgn,nhd->hgd", p, vi).flatten(0, 1)
        spread[i] = torch.einsum("hgn,nhd->hgd", p, vi.abs()).flatten(0, 1)
    return out, lse, spread

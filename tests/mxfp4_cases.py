"""Inputs and tolerances shared by the tests of the MXFP4 cache."""
import torch

from oracle import mxfp4


def make_cache(lens, page, hkv, d, dtype, seed, layout="token", spare=3):
    """Codes and scales of a paged K and V cache on the CPU, the block table and the 64-bit values.  Rows that no sequence
    holds read as NaN, table entries behind a sequence's end are no page numbers.  layout: "token" [pages, P, Hkv, ...], or
    "head", the same axes over memory ordered [pages, Hkv, P, ...]."""
    g = torch.Generator().manual_seed(seed)
    per = [(n + page - 1) // page for n in lens]
    pool = sum(per) + spare
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(max(per), 1)), 2 ** 31 - 1, dtype=torch.int32)
    table[1::2] = -1
    held = torch.zeros(pool, page, dtype=torch.bool)
    at = 0
    for i, n in enumerate(lens):
        table[i, :per[i]] = perm[at:at + per[i]]
        pos = torch.arange(n)
        held[table[i, pos // page].long(), pos % page] = True
        at += per[i]
    out = []
    for _ in range(2):
        x = torch.randn(pool, page, hkv, d, generator=g).to(dtype)
        # rows of different sizes, so that block scales differ
        x = x * 2.0 ** torch.randint(-3, 4, (pool, page, hkv, 1), generator=g).to(dtype)
        codes, scales = mxfp4.quantize(x)
        scales[~held] = 255
        values = mxfp4.dequantize(codes, scales)
        if layout == "head":
            codes = codes.transpose(1, 2).contiguous().transpose(1, 2)
            scales = scales.transpose(1, 2).contiguous().transpose(1, 2)
        out += [codes, scales, values]
    return out, table


def decode_tolerances(q, k64, spread, out64, lse64, sm_scale, dtype):
    """A logit is a sum of D products in fp32, then scaled: off by at most (D + 8) 2^-24 sum |q k|, bounded here by the
    largest rows.  A probability moves by twice that, relatively; it is rounded to 16 bits, by half a step, and so is the
    result.  fp32 sums over the tokens and the exponentials (one unit in the last place each) stay below 2^-18."""
    u = torch.finfo(dtype).eps / 2
    k = torch.nan_to_num(k64)
    logit = float(q.double().abs().amax(-1).max()) * float(k.abs().sum(-1).max()) * sm_scale
    e = (q.shape[-1] + 8) * 2.0 ** -24 * logit + 2.0 ** -18
    return u * (spread + out64.abs()) + 2 * e * spread + 2.0 ** -20, e + 2.0 ** -22 * lse64.abs().nan_to_num(0, 0, 0)

"""Timed cases of the operators around a compressed, bounded KV cache: decode attention over an MXFP4 cache, the append
with rotary positions of several axes (16-bit and MXFP4 rows), the accumulation of attention weights per cached token,
and the eviction of the tokens that attention uses least.

MXFP4: a row of D values is D/2 bytes (value 2i in the low nibble of byte i, e2m1 codes) and D/32 scale bytes, one
per block of 32 values: value = code * 2^(scale byte - 127).

``run`` computes the operators in elementary torch operations, or, where ``own`` is true, by the framework's kernels.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_MAX_EXP = {torch.bfloat16: 125, torch.float16: 13}


def _tda():
    import triton_distributed_amd
    return triton_distributed_amd


# ---- cases ---------------------------------------------------------------------------------------------------------

def _decode(name, batch, hq, hkv, d, page, lo, hi, dtype="bf16", soft_cap=0.0):
    return {"name": name, "op": "decode", "batch": batch, "hq": hq, "hkv": hkv, "d": d, "page": page, "lo": lo, "hi": hi,
            "dtype": dtype, "cache": "mxfp4", "soft_cap": soft_cap}


def _append(name, batch, new, hq, hkv, d, page, start, axes, cache, dtype="bf16", interleaved=False):
    return {"name": name, "op": "append", "batch": batch, "new": new, "hq": hq, "hkv": hkv, "d": d, "page": page, "start": start,
            "axes": axes, "cache": cache, "dtype": dtype, "interleaved": interleaved}


def _accumulate(name, batch, hq, hkv, d, page, lo, hi, cache, dtype="bf16"):
    return {"name": name, "op": "accumulate", "batch": batch, "hq": hq, "hkv": hkv, "d": d, "page": page, "lo": lo, "hi": hi,
            "cache": cache, "dtype": dtype, "soft_cap": 0.0}


def _evict(name, batch, hkv, d, page, lo, hi, keep, recent, cache, dtype="bf16"):
    return {"name": name, "op": "evict", "batch": batch, "hkv": hkv, "d": d, "page": page, "lo": lo, "hi": hi, "keep": keep,
            "recent": recent, "cache": cache, "dtype": dtype}


def listed():
    return [
        # two short conversations on pages of one token: launch and latency
        _decode("decode_b2_512_page1", 2, 8, 2, 128, 1, 512, 512),
        # a serving step at the framework's headline shape
        _decode("decode_b32_4096", 32, 32, 8, 128, 16, 4096, 4096),
        # a step of a ragged batch, one shared kv head
        _decode("decode_b64_ragged_32k", 64, 8, 1, 128, 16, 1, 32768, dtype="fp16"),
        # four very long contexts
        _decode("decode_b4_131072", 4, 64, 8, 128, 64, 131072, 131072),
        # one new token per sequence, image / video positions, 4-bit rows
        _append("append_b32_step_mxfp4", 32, 1, 32, 8, 128, 16, 100, 3, "mxfp4"),
        # one new token per sequence of a cache in 16 bits
        _append("append_b7_step_16bit", 7, 1, 32, 8, 64, 16, 77, 3, "16bit", interleaved=True),
        # two prompts with images, 4-bit rows
        _append("append_b2_prompt_mxfp4", 2, 2041, 64, 8, 128, 16, 0, 3, "mxfp4"),
        # the bookkeeping beside a serving step: 16-bit cache at the headline shape
        _accumulate("accumulate_b32_4096_16bit", 32, 32, 8, 128, 16, 4096, 4096, "16bit"),
        # ... of a ragged batch over a 4-bit cache
        _accumulate("accumulate_b16_ragged_mxfp4", 16, 64, 8, 128, 16, 100, 16384, "mxfp4"),
        # a small cache brought back to half of its tokens
        _evict("evict_b2_512_16bit", 2, 2, 128, 1, 512, 512, 256, 64, "16bit"),
        # a serving batch brought back to its budget
        _evict("evict_b32_4096_16bit", 32, 8, 128, 16, 4000, 4096, 2048, 512, "16bit"),
        # one long prompt cut down after it was read
        _evict("evict_b1_65536_16bit", 1, 8, 128, 64, 65536, 65536, 8192, 1024, "16bit", dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("decode", "append", "accumulate", "evict"))
    d = rng.choice((64, 128, 128, 256))
    hkv = rng.choice((1, 2, 3, 4, 8))
    hq = hkv * rng.choice((1, 2, 4, 5, 8, 16, 24))
    page = rng.choice((1, 7, 16, 16, 48, 64))
    batch = _log(rng, 1, 96)
    dtype = rng.choice(("bf16", "fp16"))
    if op == "append":
        new = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
        batch = min(batch, max(1, 2 ** 19 * 64 // (new * (hq + 2 * hkv) * d)))
        case = _append("", batch, new, hq, hkv, d, page, _log(rng, 1, 300), rng.choice((1, 2, 3, 3)),
                       rng.choice(("mxfp4", "mxfp4", "16bit")), dtype, rng.random() < 0.3)
    else:
        # tokens x kv heads x values: at most a quarter of the largest listed case
        hi = _log(rng, 1, 65536)
        hi = max(1, min(hi, 2 ** 27 // (batch * hkv * d)))
        lo = hi if rng.random() < 0.4 else max(1, int(hi * rng.random()))
        if op == "decode":
            case = _decode("", batch, hq, hkv, d, page, lo, hi, dtype, rng.choice((0.0, 0.0, 25.0)))
        elif op == "accumulate":
            case = _accumulate("", batch, hq, hkv, d, page, lo, hi, rng.choice(("16bit", "mxfp4")), dtype)
        else:
            keep = max(1, int(hi * rng.uniform(0.1, 1.0)))
            case = _evict("", batch, hkv, d, page, lo, hi, keep, int(keep * rng.uniform(0.0, 0.6)), "16bit", dtype)
    del case["name"]
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------

def _quantize(x, max_exp):
    """[..., D] of a 16-bit type -> codes [..., D/2] uint8, scale bytes [..., D/32] uint8.  The scale of a block is the
    smallest power of two with amax <= 7 scales (up to 7 rounds to 6, the largest code), within [2^-126, 2^max_exp]."""
    y = x.float().unflatten(-1, (-1, 32))
    man, exp = torch.frexp(y.abs().amax(-1, keepdim=True))            # amax = man * 2^exp, man in [0.5, 1)
    e = torch.where(man > 0.875, exp - 2, exp - 3).clamp(-126, max_exp)
    e = torch.where(man == 0, torch.full_like(e, -126), e)
    y = torch.ldexp(y, -e)
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)).to(torch.uint8)
    code = torch.where(torch.signbit(y), code + 8, code).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8).squeeze(-1)


def _values(codes, scales):
    """fp32 values of MXFP4 rows."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
    both = torch.stack((table.repeat(16), table.repeat_interleave(16)), -1)       # [256, 2]: low and high nibble
    v = both[codes.int()].flatten(-2)
    return torch.ldexp(v.unflatten(-1, (-1, 32)), scales.int().unsqueeze(-1) - 127).flatten(-2)


def _pages(case, gen, tokens):
    per = (tokens + case["page"] - 1) // case["page"]
    pool = per * case["batch"] + 8
    table = torch.randperm(pool, generator=gen, device=DEV)[:per * case["batch"]]
    return pool, table.view(case["batch"], per).to(torch.int32)


def _cache(case, gen, pool):
    """K and V pools of unit-variance rows: {"k", "v"} and, MXFP4, {"ks", "vs"}."""
    dt = _DTYPES[case["dtype"]]
    shape = (pool, case["page"], case["hkv"], case["d"])
    k = torch.randn(shape, generator=gen, device=DEV, dtype=dt)
    v = torch.randn(shape, generator=gen, device=DEV, dtype=dt)
    if case["cache"] == "16bit":
        return {"k": k, "v": v, "ks": None, "vs": None}
    (k, ks), (v, vs) = _quantize(k, _MAX_EXP[dt]), _quantize(v, _MAX_EXP[dt])
    return {"k": k, "v": v, "ks": ks, "vs": vs}


def _sections(case):
    """Rotary pairs per axis: an eighth and a half of them split as time / height / width usually are."""
    half, axes = case["d"] // 2, case["axes"]
    if axes == 1:
        return (half,)
    rest = (half - half // 4) // (axes - 1)
    return (half - rest * (axes - 1),) + (rest,) * (axes - 1)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    b, hkv, d = case["batch"], case["hkv"], case["d"]
    st = {"case": case, "sm_scale": d ** -0.5}
    if case["op"] == "append":
        new, start = case["new"], case["start"]
        tokens = start + new + 3
        pool, st["table"] = _pages(case, gen, tokens)
        st["lens"] = torch.randint(new, tokens + 1, (b,), generator=gen, device=DEV).to(torch.int32)
        st.update(_cache(case, gen, pool))
        st["qkv"] = torch.randn((b, new, case["hq"] + 2 * hkv, d), generator=gen, device=DEV, dtype=dt)
        st["qw"] = (1 + 0.1 * torch.randn(d, generator=gen, device=DEV)).to(dt)
        st["kw"] = (1 + 0.1 * torch.randn(d, generator=gen, device=DEV)).to(dt)
        st["positions"] = torch.randint(0, 8192, (case["axes"], b, new), generator=gen, device=DEV).to(torch.int32)
        freq = 1e6 ** (-torch.arange(d // 2, device=DEV, dtype=torch.float64) * 2 / d)
        ang = torch.arange(8192, device=DEV, dtype=torch.float64)[:, None] * freq
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        st["sections"] = _sections(case)
        return st
    pool, st["table"] = _pages(case, gen, case["hi"])
    st["lens"] = torch.randint(case["lo"], case["hi"] + 1, (b,), generator=gen, device=DEV).to(torch.int32)
    st.update(_cache(case, gen, pool))
    if case["op"] == "evict":
        # sums of attention weights: most of them small, ties among them
        w = torch.rand((b, hkv, case["hi"]), generator=gen, device=DEV) ** 6
        st["weights"] = (w * 512).round() / 64
        return st
    st["q"] = torch.randn((b, case["hq"], d), generator=gen, device=DEV, dtype=dt)
    if case["op"] == "accumulate":
        st["lse"] = torch.logsumexp(_logits(st), -1).flatten(1)
        st["weights"] = torch.rand((b, hkv, case["hi"]), generator=gen, device=DEV)
    return st


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _rows(st, tokens):
    """Pool row (page * page size + slot) of the first ``tokens`` tokens of every sequence, [B, tokens]."""
    n = torch.arange(tokens, device=DEV)
    page = st["case"]["page"]
    return st["table"].long()[:, n // page] * page + n % page


def _gather(st, rows, name, scale):
    """fp32 [B, Hkv, N, D] of the cached rows."""
    x = st[name].flatten(0, 1)[rows]
    x = x.float() if st[scale] is None else _values(x, st[scale].flatten(0, 1)[rows])
    return x.transpose(1, 2).contiguous()


def _masked(st, tokens):
    return torch.arange(tokens, device=DEV) >= st["lens"][:, None, None, None]


def _logits(st):
    """[B, Hkv, group, N] scaled (and capped) logits, -inf behind a sequence's end."""
    case = st["case"]
    k = _gather(st, _rows(st, case["hi"]), "k", "ks")
    s = st["q"].float().unflatten(1, (case["hkv"], -1)) @ k.transpose(-1, -2).contiguous() * st["sm_scale"]
    if case["soft_cap"]:
        s = case["soft_cap"] * torch.tanh(s / case["soft_cap"])
    return s.masked_fill(_masked(st, case["hi"]), -math.inf)


def _plain_decode(st):
    case = st["case"]
    s = _logits(st)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    out = p @ _gather(st, _rows(st, case["hi"]), "v", "vs") / total
    return out.flatten(1, 2).to(st["q"].dtype), (m + total.log()).flatten(1)


def _plain_append(st):
    case = st["case"]
    hq, hkv, d, new = case["hq"], case["hkv"], case["d"], case["new"]
    dt, half = st["qkv"].dtype, case["d"] // 2
    x = st["qkv"][:, :, :hq + hkv].float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    w = torch.cat((st["qw"].float().expand(hq, d), st["kw"].float().expand(hkv, d)))
    y = (w * y).to(dt).float()                                  # the halves are rounded before the rotation
    axis = _axes(case, st["sections"])
    at = st["positions"].long().permute(1, 2, 0)[..., axis]       # [B, T, D/2]: the position that turns each pair
    pair = torch.arange(half, device=DEV)
    c, s = st["cos"][at, pair][:, :, None], st["sin"][at, pair][:, :, None]
    y0, y1 = y[..., :half], y[..., half:]
    y = torch.cat((y0 * c - y1 * s, y1 * c + y0 * s), -1).to(dt)
    n = st["lens"].long()[:, None] - new + torch.arange(new, device=DEV)
    page, slot = st["table"].long().gather(1, n // case["page"]), n % case["page"]
    if st["ks"] is None:
        st["k"][page, slot] = y[:, :, hq:]
        st["v"][page, slot] = st["qkv"][:, :, hq + hkv:]
        return y[:, :, :hq], st["k"], st["v"]
    st["k"][page, slot], st["ks"][page, slot] = _quantize(y[:, :, hq:], _MAX_EXP[dt])
    st["v"][page, slot], st["vs"][page, slot] = _quantize(st["qkv"][:, :, hq + hkv:], _MAX_EXP[dt])
    return y[:, :, :hq], _values(st["k"], st["ks"]).to(dt), _values(st["v"], st["vs"]).to(dt)


def _axes(case, sections):
    """Which axis turns each of the D/2 pairs: the sections one after the other, or (interleaved) pair i by axis
    i mod A while that axis has pairs left, by axis 0 otherwise."""
    pair = torch.arange(case["d"] // 2, device=DEV)
    if not case["interleaved"]:
        return torch.bucketize(pair, torch.tensor(sections, device=DEV).cumsum(0), right=True)
    axis = pair % len(sections)
    return torch.where(pair // len(sections) < torch.tensor(sections, device=DEV)[axis], axis, 0)


def _plain_accumulate(st):
    p = torch.exp(_logits(st) - st["lse"].unflatten(1, (st["case"]["hkv"], -1))[..., None])
    st["weights"] += p.sum(2)
    return st["weights"]


def _plain_evict(st):
    case = st["case"]
    keep, n = case["keep"], case["hi"]
    slot = torch.arange(n, device=DEV)
    lens = st["lens"].long()[:, None, None]
    order = st["weights"].masked_fill((slot >= lens - case["recent"]), math.inf).masked_fill(slot >= lens, -math.inf)
    kept = torch.sort(order, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    j = torch.arange(keep, device=DEV)
    live = j < lens                                              # a sequence within the budget keeps all it has
    src = torch.where(live, kept, j)
    rows, head = _rows(st, n), torch.arange(case["hkv"], device=DEV)[:, None]
    to = rows[:, None, :keep].expand(-1, case["hkv"], -1)
    of = rows[:, None].expand(-1, case["hkv"], -1).gather(-1, src)
    for name in ("k", "v", "ks", "vs"):
        if st[name] is not None:
            pool = st[name].flatten(0, 1)
            pool[to, head] = pool[of, head]
    weights = torch.zeros_like(st["weights"])
    weights[..., :keep] = st["weights"].gather(-1, src) * live
    return (st["lens"].clamp(max=keep), torch.where(live, kept, -1).to(torch.int32), weights, st["k"], st["v"])


# ---- one pass ------------------------------------------------------------------------------------------------------

def run(state):
    st = state
    case = st["case"]
    op = case["op"]
    if not own:
        return {"decode": _plain_decode, "append": _plain_append, "accumulate": _plain_accumulate, "evict": _plain_evict}[op](st)
    tda = _tda()
    if op == "decode":
        return tda.flash_decode(st["q"], st["k"], st["v"], st["table"], st["lens"], st["sm_scale"], soft_cap=case["soft_cap"],
                                k_scale=st["ks"], v_scale=st["vs"], max_kv_len=case["hi"], min_kv_len=case["lo"])
    if op == "append":
        q = tda.qk_norm_rope_update_kvcache(st["qkv"], st["k"], st["v"], st["table"], st["lens"], st["qw"], st["kw"], st["cos"],
                                            st["sin"], k_scale=st["ks"], v_scale=st["vs"], positions=st["positions"],
                                            rope_sections=st["sections"], rope_interleaved=case["interleaved"])
        if st["ks"] is None:
            return q, st["k"], st["v"]
        return q, tda.mxfp4_dequantize(st["k"], st["ks"], q.dtype), tda.mxfp4_dequantize(st["v"], st["vs"], q.dtype)
    if op == "accumulate":
        return tda.accumulate_attention_weights(st["q"], st["k"], st["table"], st["lens"], st["lse"], st["sm_scale"], st["weights"],
                                                k_scale=st["ks"])
    lens, kept, weights = tda.evict_kvcache(st["k"], st["v"], st["table"], st["lens"], st["weights"], case["keep"], case["recent"],
                                            k_scale=st["ks"], v_scale=st["vs"])
    return lens, kept, weights, st["k"], st["v"]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def _row_bytes(case):
    return case["d"] * 2 if case["cache"] == "16bit" else case["d"] // 2 + case["d"] // 32


def work(case):
    b, hkv, d = case["batch"], case["hkv"], case["d"]
    row = _row_bytes(case)
    if case["op"] == "append":
        rows = b * case["new"]
        pool = ((case["start"] + case["new"] + 3 + case["page"] - 1) // case["page"] * b + 8) * case["page"]
        moved = rows * (2 * case["hq"] + 2 * hkv) * d * 2 + 2 * rows * hkv * row + rows * (4 * case["axes"] + 4 * d)
        if case["cache"] != "16bit":
            moved += 2 * pool * hkv * (row + 2 * d)                     # the rows as the values they stand for
        return {"bytes": moved, "flops": rows * (case["hq"] + hkv) * d * 8}
    tokens = b * (case["lo"] + case["hi"]) // 2
    if case["op"] == "evict":
        kept = b * min(case["keep"], (case["lo"] + case["hi"]) // 2)
        weights = 4 * hkv * (tokens + b * case["hi"]) + 4 * hkv * b * case["keep"]
        return {"bytes": weights + 2 * 2 * kept * hkv * row, "flops": tokens * hkv}
    q = b * case["hq"]
    if case["op"] == "decode":
        return {"bytes": 2 * tokens * hkv * row + q * (4 * d + 4) + 4 * tokens // case["page"],
                "flops": 4 * tokens * case["hq"] * d}
    return {"bytes": tokens * hkv * (row + 8) + q * (2 * d + 4) + 4 * tokens // case["page"], "flops": 2 * tokens * case["hq"] * d}


# ---- in 64 bits ----------------------------------------------------------------------------------------------------

def _values64(codes, scales):
    """MXFP4 rows from the bits of their codes: (-1)^s * (m / 2 if e = 0 else (1 + m / 2) 2^(e - 1)) * 2^(scale - 127)."""
    c = torch.stack((codes % 16, codes // 16), -1).flatten(-2).to(torch.int64)
    e, m = (c // 2) % 4, (c % 2).double() / 2
    mag = torch.where(e == 0, m, (1 + m) * 2.0 ** (e - 1).double())
    sign = 1.0 - 2.0 * (c // 8).double()
    return sign * mag * (2.0 ** (scales.double() - 127)).repeat_interleave(32, -1)


def _sequence64(st, i, name, scale, n):
    """[n, Hkv, D] rows of sequence i."""
    case = st["case"]
    x = st[name][st["table"][i].long()].flatten(0, 1)[:n]
    if st[scale] is None:
        return x.double()
    return _values64(x, st[scale][st["table"][i].long()].flatten(0, 1)[:n])


def _logits64(st, i, n):
    """[Hq, n]."""
    case = st["case"]
    group = case["hq"] // case["hkv"]
    k = _sequence64(st, i, "k", "ks", n)
    q = st["q"][i].double()
    s = torch.cat([q[h * group:(h + 1) * group] @ k[:, h].t().contiguous() for h in range(case["hkv"])]) * case["d"] ** -0.5
    return case["soft_cap"] * torch.tanh(s / case["soft_cap"]) if case["soft_cap"] else s


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    lens = st["lens"].tolist()
    if op == "evict":
        return _evict64(st, lens)
    if op == "append":
        return _append64(st, lens)
    if op == "accumulate":
        w = st["weights"].double()
        for i, n in enumerate(lens):
            p = torch.exp(_logits64(st, i, n) - st["lse"][i].double()[:, None])
            w[i, :, :n] += p.unflatten(0, (case["hkv"], -1)).sum(1)
        return w
    group = case["hq"] // case["hkv"]
    out = torch.zeros(case["batch"], case["hq"], case["d"], dtype=torch.float64, device=DEV)
    lse = torch.zeros(case["batch"], case["hq"], dtype=torch.float64, device=DEV)
    for i, n in enumerate(lens):
        s = _logits64(st, i, n)
        lse[i] = torch.logsumexp(s, -1)
        p = torch.exp(s - lse[i][:, None])
        v = _sequence64(st, i, "v", "vs", n)
        for h in range(case["hkv"]):
            out[i, h * group:(h + 1) * group] = p[h * group:(h + 1) * group] @ v[:, h]
    return out, lse


def _append64(st, lens):
    case = st["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    dt, half, new = st["qkv"].dtype, d // 2, case["new"]
    owner = []
    for i in range(half):
        a = len(st["sections"])
        if case["interleaved"]:
            owner.append(i % a if i // a < st["sections"][i % a] else 0)
        else:
            owner.append(next(x for x in range(a) if i < sum(st["sections"][:x + 1])))
    rows = st["qkv"].double()
    norm = torch.empty_like(rows[:, :, :hq + hkv])
    for heads, w in ((slice(0, hq), st["qw"]), (slice(hq, hq + hkv), st["kw"])):
        x = rows[:, :, heads]
        norm[:, :, heads] = (x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + 1e-6) * w.double()).to(dt).double()
    turned = torch.empty_like(norm)
    for i in range(half):
        at = st["positions"][owner[i]].long()
        c, s = st["cos"][:, i].double()[at][..., None], st["sin"][:, i].double()[at][..., None]
        turned[..., i] = norm[..., i] * c - norm[..., i + half] * s
        turned[..., i + half] = norm[..., i + half] * c + norm[..., i] * s
    if st["ks"] is not None:                                    # (4-bit rows: a value next to a border has no error to speak of)
        return [turned[:, :, :hq], None, None]
    k, v = st["k"].double(), st["v"].double()
    for b, n in enumerate(lens):
        for t in range(new):
            at = n - new + t
            page = int(st["table"][b, at // case["page"]])
            k[page, at % case["page"]] = turned[b, t, hq:]
            v[page, at % case["page"]] = rows[b, t, hq + hkv:]
    return [turned[:, :, :hq], k, v]


def _evict64(st, lens):
    case = st["case"]
    keep, recent, page = case["keep"], case["recent"], case["page"]
    w = st["weights"].cpu().numpy().astype(np.float64)
    new_w, kept = np.zeros_like(w), np.full(w.shape[:2] + (keep,), -1)
    k, v = st["k"].double(), st["v"].double()
    for b, n in enumerate(lens):
        for h in range(case["hkv"]):
            old = max(n - recent, 0)
            heavy = np.lexsort((np.arange(old), -w[b, h, :old]))[:max(min(keep, n) - min(recent, n), 0)]
            stay = np.concatenate((np.sort(heavy), np.arange(old, n)))
            kept[b, h, :len(stay)] = stay
            new_w[b, h, :len(stay)] = w[b, h, stay]
            of, to = torch.from_numpy(stay).to(DEV), torch.arange(len(stay), device=DEV)
            table = st["table"][b].long()
            for pool in (k, v):
                pool[table[to // page], to % page, h] = pool[table[of // page], of % page, h]
    return [torch.tensor([min(n, keep) for n in lens], device=DEV, dtype=torch.int32), torch.from_numpy(kept).to(torch.int32),
            torch.from_numpy(new_w), k, v]

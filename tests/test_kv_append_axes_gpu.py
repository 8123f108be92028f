"""The append with explicit positions (one to four axes) and into MXFP4 caches, on the GPU.

The 16-bit rows are compared with 64 bits: the kernel and the oracle round at the same two points, and an fp32 difference in
the last bits can flip either rounding by one step, eps: an element is off by at most eps (|y0| + |y1|) from flipped halves,
and by eps |result| from the result's own rounding (plus what fp32 itself loses, 2^-20 of that).  The fp8 and 4-bit rows are
then the codes of the kernel's own 16-bit rows, bit for bit."""
import pytest
import torch

from oracle import mxfp4, rope_axes

pytestmark = pytest.mark.gpu

HQ, HKV = 6, 2


def _inputs(seed, lens, new, d, page, dtype, axes, hq=HQ, hkv=HKV, max_pos=500, tables=None):
    g = torch.Generator().manual_seed(seed)
    b = len(lens)
    per = [max((n + page - 1) // page, 1) for n in lens]
    pool = sum(per) + 2
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((b, max(per) + 1), 2 ** 31 - 1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = perm[at:at + n]
        at += n
    qkv = (torch.randn(b, new, hq + 2 * hkv, d, generator=g) * 2).to(dtype)
    wq = (1 + 0.2 * torch.randn(d, generator=g)).to(dtype)
    wk = (1 + 0.2 * torch.randn(d, generator=g)).to(dtype)
    shape = (max_pos, d // 2) if tables is None else (tables, max_pos, d)
    ang = torch.rand(shape, generator=g) * 6.28
    positions = torch.randint(0, max_pos, (axes, b, new), generator=g).to(torch.int32)
    return qkv, wq, wk, table, pool, ang.cos(), ang.sin(), positions


def _targets(table, lens, new, page):
    """(b, t, page, slot) of the rows that are written."""
    for b, n in enumerate(lens):
        for t in range(new):
            at = n - new + t
            yield b, t, int(table[b, at // page]), at % page


def _check_rows(got, want, pair, dtype, tag):
    eps = torch.finfo(dtype).eps
    got = got.cpu().double()
    tol = (eps + 2.0 ** -20) * (pair + want.abs()) + 2.0 ** -24
    off = (got - want).abs()
    assert (off <= tol).all(), f"{tag}: off by {float(off.max())}, {float((off - tol).max())} over the tolerance"
    # flipped roundings are rare: nearly everything is the nearest 16-bit value
    assert float((got != want.to(dtype).double()).double().mean()) < 0.02, tag


def _append(x, lens, page, kind, dtype, dev, pos_arg, sections, interleaved, hq=HQ, hkv=HKV, pools=None):
    import triton_distributed_amd as tda
    qkv, wq, wk, table, pool, cos, sin, _ = x
    d = qkv.shape[-1]
    if kind == "16bit":
        k = torch.full((pool, page, hkv, d), 77.0, dtype=dtype, device=dev)
        v, ks, vs = k.clone(), None, None
    elif kind == "fp8":
        k = torch.full((pool, page, hkv, d), 1.5, device=dev).to(torch.float8_e4m3fn)
        v = k.clone()
        ks, vs = (torch.tensor([0.01, 0.03, 1.0, 0.5][:hkv], device=dev) for _ in range(2))
    else:
        k = torch.full((pool, page, hkv, d // 2), 0x5A, dtype=torch.uint8, device=dev)
        v = k.clone()
        ks = torch.full((pool, page, hkv, d // 32), 0xA5, dtype=torch.uint8, device=dev)
        vs = ks.clone()
    q = tda.qk_norm_rope_update_kvcache(qkv.to(dev), k, v, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                                        wq.to(dev), wk.to(dev), cos.to(dev), sin.to(dev), k_scale=ks, v_scale=vs,
                                        positions=pos_arg, rope_sections=sections, rope_interleaved=interleaved)
    torch.cuda.synchronize()
    return q, k, v, ks, vs


def _check(seed, lens, new, d, page, dtype, sections, interleaved, dev, hq=HQ, hkv=HKV, tables=None):
    x = _inputs(seed, lens, new, d, page, dtype, len(sections), hq, hkv, tables=tables)
    qkv, wq, wk, table, pool, cos, sin, positions = x
    pos = positions.to(dev)
    q, k, v, _, _ = _append(x, lens, page, "16bit", dtype, dev, pos, sections, interleaved, hq, hkv)
    want_q, pair_q = rope_axes.norm_rope(qkv[:, :, :hq], wq, 1e-6, cos, sin, positions, sections, interleaved)
    want_k, pair_k = rope_axes.norm_rope(qkv[:, :, hq:hq + hkv], wk, 1e-6, cos, sin, positions, sections, interleaved)
    if hq:
        _check_rows(q, want_q, pair_q, dtype, "q")
    k, v = k.cpu(), v.cpu()
    mine_k = torch.empty(len(lens), new, hkv, d, dtype=dtype)
    mine_v = torch.empty_like(mine_k)
    for b, t, pg, slot in _targets(table, lens, new, page):
        mine_k[b, t], mine_v[b, t] = k[pg, slot], v[pg, slot]
        k[pg, slot] = v[pg, slot] = 77.0
    assert (k == 77).all() and (v == 77).all()                         # nothing else was written
    _check_rows(mine_k, want_k, pair_k, dtype, "k")
    assert torch.equal(mine_v, qkv[:, :, hq + hkv:])
    # fp8
    q8, k8, v8, ks, vs = _append(x, lens, page, "fp8", dtype, dev, pos, sections, interleaved, hq, hkv)
    assert torch.equal(q8, q)
    e4m3 = lambda r, s: (r.float() / s.cpu()[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    k8, v8 = k8.cpu().view(torch.uint8), v8.cpu().view(torch.uint8)
    fill = k8.new_tensor([1.5], dtype=torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)
    for b, t, pg, slot in _targets(table, lens, new, page):
        assert torch.equal(k8[pg, slot], e4m3(mine_k[b, t], ks)) and torch.equal(v8[pg, slot], e4m3(mine_v[b, t], vs))
        k8[pg, slot] = v8[pg, slot] = fill
    assert (k8 == fill).all() and (v8 == fill).all()
    # MXFP4
    q4, k4, v4, ks, vs = _append(x, lens, page, "mxfp4", dtype, dev, pos, sections, interleaved, hq, hkv)
    assert torch.equal(q4, q)
    k4, v4, ks, vs = k4.cpu(), v4.cpu(), ks.cpu(), vs.cpu()
    (kc, kb), (vc, vb) = mxfp4.quantize(mine_k), mxfp4.quantize(mine_v)
    for b, t, pg, slot in _targets(table, lens, new, page):
        assert torch.equal(k4[pg, slot], kc[b, t]) and torch.equal(ks[pg, slot], kb[b, t])
        assert torch.equal(v4[pg, slot], vc[b, t]) and torch.equal(vs[pg, slot], vb[b, t])
        k4[pg, slot] = v4[pg, slot] = 0x5A
        ks[pg, slot] = vs[pg, slot] = 0xA5
    assert (k4 == 0x5A).all() and (v4 == 0x5A).all() and (ks == 0xA5).all() and (vs == 0xA5).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page,new", [(1, 1), (16, 1), (7, 3), (16, 19)])
def test_three_axes(cuda_device, dtype, d, page, new):
    third = d // 2 // 3
    _check(d + page, [new, 40 + new, 17 + new], new, d, page, dtype, (d // 2 - 2 * third, third, third), False, cuda_device)


@pytest.mark.parametrize("sections,interleaved", [((64,), False), ((64,), True), ((1, 63), False), ((0, 64, 0), False), ((24, 20, 20), True),
                                                  ((40, 12, 12), True), ((10, 20, 30, 4), False), ((16, 16, 16, 16), True), ((5, 0, 59), True)])
def test_sections(cuda_device, sections, interleaved):
    _check(3, [9, 1, 30], 1, 128, 16, torch.bfloat16, sections, interleaved, cuda_device)


def test_many_rows_and_head_layouts(cuda_device):
    """More rows than are resident at once (four rounds a wavefront), head counts that leave the last round partly empty, no
    q heads at all, tables per sequence."""
    _check(4, [160, 150], 140, 128, 16, torch.bfloat16, (20, 22, 22), False, cuda_device, hq=127, hkv=1)
    _check(5, [600, 590], 577, 64, 16, torch.float16, (12, 10, 10), False, cuda_device, hq=5, hkv=3)
    _check(6, [300], 257, 256, 8, torch.bfloat16, (128,), False, cuda_device, hq=35, hkv=4)
    _check(7, [3, 9], 2, 128, 16, torch.bfloat16, (30, 34), False, cuda_device, hq=0, hkv=3)
    _check(8, [3, 9, 30], 2, 128, 16, torch.bfloat16, (30, 34), False, cuda_device, tables=3)


def test_default_positions_are_the_places_in_the_cache(cuda_device):
    """An MXFP4 cache without positions: the q rows and codes of the same call with the places spelled out."""
    lens, new = [21, 5], 5
    x = _inputs(9, lens, new, 128, 16, torch.bfloat16, 1)
    places = torch.tensor([[n - new + t for t in range(new)] for n in lens], dtype=torch.int32, device=cuda_device)
    a = _append(x, lens, 16, "mxfp4", torch.bfloat16, cuda_device, None, None, False)
    b = _append(x, lens, 16, "mxfp4", torch.bfloat16, cuda_device, places, None, False)
    for s, t in zip(a, b):
        assert torch.equal(s, t)


def test_positions_and_rows_of_any_layout(cuda_device):
    """Transposed and broadcast positions, rows that start between the 8-byte marks, wide strides."""
    import triton_distributed_amd as tda
    dev, lens, new = cuda_device, [21, 5, 12], 4
    x = _inputs(10, lens, new, 128, 16, torch.bfloat16, 3)
    qkv, wq, wk, table, pool, cos, sin, positions = x
    want = _append(x, lens, 16, "16bit", torch.bfloat16, dev, positions.to(dev), (24, 20, 20), False)
    base = torch.zeros(3, new, HQ + 2 * HKV, 133, dtype=torch.bfloat16, device=dev)
    odd = base[..., 3:131]
    odd.copy_(qkv)
    pos = positions.to(dev).permute(2, 1, 0).contiguous().permute(2, 1, 0)
    kbase = torch.full((pool, 16, HKV, 131), 77.0, dtype=torch.bfloat16, device=dev)
    vbase = kbase.clone()
    qbase = torch.zeros(3, new, HQ, 129, dtype=torch.bfloat16, device=dev)
    q = tda.qk_norm_rope_update_kvcache(odd, kbase[..., 1:129], vbase[..., 1:129], table.to(dev),
                                        torch.tensor(lens, dtype=torch.int32, device=dev), wq.to(dev), wk.to(dev), cos.to(dev),
                                        sin.to(dev), qbase[..., 1:], positions=pos, rope_sections=(24, 20, 20))
    assert torch.equal(q, want[0]) and torch.equal(kbase[..., 1:129], want[1]) and torch.equal(vbase[..., 1:129], want[2])
    assert (qbase[..., 0] == 0).all() and (kbase[..., 0] == 77).all() and (kbase[..., 129:] == 77).all()
    one = positions[:1, :1, :1].to(dev).expand(3, 3, new)
    a = _append(x, lens, 16, "mxfp4", torch.bfloat16, dev, one, (24, 20, 20), False)
    b = _append(x, lens, 16, "mxfp4", torch.bfloat16, dev, one.contiguous(), (24, 20, 20), False)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_places_outside_the_cache_are_not_written(cuda_device):
    """A length that does not count all new tokens, table entries that are no pages, positions outside the tables."""
    lens, new = [2, 40], 5
    x = _inputs(11, [40, 40], new, 128, 16, torch.bfloat16, 2)
    qkv, wq, wk, table, pool, cos, sin, positions = x
    table[1, 2] = -1
    positions[0, 0, 0], positions[1, 0, 1] = -7, 100000
    q, k, v, _, _ = _append(x, lens, 16, "16bit", torch.bfloat16, cuda_device, positions.to(cuda_device), (32, 32), False)
    want_q, pair_q = rope_axes.norm_rope(qkv[:, :, :HQ], wq, 1e-6, cos, sin, positions, (32, 32), False)
    _check_rows(q, want_q, pair_q, torch.bfloat16, "q")
    v = v.cpu()
    for t in (3, 4):                                            # the only ones with a place: 2 - 5 + t >= 0
        pg, slot = int(table[0, 0]), t - 3
        assert torch.equal(v[pg, slot], qkv[0, t, HQ + HKV:])
        v[pg, slot] = 77.0
    assert (v == 77).all()


def test_infinite_and_nan_rows_read_as_nan(cuda_device):
    import triton_distributed_amd as tda
    lens, new = [3], 3
    x = _inputs(12, lens, new, 128, 16, torch.bfloat16, 1)
    x[0][0, 0, HQ + HKV, 40] = float("inf")
    x[0][0, 1, HQ + HKV + 1, 0] = float("nan")
    _, k, v, ks, vs = _append(x, lens, 16, "mxfp4", torch.bfloat16, cuda_device, x[7].to(cuda_device), None, False)
    back = tda.mxfp4_dequantize(v, vs).cpu()
    pg = int(x[3][0, 0])
    nan = back[pg, :3].isnan()
    assert nan[0, 0, 32:64].all() and nan[1, 1, :32].all() and int(nan.sum()) == 64


def test_captured_append(cuda_device):
    """Replays follow the lengths and the positions on the device."""
    import triton_distributed_amd as tda
    dev, lens, new = cuda_device, [21, 5], 1
    x = _inputs(13, [64, 64], new, 128, 16, torch.bfloat16, 3)
    qkv, wq, wk, table, pool, cos, sin, positions = [t.to(dev) if isinstance(t, torch.Tensor) else t for t in x]
    k = torch.zeros(pool, 16, HKV, 64, dtype=torch.uint8, device=dev)
    v, ks = k.clone(), torch.zeros(pool, 16, HKV, 4, dtype=torch.uint8, device=dev)
    vs, n = ks.clone(), torch.tensor(lens, dtype=torch.int32, device=dev)
    out = torch.empty(2, new, HQ, 128, dtype=torch.bfloat16, device=dev)
    call = lambda: tda.qk_norm_rope_update_kvcache(qkv, k, v, table, n, wq, wk, cos, sin, out, k_scale=ks, v_scale=vs,
                                                   positions=positions, rope_sections=(24, 20, 20))
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step in range(3):
        n.copy_(torch.tensor([22 + step, 6 + step], dtype=torch.int32))
        positions.add_(1)
        call()
        torch.cuda.synchronize()
        eager = [t.clone() for t in (out, k, v, ks, vs)]
        for t in (out, k, v, ks, vs):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0])
        for b, length in enumerate((22 + step, 6 + step)):
            pg, slot = int(table[b, (length - 1) // 16]), (length - 1) % 16
            for got, want in zip((k, v, ks, vs), eager[1:]):
                assert torch.equal(got[pg, slot], want[pg, slot])

"""MXFP4 caches on the GPU: the conversions against the format's definition, the decode against attention in 64 bits over
the values that the codes stand for."""
import ctypes as C
import math

import pytest
import torch

from oracle import mxfp4
from tests.mxfp4_cases import decode_tolerances, make_cache

pytestmark = pytest.mark.gpu


def _close(got, want, tol):
    """|got - want| <= tol, infinities and NaN in the same places."""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    same = (got == want) | torch.isnan(want)
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    worst = float((off - tol).max())
    assert worst <= 0, f"off by {float(off.max()):.3g}, {worst:.3g} over the tolerance"


def _run(lens, hq, hkv, d, page, dtype, seed, layout="token", soft_cap=0.0, cuda_device=None, **kw):
    import triton_distributed_amd as tda
    (kc, ks, k64, vc, vs, v64), table = make_cache(lens, page, hkv, d, dtype, seed, layout)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(len(lens), hq, d, generator=g).to(dtype)
    sm_scale = d ** -0.5
    dev = lambda t: t.to(cuda_device)
    # (.to keeps the strides of the "head" layout)
    out, lse = tda.flash_decode(dev(q), dev(kc), dev(vc), dev(table), torch.tensor(lens, dtype=torch.int32, device=cuda_device),
                                sm_scale, soft_cap=soft_cap, k_scale=dev(ks), v_scale=dev(vs), **kw)
    torch.cuda.synchronize()
    o64, l64, spread = mxfp4.decode(q, k64, v64, table, lens, sm_scale, soft_cap)
    tol_o, tol_l = decode_tolerances(q, k64, spread, o64, l64, sm_scale, dtype)
    _close(out, o64, tol_o)
    _close(lse, l64, tol_l)
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_code_and_scale_dequantizes_exactly(cuda_device, dtype):
    import triton_distributed_amd as tda
    codes = torch.arange(256, dtype=torch.uint8).view(1, 16, 16).expand(256, 16, 16).contiguous()
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1, 1).expand(256, 16, 1).contiguous()
    got = tda.mxfp4_dequantize(codes.to(cuda_device), scales.to(cuda_device), dtype).cpu()
    want = mxfp4.dequantize(codes, scales).to(dtype)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_matches_the_definition(cuda_device, dtype):
    """Random rows over the whole range of exponents, every 16-bit pattern, zeros, infinities and NaN."""
    import triton_distributed_amd as tda
    g = torch.Generator().manual_seed(5)
    lo, hi = (-130, 128) if dtype == torch.bfloat16 else (-24, 16)
    x = torch.randn(3000, 64, generator=g).double() * 2.0 ** torch.randint(lo, hi, (3000, 1), generator=g).double()
    top = torch.finfo(dtype).max
    x = x.clamp(-top, top).to(dtype)
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).view(1024, 64)
    zeros = torch.zeros(2, 64, dtype=dtype)
    zeros[1] = -0.0
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, -0.25, -5.0, 1.0] + [0.0] * 52, dtype=dtype)
    x = torch.cat((x, every, zeros, ties[None], ties[None] * 2.0 ** 8))
    codes, scales = tda.mxfp4_quantize(x.to(cuda_device))
    want_c, want_s = mxfp4.quantize(x)
    assert torch.equal(scales.cpu(), want_s)
    fine = (want_s != 255).repeat_interleave(16, -1)
    assert torch.equal(codes.cpu()[fine], want_c[fine])
    back = tda.mxfp4_dequantize(codes, scales, dtype).cpu()
    assert torch.isfinite(back[(want_s != 255).repeat_interleave(32, -1)]).all()
    assert back[(want_s == 255).repeat_interleave(32, -1)].isnan().all()


def test_conversions_of_strided_rows(cuda_device):
    """Rows of a cache laid out by heads, a slice of wider rows; what lies between them stays."""
    import triton_distributed_amd as tda
    x = torch.randn(5, 3, 7, 192, device=cuda_device, dtype=torch.bfloat16)[..., 64:160]
    codes = torch.full((5, 7, 3, 64), 99, dtype=torch.uint8, device=cuda_device)
    view = codes.transpose(1, 2)[..., 4:52]
    scales = torch.full((5, 3, 7, 5), 98, dtype=torch.uint8, device=cuda_device)
    tda.mxfp4_quantize(x, view, scales[..., 1:4])
    want_c, want_s = mxfp4.quantize(x.cpu())
    assert torch.equal(view.cpu(), want_c) and torch.equal(scales[..., 1:4].cpu(), want_s)
    assert (codes[..., :4] == 99).all() and (codes[..., 52:] == 99).all()
    assert (scales[..., 0] == 98).all() and (scales[..., 4] == 98).all()
    out = torch.zeros(5, 3, 7, 192, device=cuda_device, dtype=torch.float16)
    tda.mxfp4_dequantize(view, scales[..., 1:4], out=out[..., 64:160])
    assert torch.equal(out[..., 64:160].cpu(), mxfp4.dequantize(want_c, want_s).half())
    assert (out[..., :64] == 0).all() and (out[..., 160:] == 0).all()
    assert tda.mxfp4_quantize(x[:0])[0].shape == (0, 3, 7, 48)


LENS = [0, 1, 15, 16, 17, 31, 32, 33, 255, 256, 257, 511, 700, 1029]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 5, 16, 48, 64])
def test_lengths_pages_head_dims(cuda_device, dtype, d, page):
    _run(LENS, 8, 2, d, page, dtype, 10 * d + page, cuda_device=cuda_device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hkv", [2, 4, 8, 12])
@pytest.mark.parametrize("page", [16, 64])
def test_pairs_of_neighbouring_heads(cuda_device, dtype, d, hkv, page):
    """Pairs of kv heads, staged through LDS (d = 128) or in registers: chunks, a single pass, equal shares; groups that leave
    columns empty and groups of more than one tile of q heads."""
    _run(LENS, 2 * hkv, hkv, d, page, dtype, 50 + hkv, cuda_device=cuda_device)
    _run([100, 0, 17, 260, 129], 20 * hkv, hkv, d, page, dtype, 51 + hkv, kv_split=1, cuda_device=cuda_device)
    _run([1500, 3, 0, 640], 3 * hkv, hkv, d, page, dtype, 52 + hkv, force_balanced=True, cuda_device=cuda_device)
    _run([700, 2100], hkv, hkv, d, page, dtype, 53 + hkv, kv_split=5, soft_cap=20.0, cuda_device=cuda_device)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (6, 2), (16, 1), (17, 1), (40, 1), (96, 3), (64, 8), (20, 4)])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_head_layouts(cuda_device, hq, hkv, layout):
    _run([300, 0, 77, 1], hq, hkv, 128, 16, torch.bfloat16, 100 + hq, layout, cuda_device=cuda_device)


@pytest.mark.parametrize("kv_split", [-1, 1, 7, 64])
@pytest.mark.parametrize("page", [3, 16])
def test_split_counts(cuda_device, kv_split, page):
    _run([2000, 5, 0, 1111], 8, 2, 128, page, torch.bfloat16, 7, kv_split=kv_split, cuda_device=cuda_device)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [7, 32])
def test_equal_shares(cuda_device, d, page):
    """The plan that cuts the whole batch into equal shares, whatever the planner would choose."""
    _run([3000, 1, 0, 64, 1700, 33, 0, 900], 10, 2, d, page, torch.bfloat16, 8, force_balanced=True, cuda_device=cuda_device)


def test_soft_cap_and_known_lengths(cuda_device):
    _run([600, 590, 600], 4, 1, 128, 16, torch.float16, 9, soft_cap=5.0, cuda_device=cuda_device)
    _run([640] * 40, 32, 8, 128, 16, torch.bfloat16, 9, max_kv_len=640, min_kv_len=640, cuda_device=cuda_device)


def test_one_dominant_token(cuda_device):
    """Logits over a range of several hundred: the running maximum moves by more and by less than the step at which the
    accumulators are rescaled."""
    import triton_distributed_amd as tda
    lens = [777]
    (kc, ks, k64, vc, vs, v64), table = make_cache(lens, 16, 1, 128, torch.bfloat16, 4)
    q = torch.randn(1, 4, 128, generator=torch.Generator().manual_seed(3)).bfloat16() * 8
    out, lse = tda.flash_decode(q.to(cuda_device), kc.to(cuda_device), vc.to(cuda_device), table.to(cuda_device),
                                torch.tensor(lens, dtype=torch.int32, device=cuda_device), 0.5, k_scale=ks.to(cuda_device),
                                v_scale=vs.to(cuda_device))
    o64, l64, spread = mxfp4.decode(q, k64, v64, table, lens, 0.5)
    tol_o, tol_l = decode_tolerances(q, k64, spread, o64, l64, 0.5, torch.bfloat16)
    _close(out, o64, tol_o)
    _close(lse, l64, tol_l)


def test_typed_caches_packed_result_static_scratch(cuda_device):
    """float4 / e8m0 spelling of the types, the packed drop-in result and the entry that allocates nothing: same bits."""
    import triton_distributed_amd as tda
    from triton_distributed_amd import _lib
    lens = [1500, 40, 0]
    (kc, ks, k64, vc, vs, v64), table = make_cache(lens, 16, 2, 128, torch.bfloat16, 12)
    dev = lambda t: t.to(cuda_device)
    q = dev(torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(3)).bfloat16())
    kc, ks, vc, vs, table = dev(kc), dev(ks), dev(vc), dev(vs), dev(table)
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    out, lse = tda.flash_decode(q, kc, vc, table, n, 0.1, k_scale=ks, v_scale=vs)
    f4, e8 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
    out2, lse2 = tda.flash_decode(q, kc.view(f4), vc.view(f4), table, n, 0.1, k_scale=ks.view(e8), v_scale=vs.view(e8))
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    call = tda.prepare_decode(q, kc, vc, table, n, 0.1, k_scale=ks, v_scale=vs, static_scratch=True)
    assert call.plan.num_splits > 1
    out3, lse3 = call.run_static()
    assert torch.equal(out, out3) and torch.equal(lse, lse3)
    packed = torch.empty(3, 8, 129, dtype=torch.bfloat16, device=cuda_device)
    tda.prepare_decode(q, kc, vc, table, n, 0.1, k_scale=ks, v_scale=vs, packed_out=packed, want_lse=False).run()
    assert torch.equal(packed[..., :128], out) and torch.equal(packed[..., 128], lse.bfloat16())
    # counters are accepted (and left at zero): one workgroup per piece
    call = tda.prepare_decode(q, kc, vc, table, n, 0.1, k_scale=ks, v_scale=vs, kv_split=20)
    out4, lse4 = call.run()
    torch.testing.assert_close(out4.float(), out.float(), atol=2e-2, rtol=2e-2)
    rc = _lib.load().fdk_decode_splitkv(C.byref(call.args), torch.cuda.current_stream().cuda_stream)
    rc2 = _lib.load().fdk_combine(C.byref(call.args), torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and rc2 == 0
    assert torch.equal(call.out, out4) and torch.equal(call.lse, lse4)


def test_captured_and_replayed_on_another_stream(cuda_device):
    """A captured call, replayed while eager calls of other shapes run in between, follows the lengths on the device."""
    import triton_distributed_amd as tda
    (kc, ks, k64, vc, vs, v64), table = make_cache([900, 900], 16, 2, 128, torch.bfloat16, 13)
    dev = lambda t: t.to(cuda_device)
    qc = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(3)).bfloat16()
    q, kc, ks, vc, vs, tb = dev(qc), dev(kc), dev(ks), dev(vc), dev(vs), dev(table)
    n = torch.tensor([5, 5], dtype=torch.int32, device=cuda_device)
    call = tda.prepare_decode(q, kc, vc, tb, n, 0.1, k_scale=ks, v_scale=vs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call.run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call.run()
    for lens in ([900, 1], [0, 333], [512, 512]):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        tda.flash_decode(q, kc, vc, tb, n, 0.1, k_scale=ks, v_scale=vs, kv_split=9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        o64, l64, spread = mxfp4.decode(qc, k64, v64, table, lens, 0.1)
        tol_o, tol_l = decode_tolerances(qc, k64, spread, o64, l64, 0.1, torch.bfloat16)
        _close(call.out, o64, tol_o)
        _close(call.lse, l64, tol_l)
        assert math.isfinite(float(call.out.float().sum()))


@pytest.mark.parametrize("d,page,hkv", [(128, 16, 2), (128, 16, 1), (128, 24, 2), (64, 16, 2), (256, 16, 2)])
def test_pages_past_32_bit_offsets(cuda_device, d, page, hkv):
    """Pools of which most pages lie more than 4 GiB behind the first: append, decode, attention weights and eviction leave
    the same bits as on the same pages side by side."""
    import triton_distributed_amd as tda
    dev, pages, far = cuda_device, 12, 700 << 20
    buf = torch.empty(pages * far, dtype=torch.uint8, device=dev)
    shapes = [(pages, page, hkv, n) for n in (d // 2, d // 2, d // 32, d // 32)]
    at = (0, 200 << 20, 400 << 20, 500 << 20)
    wide = [torch.as_strided(buf, s, (far, hkv * s[3], s[3], 1), o) for s, o in zip(shapes, at)]
    g = torch.Generator().manual_seed(d + page)
    near = [torch.randint(0, 256, s, dtype=torch.uint8, generator=g).to(dev) for s in shapes[:2]]
    near += [torch.randint(118, 130, s, dtype=torch.uint8, generator=g).to(dev) for s in shapes[2:]]
    for w, n in zip(wide, near):
        w.copy_(n)
    table = torch.randperm(pages, generator=g).to(torch.int32).view(2, 6).to(dev)
    lens = torch.tensor([6 * page - 3, 2 * page + 5], dtype=torch.int32, device=dev)
    ang = torch.rand(300, d // 2, generator=g) * 6.28
    cos, sin = (torch.cat((t, t), -1).to(dev) for t in (ang.cos(), ang.sin()))
    ones = torch.ones(d, dtype=torch.bfloat16, device=dev)
    qkv = torch.randn(2, 4, 6 * hkv, d, generator=g).bfloat16().to(dev)
    got = []
    for k, v, ks, vs in (near, wide):
        q = tda.qk_norm_rope_update_kvcache(qkv, k, v, table, lens, ones, ones, cos, sin, k_scale=ks, v_scale=vs)[:, -1]
        out, lse = tda.flash_decode(q, k, v, table, lens, 0.1, k_scale=ks, v_scale=vs)
        w = tda.accumulate_attention_weights(q, k, table, lens, lse, 0.1, torch.zeros(2, hkv, 6 * page, device=dev), k_scale=ks)
        n, kept, w2 = tda.evict_kvcache(k, v, table, lens, w, 2 * page, 7, k_scale=ks, v_scale=vs)
        got.append([q, out, lse, w, n, kept, w2, k, v, ks, vs])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert torch.isfinite(got[0][1]).all() and int(got[0][4][0]) == 2 * page


@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (128, 7), (256, 32)])
def test_scales_and_rows_laid_out_apart(cuda_device, d, page):
    """Block scales in the middle of wider rows, tokens with room between them: the same bits as side by side."""
    import triton_distributed_amd as tda
    lens, hkv, hq = [300, 1, 77], 2, 6
    (kc, ks, _, vc, vs, _), table = make_cache(lens, page, hkv, d, torch.bfloat16, d)
    dev = [t.to(cuda_device) for t in (kc, vc, ks, vs)]
    apart = []
    for i, t in enumerate(dev):
        room = torch.full(t.shape[:2] + (hkv + 2, t.shape[3] + (0 if i < 2 else 8)), 0xFF, dtype=torch.uint8, device=cuda_device)
        view = room[:, :, 1:1 + hkv, :t.shape[3]] if i < 2 else room[:, :, 1:1 + hkv, 4:4 + t.shape[3]]
        apart.append(view.copy_(t))
    q = torch.randn(3, hq, d, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda_device)
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    for kw in ({}, dict(kv_split=3), dict(force_balanced=True)):
        a, b = (tda.flash_decode(q, k, v, table.to(cuda_device), n, 0.1, k_scale=s, v_scale=t, **kw) for k, v, s, t in (dev, apart))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (128, 5)])
def test_scales_of_a_head_past_32_bit_offsets(cuda_device, d, page):
    """Block scales laid out by head, the second head's more than 4 GiB behind the first's."""
    import triton_distributed_amd as tda
    lens, hkv = [90, 33], 2
    (kc, ks, _, vc, vs, _), table = make_cache(lens, page, hkv, d, torch.float16, d)
    k, v, ks, vs, table = (t.to(cuda_device) for t in (kc, vc, ks, vs, table))
    buf = torch.empty((4 << 30) + (64 << 20), dtype=torch.uint8, device=cuda_device)
    far = [torch.as_strided(buf, t.shape, (page * d // 32, d // 32, (4 << 30) + 256, 1), o).copy_(t) for t, o in ((ks, 0), (vs, 32 << 20))]
    q = torch.randn(2, 6, d, generator=torch.Generator().manual_seed(1)).half().to(cuda_device)
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    got = []
    for s, t in ((ks, vs), far):
        out, lse = tda.flash_decode(q, k, v, table, n, 0.1, k_scale=s, v_scale=t)
        got.append([out, lse, tda.accumulate_attention_weights(q, k, table, n, lse, 0.1, torch.zeros(2, hkv, 90, device=cuda_device), k_scale=s)])
        kk, vv = k.clone(), v.clone()
        tda.evict_kvcache(kk, vv, table, n, got[-1][-1], 20, 5, k_scale=s, v_scale=t)
        got[-1] += [kk, vv, s, t]
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_conversion_results_belong_to_the_stream_they_are_written_on(cuda_device):
    """A result that is dropped while its kernel still has to run goes back to that stream's pool: the next tensor of the
    current stream is another one, and keeps what is written to it."""
    import triton_distributed_amd as tda
    dev, side = cuda_device, torch.cuda.Stream()
    x = torch.randn(4096, 8192, device=dev, dtype=torch.bfloat16)
    codes, scales = tda.mxfp4_quantize(x)
    torch.cuda.synchronize()
    for convert in (lambda: tda.mxfp4_quantize(x, stream=side), lambda: (tda.mxfp4_dequantize(codes, scales, stream=side),)):
        torch.cuda.empty_cache()
        with torch.cuda.stream(side):
            torch.cuda._sleep(int(2e7))
        made = convert()
        at = [t.data_ptr() for t in made]
        shapes = [(t.shape, t.dtype) for t in made]
        del made
        mine = [torch.full(s, 5, dtype=t, device=dev) for s, t in shapes]
        torch.cuda.synchronize()
        assert not set(at) & {t.data_ptr() for t in mine}
        assert all((t == 5).all() for t in mine)
    c, s = tda.mxfp4_quantize(x, stream=side)
    y = tda.mxfp4_dequantize(c, s, stream=side)
    side.synchronize()
    assert torch.equal(c, codes) and torch.equal(s, scales) and torch.equal(y, tda.mxfp4_dequantize(codes, scales))

"""Attention weights per cached token, eviction, and the two with append and decode as a serving loop runs them, on the GPU."""
import math

import pytest
import torch

from oracle import kv_evict as okv
from oracle import mxfp4
from oracle.fp8 import dequant_per_head, quant_per_head
from tests.mxfp4_cases import make_cache

pytestmark = pytest.mark.gpu


def _cache(kind, lens, page, hkv, d, dtype, seed, dv=None):
    """{"k", "v", "ks", "vs"} on the CPU, the table, and K and V in 64 bits."""
    if kind == "mxfp4":
        (kc, ks, k64, vc, vs, v64), table = make_cache(lens, page, hkv, d, dtype, seed)
        return {"k": kc, "v": vc, "ks": ks, "vs": vs}, table, k64, v64
    g = torch.Generator().manual_seed(seed)
    per = [(n + page - 1) // page for n in lens]
    pool = sum(per) + 3
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(max(per), 1)), 2 ** 31 - 1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = perm[at:at + n]
        at += n
    k = torch.randn(pool, page, hkv, d, generator=g).to(dtype)
    v = torch.randn(pool, page, hkv, dv or d, generator=g).to(dtype)
    if kind == "16bit":
        return {"k": k, "v": v, "ks": None, "vs": None}, table, k.double(), v.double()
    (k8, ks), (v8, vs) = quant_per_head(k), quant_per_head(v)
    return {"k": k8, "v": v8, "ks": ks, "vs": vs}, table, dequant_per_head(k8, ks, dtype).double(), dequant_per_head(v8, vs, dtype).double()


def _accumulate(kind, lens, hq, hkv, d, page, dtype, seed, dev, soft_cap=0.0, length=None):
    import triton_distributed_amd as tda
    c, table, k64, _ = _cache(kind, lens, page, hkv, d, dtype, seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(len(lens), hq, d, generator=g).to(dtype)
    sm_scale = d ** -0.5
    lse = torch.full((len(lens), hq), -math.inf)
    for i, n in enumerate(lens):
        if n:
            pos = torch.arange(n)
            s = torch.einsum("hgd,nhd->hgn", q[i].double().unflatten(0, (hkv, -1)), k64[table[i].long()[pos // page], pos % page]) * sm_scale
            s = soft_cap * torch.tanh(s / soft_cap) if soft_cap else s
            lse[i] = torch.logsumexp(s, -1).flatten().float()
    length = length or max(lens) + 5
    before = torch.rand(len(lens), hkv, length, generator=g)
    w = before.to(dev)
    ks = None if c["ks"] is None else c["ks"].to(dev)
    got = tda.accumulate_attention_weights(q.to(dev), c["k"].to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                                           lse.to(dev), sm_scale, w, soft_cap=soft_cap, k_scale=ks)
    torch.cuda.synchronize()
    assert got.data_ptr() == w.data_ptr()
    add, big = okv.token_weights(q, torch.nan_to_num(k64), table, lens, lse, sm_scale, soft_cap, length)
    # a logit: D products summed in fp32 and the scale; logit and lse scaled to powers of two (2^-22 of each); the exponential
    # and the sums over the heads (below 2^-18), then the addition to what was there
    k = torch.nan_to_num(k64).abs()
    e = (d + 8) * 2.0 ** -24 * float(q.double().abs().amax(-1).max()) * float(k.sum(-1).max()) * sm_scale
    tol = add * (e + 2.0 ** -22 * big + 2.0 ** -18) + 2.0 ** -23 * (before.double() + add)
    off = (got.cpu().double() - (before.double() + add)).abs()
    assert (off <= tol).all(), f"off by {float((off - tol).max())} over the tolerance"
    for i, n in enumerate(lens):
        assert torch.equal(got[i, :, n:].cpu(), before[i, :, n:])          # behind the end: nothing
    return got


LENS = [0, 1, 15, 16, 17, 33, 127, 128, 129, 700]


@pytest.mark.parametrize("kind", ["16bit", "fp8", "mxfp4"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 7, 16, 48])
def test_weights_of_lengths_and_pages(cuda_device, kind, d, page):
    _accumulate(kind, LENS, 8, 2, d, page, torch.bfloat16, d + page, cuda_device)


@pytest.mark.parametrize("batch", [2, 63, 64, 65, 130])
@pytest.mark.parametrize("kind,hkv", [("16bit", 1), ("mxfp4", 4)])
def test_weights_of_ragged_batches(cuda_device, kind, hkv, batch):
    """Tables that may hold long sequences: workgroups by length.  One long sequence, empty ones, ones of one token; many
    alike; all empty."""
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 90, (batch,), generator=g).tolist()
    lens[-1], lens[batch // 2], lens[0] = 2100, 0, 1
    _accumulate(kind, lens, 2 * hkv, hkv, 64, 16, torch.bfloat16, batch, cuda_device)
    _accumulate(kind, [lens[0]] + [300] * (batch - 2) + [2048], hkv, hkv, 64, 16, torch.float16, batch, cuda_device, length=2048)
    q = torch.randn(batch, hkv, 64, device=cuda_device, dtype=torch.float16)
    w = torch.rand(batch, hkv, 3200, device=cuda_device)
    before = w.clone()
    import triton_distributed_amd as tda
    tda.accumulate_attention_weights(q, torch.zeros(1, 16, hkv, 64, device=cuda_device, dtype=torch.float16),
                                     torch.zeros(batch, 200, dtype=torch.int32, device=cuda_device),
                                     torch.zeros(batch, dtype=torch.int32, device=cuda_device),
                                     torch.zeros(batch, hkv, device=cuda_device), 0.1, w)
    assert torch.equal(w, before)


@pytest.mark.parametrize("kind,d", [("16bit", 192), ("16bit", 576), ("fp8", 192), ("fp8", 576)])
def test_weights_of_two_segment_rows(cuda_device, kind, d):
    _accumulate(kind, [300, 17, 0], 16, 1, d, 16, torch.float16, d, cuda_device)


@pytest.mark.parametrize("kind", ["16bit", "fp8", "mxfp4"])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (16, 1), (17, 1), (40, 1), (128, 2), (64, 8), (9, 9)])
def test_weights_of_head_layouts(cuda_device, kind, hq, hkv):
    _accumulate(kind, [300, 0, 77, 1], hq, hkv, 128, 16, torch.float16, hq, cuda_device)


def test_weights_soft_cap_long_and_short_rows(cuda_device):
    _accumulate("16bit", [5000, 3], 8, 2, 128, 16, torch.bfloat16, 3, cuda_device, soft_cap=3.0)
    _accumulate("mxfp4", [40, 200], 8, 2, 128, 16, torch.bfloat16, 3, cuda_device, length=200)
    # weights shorter than a sequence: the tokens behind them are left out
    import triton_distributed_amd as tda
    dev = cuda_device
    c, table, k64, _ = _cache("16bit", [100], 16, 1, 64, torch.bfloat16, 5)
    q = torch.randn(1, 4, 64).bfloat16()
    lse = torch.full((1, 4), 3.0)
    buf = torch.zeros(1, 1, 64, device=dev)
    tda.accumulate_attention_weights(q.to(dev), c["k"].to(dev), table.to(dev), torch.tensor([100], dtype=torch.int32, device=dev),
                                     lse.to(dev), 0.125, buf[..., :50])
    want, _ = okv.token_weights(q, k64, table, [100], lse, 0.125, length=50)
    torch.testing.assert_close(buf[..., :50].cpu().double(), want, rtol=1e-4, atol=1e-6)
    assert (buf[..., 50:] == 0).all()


def test_weights_repeat_bit_for_bit_and_sum_to_the_heads(cuda_device):
    """Two runs give the same bits; with the decode's own lse the weights of a sequence add up to its q heads."""
    import triton_distributed_amd as tda
    dev = cuda_device
    for kind in ("16bit", "mxfp4"):
        lens = [3000, 64, 1]
        c, table, _, _ = _cache(kind, lens, 16, 2, 128, torch.bfloat16, 21)
        c = {n: None if t is None else t.to(dev) for n, t in c.items()}
        q, n, tb = torch.randn(3, 8, 128, device=dev).bfloat16(), torch.tensor(lens, dtype=torch.int32, device=dev), table.to(dev)
        _, lse = tda.flash_decode(q, c["k"], c["v"], tb, n, 0.1, k_scale=c["ks"], v_scale=c["vs"])
        runs = [tda.accumulate_attention_weights(q, c["k"], tb, n, lse, 0.1, torch.zeros(3, 2, 3000, device=dev), k_scale=c["ks"])
                for _ in range(2)]
        assert torch.equal(*runs)
        # (each weight is off by at most 2^-12 of itself)
        torch.testing.assert_close(runs[0].double().sum(-1).cpu(), torch.full((3, 2), 4.0, dtype=torch.float64), rtol=2.0 ** -12, atol=0)


def _evict(kind, lens, hkv, d, page, keep, recent, dtype, seed, dev, weights=None, dv=None, length=None, in_place=False, **kw):
    import triton_distributed_amd as tda
    c, table, _, _ = _cache(kind, lens, page, hkv, d, dtype, seed, dv)
    if kind != "mxfp4":
        c["ks"] = c["vs"] = None
    length = length or max(max(lens), 1) + 3
    g = torch.Generator().manual_seed(seed + 2)
    if weights is None:
        weights = (torch.rand(len(lens), hkv, length, generator=g) ** 4 * 64).round() / 64      # many ties
    on = {n: None if t is None else t.to(dev) for n, t in c.items()}
    w, n, tb = weights.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), table.to(dev)
    if in_place:
        kw = dict(kw, weights_out=w, kv_lens_out=n)
    new, kept, wo = tda.evict_kvcache(on["k"], on["v"], tb, n, w, keep, recent, k_scale=on["ks"], v_scale=on["vs"], **kw)
    torch.cuda.synchronize()
    names = [x for x in ("k", "v", "ks", "vs") if c[x] is not None]
    raw = lambda t: t.cpu().view(torch.uint8)
    rows, want_new, want_kept, want_w = okv.evict([raw(c[x]) for x in names], table, lens, weights, keep, recent)
    assert torch.equal(new.cpu(), want_new)
    assert torch.equal(kept.cpu(), want_kept)
    assert torch.equal(wo.cpu().view(torch.int32), want_w.view(torch.int32))
    for x, want in zip(names, rows):
        assert torch.equal(raw(on[x]), want), x                            # moved rows, and every other byte as it was
    if in_place:
        assert wo.data_ptr() == w.data_ptr() and new.data_ptr() == n.data_ptr()
    else:
        assert torch.equal(n.cpu(), torch.tensor(lens, dtype=torch.int32))


@pytest.mark.parametrize("kind", ["16bit", "fp8", "mxfp4"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 7, 16])
def test_evictions(cuda_device, kind, d, page):
    _evict(kind, [0, 1, 39, 40, 41, 64, 300, 517], 2, d, page, 40, 10, torch.bfloat16, d + page, cuda_device)


@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (30, 0), (30, 30), (30, 29), (299, 5), (300, 0), (303, 100)])
@pytest.mark.parametrize("in_place", [False, True])
def test_budgets(cuda_device, keep, recent, in_place):
    _evict("16bit", [300, 31, 299], 3, 64, 16, keep, recent, torch.float16, keep + recent, cuda_device, in_place=in_place)


def test_rows_of_other_lengths(cuda_device):
    _evict("16bit", [200, 90], 1, 576, 16, 60, 7, torch.bfloat16, 1, cuda_device, dv=512)
    _evict("16bit", [200, 90], 2, 192, 16, 60, 7, torch.bfloat16, 2, cuda_device, dv=128)
    _evict("fp8", [200, 90], 2, 192, 5, 60, 7, torch.bfloat16, 3, cuda_device)


@pytest.mark.parametrize("kind,batch,keep", [("16bit", 1, 3000), ("mxfp4", 1, 3000), ("16bit", 80, 300)])
def test_long_rows_and_many_sequences(cuda_device, kind, batch, keep):
    """Chunks that follow each other, one launch for all moves and two."""
    lens = [5000] if batch == 1 else [(37 * i) % 700 for i in range(batch)]
    _evict(kind, lens, 2 if batch == 1 else 8, 64, 16, keep, 100, torch.bfloat16, 5, cuda_device, in_place=batch > 1)


@pytest.mark.parametrize("b,hkv,length,keep,recent,d", [(1, 1, 70000, 9000, 100, 64), (1, 3, 40000, 39000, 0, 64), (4, 16, 60000, 5000, 5000, 64),
                                                        (4, 16, 60000, 3000, 17, 64), (2, 100, 90000, 700, 10, 32), (1, 1, 270000, 1000, 500, 32)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rows_spread_over_workgroups(cuda_device, b, hkv, length, keep, recent, d, in_place):
    """Long rows, whose weights several workgroups share: a few of them, many, and so many that each holds its weights in
    registers no more; ragged lengths with one that needs no eviction.  Against a stable sort."""
    import triton_distributed_amd as tda
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(length + hkv)
    page, per = 64, (length + 63) // 64
    table = torch.randperm(b * per, generator=g, device=dev).to(torch.int32).view(b, per)
    k = torch.randint(0, 256, (b * per, page, hkv, d), generator=g, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn)
    v = torch.randint(0, 256, (b * per, page, hkv, d), generator=g, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn)
    lens = torch.tensor([length, keep - 1, keep + 1, length // 2][:b], dtype=torch.int32, device=dev)
    w = (torch.rand(b, hkv, length, generator=g, device=dev) ** 8 * 1000).round() / 8                  # many zeros, many ties
    w[0, 0] = w[0, 0, 0]                                                                              # a row of equal weights
    want_k, want_v, want_w = k.view(torch.uint8).clone(), v.view(torch.uint8).clone(), torch.zeros_like(w)
    want_kept = torch.full((b, hkv, keep), -1, dtype=torch.int32, device=dev)
    for i, n in enumerate(lens.tolist()):
        order = w[i, :, :n].clone()
        order[:, max(n - recent, 0):] = math.inf
        stay = torch.sort(order, dim=-1, descending=True, stable=True).indices[:, :keep].sort(-1).values
        m = stay.shape[1]
        want_kept[i, :, :m] = stay.to(torch.int32)
        want_w[i, :, :m] = w[i].gather(-1, stay)
        head, to = torch.arange(hkv, device=dev)[:, None], torch.arange(m, device=dev)
        row = table[i].long()
        for pool in (want_k, want_v):
            pool[row[to // page], to % page, head] = pool[row[stay // page], stay % page, head]
    new, kept, wo = tda.evict_kvcache(k, v, table, lens, w, keep, recent, weights_out=w if in_place else None)
    assert torch.equal(kept, want_kept)
    assert torch.equal(wo, want_w) and (wo.data_ptr() == w.data_ptr()) == in_place
    assert torch.equal(new, lens.clamp(max=keep))
    assert torch.equal(k.view(torch.uint8), want_k) and torch.equal(v.view(torch.uint8), want_v)


def test_weights_that_order_awkwardly(cuda_device):
    """All alike, all zero, both zeros, negative, infinite, NaN, subnormal, apart in the last bit only."""
    n = 400
    base = torch.ones(1, 1, n)
    cases = [base, base * 0, torch.where(torch.arange(n) % 3 == 0, 0.0, -0.0)[None, None], -torch.rand(1, 1, n),
             torch.rand(1, 1, n), torch.rand(1, 1, n) * 1e-40, base + torch.arange(n).flip(0) % 7 * 2.0 ** -23,
             (torch.arange(n) * 1.0)[None, None], (torch.arange(n).flip(0) * 1.0)[None, None]]
    cases[4][0, 0, ::7] = math.inf
    cases[4][0, 0, 1::9] = -math.inf
    cases[4][0, 0, 2::11] = math.nan
    cases[4][0, 0, 5] = -math.nan
    for i, w in enumerate(cases):
        for keep, recent in ((100, 20), (1, 0), (399, 0)):
            _evict("16bit", [n], 1, 64, 16, keep, recent, torch.bfloat16, 40 + i, cuda_device, weights=w.float().contiguous(), length=n)


def test_weights_laid_out_apart(cuda_device):
    """Weights that are views: heads outermost, a slice of longer rows; a length beyond what the weights cover."""
    import triton_distributed_amd as tda
    dev, lens = cuda_device, [120, 64]
    c, table, _, _ = _cache("16bit", lens, 16, 2, 64, torch.bfloat16, 8)
    w = torch.rand(2, 2, 110, generator=torch.Generator().manual_seed(1))
    base = torch.full((2, 2, 130), 9.0, device=dev)
    view = base.transpose(0, 1)[..., 7:117]
    view.copy_(w)
    k, v = c["k"].to(dev), c["v"].to(dev)
    new, kept, wo = tda.evict_kvcache(k, v, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), view, 50, 10, weights_out=view)
    rows, want_new, want_kept, want_w = okv.evict([c["k"], c["v"]], table, lens, w, 50, 10)
    assert torch.equal(new.cpu(), want_new) and torch.equal(kept.cpu(), want_kept) and torch.equal(view.cpu(), want_w)
    assert torch.equal(k.cpu(), rows[0]) and torch.equal(v.cpu(), rows[1])
    assert (base[..., :7] == 9).all() and (base[..., 117:] == 9).all()


def test_captured_bookkeeping(cuda_device):
    """Weights and eviction in a graph: replays follow the lengths and weights on the device."""
    import triton_distributed_amd as tda
    dev = cuda_device
    c, table, k64, _ = _cache("16bit", [400, 400], 16, 2, 64, torch.bfloat16, 31)
    k, v, tb = c["k"].to(dev), c["v"].to(dev), table.to(dev)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(2)).bfloat16()
    qd, n = q.to(dev), torch.tensor([50, 60], dtype=torch.int32, device=dev)
    lse, w = torch.full((2, 4), 4.0, device=dev), torch.zeros(2, 2, 400, device=dev)
    wo, new = torch.empty_like(w), torch.empty_like(n)
    kept = torch.empty(2, 2, 100, dtype=torch.int32, device=dev)

    def step():
        tda.accumulate_attention_weights(qd, k, tb, n, lse, 0.125, w)
        return tda.evict_kvcache(k, v, tb, n, w, 100, 20, weights_out=wo, kv_lens_out=new, kept=kept)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lens in ([400, 120], [0, 399], [100, 101]):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        w.zero_()
        k.copy_(c["k"])
        v.copy_(c["v"])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (w, wo, new, kept, k, v)]
        w.zero_()
        k.copy_(c["k"])
        v.copy_(c["v"])
        step()
        torch.cuda.synchronize()
        for a, b in zip(replayed, (w, wo, new, kept, k, v)):
            assert torch.equal(a, b)
        rows, want_new, want_kept, _ = okv.evict([c["k"], c["v"]], table, lens, w.cpu(), 100, 20)
        assert torch.equal(new.cpu(), want_new) and torch.equal(kept.cpu(), want_kept) and torch.equal(k.cpu(), rows[0])


def test_another_stream_than_the_current_one(cuda_device):
    import triton_distributed_amd as tda
    dev, side = cuda_device, torch.cuda.Stream()
    c, table, _, _ = _cache("16bit", [400], 16, 2, 64, torch.bfloat16, 33)
    w = torch.rand(1, 2, 400, generator=torch.Generator().manual_seed(1))
    k, v, tb, n, wd = c["k"].to(dev), c["v"].to(dev), table.to(dev), torch.tensor([400], dtype=torch.int32, device=dev), w.to(dev)
    torch.cuda.synchronize()
    new, kept, wo = tda.evict_kvcache(k, v, tb, n, wd, 100, 20, stream=side)
    side.synchronize()
    rows, want_new, want_kept, want_w = okv.evict([c["k"], c["v"]], table, [400], w, 100, 20)
    assert torch.equal(new.cpu(), want_new) and torch.equal(kept.cpu(), want_kept) and torch.equal(wo.cpu(), want_w)
    assert torch.equal(k.cpu(), rows[0]) and torch.equal(v.cpu(), rows[1])


@pytest.mark.parametrize("kind", ["16bit", "mxfp4"])
@pytest.mark.parametrize("bad", [-1, -2 ** 31, 12, 2 ** 31 - 1])
def test_rows_of_pages_outside_the_pool_are_left_out(cuda_device, kind, bad):
    """64 tokens on four pages, the last 32 stay: a source page and, in another sequence, a target page that the pool of
    12 does not have."""
    import triton_distributed_amd as tda
    dev, shape = cuda_device, (12, 16, 2, 64)
    g = torch.Generator().manual_seed(3)
    if kind == "mxfp4":
        pools = [torch.randint(0, 256, shape[:3] + (n,), dtype=torch.uint8, generator=g) for n in (32, 32, 2, 2)]
    else:
        pools = [torch.randn(shape, generator=g).bfloat16() for _ in range(2)]
    table = torch.tensor([[3, 5, bad, 7], [1, bad, 0, 2], [4, 6, 8, 9]], dtype=torch.int32)
    want = [t.clone() for t in pools]
    for t, before in zip(want, pools):
        t[5] = before[7]                       # (slots 0 .. 15 of sequence 0 would come from the bad page)
        t[1] = before[0]                       # (slots 16 .. 31 of sequence 1 would go to it)
        t[4], t[6] = before[8], before[9]
    got = [t.to(dev) for t in pools]
    weights = torch.arange(64, dtype=torch.float32, device=dev).expand(3, 2, 64).contiguous()
    scales = dict(k_scale=got[2], v_scale=got[3]) if kind == "mxfp4" else {}
    lens, kept, _ = tda.evict_kvcache(got[0], got[1], table.to(dev), torch.full((3,), 64, dtype=torch.int32, device=dev), weights, 32, 4, **scales)
    assert lens.tolist() == [32] * 3 and kept[0, 0].tolist() == list(range(32, 64))
    for t, w in zip(got, want):
        assert torch.equal(t.cpu(), w)


@pytest.mark.parametrize("dk,dv,first,hkv", [(576, 512, 0, 1), (576, 512, 64, 1), (128, 128, 0, 4), (64, 128, 0, 2)])
@pytest.mark.parametrize("lens,keep", [([700, 90, 300], 200), ([5000], 3000)])
def test_v_rows_that_are_a_part_of_the_k_rows(cuda_device, dk, dv, first, hkv, lens, keep):
    """Latent attention holds V inside K (and, the other way round, K inside V): every row moves once, whole."""
    import triton_distributed_amd as tda
    dev, page, d = cuda_device, 16, max(dk, dv)
    c, table, _, _ = _cache("16bit", lens, page, hkv, d, torch.bfloat16, dk + first)
    pool = c["k"].to(dev)
    k, v = (pool, pool[..., first:first + dv]) if dk >= dv else (pool[..., first:first + dk], pool)
    w = (torch.rand(len(lens), hkv, max(lens), generator=torch.Generator().manual_seed(4)) ** 4 * 64).round() / 64
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    new, kept, wo = tda.evict_kvcache(k, v, table.to(dev), n, w.to(dev), keep, 50)
    (want,), want_new, want_kept, want_w = okv.evict([c["k"]], table, lens, w, keep, 50)
    assert torch.equal(new.cpu(), want_new) and torch.equal(kept.cpu(), want_kept) and torch.equal(wo.cpu(), want_w)
    assert torch.equal(pool.cpu(), want)


def test_mxfp4_rows_and_scales_that_are_v_and_k_at_once(cuda_device):
    import triton_distributed_amd as tda
    dev, lens = cuda_device, [400, 77]
    c, table, _, _ = _cache("mxfp4", lens, 16, 2, 128, torch.bfloat16, 6)
    rows, scales = c["k"].to(dev), c["ks"].to(dev)
    w = torch.rand(2, 2, 400, generator=torch.Generator().manual_seed(4))
    tda.evict_kvcache(rows, rows, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), w.to(dev), 60, 5, k_scale=scales, v_scale=scales)
    (want_rows, want_scales), _, _, _ = okv.evict([c["k"], c["ks"]], table, lens, w, 60, 5)
    assert torch.equal(rows.cpu(), want_rows) and torch.equal(scales.cpu(), want_scales)


@pytest.mark.parametrize("b,hkv,length,keep,recent,d", [(1, 1, 4097, 4000, 100, 32), (1, 3, 16384, 16000, 0, 32), (2, 16, 12001, 300, 300, 32),
                                                        (4, 64, 9000, 2000, 17, 32), (4, 64, 20000, 19000, 17, 32), (2, 40, 70000, 1000, 10, 32)])
@pytest.mark.parametrize("in_place", [False, True])
def test_long_rows_of_one_workgroup_each(cuda_device, b, hkv, length, keep, recent, d, in_place):
    """Up to 16384 weights out of registers; longer rows, of which there are many, read in every pass."""
    test_rows_spread_over_workgroups(cuda_device, b, hkv, length, keep, recent, d, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_segments_that_are_read_in_every_pass(cuda_device, in_place):
    """Eight workgroups to a row, of more than 16384 weights each."""
    test_rows_spread_over_workgroups(cuda_device, 1, 64, 140000, 700, 10, 32, in_place)

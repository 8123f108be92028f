"""A paged cache in 4 bits, kept at a budget: bookkeeping on the CPU, and a serving loop - append with positions of three
axes, decode, attention weights, eviction - against 64 bits on the GPU."""
import pytest
import torch

from oracle import kv_evict as okv
from oracle import mxfp4, rope_axes
from triton_distributed_amd.paged_kv_cache import PagedKVCache


def _cache(device, dtype=torch.float4_e2m1fn_x2, layers=2, batch=3, **kw):
    return PagedKVCache(PAGE_SIZE=4, num_layers=layers, batch_size=batch, max_length=64, num_kv_heads=2, head_dim=64, dtype=dtype,
                        device=device, generator=torch.Generator().manual_seed(1), **kw)


def test_mxfp4_pools():
    c = _cache("cpu")
    blocks = 16 * 3 * 2
    assert tuple(c.key_cache.shape) == (blocks, 4, 2, 32) == tuple(c.value_cache.shape)
    assert c.key_cache.dtype == torch.float4_e2m1fn_x2
    assert tuple(c.k_block_scale.shape) == (blocks, 4, 2, 2) == tuple(c.v_block_scale.shape)
    assert c.nbytes == 2 * blocks * 4 * 2 * 34
    assert c.layer_scales(1) == (c.k_block_scale, c.v_block_scale)
    assert not c.key_cache.view(torch.uint8).any() and (c.value_cache.data_ptr() - c.key_cache.data_ptr()) % 512 == 256
    with pytest.raises(ValueError, match="zeroed"):
        _cache("cpu", fill="randn")
    with pytest.raises(ValueError, match="multiple of 32"):
        PagedKVCache(head_dim=48, max_length=8, num_layers=1, dtype=torch.float4_e2m1fn_x2, device="cpu")


def test_positions_and_refusals_without_a_gpu():
    c = _cache("cpu")
    c.inc_offset(5)
    c.inc_offset(2)
    assert c.next_positions(2).tolist() == [[5, 6]] * 3 and c.next_positions(2).dtype == torch.int32
    w = torch.zeros(2, 3, 2, 7)
    assert c.evict(w, 7, 2) is None and c.max_kv_len == 7                  # nothing has to go
    for bad in (w[0], w[:1], w[..., :6]):
        with pytest.raises(ValueError, match="weights"):
            c.evict(bad, 3, 1)
    with pytest.raises(ValueError, match="GPU"):
        c.evict(w, 3, 1)
    assert c.max_kv_len == 7 and c.next_positions(1).tolist() == [[6]] * 3


def _evict_on_the_host(monkeypatch):
    """Stand-ins for the operators: lengths as the eviction leaves them; what the append is given."""
    import triton_distributed_amd as tda
    given = []

    def evict(k, v, table, lens, w, keep, recent, kv_lens_out=None, **kw):
        if kv_lens_out is not None:
            kv_lens_out.clamp_(max=keep)

    def append(*args, positions=None, **kw):
        given.append(positions)
    monkeypatch.setattr(tda, "evict_kvcache", evict, raising=False)
    monkeypatch.setattr(tda, "qk_norm_rope_update_kvcache", append, raising=False)
    return given


def test_positions_behind_the_rotary_tables_are_refused(monkeypatch):
    """A cache at a budget sees more tokens than it holds: from the first that the tables have no row for, an append that
    would take its position from the count is refused, on the host; one with positions of its own is not."""
    given = _evict_on_the_host(monkeypatch)
    c = _cache("cpu")
    w, table = torch.zeros(2, 3, 2, 64), torch.zeros(1, 40, 64)
    x = torch.zeros(3, 1, 8, 64, dtype=torch.bfloat16)
    c.inc_offset(30)
    c.evict(w, 20, 5)
    for seen in range(31, 41):
        c.inc_offset(1)
        c.append(0, x, None, None, table, table)
        assert given[-1].tolist() == [[seen - 1]] * 3
        if seen == 35:
            c.evict(w, 20, 5)
    assert c.max_kv_len == 25 < 40
    c.inc_offset(1)
    n = len(given)
    for cos, sin in ((table, table), (table.expand(3, 40, 64), table[0]), (torch.zeros(50, 64), table)):
        with pytest.raises(ValueError, match="positions"):
            c.append(0, x, None, None, cos, sin)
    assert len(given) == n
    c.append(0, x, None, None, table, table, positions=torch.zeros(3, 1, dtype=torch.int32))
    c.append(0, x, None, None, torch.zeros(41, 64), torch.zeros(41, 64))
    assert len(given) == n + 2 and given[-1].tolist() == [[40]] * 3
    c.reset()
    c.inc_offset(2)
    c.append(0, x, None, None, table[:, :1], table[:, :1])                  # (as ever without an eviction: places in the cache)
    assert given[-1] is None and c.next_positions(1).tolist() == [[1]] * 3


def test_an_eviction_is_not_captured(monkeypatch):
    """A replay would shorten the sequences once more and count the tokens seen from the shortened lengths, while the host
    goes on from what it knew at the capture."""
    import sys
    _evict_on_the_host(monkeypatch)
    c = _cache("cpu")
    w = torch.zeros(2, 3, 2, 64)
    c.inc_offset(30)
    monkeypatch.setattr(sys.modules["triton_distributed_amd.flash_decode"], "_capturing", lambda: True)
    with pytest.raises(ValueError, match="capture"):
        c.evict(w, 20, 5)
    assert c.max_kv_len == 30 and c.kv_lens.tolist() == [30] * 3 and c.next_positions(1).tolist() == [[29]] * 3
    assert c.evict(w, 30, 5) is None
    monkeypatch.undo()
    _evict_on_the_host(monkeypatch)
    assert tuple(c.evict(w, 20, 5).shape) == (2, 3, 2, 20) and c.max_kv_len == 20


@pytest.mark.gpu
def test_an_eviction_under_capture_leaves_the_cache_as_it_was(cuda_device):
    c = _cache(cuda_device)
    c.inc_offset(30)
    w = torch.rand(2, 3, 2, 64, device=cuda_device)
    x = torch.zeros(1, device=cuda_device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(ValueError, match="capture"):
            c.evict(w, 20, 5)
    graph.replay()
    torch.cuda.synchronize()
    assert c.max_kv_len == 30 and c.kv_lens.tolist() == [30] * 3 and float(x) == 1
    assert tuple(c.evict(w, 20, 5).shape) == (2, 3, 2, 20) and c.kv_lens.tolist() == [20] * 3


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float4_e2m1fn_x2, torch.bfloat16])
def test_a_serving_loop_at_a_budget(cuda_device, dtype):
    """Prompt, then single tokens; after every decode the weights, an eviction whenever the budget is exceeded by four
    tokens.  Every step's decode, weights, survivors and rows against the oracle, which carries its own copy of the cache."""
    dev, b, hq, hkv, d, layers, keep, recent = cuda_device, 3, 4, 2, 64, 2, 20, 6
    c = _cache(dev, dtype)
    g = torch.Generator().manual_seed(2)
    sections, scale = (12, 10, 10), 0.125
    ang = torch.rand(200, d // 2, generator=g) * 6.28
    cos, sin = ang.cos(), ang.sin()
    wq, wk = ((1 + 0.1 * torch.randn(d, generator=g)).bfloat16() for _ in range(2))
    S = 40
    weights = torch.zeros(layers, b, hkv, S, device=dev)
    seen, evictions = 0, 0
    tables = c.block_tables.cpu()

    def values():
        """K and V of the pools in 64 bits."""
        if c.mxfp4:
            return [mxfp4.dequantize(x, s) for x, s in ((c.key_cache, c.k_block_scale), (c.value_cache, c.v_block_scale))]
        return [x.cpu().double() for x in (c.key_cache, c.value_cache)]

    for step in range(14):
        new = 17 if step == 0 else 1
        c.inc_offset(new)
        lens = [c.max_kv_len] * b
        time = torch.arange(seen, seen + new, dtype=torch.int32).expand(b, new)
        assert torch.equal(c.next_positions(new).cpu(), time)
        positions = torch.stack((time, time // 3 + 1, time % 5))
        seen += new
        for layer in range(layers):
            qkv = torch.randn(b, new, hq + 2 * hkv, d, generator=g).bfloat16()
            before = values()
            q = c.append(layer, qkv.to(dev), wq.to(dev), wk.to(dev), cos.to(dev), sin.to(dev), positions=positions.to(dev),
                         rope_sections=sections)
            want, pair = rope_axes.norm_rope(qkv[:, :, :hq], wq, 1e-6, cos, sin, positions, sections, False)
            assert ((q.cpu().double() - want).abs() <= 2.0 ** -7 * (pair + want.abs()) + 2.0 ** -20).all()
            after = values()
            v16 = qkv[:, :, hq + hkv:]
            v_want = mxfp4.dequantize(*mxfp4.quantize(v16)) if c.mxfp4 else v16.double()
            for i in range(b):
                for t in range(new):
                    at = lens[i] - new + t
                    pg, slot = int(tables[layer, i, at // 4]), at % 4
                    assert torch.equal(after[1][pg, slot], v_want[i, t])
                    before[1][pg, slot] = v_want[i, t]
            assert torch.equal(after[1], before[1])                       # nothing else moved
            q1 = q[:, -1].contiguous()
            out, lse = c.decode(layer, q1, scale)
            o64, l64, spread = mxfp4.decode(q1, after[0], after[1], tables[layer], lens, scale)
            assert ((out.cpu().double() - o64).abs() <= 2.0 ** -8 * (spread + o64.abs()) + 2.0 ** -12 * spread + 2.0 ** -20).all()
            torch.testing.assert_close(lse.cpu().double(), l64, atol=2.0 ** -14, rtol=2.0 ** -20)
            w_before = weights[layer].cpu().double()
            c.accumulate(layer, q1, lse, scale, weights[layer])
            add, _ = okv.token_weights(q1, after[0], tables[layer], lens, lse, scale, length=S)
            torch.testing.assert_close(weights[layer].cpu().double(), w_before + add, rtol=2.0 ** -12, atol=2.0 ** -20)
        if c.max_kv_len >= keep + 4:
            pools = [x.cpu().view(torch.uint8) if x is not None else None for x in (c.key_cache, c.value_cache, c.k_block_scale, c.v_block_scale)]
            pools = [x for x in pools if x is not None]
            w_before = weights.cpu()
            kept = c.evict(weights, keep, recent)
            for layer in range(layers):
                pools, new_lens, want_kept, want_w = okv.evict(pools, tables[layer], lens, w_before[layer], keep, recent)
                assert torch.equal(kept[layer].cpu(), want_kept) and torch.equal(weights[layer].cpu(), want_w)
            assert torch.equal(c.kv_lens.cpu(), new_lens) and c.max_kv_len == keep
            got = [x.cpu().view(torch.uint8) for x in (c.key_cache, c.value_cache, c.k_block_scale, c.v_block_scale) if x is not None]
            assert all(torch.equal(a, w) for a, w in zip(got, pools))
            evictions += 1
    assert evictions >= 2
    # one more token, at the position that follows all that were seen
    c.inc_offset(1)
    assert c.next_positions(1).tolist() == [[seen]] * b
    qkv = torch.randn(b, 1, hq + 2 * hkv, d, generator=g).bfloat16()
    q = c.append(0, qkv.to(dev), wq.to(dev), wk.to(dev), cos.to(dev), sin.to(dev))
    want, pair = rope_axes.norm_rope(qkv[:, :, :hq], wq, 1e-6, cos, sin, torch.full((1, b, 1), seen), (d // 2,), False)
    assert ((q.cpu().double() - want).abs() <= 2.0 ** -7 * (pair + want.abs()) + 2.0 ** -20).all()


@pytest.mark.gpu
def test_eviction_and_append_on_another_stream(cuda_device):
    """What the cache works out with torch goes with the kernels, while the current stream is busy with something else."""
    dev = cuda_device
    c = _cache(dev)
    c.inc_offset(30)
    w = torch.rand(2, 3, 2, 64, device=dev)
    ang = torch.rand(200, 32, device=dev) * 6.28
    qkv = torch.randn(3, 1, 8, 64, device=dev).bfloat16()
    ones = torch.ones(64, device=dev, dtype=torch.bfloat16)
    cos, sin = (torch.cat([t, t], -1) for t in (ang.cos(), ang.sin()))
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(int(2e7))
    assert tuple(c.evict(w, 20, 5, stream=other).shape) == (2, 3, 2, 20)
    with torch.cuda.stream(other):
        c.inc_offset(1)
    q = c.append(0, qkv, ones, ones, cos, sin, stream=other)
    other.synchronize()
    assert c.kv_lens.tolist() == [21] * 3
    torch.cuda.synchronize()
    assert c.next_positions(1).tolist() == [[30]] * 3
    want = c.append(0, qkv, ones, ones, cos, sin, positions=torch.full((3, 1), 30, dtype=torch.int32, device=dev))
    assert torch.equal(q, want)


@pytest.mark.gpu
def test_two_caches_at_once_on_two_streams_and_threads(cuda_device):
    """The loop of two caches on two streams, from two threads, gives the bits that each gives by itself."""
    import threading
    dev = cuda_device
    ang = torch.rand(400, 64, generator=torch.Generator().manual_seed(9)) * 6.28
    cos, sin = (torch.cat([t, t], -1).to(dev) for t in (ang.cos(), ang.sin()))
    ones = torch.ones(128, device=dev, dtype=torch.bfloat16)
    prompts = [torch.randn(4, 300, 12, 128, generator=torch.Generator().manual_seed(i)).bfloat16().to(dev) for i in range(2)]
    steps = [torch.randn(24, 4, 1, 12, 128, generator=torch.Generator().manual_seed(7 + i)).bfloat16().to(dev) for i in range(2)]
    torch.cuda.synchronize()

    def loop(i, got):
        with torch.cuda.stream(torch.cuda.Stream()):
            c = PagedKVCache(PAGE_SIZE=16, num_layers=1, batch_size=4, max_length=400, num_kv_heads=2, head_dim=128,
                             dtype=torch.float4_e2m1fn_x2, device=dev, generator=torch.Generator().manual_seed(i))
            w = torch.zeros(1, 4, 2, 400, device=dev)
            for x in [prompts[i], *steps[i]]:
                c.inc_offset(x.shape[1])
                q = c.append(0, x, ones, ones, cos, sin)[:, -1].contiguous()
                out, lse = c.decode(0, q, 0.09)
                c.accumulate(0, q, lse, 0.09, w[0])
                got += [out, lse, w.clone()]
                if c.max_kv_len > 200 + 4 * i:
                    got.append(c.evict(w, 190, 30))
            torch.cuda.current_stream().synchronize()
    alone, together = ([], []), ([], [])
    for i in range(2):
        loop(i, alone[i])
    threads = [threading.Thread(target=loop, args=(i, together[i])) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, together):
        assert len(a) == len(b) > 75
        for x, y in zip(a, b):
            assert torch.equal(x, y)

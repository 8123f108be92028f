"""Attention weights and eviction, without a GPU: what is refused, and the oracle against a case worked out by hand."""
import ctypes as C
import math

import pytest
import torch

import triton_distributed_amd as tda
from oracle import kv_evict as okv
from triton_distributed_amd import _lib
from triton_distributed_amd._lib import FdkAttnWeightsArgs, FdkKvEvictArgs


def _weights_args(**kw):
    a = FdkAttnWeightsArgs()
    a.struct_size, a.flags = C.sizeof(FdkAttnWeightsArgs), _lib.FDK_FLAG_DRY_RUN
    a.q, a.q_stride_b, a.q_stride_h, a.q_dtype = 0x10000, 32 * 128, 128, _lib.FDK_BF16
    a.kv_dtype, a.k_cache = _lib.FDK_BF16, 0x20000
    a.k_stride_page, a.k_stride_tok, a.k_stride_head = 16 * 8 * 128, 8 * 128, 128
    a.k_block_scale, a.kbs_stride_page, a.kbs_stride_tok, a.kbs_stride_head = 0x30001, 512, 32, 4
    a.block_table, a.table_stride_b, a.kv_lens, a.lse, a.lse_stride_b = 0x40000, 256, 0x50000, 0x60000, 32
    a.weights, a.weights_stride_b, a.weights_stride_h = 0x70000, 8 * 4096, 4096
    a.batch, a.num_q_heads, a.num_kv_heads, a.head_dim = 32, 32, 8, 128
    a.page_size, a.max_pages, a.weights_len, a.sm_scale = 16, 256, 4096, 0.1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


MX = dict(kv_dtype=_lib.FDK_MXFP4, k_stride_page=16 * 8 * 64, k_stride_tok=8 * 64, k_stride_head=64)


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (MX, 0), (dict(kv_dtype=_lib.FDK_FP8_E4M3), 0), (dict(batch=0, q=None), 0),
    (dict(struct_size=8), _lib.FDK_EABI), (dict(q=None), _lib.FDK_ENULL), (dict(lse=None), _lib.FDK_ENULL), (dict(weights=None), _lib.FDK_ENULL),
    (dict(k_cache=None), _lib.FDK_ENULL), (dict(block_table=None), _lib.FDK_ENULL), (dict(MX, k_block_scale=None), _lib.FDK_ENULL),
    (dict(q=0x10008), _lib.FDK_EALIGN), (dict(q_stride_h=132), _lib.FDK_EALIGN), (dict(k_stride_tok=8 * 128 + 4), _lib.FDK_EALIGN),
    (dict(weights=0x70002), _lib.FDK_EALIGN), (dict(num_q_heads=33), _lib.FDK_ESHAPE), (dict(num_kv_heads=0), _lib.FDK_ESHAPE),
    (dict(head_dim=96), _lib.FDK_EUNSUPPORTED), (dict(MX, head_dim=192), _lib.FDK_EUNSUPPORTED), (dict(kv_dtype=_lib.FDK_FP16), _lib.FDK_EUNSUPPORTED),
    (dict(weights_len=0), _lib.FDK_ESHAPE), (dict(weights_stride_h=4095), _lib.FDK_ESHAPE), (dict(weights_stride_b=4095), _lib.FDK_ESHAPE),
    (dict(lse_stride_b=31), _lib.FDK_ESHAPE), (dict(page_size=0), _lib.FDK_ESHAPE), (dict(max_pages=1 << 27), _lib.FDK_ESHAPE),
    (dict(table_stride_b=255), _lib.FDK_ESHAPE), (dict(sm_scale=math.inf), _lib.FDK_ESHAPE), (dict(soft_cap=math.nan), _lib.FDK_ESHAPE),
    (dict(k_stride_head=120), _lib.FDK_ESHAPE), (dict(batch=70000), _lib.FDK_ESHAPE), (dict(MX, kbs_stride_head=3), _lib.FDK_ESHAPE),
    (dict(k_stride_page=1 << 31), _lib.FDK_ESHAPE), (dict(k_stride_tok=1 << 27), _lib.FDK_ESHAPE),
])
def test_weights_refusals(kw, code):
    assert _lib.load().fdk_accumulate_weights(C.byref(_weights_args(**kw)), None) == code, _lib.load().fdk_last_error()


def _evict_args(**kw):
    a = FdkKvEvictArgs()
    a.struct_size, a.flags, a.kv_dtype = C.sizeof(FdkKvEvictArgs), _lib.FDK_FLAG_DRY_RUN, _lib.FDK_BF16
    a.k_cache, a.v_cache = 0x10000, 0x20000
    a.k_stride_page, a.k_stride_tok, a.k_stride_head = 16 * 8 * 128, 8 * 128, 128
    a.v_stride_page, a.v_stride_tok, a.v_stride_head = 16 * 8 * 128, 8 * 128, 128
    a.block_table, a.table_stride_b, a.kv_lens = 0x30000, 256, 0x40000
    a.weights, a.weights_stride_b, a.weights_stride_h = 0x50000, 8 * 4096, 4096
    a.weights_out, a.weights_out_stride_b, a.weights_out_stride_h = 0x60000, 8 * 4096, 4096
    a.kept, a.kv_lens_out, a.workspace, a.workspace_bytes = 0x70000, 0x80000, 0x90000, 32 * 8 * 16
    a.batch, a.num_kv_heads, a.head_dim = 32, 8, 128
    a.page_size, a.max_pages, a.weights_len, a.keep, a.recent, a.num_pages = 16, 256, 4096, 2048, 256, 8192
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (dict(batch=0, k_cache=None), 0), (dict(weights_out=0x50000, kv_lens_out=0x40000), 0), (dict(keep=4096, recent=4096), 0),
    (dict(kv_dtype=_lib.FDK_FP8_E4M3), 0), (dict(struct_size=16), _lib.FDK_EABI), (dict(kv_dtype=_lib.FDK_FP32), _lib.FDK_EUNSUPPORTED),
    (dict(kv_dtype=_lib.FDK_MXFP4), _lib.FDK_ENULL), (dict(head_dim=40), _lib.FDK_EUNSUPPORTED), (dict(v_head_dim=8192), _lib.FDK_EUNSUPPORTED),
    (dict(keep=0), _lib.FDK_ESHAPE), (dict(keep=4097), _lib.FDK_ESHAPE), (dict(num_pages=0), _lib.FDK_ESHAPE), (dict(recent=-1), _lib.FDK_ESHAPE), (dict(recent=2049), _lib.FDK_ESHAPE),
    (dict(v_cache=0x20008), _lib.FDK_EALIGN), (dict(v_cache=None), _lib.FDK_ENULL), (dict(kept=None), _lib.FDK_ENULL),
    (dict(weights_out=None), _lib.FDK_ENULL), (dict(kv_lens_out=None), _lib.FDK_ENULL), (dict(workspace=None), _lib.FDK_EWORKSPACE),
    (dict(workspace_bytes=32 * 8 * 16 - 1), _lib.FDK_EWORKSPACE), (dict(workspace=0x90008), _lib.FDK_EALIGN), (dict(kept=0x70001), _lib.FDK_EALIGN),
    (dict(weights_out_stride_h=4000), _lib.FDK_ESHAPE), (dict(weights_out=0x50000, weights_stride_h=5000), _lib.FDK_ESHAPE),
    (dict(weights_stride_b=-1), _lib.FDK_ESHAPE), (dict(v_stride_tok=8 * 128 + 2), _lib.FDK_EALIGN), (dict(v_head_dim=160), _lib.FDK_ESHAPE),
])
def test_evict_refusals(kw, code):
    assert _lib.load().fdk_kv_evict(C.byref(_evict_args(**kw)), None) == code, _lib.load().fdk_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(v_cache=0x10000), 0), (dict(v_cache=0x10000, v_head_dim=64), 0), (dict(v_cache=0x10080, v_head_dim=64), 0),
    (dict(k_cache=0x10080, v_cache=0x10000, head_dim=64), 0), (dict(v_cache=0x10100), 0), (dict(v_cache=0x10080), _lib.FDK_ESHAPE),
    (dict(v_cache=0x0FF80), _lib.FDK_ESHAPE), (dict(v_cache=0x0FF00), 0),
    (dict(v_cache=0x10080, batch=1, num_kv_heads=1, v_stride_head=999), _lib.FDK_ESHAPE),
])
def test_rows_that_share_memory(kw, code):
    """V rows that are a part of the K rows, or the other way round, are one thing to move; rows of which parts overlap are refused."""
    assert _lib.load().fdk_kv_evict(C.byref(_evict_args(**kw)), None) == code, _lib.load().fdk_last_error()


def test_weights_rows_that_share_elements_are_refused():
    """Every layout of three sequences x four heads with strides up to 60 elements, rows of 5: against the elements themselves."""
    lib = _lib.load()
    for sb in range(5, 60):
        for sh in range(5, 60):
            at = [b * sb + h * sh + i for b in range(3) for h in range(4) for i in range(5)]
            want = 0 if len(set(at)) == len(at) else _lib.FDK_ESHAPE
            a = _weights_args(batch=3, num_kv_heads=4, num_q_heads=4, weights_len=5, weights_stride_b=sb, weights_stride_h=sh, lse_stride_b=4)
            assert lib.fdk_accumulate_weights(C.byref(a), None) == want, (sb, sh)
            e = _evict_args(batch=3, num_kv_heads=4, weights_len=5, keep=3, recent=1, weights_out_stride_b=sb, weights_out_stride_h=sh)
            assert lib.fdk_kv_evict(C.byref(e), None) == want, (sb, sh)
    # large strides, one axis alone
    assert lib.fdk_accumulate_weights(C.byref(_weights_args(weights_stride_b=4096, weights_stride_h=4096 * 31)), None) == _lib.FDK_ESHAPE
    assert lib.fdk_accumulate_weights(C.byref(_weights_args(weights_stride_b=4096, weights_stride_h=4096 * 32)), None) == 0
    assert lib.fdk_accumulate_weights(C.byref(_weights_args(batch=1, weights_stride_b=0)), None) == 0
    assert lib.fdk_accumulate_weights(C.byref(_weights_args(weights_stride_b=1 << 61, weights_stride_h=1 << 60)), None) == _lib.FDK_ESHAPE


def test_workspace_of_long_rows():
    """One plan entry a row; rows that few workgroups would have to themselves need room for counts and weights."""
    lib = _lib.load()
    of = lambda **kw: lib.fdk_kv_evict_workspace_bytes(C.byref(_evict_args(**kw)))
    assert of() == 32 * 8 * 16
    long = dict(batch=1, max_pages=4096, table_stride_b=4096, weights_len=65536, weights_stride_h=65536, weights_out_stride_h=65536)
    need = of(**long)
    assert need > 8 * 2048 * 4 and of(**dict(long, keep=4096)) == need + 8 * 2048 * 4
    assert lib.fdk_kv_evict(C.byref(_evict_args(**dict(long, workspace_bytes=need - 1))), None) == _lib.FDK_EWORKSPACE
    assert lib.fdk_kv_evict(C.byref(_evict_args(**dict(long, workspace_bytes=need))), None) == 0
    assert of(batch=0) == 0 and of(struct_size=4) == 0 and of(max_pages=1 << 30) == 0
    assert lib.fdk_kv_evict_workspace_bytes(None) == 0


def test_workspace_says_which_rows_are_shared_out():
    """Rows that one workgroup holds in registers, and rows of which there are enough for the compute units, stay one workgroup's."""
    lib = _lib.load()

    def shared(batch, length):
        a = _evict_args(batch=batch, max_pages=length // 16 + 1, table_stride_b=length // 16 + 1, weights_len=length)
        return lib.fdk_kv_evict_workspace_bytes(C.byref(a)) > batch * 8 * 16
    assert [shared(1, n) for n in (4097, 8192, 16384, 16385, 65536, 1 << 20)] == [False, False, False, True, True, True]
    assert [shared(b, 65536) for b in (8, 9, 16, 32, 200)] == [True, False, False, False, False]
    assert [shared(1, n) for n in (64 * 65471, 64 * 65471 + 1)] == [True, False]              # (counts of 16 bits)


def test_python_refusals():
    k = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    table, n, w = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(1, 2, 64)
    with pytest.raises(ValueError, match="live on the GPU"):
        tda.evict_kvcache(k, k, table, n, w, 10, 2)
    for kw, what in ((dict(keep=0), "keep"), (dict(keep=65), "keep"), (dict(recent=11), "recent"), (dict(weights=w[:, :1]), "weights"),
                     (dict(weights=w.double()), "weights"), (dict(value_cache=k[:2]), "caches"), (dict(kv_lens=n.long()), "kv_lens"),
                     (dict(block_table=table[0]), "block_table"), (dict(key_cache=k[0]), "caches")):
        args = dict(key_cache=k, value_cache=k, block_table=table, kv_lens=n, weights=w, keep=10, recent=2)
        args.update(kw)
        with pytest.raises(ValueError, match=what):
            tda.evict_kvcache(**args)
    q, lse = torch.zeros(1, 4, 64, dtype=torch.bfloat16), torch.zeros(1, 4)
    with pytest.raises(ValueError, match="live on the GPU"):
        tda.accumulate_attention_weights(q, k, table, n, lse, 0.1, w)
    for kw, what in ((dict(q=q[:, :3]), "multiple"), (dict(q=q[..., :32]), "q must"), (dict(lse=lse[:, :3]), "lse"), (dict(lse=lse.double()), "lse"),
                     (dict(weights=w[0]), "weights"), (dict(kv_lens=n[:0]), "kv_lens")):
        args = dict(q=q, k_cache=k, block_table=table, kv_lens=n, lse=lse, sm_scale=0.1, weights=w)
        args.update(kw)
        with pytest.raises(ValueError, match=what):
            tda.accumulate_attention_weights(**args)


def test_oracle_by_hand():
    w = torch.tensor([5.0, 1.0, 3.0, 3.0, 0.0, 3.0, 9.0])
    assert okv.survivors(w, 7, 7, 0) == list(range(7))
    assert okv.survivors(w, 7, 4, 1) == [0, 2, 3, 6]                   # 5, then the first two of the 3s, and the last token
    assert okv.survivors(w, 7, 3, 3) == [4, 5, 6]
    assert okv.survivors(torch.tensor([1.0, math.nan, 2.0, -math.inf]), 4, 2, 0) == [1, 2]
    assert okv.survivors(torch.tensor([-0.0, 0.0, 0.0]), 3, 1, 0) == [0]
    rows = torch.arange(8.0).view(4, 2, 1, 1)                          # pages of two tokens, one head
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)               # tokens 0..4 hold 4, 5, 0, 1, 6
    (moved,), lens, kept, out = okv.evict([rows], table, [5], torch.tensor([[[1.0, 4.0, 2.0, 8.0, 0.0]]]), 3, 1)
    assert kept.tolist() == [[[1, 3, 4]]] and lens.tolist() == [3] and out.tolist() == [[[4.0, 8.0, 0.0, 0.0, 0.0]]]
    assert moved.flatten().tolist() == [6.0, 1.0, 2.0, 3.0, 5.0, 1.0, 6.0, 7.0]

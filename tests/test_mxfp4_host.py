"""MXFP4 caches, without a GPU: what the entry points refuse, how calls are planned, and the oracle itself."""
import ctypes as C

import pytest
import torch

from oracle import mxfp4
from triton_distributed_amd import _lib
from triton_distributed_amd._lib import FdkDecodeArgs, FdkKvAppendArgs, FdkKvAppendAxesArgs, FdkMxfp4Args, FdkPlan
import triton_distributed_amd as tda


def _args(**kw):
    """A valid dry-run argument block on fake (never dereferenced) pointers: B32 32q/8kv P16 N4096, 4-bit cache."""
    a = FdkDecodeArgs()
    a.struct_size = C.sizeof(FdkDecodeArgs)
    a.flags = _lib.FDK_FLAG_DRY_RUN
    a.q, a.k_cache, a.v_cache = 0x10000, 0x20000, 0x30000
    a.block_table, a.kv_lens, a.out, a.lse = 0x40000, 0x50000, 0x60000, 0x70000
    a.q_dtype = a.out_dtype = _lib.FDK_BF16
    a.kv_dtype = _lib.FDK_MXFP4
    a.batch, a.num_q_heads, a.num_kv_heads, a.head_dim = 32, 32, 8, 128
    a.page_size, a.max_pages = 16, 256
    a.q_stride_b, a.q_stride_h = 32 * 128, 128
    a.k_stride_page, a.k_stride_tok, a.k_stride_head = 16 * 8 * 64, 8 * 64, 64
    a.v_stride_page, a.v_stride_tok, a.v_stride_head = 16 * 8 * 64, 8 * 64, 64
    a.k_block_scale, a.v_block_scale = 0x80004, 0x9000C
    a.kbs_stride_page, a.kbs_stride_tok, a.kbs_stride_head = 16 * 8 * 4, 8 * 4, 4
    a.vbs_stride_page, a.vbs_stride_tok, a.vbs_stride_head = 16 * 8 * 4, 8 * 4, 4
    a.table_stride_b = 256
    a.sm_scale = 0.088
    a.out_stride_b, a.out_stride_h, a.lse_stride_b = 32 * 128, 128, 32
    a.max_kv_len = a.min_kv_len = 4096
    a.workspace, a.workspace_bytes = 0xA0000, 1 << 40
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _rc(a):
    return _lib.load().fdk_decode(C.byref(a), None)


def test_valid_calls_pass_a_dry_run():
    assert _rc(_args()) == 0
    assert _rc(_args(q_dtype=_lib.FDK_FP16)) == 0
    for d in (64, 256):
        a = _args(head_dim=d, k_stride_head=d // 2, v_stride_head=d // 2, k_stride_tok=4 * d, v_stride_tok=4 * d,
                  k_stride_page=64 * d, v_stride_page=64 * d, kbs_stride_head=d // 32, vbs_stride_head=d // 32,
                  q_stride_h=d, q_stride_b=32 * d, out_stride_h=d, out_stride_b=32 * d)
        assert _rc(a) == 0, _lib.load().fdk_last_error()


@pytest.mark.parametrize("field,value,code", [
    ("k_block_scale", 0, _lib.FDK_ENULL), ("v_block_scale", 0, _lib.FDK_ENULL),
    ("algo", _lib.FDK_ALGO_VALU, _lib.FDK_EUNSUPPORTED),
    ("flags", _lib.FDK_FLAG_DRY_RUN | _lib.FDK_FLAG_SINGLE_LAUNCH, _lib.FDK_EUNSUPPORTED),
    ("head_dim", 192, _lib.FDK_EUNSUPPORTED), ("v_head_dim", 64, _lib.FDK_EUNSUPPORTED),
    ("q_dtype", _lib.FDK_MXFP4, _lib.FDK_EUNSUPPORTED), ("out_dtype", _lib.FDK_MXFP4, _lib.FDK_EUNSUPPORTED),
    ("k_stride_head", 32, _lib.FDK_ESHAPE), ("k_stride_tok", 8 * 64 + 8, _lib.FDK_EALIGN),
    ("kbs_stride_head", 3, _lib.FDK_ESHAPE), ("vbs_stride_tok", -1, _lib.FDK_ESHAPE),
    ("k_block_scale", 0x80002, _lib.FDK_EALIGN), ("v_block_scale", 0x90001, _lib.FDK_EALIGN), ("kbs_stride_tok", 34, _lib.FDK_EALIGN),
    ("kbs_stride_page", 1 << 32, _lib.FDK_ESHAPE), ("vbs_stride_tok", 1 << 62, _lib.FDK_ESHAPE),
])
def test_refusals(field, value, code):
    assert _rc(_args(**{field: value})) == code


def test_a_caller_of_the_previous_revision_is_asked_for_scales():
    a = _args(struct_size=FdkDecodeArgs.k_block_scale.offset)
    assert _rc(a) == _lib.FDK_ENULL
    a.kv_dtype = _lib.FDK_BF16
    for f in ("k_stride_head", "v_stride_head"):
        setattr(a, f, 128)
    assert _rc(a) == 0


def test_plans():
    """Two kv heads per workgroup where their rows share lines (heads side by side, rows below 128 bytes), unless the call is short
    and only one each fills the compute units; short batches are cut into chunks, long ragged ones into equal shares."""
    plan = FdkPlan()
    lib = _lib.load()

    def of(**kw):
        assert lib.fdk_plan(C.byref(_args(**kw)), 0, C.byref(plan)) == 0
        assert plan.algo == _lib.FDK_ALGO_MFMA and (not plan.balanced or plan.workgroups % (8 // plan.kv_heads_per_wg) == 0)
        return plan
    short = dict(max_pages=64, table_stride_b=64, max_kv_len=1024, min_kv_len=1024)
    assert (of(**short).num_splits, plan.kv_heads_per_wg, plan.balanced) == (1, 1, 0)
    long = dict(max_pages=512, table_stride_b=512, max_kv_len=8192, min_kv_len=8192)
    assert (of(**long).num_splits, plan.kv_heads_per_wg, plan.balanced) == (2, 2, 0)
    assert (of(batch=64).num_splits, plan.kv_heads_per_wg, plan.balanced) == (1, 2, 0)
    assert of(batch=48, **short).kv_heads_per_wg == 2                  # (384 single heads would fill 256 compute units unevenly)
    assert of(page_size=1, max_pages=4096, table_stride_b=4096, batch=64).kv_heads_per_wg == 2
    assert of(batch=64, num_kv_heads=3, num_q_heads=6).kv_heads_per_wg == 1
    by_head = dict(k_stride_head=16 * 64, k_stride_tok=64, v_stride_head=16 * 64, v_stride_tok=64)
    assert of(batch=64, **by_head).kv_heads_per_wg == 1
    assert (of(**by_head).num_splits, plan.kv_heads_per_wg) == (1, 1)
    wide = dict(head_dim=256, k_stride_head=128, v_stride_head=128, k_stride_tok=1024, v_stride_tok=1024)
    assert of(batch=64, **wide).kv_heads_per_wg == 1
    assert of(batch=64, num_kv_heads=1, num_q_heads=8).kv_heads_per_wg == 1
    for kw in (dict(batch=2), dict(batch=3, min_kv_len=0), dict(batch=40, min_kv_len=0, max_kv_len=0, max_pages=8192, table_stride_b=8192),
               dict(batch=4, max_pages=16384, table_stride_b=16384, max_kv_len=0, min_kv_len=0)):
        assert of(**kw).num_splits > 1


def _conv(**kw):
    a = FdkMxfp4Args()
    a.struct_size = C.sizeof(FdkMxfp4Args)
    a.flags = _lib.FDK_FLAG_DRY_RUN
    a.x, a.codes, a.scales = 0x10000, 0x20000, 0x30001
    a.x_stride, a.codes_stride, a.scales_stride = (C.c_int64 * 3)(0, 0, 128), (C.c_int64 * 3)(0, 0, 64), (C.c_int64 * 3)(0, 0, 4)
    a.n = (C.c_int32 * 3)(1, 1, 1000)
    a.num_values, a.x_dtype = 128, _lib.FDK_BF16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (dict(num_values=100), _lib.FDK_ESHAPE), (dict(num_values=0), _lib.FDK_ESHAPE), (dict(x_dtype=_lib.FDK_FP32), _lib.FDK_EUNSUPPORTED),
    (dict(x=0), _lib.FDK_ENULL), (dict(x=0x10008), _lib.FDK_EALIGN), (dict(codes=0x20002), _lib.FDK_EALIGN),
    (dict(x_stride=(C.c_int64 * 3)(0, 0, 132)), _lib.FDK_EALIGN), (dict(codes_stride=(C.c_int64 * 3)(0, 0, 66)), _lib.FDK_EALIGN),
    (dict(n=(C.c_int32 * 3)(1, -1, 1)), _lib.FDK_ESHAPE), (dict(n=(C.c_int32 * 3)(0, 1, 1), x=0), 0),
    (dict(n=(C.c_int32 * 3)(2 ** 31 - 1, 2 ** 31 - 1, 4)), _lib.FDK_ESHAPE), (dict(n=(C.c_int32 * 3)(2 ** 20, 2 ** 10, 4)), _lib.FDK_ESHAPE), (dict(struct_size=8), _lib.FDK_EABI),
])
def test_conversion_refusals(kw, code):
    lib = _lib.load()
    for fn in (lib.fdk_mx_quantize, lib.fdk_mx_dequantize):
        assert fn(C.byref(_conv(**kw)), None) == code


@pytest.mark.parametrize("name,row", [("codes_stride", 64), ("scales_stride", 4), ("x_stride", 128)])
@pytest.mark.parametrize("axis", [0, 1, 2])
def test_conversion_results_whose_rows_overlap(name, row, axis):
    """A row that is read may stand for many (stride 0); rows that are written have memory of their own."""
    lib = _lib.load()
    strides = dict(x_stride=[128] * 3, codes_stride=[64] * 3, scales_stride=[4] * 3)
    n = [1, 1, 1]
    n[axis] = 7
    for stride, apart in ((0, False), (row // 2, False), (row, True)):
        st = {k: list(v) for k, v in strides.items()}
        st[name][axis] = stride
        a = _conv(n=(C.c_int32 * 3)(*n), **{k: (C.c_int64 * 3)(*v) for k, v in st.items()})
        writes = lib.fdk_mx_dequantize if name == "x_stride" else lib.fdk_mx_quantize
        reads = lib.fdk_mx_quantize if name == "x_stride" else lib.fdk_mx_dequantize
        assert reads(C.byref(a), None) == 0
        assert writes(C.byref(a), None) == (0 if apart else _lib.FDK_ESHAPE)
        a.n[axis] = 1                                               # (one row: its stride is not used)
        assert writes(C.byref(a), None) == 0


def test_python_refusals():
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="live on the GPU"):
        tda.mxfp4_quantize(x)
    with pytest.raises(ValueError, match="bf16 / fp16"):
        tda.mxfp4_quantize(x.float())
    with pytest.raises(ValueError, match="multiple of 32"):
        tda.mxfp4_quantize(x[:, :48])
    with pytest.raises(ValueError, match="codes"):
        tda.mxfp4_quantize(x, torch.zeros(4, 32, dtype=torch.uint8))
    with pytest.raises(ValueError, match="scales"):
        tda.mxfp4_dequantize(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 3, dtype=torch.uint8))
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    cache, scale = torch.zeros(2, 16, 2, 64, dtype=torch.uint8), torch.zeros(2, 16, 2, 4, dtype=torch.uint8)
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="live on the GPU"):
        tda.flash_decode(q, cache, cache, table, n, 0.1, k_scale=scale, v_scale=scale)
    plan = tda.get_split_kv_plan(q, cache, cache, table, n, num_cus=256)
    assert plan.algo == "mfma"
    from triton_distributed_amd.flash_decode import _check_block_scales
    for bad in (None, scale[..., :3], scale.float(), scale[:1], scale.transpose(1, 3)):
        with pytest.raises(ValueError, match="k_scale"):
            _check_block_scales("k_scale", bad, cache)


def test_oracle_by_hand():
    """Codes and scales worked out by hand."""
    x = torch.zeros(1, 64, dtype=torch.bfloat16)
    x[0, :6] = torch.tensor([7.0, -6.5, 0.25, 0.75, 2.5, -1.0])              # amax 7: scale 1
    x[0, 32:36] = torch.tensor([7.0625, 1.0, -14.0, 5.0])                    # amax 14: scale 2
    codes, scales = mxfp4.quantize(x)
    assert scales.tolist() == [[127, 128]]
    assert codes[0, :3].tolist() == [7 | (15 << 4), 0 | (2 << 4), 4 | (10 << 4)]
    assert codes[0, 16:18].tolist() == [6 | (1 << 4), 15 | (4 << 4)]
    v = mxfp4.dequantize(codes, scales)
    assert v[0, :6].tolist() == [6.0, -6.0, 0.0, 1.0, 2.0, -1.0] and v[0, 32:36].tolist() == [8.0, 1.0, -12.0, 4.0]
    x[0, 3] = float("inf")
    assert mxfp4.quantize(x)[1].tolist() == [[255, 128]]
    assert mxfp4.quantize(torch.full((1, 32), 65504.0, dtype=torch.float16))[1].tolist() == [[127 + 13]]
    assert mxfp4.quantize(torch.zeros(1, 32, dtype=torch.float16))[1].tolist() == [[1]]


def _append_args(kw):
    """A valid dry-run fdk_kv_append block on fake pointers: B32, 1 new token, 32q/8kv, D128, P16, 4-bit cache, three axes."""
    a = FdkKvAppendArgs()
    a.struct_size = C.sizeof(FdkKvAppendArgs)
    a.flags = _lib.FDK_FLAG_DRY_RUN
    a.qkv, a.q_weight, a.k_weight, a.cos, a.sin = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000
    a.qkv_stride_b, a.qkv_stride_t, a.qkv_stride_h = 48 * 128, 48 * 128, 128
    a.qkv_dtype, a.kv_dtype = _lib.FDK_BF16, _lib.FDK_MXFP4
    a.q_eps = a.k_eps = 1e-6
    a.cs_stride_b, a.cs_stride_pos, a.max_positions = 0, 128, 8192
    a.batch, a.new_tokens, a.num_q_heads, a.num_kv_heads, a.head_dim = 32, 1, 32, 8, 128
    a.block_table, a.table_stride_b, a.kv_lens = 0x60000, 256, 0x70000
    a.page_size, a.max_pages, a.num_pages = 16, 256, 9000
    a.k_cache, a.v_cache = 0x80000, 0x90000
    a.k_stride_page = a.v_stride_page = 16 * 8 * 64
    a.k_stride_tok = a.v_stride_tok = 8 * 64
    a.k_stride_head = a.v_stride_head = 64
    a.q_out, a.q_out_stride_b, a.q_out_stride_t, a.q_out_stride_h = 0xA0000, 32 * 128, 32 * 128, 128
    x = FdkKvAppendAxesArgs()
    x.struct_size = C.sizeof(FdkKvAppendAxesArgs)
    x.append = C.addressof(a)
    x.k_block_scale, x.v_block_scale = 0xB0001, 0xC0001
    x.kbs_stride_page, x.kbs_stride_tok, x.kbs_stride_head = 16 * 8 * 4, 8 * 4, 4
    x.vbs_stride_page, x.vbs_stride_tok, x.vbs_stride_head = 16 * 8 * 4, 8 * 4, 4
    x.positions, x.pos_stride_axis, x.pos_stride_b, x.pos_stride_t = 0xD0000, 32, 1, 1
    x.num_axes, x.rope_sections = 3, (C.c_int32 * 4)(24, 20, 20, 0)
    for k, v in kw.items():
        setattr(x if hasattr(x, k) and k not in ("struct_size", "flags") else a, k, v)
    return a, x


def _append_rc(**kw):
    a, x = _append_args(kw)
    return _lib.load().fdk_kv_append_axes(C.byref(x), None)


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (dict(num_axes=0), _lib.FDK_ESHAPE), (dict(num_axes=5), _lib.FDK_ESHAPE), (dict(num_axes=2), _lib.FDK_ESHAPE),
    (dict(rope_sections=(C.c_int32 * 4)(64, 20, -20, 0)), _lib.FDK_ESHAPE), (dict(positions=0xD0002), _lib.FDK_EALIGN),
    (dict(positions=None), _lib.FDK_ENULL), (dict(positions=None, num_axes=0), 0),
    (dict(positions=None, num_axes=0, rope_interleaved=1), _lib.FDK_ENULL),
    (dict(k_block_scale=None), _lib.FDK_ENULL), (dict(kbs_stride_head=3), _lib.FDK_ESHAPE), (dict(v_stride_head=63), _lib.FDK_ESHAPE),
    (dict(k_cache=0x80001), _lib.FDK_EALIGN), (dict(v_stride_tok=8 * 64 + 1), _lib.FDK_EALIGN),
    (dict(kv_dtype=_lib.FDK_BF16, k_stride_head=128, v_stride_head=128), 0),
    (dict(kv_dtype=_lib.FDK_FP16), _lib.FDK_EUNSUPPORTED),
])
def test_append_refusals(kw, code):
    assert _append_rc(**kw) == code


def test_append_blocks():
    """The block of fdk_kv_append alone knows no 4-bit rows; the block around it is checked like the others."""
    lib = _lib.load()
    a, x = _append_args({})
    assert lib.fdk_kv_append(C.byref(a), None) == _lib.FDK_EUNSUPPORTED
    assert lib.fdk_kv_append_axes(None, None) == _lib.FDK_ENULL
    x.struct_size -= 8
    assert lib.fdk_kv_append_axes(C.byref(x), None) == _lib.FDK_EABI
    x.struct_size += 8
    a.struct_size -= 8
    assert lib.fdk_kv_append_axes(C.byref(x), None) == _lib.FDK_EABI
    x.append = None
    assert lib.fdk_kv_append_axes(C.byref(x), None) == _lib.FDK_ENULL
    # neither positions nor 4-bit rows: the plain append
    a, x = _append_args(dict(positions=None, num_axes=0, kv_dtype=_lib.FDK_BF16, k_stride_head=128, v_stride_head=128,
                             k_block_scale=None))
    assert lib.fdk_kv_append_axes(C.byref(x), None) == 0


def test_entry_points_without_block_scales_say_so():
    """The drop-ins for the reference's functions, and the layer over them, cannot be given the scales of a 4-bit cache."""
    from triton_distributed_amd.sp_flash_decode_layer import SpGQAFlashDecodeAttention
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    layer = SpGQAFlashDecodeAttention(0, 0, 1, 1, 4, 2, 128, 128)
    for cache in (torch.zeros(2, 16, 2, 64, dtype=torch.uint8), torch.zeros(2, 16, 2, 64, dtype=torch.uint8).view(torch.float4_e2m1fn_x2)):
        for fn in (tda.gqa_fwd_batch_decode, tda.gqa_fwd_batch_decode_intra_rank, tda.gqa_fwd_batch_decode_persistent):
            with pytest.raises(ValueError, match=f"{fn.__name__} takes no block scales"):
                fn(q, cache, cache, None, [1], n, table, 0.1)
            with pytest.raises(ValueError, match="flash_decode"):
                getattr(tda, fn.__name__ + "_aot")(None, q, cache, cache, None, [1], n, table, 0.1)
        with pytest.raises(ValueError, match="flash_decode_bsnh takes no block scales"):
            tda.flash_decode_bsnh(q[:, None], cache, cache, table, n)
        with pytest.raises(ValueError, match="takes no block scales"):
            layer(q, cache, cache, n[None], table)

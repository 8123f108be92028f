"""How exact the probabilities of a decode over an MXFP4 cache are: with V rows of one 1 each, a value of the result is a sum of
probabilities, and the one rounding to 16 bits that the result itself needs is all that may be seen in it."""
import pytest
import torch

from oracle import mxfp4
from tests.mxfp4_cases import make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hkv,page,layout", [(64, 2, 16, "token"), (64, 1, 5, "token"), (128, 2, 16, "token"), (128, 2, 5, "token"),
                                               (128, 2, 16, "head"), (256, 2, 32, "token")])
@pytest.mark.parametrize("group", [3, 8, 12])
@pytest.mark.parametrize("kw", [{}, dict(kv_split=1), dict(force_balanced=True)])
def test_the_result_is_rounded_once(cuda_device, dtype, d, hkv, page, layout, group, kw):
    import triton_distributed_amd as tda
    lens, hq, sm_scale = [d, 700, 37], group * hkv, 0.002
    (kc, ks, k64, vc, vs, _), table = make_cache(lens, page, hkv, d, dtype, 77, layout)
    v = torch.zeros(vc.shape[:3] + (d,), dtype=dtype)
    for i, n in enumerate(lens):
        pos = torch.arange(n)
        v[table[i, pos // page].long(), pos % page, :, pos % d] = 1                  # token n: a 1 at value n mod D
    held = ~k64[..., 0, 0].isnan()
    codes, scales = mxfp4.quantize(v)
    scales[~held] = 255
    vc.copy_(codes), vs.copy_(scales)
    v64 = mxfp4.dequantize(vc, vs)
    assert torch.equal(v64[held], v.double()[held])
    q = torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(5)).to(dtype)
    dev = lambda t: t.to(cuda_device)
    out, _ = tda.flash_decode(dev(q), dev(kc), dev(vc), dev(table), torch.tensor(lens, dtype=torch.int32, device=cuda_device), sm_scale,
                              k_scale=dev(ks), v_scale=dev(vs), **kw)
    o64, _, _ = mxfp4.decode(q, k64, v64, table, lens, sm_scale)
    # A logit is a sum of D products in fp32: off by at most e = (D + 8) 2^-24 sum |q k| sm_scale, a probability by 2 e of itself;
    # fp32 sums over the tokens n 2^-24; exponentials, reciprocal, scaling of the parts 2^-18; 16-bit parts of a probability whose
    # rest is below 2^-16 of it.  Then the result's own rounding, half a step.
    size = max(float(torch.einsum("hgd,nhd->hgn", q[i].double().abs().unflatten(0, (hkv, -1)),
                                  k64[table[i, torch.arange(n) // page].long(), torch.arange(n) % page].abs()).max()) for i, n in enumerate(lens))
    e = (d + 8) * 2.0 ** -24 * size * sm_scale
    step = 2.0 ** torch.floor(torch.log2(o64.clamp_min(2.0 ** -60))) * torch.finfo(dtype).eps
    tol = step.clamp_min(torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps) / 2 + o64 * (2 * e + max(lens) * 2.0 ** -24 + 2.0 ** -16 + 2.0 ** -18)
    off = (out.cpu().double() - o64).abs()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()} values off by up to {float((off / step).max()):.3f} steps"

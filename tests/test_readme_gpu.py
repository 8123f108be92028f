"""The README's lines for a cache in 4 bits, run as they stand there."""
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_lines_for_a_cache_in_4_bits(cuda_device):
    import triton_distributed_amd as tda
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")) as f:
        code = next(block for block in f.read().split("```") if block.startswith("python") and "evict_kvcache" in block)
    dev, b, hkv, length = cuda_device, 2, 2, 2060
    pages = (length + 15) // 16
    pool = lambda n: torch.zeros(b * pages, 16, hkv, n, dtype=torch.uint8, device=dev)
    angles = torch.rand(length, 64, device=dev)
    ones = torch.ones(128, dtype=torch.bfloat16, device=dev)
    names = dict(tda=tda, torch=torch, rows=torch.randn(4, 128, device=dev).bfloat16(), k=pool(64), v=pool(64), ks=pool(4), vs=pool(4),
                 table=torch.arange(b * pages, dtype=torch.int32, device=dev).view(b, pages),
                 kv_lens=torch.full((b,), length, dtype=torch.int32, device=dev), wq=ones, wk=ones,
                 cos=torch.cat((angles, angles), -1).cos(), sin=torch.cat((angles, angles), -1).sin(),
                 qkv=torch.randn(b, 1, 8 + 2 * hkv, 128, device=dev).bfloat16(),
                 pos=torch.randint(0, length, (3, b, 1), dtype=torch.int32, device=dev), sm_scale=128 ** -0.5,
                 weights=torch.zeros(b, hkv, length, device=dev))
    exec(code[len("python"):], names)
    torch.cuda.synchronize()
    assert names["lens"].tolist() == [2048] * b and tuple(names["kept"].shape) == (b, hkv, 2048)
    assert torch.isfinite(names["out"].float()).all() and torch.isfinite(names["lse"]).all()
    # (every q head's weights add up to 1 over the tokens; what the twelve that left had is gone)
    assert (names["weights"].sum(-1) <= 4 + 1e-3).all() and (names["weights"][..., :2048] >= 0).all()

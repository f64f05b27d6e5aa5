"""`block_append` against the framework's other writer of the same pools, byte by byte."""
import pytest
import torch

from inference_optimizations_b200.ops import block_sparse as S
from inference_optimizations_b200.ops import kvcache as K

pytestmark = pytest.mark.gpu

FMTS = {"bf16": K.FMT_BF16, "fp8": K.FMT_FP8, "nvfp4": K.FMT_NVFP4}


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("d", [128, 256, 512])
@pytest.mark.parametrize("ks,vs", [(1.0, 1.0), (0.75, 1.25), (0.0371, 3.3), (0.875, 7.0), (2.0 ** 100, 2.0 ** -100)])
@pytest.mark.parametrize("t", [5, 700])
def test_append_writes_the_bytes_of_the_other_writer(cuda, fmt, d, ks, vs, t):
    """V always (it is bf16 on both sides); K without norm and at rotation angle 0, where every key is a bf16 value."""
    fmt = FMTS[fmt]
    hq, hk = 4, 2
    g = torch.Generator().manual_seed(d + t)
    qkv = torch.randn(t, (hq + 2 * hk) * d, generator=g).to(torch.bfloat16).to(cuda)
    pos = torch.arange(t, dtype=torch.int32, device=cuda)
    cs = torch.cat([torch.ones(t, d // 2), torch.zeros(t, d // 2)], 1).to(cuda)
    pages = (t + 63) // 64 + 1
    p1 = torch.zeros(pages, hk, 2, K.part_bytes(fmt, d), dtype=torch.uint8, device=cuda)
    p2 = p1.clone()
    S.block_append(qkv, None, None, cs, pos, pos + 64, p1, *S.alloc_bounds(pages, hk, d, cuda), fmt, hq, hk, d, 1e-6, True,
                   ks, vs)
    K.gqa_prep(qkv, None, None, cs, pos, pos + 64, p2, fmt, hq, hk, d, 1e-6, True, ks, vs)
    assert torch.equal(p1, p2)


@pytest.mark.parametrize("fmt", ["fp8", "nvfp4"])
@pytest.mark.parametrize("d", [128, 512])
@pytest.mark.parametrize("vs", [1.0, 0.875, 1e-30])
def test_values_that_are_not_finite(cuda, fmt, d, vs):
    """Infinite and NaN V, and V that overflows in units of the scale, give the other writer's bytes."""
    fmt = FMTS[fmt]
    qkv = torch.randn(64, 4 * d, generator=torch.Generator().manual_seed(d)).to(torch.bfloat16)
    qkv[3, 3 * d + 5], qkv[4, 3 * d + 40], qkv[5, 4 * d - 1], qkv[6, 3 * d + 17] = \
        float("inf"), -float("inf"), float("nan"), 3e38
    qkv = qkv.to(cuda)
    pos = torch.arange(64, dtype=torch.int32, device=cuda)
    cs = torch.cat([torch.ones(64, d // 2), torch.zeros(64, d // 2)], 1).to(cuda)
    p1 = torch.zeros(1, 1, 2, K.part_bytes(fmt, d), dtype=torch.uint8, device=cuda)
    p2 = p1.clone()
    S.block_append(qkv, None, None, cs, pos, pos, p1, *S.alloc_bounds(1, 1, d, cuda), fmt, 2, 1, d, 1e-6, True, 1.0, vs)
    K.gqa_prep(qkv, None, None, cs, pos, pos, p2, fmt, 2, 1, d, 1e-6, True, 1.0, vs)
    assert torch.equal(p1[:, :, 1], p2[:, :, 1])

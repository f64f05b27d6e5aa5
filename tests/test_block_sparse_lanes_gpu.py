"""Block-sparse attention on SM partitions of the GPU: clusters on a lane of 8 SMs, the engine's prefill / decode lanes."""
import pytest
import torch

from inference_optimizations_b200.engine.pdmux import Lanes, PdmuxEngine
from inference_optimizations_b200.ops import block_sparse as S
from inference_optimizations_b200.ops import kvcache as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,d,n_q", [(K.FMT_BF16, 512, 1), (K.FMT_BF16, 128, 4), (K.FMT_NVFP4, 512, 4)])
def test_one_list_on_eight_sms(cuda, fmt, d, n_q):
    """One list wants a cluster of 8; at head_dim 512 over a bf16 cache each of its CTAs takes an SM."""
    total = torch.cuda.get_device_properties(0).multi_processor_count
    lanes = Lanes("cuda:0", 3, [(total, 0), (total - 8, 8), (0, total)])
    streams = lanes.streams(1)
    assert lanes.sms[1][1] == 8
    pages = 40
    g = torch.Generator().manual_seed(d + n_q)
    pool = torch.randint(0, 256, (pages + 1, 1, 2, K.part_bytes(fmt, d)), generator=g, dtype=torch.uint8)
    if fmt == K.FMT_BF16:
        pool.view(torch.bfloat16).copy_(torch.randn(pages + 1, 1, 2, 64 * d, generator=g))
    else:
        pool[..., 32 * d:] &= 0x0F
        pool[..., 32 * d:] |= 0x28
    pool = pool.to(cuda)
    codes, scale = S.alloc_bounds(pages + 1, 1, d, cuda)
    S.block_summarize(pool, torch.arange(pages + 1, dtype=torch.int32, device=cuda), codes, scale, fmt, 1, d)
    table = (torch.randperm(pages, generator=g) + 1)[None].int().to(cuda)
    kv = torch.tensor([pages * 64 - 3], dtype=torch.int32, device=cuda)
    q = torch.randn(n_q, 2, d, generator=g).to(torch.bfloat16).to(cuda)
    all_pages = torch.arange(pages, dtype=torch.int32, device=cuda).view(1, 1, pages)

    def step():
        blocks, count = S.block_select(q, codes, scale, table, kv, n_q, 1, 9)
        return (blocks, count, *S.block_decode(q, pool, table, kv, all_pages, n_q, 1, fmt, d ** -0.5))
    want = step()
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            got = step()
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kv", ["nvfp4", "bf16"])
def test_engine_lanes_with_selected_pages(cuda, kv):
    from inference_optimizations_b200.config import EngineConfig
    from inference_optimizations_b200.engine.engine import Engine
    from inference_optimizations_b200.engine.scheduler import SamplingParams
    prompts = [list(range(3, 160)), list(range(7, 16)), list(range(100, 490)), list(range(1, 33))]
    params = SamplingParams(max_new_tokens=8, ignore_eos=True)
    ecfg = EngineConfig(model="tiny_gqa", device="cuda:0", kv_dtype=kv, max_running=4, chunked_prefill=128, sparse_pages=4)
    ref = Engine(ecfg, max_seq=1024).generate(prompts, params)
    pm = PdmuxEngine(Engine(ecfg, max_seq=1024), token_budget=256)
    assert pm.generate(prompts, params) == ref
    assert any(g == 1 and s is not None and n > 0 for g, s, n in pm.log)
    kvc = pm.engine.runner.kv
    assert kvc.sparse_status.item() == 0 and kvc.alloc["global"].used == 0

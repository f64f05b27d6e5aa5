"""Speculation with a small budget of pages on the GPU: graphs, bounds after accepted and rejected drafts (of finished
pages: an unfinished one's are not used, and may be those of a rejected token that reached the page's end)."""
import pytest
import torch

from inference_optimizations_b200.config import EngineConfig
from inference_optimizations_b200.engine.engine import Engine
from inference_optimizations_b200.engine.scheduler import SamplingParams
from inference_optimizations_b200.ops import block_sparse as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["bf16", "fp8", "nvfp4"])
def test_speculation_keeps_the_bounds_of_what_the_pages_hold(cuda, kv):
    prompts = [[(13 * i + 7 * j) % 500 + 1 for j in range(n)] for i, n in enumerate((700, 30, 381))]
    params = SamplingParams(max_new_tokens=150, ignore_eos=True)

    def engine():
        return Engine(EngineConfig(model="tiny_gqa", device="cuda:0", kv_dtype=kv, max_running=4, chunked_prefill=128,
                                   graph_batch_sizes="1,2,4", spec=True, spec_policy="always", sparse_pages=4),
                      max_seq=1024)
    plain = engine().generate(prompts, params)
    eng = engine()
    run, at = eng.runner, {}

    def script(r, length):                                  # right drafts, then one wrong token after 0 .. 3 of them
        known = plain[at.setdefault(r.rid, len(at))]
        done = length - r.prompt_len + 1
        return [(known[done + k] if done + k < len(known) and k < length % 4 else 499, True) for k in range(3)]
    run.draft_script = script
    reqs = [eng.add_request(p, params) for p in prompts]
    steps, pages = 0, 0
    while eng.has_work():
        eng.step()
        steps += 1
        if steps % 10 or not eng.sched.running:
            continue
        full = [run.pages[r.rid]["global"].pages[j] for r in eng.sched.running for j in range(r.kv_len // 64)]
        ids = torch.tensor(full, dtype=torch.int32, device=cuda)
        pages += len(full)
        for pool, b in zip(run.kv.pools, run.kv.bounds):
            if b is not None:
                c, s = b[0].clone(), b[1].clone()
                S.block_summarize(pool, ids, c, s, run.kv.fmt, c.shape[1], c.shape[3], run.kv.k_scale)
                assert torch.equal(c, b[0]) and torch.equal(s, b[1])
    assert all(len(r.output) == 150 for r in reqs)
    taken, steps = sum(r.accepted for r in reqs), sum(r.spec_steps for r in reqs)
    assert 0.1 * 3 * steps < taken < 0.95 * 3 * steps       # accepted and rejected drafts both
    assert pages >= 100
    assert run.kv.sparse_status.item() == 0

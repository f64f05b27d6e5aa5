"""Block-sparse decode in the GQA engine beyond single tokens on one rank: speculation with a small budget, tensor
parallelism."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from inference_optimizations_b200.config import EngineConfig
from inference_optimizations_b200.engine.engine import Engine
from inference_optimizations_b200.engine.scheduler import SamplingParams
from inference_optimizations_b200.ops import block_sparse as S

PROMPTS = [[(13 * i + 7 * j) % 500 + 1 for j in range(n)] for i, n in enumerate((250, 30, 381))]


def _engine(tp=1, rank=0, **kw):
    from inference_optimizations_b200.parallel import dist as D
    ecfg = EngineConfig(**{**dict(model="tiny_gqa", device="cpu", kv_dtype="bf16", max_running=4, chunked_prefill=100,
                                  cuda_graphs=False, sparse_pages=3, tp=tp), **kw})
    return Engine(ecfg, max_seq=512, tp_rank=rank, tp=tp, all_reduce=D.host_all_reduce if tp > 1 else None,
                  argmax_merge=D.argmax_merge if tp > 1 else None)


@pytest.mark.parametrize("kv", ["bf16", "nvfp4"])
def test_verify_ranks_pages_by_the_bounds_of_what_they_hold(kv, monkeypatch):
    """Drafts of which none, some and all are accepted, over several page ends: whenever a list is made, the bounds of
    the pages before the group's first token are those of the keys stored there."""
    eng = _engine(spec=True, kv_dtype=kv)
    run, real, lists = eng.runner, S.block_select, [0, 0]

    def spy(q, codes, scale, table, kv_len, n_q, hk, budget, sink=1, local=1, req_idx=None, out=None):
        layer = next(i for i, b in enumerate(run.kv.bounds) if b is not None and b[0] is codes)
        for b, n in enumerate(kv_len.tolist()):
            done = max(0, n - n_q) // 64
            last = table[int(req_idx[b]), max(0, done - 2):done].contiguous()       # (older ones were last once)
            c, s = codes.clone(), scale.clone()
            S.block_summarize(run.kv.pools[layer], last, c, s, run.kv.fmt, hk, codes.shape[3], run.kv.k_scale)
            assert torch.equal(c, codes) and torch.equal(s, scale)
            lists[0] += done > budget
            lists[1] += n_q == 4
        return real(q, codes, scale, table, kv_len, n_q, hk, budget, sink, local, req_idx, out)
    plain = _engine(spec=True, kv_dtype=kv).generate(PROMPTS, SamplingParams(max_new_tokens=70))
    monkeypatch.setattr(S, "block_select", spy)
    at = {}

    def script(r, length):                                  # right drafts, then one wrong token after 0 .. 3 of them
        known = plain[at.setdefault(r.rid, len(at))]
        done = length - r.prompt_len + 1
        return [(known[done + k] if done + k < len(known) and k < length % 4 else 499, True) for k in range(3)]
    run.draft_script = script
    reqs = [eng.add_request(p, SamplingParams(max_new_tokens=70)) for p in PROMPTS]
    while eng.has_work():
        eng.step()
    assert all(len(r.output) == 70 for r in reqs)
    taken, steps = sum(r.accepted for r in reqs), sum(r.spec_steps for r in reqs)
    assert 0.2 * 3 * steps < taken < 0.9 * 3 * steps        # accepted and rejected drafts both
    assert lists[0] > 20 and lists[1] > 20


def _worker(rank, port, q):
    torch.set_num_threads(2)                                # (two ranks share the cores)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2")
    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        res = {}
        for pages in (8, 3):
            eng = _engine(2, rank, sparse_pages=pages)
            outs = eng.generate(PROMPTS, SamplingParams(max_new_tokens=6))
            kv = eng.runner.kv
            before = [(c.clone(), s.clone()) for c, s in (b for b in kv.bounds if b is not None)]
            kv.summarize()
            same = all(torch.equal(c[d], c2[d]) and torch.equal(s[d], s2[d]) and int(d.sum()) >= 8
                       for (c, s), (c2, s2) in zip(before, (b for b in kv.bounds if b is not None))
                       for d in [s.ne(0).all(1)])
            res[pages] = outs, same, kv.bounds[next(i for i, b in enumerate(kv.bounds) if b is not None)][0].shape[1]
        q.put((rank, res))
        dist.barrier()
    finally:
        dist.destroy_process_group()


def test_two_ranks():
    """Each rank keeps the bounds of its own kv heads and both give the same tokens; with room for every page the tokens
    are the cache-free forward's wherever that is no tie (sums over ranks round differently)."""
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    procs = [ctx.Process(target=_worker, args=(r, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = dict(q.get(timeout=600) for _ in procs)
    for p in procs:
        p.join(timeout=120)
    one = _engine()
    heads = one.cfg.num_kv_heads_global
    for pages in (8, 3):
        (o0, same0, h0), (o1, same1, h1) = res[0][pages], res[1][pages]
        assert o0 == o1 and all(len(o) == 6 for o in o0) and same0 and same1 and h0 == h1 == heads // 2
    checked = 0
    for p, o in zip(PROMPTS, res[0][8][0]):
        for i, tok in enumerate(o):
            ref = one.runner.model.reference_logits(p + o[:i])[-1]
            top = torch.topk(ref, 2).values
            if (top[0] - top[1]).item() > 0.05:
                assert tok == int(ref.argmax())
                checked += 1
    assert checked >= 6


def test_a_captured_step_keeps_the_tensors_that_it_reads(monkeypatch):
    """A graph holds addresses: what a step body made before its capture must not be freed while the graph can replay."""
    import contextlib
    import gc
    import weakref
    fake = type("Fake", (), {"wait_stream": lambda *a: None, "replay": lambda *a: None})
    monkeypatch.setattr(torch.cuda, "Stream", lambda *a, **k: fake())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a, **k: fake())
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "graph", lambda g, pool=None: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "CUDAGraph", fake)
    monkeypatch.setattr(torch.cuda, "graph_pool_handle", lambda: 0)
    run = _engine().runner
    rows = torch.arange(4)
    ran = []

    def body(rows=rows):
        ran.append(rows.sum().item())
    left = weakref.ref(rows)
    step = run._capture(body)
    del rows, body
    gc.collect()
    assert left() is not None and ran == [6, 6]
    step()
    del step
    gc.collect()
    assert left() is None

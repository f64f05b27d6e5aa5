"""Block-sparse attention oracles: the bounds hold, the selection follows its rules, full lists are dense attention,
refusals."""
import math

import pytest
import torch

from inference_optimizations_b200.ops import attention as A
from inference_optimizations_b200.ops import block_sparse as S
from inference_optimizations_b200.ops import kvcache as K
from inference_optimizations_b200.ops.basic import rope_table

FMTS = (K.FMT_BF16, K.FMT_FP8, K.FMT_NVFP4)


def session(fmt, n, d=128, hq=4, hk=2, seed=0, step=None, ks=0.5, vs=0.5):
    """A request of n tokens appended `step` rows at a time: (last q, pool, table, codes, scale)."""
    g = torch.Generator().manual_seed(seed)
    if fmt == K.FMT_BF16:
        ks = vs = 1.0
    npg = (n + 63) // 64
    pool = torch.zeros(npg + 1, hk, 2, K.part_bytes(fmt, d), dtype=torch.uint8)
    codes, sc = S.alloc_bounds(npg + 1, hk, d, "cpu")
    table = (torch.randperm(npg, generator=g) + 1)[None].int()
    qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g).to(torch.bfloat16)
    cs = rope_table(n + 64, d, 10000.0)
    qs = []
    for lo in range(0, n, step or n):
        pos = torch.arange(lo, min(n, lo + (step or n)), dtype=torch.int32)
        slot = (table[0, (pos // 64).long()] * 64 + pos % 64).int()
        qs.append(S.block_append(qkv[pos.long()], None, None, cs, pos, slot, pool, codes, sc, fmt, hq, hk, d, 1e-6,
                                 True, ks, vs))
    return torch.cat(qs), pool, table, codes, sc, ks, vs


@pytest.mark.parametrize("fmt", FMTS)
def test_append_writes_what_the_existing_writer_writes(fmt):
    """Without norm and at rotation angle 0 every key is a bf16 value, and the bytes of both writers are the same
    (elsewhere `gqa_prep` rounds the rotated key to bf16 before it encodes it, `block_append` does not)."""
    d, hq, hk, n = 128, 4, 2, 150
    ks, vs = (1.0, 1.0) if fmt == K.FMT_BF16 else (0.5, 0.5)
    qkv = torch.randn(n, (hq + 2 * hk) * d, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    pos = torch.arange(n, dtype=torch.int32)
    cs = torch.cat([torch.ones(n, d // 2), torch.zeros(n, d // 2)], 1)
    p1 = torch.zeros(4, hk, 2, K.part_bytes(fmt, d), dtype=torch.uint8)
    p2 = p1.clone()
    q1 = S.block_append(qkv, None, None, cs, pos, pos + 64, p1, *S.alloc_bounds(4, hk, d, "cpu"), fmt, hq, hk, d, 1e-6,
                        True, ks, vs)
    q2 = K.gqa_prep(qkv, None, None, cs, pos, pos + 64, p2, fmt, hq, hk, d, 1e-6, True, ks, vs)
    assert torch.equal(p1, p2) and torch.equal(q1, q2)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("step", [1, 7, 64, 100])
def test_bounds_do_not_depend_on_the_calls(fmt, step):
    a, b = session(fmt, 200), session(fmt, 200, step=step)
    for x, y in zip(a[:5], b[:5]):
        assert torch.equal(x, y)
    assert (a[4][a[2][0, :3].long()] > 0).all() and not a[4][a[2][0, 3].long()].any()


@pytest.mark.parametrize("fmt", FMTS)
def test_scores_bound_every_key_of_the_page(fmt):
    d, hk = 128, 2
    q, pool, table, codes, sc, ks, vs = session(fmt, 320)
    keys, _ = K.gqa_pool_read_ref(pool, table[0], 320, fmt, d, ks, vs)
    rows = q[-1].float()
    for j in range(5):
        p = int(table[0, j])
        for h in range(hk):
            c = codes[p, h].double() * float(sc[p, h])
            for r in rows[2 * h:2 * h + 2].double():
                top = (keys[64 * j:64 * j + 64, h].double() @ r).max()
                # a code is at most half a step off (one step where it was clamped)
                assert (r * c[0] + r.abs() * c[1]).sum() + r.abs().sum() * 2 * float(sc[p, h]) >= top


def test_select_rules():
    d, hk, hq = 128, 1, 1
    q, pool, table, codes, sc, *_ = session(K.FMT_BF16, 64 * 20 + 10, hq=hq, hk=hk)
    kv = torch.tensor([64 * 20 + 10], dtype=torch.int32)
    phys = table[0].long()
    scores = torch.stack([(q[-1, 0].float() * codes[p, 0, 0] + q[-1, 0].float().abs() * codes[p, 0, 1]).sum() * sc[p, 0]
                          for p in phys])
    for budget, sink, local in ((3, 1, 1), (8, 0, 2), (10, 3, 1), (21, 1, 1), (64, 1, 1)):
        blocks, count = S.block_select(q[-1:], codes, sc, table, kv, 1, hk, budget, sink, local)
        got = [x for x in blocks[0, 0].tolist() if x >= 0]
        assert len(got) == count.item() == min(21, budget) and got == sorted(got)
        assert set(range(sink)) <= set(got) and set(range(21 - local, 21)) <= set(got)
        rest = [x for x in range(sink, 21 - local) if x not in got]
        mid = [x for x in got if sink <= x < 21 - local]
        if rest and mid:                                  # (codes of q round by up to 2^-7 of a step each)
            assert min(scores[mid]) >= max(scores[rest]) * 0.97
    # a verify group whose tokens straddle two pages keeps both
    q4 = q[-14:-10].contiguous()
    blocks, _ = S.block_select(q4, codes, sc, table, torch.tensor([64 * 20 + 2], dtype=torch.int32), 4, hk, 3)
    assert blocks[0, 0].tolist() == [0, 19, 20]
    empty, count = S.block_select(q[-1:], codes, sc, table, torch.tensor([0], dtype=torch.int32), 1, hk, 4)
    assert count.item() == 0 and (empty == -1).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_full_lists_are_dense_attention(fmt):
    q, pool, table, codes, sc, ks, vs = session(fmt, 200)
    kv = torch.tensor([200], dtype=torch.int32)
    for n_q in (1, 4):
        blocks, _ = S.block_select(q[-n_q:], codes, sc, table, kv, n_q, 2, 4)
        out, lse = S.block_decode(q[-n_q:], pool, table, kv, blocks, n_q, 2, fmt, 0.1, ks, vs)
        want = A.gqa_decode_ref(q[-n_q:], pool, table, kv, n_q, 2, fmt, 0.1, 0, ks, vs)
        assert (out.float() - want).abs().max() <= want.abs().max() * 2 ** -8 + 1e-6
        assert torch.isfinite(lse).all()


def test_empty_groups_and_garbage_past_the_end():
    q, pool, table, codes, sc, ks, vs = session(K.FMT_BF16, 70)
    pool.view(torch.bfloat16).view(-1, 2, 2, 64, 128)[int(table[0, 1]), :, :, 6:] = math.nan
    kv = torch.tensor([70, 0], dtype=torch.int32)
    blocks = torch.full((2, 2, 3), -1, dtype=torch.int32)
    blocks[0, :, 1:] = torch.tensor([1, 0])
    out, lse = S.block_decode(torch.cat([q[-1:], q[:1]]), pool, table.repeat(2, 1), kv, blocks, 1, 2, 0, 0.1)
    assert torch.isfinite(out).all() and not out[1].any()
    assert torch.isfinite(lse[0]).all() and (lse[1] == -math.inf).all()


def test_refusals():
    q, pool, table, codes, sc, *_ = session(K.FMT_BF16, 70)
    kv = torch.tensor([70], dtype=torch.int32)
    for kw in (dict(budget=2), dict(budget=4, sink=-1), dict(budget=4, local=0), dict(budget=S.MAX_LIST + 1)):
        with pytest.raises(RuntimeError):
            S.block_select(q[-1:], codes, sc, table, kv, 1, 2, **kw)
    with pytest.raises(RuntimeError):
        S.block_select(q[-9:], codes, sc, table, kv, 9, 2, 4)              # 18 rows
    with pytest.raises(RuntimeError):
        S.block_decode(q[-1:], pool, table, kv, torch.zeros(1, 3, 4, dtype=torch.int32), 1, 2, 0, 0.1)
    with pytest.raises(RuntimeError):
        S.block_decode(q[-1:], pool, table, kv, torch.zeros(1, 2, 4, dtype=torch.int32), 1, 2, 1, 0.1)
    with pytest.raises(RuntimeError):
        S.block_summarize(pool, torch.tensor([1]), codes[:1], sc, 0, 2, 128)
    for kw in (dict(sm_scale=0.0), dict(sm_scale=-0.1), dict(sm_scale=float("nan"))):
        with pytest.raises(RuntimeError):
            S.block_decode(q[-1:], pool, table, kv, torch.zeros(1, 2, 4, dtype=torch.int32), 1, 2, 0, **kw)
    q, pool, table, codes, sc, *_ = session(K.FMT_FP8, 70)
    with pytest.raises(RuntimeError):
        S.block_decode(q[-1:], pool, table, kv, torch.zeros(1, 2, 4, dtype=torch.int32), 1, 2, 1, 0.1, k_scale=0.0)
    with pytest.raises(RuntimeError):
        S.block_summarize(pool, torch.tensor([1]), codes, sc, 1, 2, 128, k_scale=-1.0)
    with pytest.raises(RuntimeError):
        S.block_append(torch.zeros(1, 8 * 128, dtype=torch.bfloat16), None, None, rope_table(4, 128, 1e4),
                       torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), pool, codes, sc, 1, 4, 2,
                       128, 1e-6, True, 1.0, 0.0)



def test_selection_over_bounds_of_no_page_is_refused():
    q, pool, table, codes, sc, *_ = session(K.FMT_BF16, 64 * 9)
    for n in (64 * 9, 64):                                  # with candidates to score and without
        with pytest.raises(RuntimeError, match="at least one page"):
            S.block_select(q[-1:], codes[:0], sc[:0], table, torch.tensor([n], dtype=torch.int32), 1, 2, 3)


# ------------------------------------------------------------------------------------------------ engine
def _engine(**kw):
    from inference_optimizations_b200.config import EngineConfig
    from inference_optimizations_b200.engine.engine import Engine
    kw = {**dict(model="tiny_gqa", device="cpu", kv_dtype="bf16", max_running=4, chunked_prefill=100, cuda_graphs=False),
          **kw}
    return Engine(EngineConfig(**kw), max_seq=512)


def _follows_reference(eng, prompts, outs, gap=1e-2):
    n = 0
    for p, o in zip(prompts, outs):
        seq = list(p)
        for tok in o:
            ref = eng.runner.model.reference_logits(seq)[-1]
            top = torch.topk(ref, 2).values
            if (top[0] - top[1]).item() > gap:           # not a numerical tie
                assert tok == int(ref.argmax())
                n += 1
            seq.append(tok)
    return n


@pytest.mark.parametrize("spec", [False, True])
def test_engine_with_room_for_every_page_is_the_dense_engine(spec):
    from inference_optimizations_b200.engine.scheduler import SamplingParams
    torch.manual_seed(0)
    eng = _engine(sparse_pages=8, spec=spec)
    prompts = [torch.randint(1, 500, (n,)).tolist() for n in (190, 9, 130)]
    outs = eng.generate(prompts, SamplingParams(max_new_tokens=6))
    assert _follows_reference(eng, prompts, outs) >= 6


def test_engine_attends_to_the_selected_pages(monkeypatch):
    from inference_optimizations_b200.engine.scheduler import SamplingParams
    torch.manual_seed(1)
    eng = _engine(sparse_pages=3)
    seen = []
    real = S.block_select

    def spy(*a, **k):
        r = real(*a, **k)
        seen.append((a[4].clone(), r[0].clone(), r[1].clone()))
        return r
    monkeypatch.setattr(S, "block_select", spy)
    outs = eng.generate([torch.randint(1, 500, (450,)).tolist(), [7] * 20], SamplingParams(max_new_tokens=5))
    assert all(len(o) == 5 for o in outs)
    assert len(seen) >= 2 * 4                              # both global layers, every decode step
    for kv, blocks, count in seen:
        for b, n in enumerate(kv.tolist()):
            npg = (n + 63) // 64
            assert (count[b] == min(npg, 3)).all()
            assert (blocks[b, :, min(npg, 3) - 1] == npg - 1).all() and (blocks[b, :, 0] == 0).all()
    # every finished page of the requests had its bounds when it was ranked: recomputing them changes nothing
    kv = eng.runner.kv
    before = [(c.clone(), s.clone()) for c, s in (b for b in kv.bounds if b is not None)]
    kv.summarize()
    for (c, s), (c2, s2) in zip(before, (b for b in kv.bounds if b is not None)):
        done = s.ne(0).all(1)
        assert done.sum() >= 7 and torch.equal(c[done], c2[done]) and torch.equal(s[done], s2[done])


def test_engine_refuses_what_it_cannot_serve():
    for kw in (dict(sparse_pages=2), dict(sparse_pages=4000), dict(sparse_pages=4, sparse_local=0),
               dict(sparse_pages=4, model="tiny_mla", kv_dtype="nvfp4")):
        with pytest.raises(ValueError):
            _engine(**kw)


@pytest.mark.parametrize("spec", [False, True])
def test_engine_reports_a_wait_that_ran_out(spec):
    """A status word of the attention ends the step with an error; the step can be repeated."""
    from inference_optimizations_b200.engine.scheduler import SamplingParams
    from inference_optimizations_b200.parallel.health import DeviceWaitTimeout
    torch.manual_seed(3)
    prompts = [torch.randint(1, 500, (n,)).tolist() for n in (260, 70)]
    want = _engine(sparse_pages=4, spec=spec).generate(prompts, SamplingParams(max_new_tokens=8))
    eng = _engine(sparse_pages=4, spec=spec)
    reqs = [eng.add_request(p, SamplingParams(max_new_tokens=8)) for p in prompts]
    while len(eng.sched.running) < 2 or any(len(r.output) < 2 for r in reqs):
        eng.step()
    for _ in range(2):
        eng.runner.kv.sparse_status.fill_(1)
        before = [list(r.output) for r in reqs]
        with pytest.raises(DeviceWaitTimeout):
            eng.step()
        assert [r.output for r in reqs] == before
        eng.step()
    while eng.has_work():
        eng.step()
    assert [r.output for r in reqs] == want


def test_engine_refuses_tables_wider_than_the_selection():
    from inference_optimizations_b200.config import EngineConfig
    from inference_optimizations_b200.engine.engine import Engine
    ecfg = EngineConfig(model="tiny_gqa", device="cpu", kv_dtype="bf16", max_running=1, chunked_prefill=64,
                        cuda_graphs=False, sparse_pages=8)
    widest = 64 * (S.MAX_PAGES - 2)                          # one page of growth, one spare entry
    assert Engine(ecfg, max_seq=widest, global_pages=8).runner.kv.tables["global"].dev.shape[1] == S.MAX_PAGES
    with pytest.raises(ValueError, match="max_seq"):
        Engine(ecfg, max_seq=widest + 1, global_pages=8)

"""What `block_decode` and `block_select` do at their limits.

A copy that does not arrive: `block_decode` gives up after its wait limit (~2 s), waits for its other copies with the
same limit, marks the group's output NaN, records a status and leaves the context usable.  No copy is really lost: every
barrier awaits a few bytes more than its copy brings."""
import time

import pytest
import torch

from inference_optimizations_b200.ops import block_sparse as S
from inference_optimizations_b200.ops import kvcache as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,d,hq,n_q,pages", [(K.FMT_BF16, 128, 4, 1, 40), (K.FMT_FP8, 256, 4, 4, 3),
                                                (K.FMT_NVFP4, 512, 2, 1, 1), (K.FMT_BF16, 512, 2, 8, 24)])
def test_decode_gives_up_on_a_copy_that_does_not_arrive(cuda, fmt, d, hq, n_q, pages):
    from inference_optimizations_b200._ext import ext
    from inference_optimizations_b200.parallel import health as HL
    pool = torch.zeros(pages + 1, 1, 2, K.part_bytes(fmt, d), dtype=torch.uint8, device=cuda)
    table = torch.arange(1, pages + 1, dtype=torch.int32, device=cuda)[None].repeat(2, 1)
    kv = torch.tensor([pages * 64, 0], dtype=torch.int32, device=cuda)           # the second group has nothing to wait for
    blocks = torch.arange(pages, dtype=torch.int32, device=cuda).repeat(2, 1, 1)
    q = torch.randn(2 * n_q, hq, d, device=cuda).to(torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    args = (q, pool, table, None, kv, blocks, None, None, status, n_q, 1, fmt, 0.1, 1.0, 1.0)
    t0 = time.time()
    out, lse = ext().block_decode(*args, never_bytes=16)
    torch.cuda.synchronize()
    assert time.time() - t0 < 15
    assert status.item() == 1 and out[:n_q].isnan().all() and lse[:n_q].isnan().all()
    assert not out[n_q:].any() and (lse[n_q:] == -float("inf")).all()
    with pytest.raises(HL.DeviceWaitTimeout):
        HL.check_status([status])
    status.zero_()
    out, lse = ext().block_decode(*args)
    assert status.item() == 0 and not out.any() and lse[:n_q].isfinite().all()
    assert torch.equal(S.block_decode(q, pool, table, kv, blocks, n_q, 1, fmt, 0.1)[1], lse)


def test_selection_over_bounds_of_no_page_is_refused(cuda):
    codes, sc = S.alloc_bounds(0, 2, 128, cuda)
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device=cuda)
    table = torch.zeros(1, 9, dtype=torch.int32, device=cuda)
    for n in (64 * 9, 64):
        with pytest.raises(RuntimeError, match="at least one page"):
            S.block_select(q, codes, sc, table, torch.tensor([n], dtype=torch.int32, device=cuda), 1, 2, 3)


@pytest.mark.parametrize("fmt,d,hq,n_q", [(K.FMT_BF16, 512, 2, 1), (K.FMT_FP8, 128, 8, 2), (K.FMT_NVFP4, 512, 2, 8),
                                          (K.FMT_BF16, 256, 8, 2)])
def test_long_and_short_lists_from_two_threads(cuda, fmt, d, hq, n_q):
    """The longest list (every form's largest shared memory) and the shortest one, called in turn by two host threads."""
    import threading
    pool = torch.zeros(9, 1, 2, K.part_bytes(fmt, d), dtype=torch.uint8, device=cuda)
    codes, sc = S.alloc_bounds(9, 1, d, cuda)
    q = torch.randn(n_q, hq, d, device=cuda).to(torch.bfloat16)
    torch.cuda.synchronize()
    failed = []

    def calls(width, budget):
        try:
            table = torch.ones(1, width, dtype=torch.int32, device=cuda)
            kv = torch.tensor([8 * 64], dtype=torch.int32, device=cuda)
            for _ in range(50):
                blocks, count = S.block_select(q, codes, sc, table, kv, n_q, 1, budget)
                out, lse = S.block_decode(q, pool, table, kv, blocks, n_q, 1, fmt, 0.1)
            torch.cuda.synchronize()
            if count.item() != min(8, budget) or out.any() or not lse.isfinite().all():
                failed.append((width, budget))
        except RuntimeError as e:
            failed.append(e)
    threads = [threading.Thread(target=calls, args=a) for a in ((S.MAX_PAGES, S.MAX_LIST), (9, 3))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed

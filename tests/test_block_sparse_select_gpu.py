"""Selection at the ends of the scores' range: products that underflow, products that overflow."""
import pytest
import torch

from inference_optimizations_b200.ops import block_sparse as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,hq,n_q", [(128, 4, 1), (256, 8, 2), (512, 2, 4)])
@pytest.mark.parametrize("q_exp,k_exp", [(-80, -100), (-45, -95), (-20, -100), (100, 60), (100, 20)])
def test_scores_that_leave_the_range_tie(cuda, d, hq, n_q, q_exp, k_exp):
    """Scores of either sign that become 0 are equal, and so are those that become infinite: the lowest pages win."""
    pages, hk = 70, 2
    g = torch.Generator().manual_seed(d + q_exp)
    codes = torch.randint(-127, 128, (pages, hk, 2, d), generator=g, dtype=torch.int8)
    codes[:, :, 1] = torch.randint(0, 9, (pages, hk, d), generator=g)
    sc = torch.full((pages, hk), 2.0 ** k_exp, dtype=torch.bfloat16)
    q = (torch.randn(2 * n_q, hq, d, generator=g) * 2.0 ** q_exp).to(torch.bfloat16)
    table = torch.stack([torch.randperm(pages, generator=g) for _ in range(2)]).int()
    kv = torch.tensor([pages * 64, pages * 64 - 77], dtype=torch.int32)
    for budget in (3, 12, 50):
        want = S.block_select(q, codes, sc, table, kv, n_q, hk, budget)
        got = S.block_select(*[x.to(cuda) for x in (q, codes, sc, table, kv)], n_q, hk, budget)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])

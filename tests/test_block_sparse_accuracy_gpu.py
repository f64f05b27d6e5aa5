"""Accuracy of `block_decode` element by element against 64 bits, with a bound for each way the weights are held:
requests with one dominating token, block scales from the smallest to the largest, queries that make scores large."""
import functools
import math

import pytest
import torch

from inference_optimizations_b200.ops import block_sparse as S
from inference_optimizations_b200.ops import kvcache as K

pytestmark = pytest.mark.gpu

FMTS = {"bf16": K.FMT_BF16, "fp8": K.FMT_FP8, "nvfp4": K.FMT_NVFP4}
KS, VS = 0.75, 1.25
# Relative rounding of a weight for the second product: 11 bits over 8-bit and 4-bit caches, 16 (8 and what they leave,
# 8 more) over bf16 ones.
UNIT = {K.FMT_BF16: 2.0 ** -16, K.FMT_FP8: 2.0 ** -11, K.FMT_NVFP4: 2.0 ** -11}


def part_abs(pool, fmt, d):
    """The pool with |V|, and with |V| and |K|."""
    out = []
    for parts in (slice(1, 2), slice(0, 2)):
        p = pool.clone()
        if fmt == K.FMT_BF16:
            p.view(torch.bfloat16)[:, :, parts].abs_()
        elif fmt == K.FMT_FP8:
            p[:, :, parts] &= 0x7F
        else:
            p[:, :, parts, :K.PAGE * d // 2] &= 0x77
        out.append(p)
    return out


def check(out, lse, q, pool, table, kv, blocks, n_q, hk, fmt, sm):
    """out: its own rounding to bf16 (2^-8), of each weight UNIT and twice the score's error, and where weights are f16
    2^-37 of the largest for each of them (the last step of an f16 that carries 2^12).  Scores: an fp32 sum of D exact
    products, at most D 2^-23 of the sum of their sizes, and the exponent's rounding, 2^-22 of the score each for its
    scale and its difference.  lse: the scores' error, and 2^-20 of a sum of fp32 terms."""
    d = q.shape[2]
    c = [x.cpu() for x in (q, pool, table, kv, blocks)]

    def ref(q_, pool_):
        return S.block_decode_ref(q_, pool_, *c[2:], n_q, hk, fmt, sm, KS, VS, None, torch.float64)
    want, wlse = ref(c[0], c[1])
    va, ka = part_abs(c[1], fmt, d)
    mag, _ = ref(c[0], va)
    zero = torch.zeros_like(c[0])
    total, count = ref(zero, va)
    total = total * count.exp()[..., None]                            # sum of |v| over what a row sees
    size = ref(c[0].abs(), ka)[1].clamp(min=0)                        # at least the largest sum of |q||k| sm
    ds = (size * (d * 2.0 ** -23 + 2.0 ** -21) + 2.0 ** -20)[..., None]
    tiny = 0.0 if fmt == K.FMT_BF16 else 2.0 ** -37
    tol = want.abs() * 2.0 ** -8 + mag * (UNIT[fmt] + 2 * ds) + total * tiny + 1e-30
    got = out.cpu().double()
    off = (got - want).abs()
    same = (got == want) | (want.isnan() & got.isnan())               # (infinities and NaN)
    assert ((off <= tol) | same).all(), f"{(off / tol).max()} of the bound"
    near = (lse.cpu().double() - wlse).abs() <= ds[..., 0] + 2.0 ** -20 * (1 + wlse.abs())
    assert (near | (lse.cpu() == wlse)).all()                         # (a row that sees nothing: -inf)


@functools.lru_cache(maxsize=1)
def dominated_pool(fmt, d, scale, seed):
    g = torch.Generator().manual_seed(seed)
    pages, n = 64, 4096
    codes = torch.tensor([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -1.0])
    v = codes[torch.randint(0, 8, (n, 1, d), generator=g)]
    v[:, :, ::16] = 6.0                                               # every block of 16 has the largest code
    v = v * scale
    v[17] = 0
    k = torch.zeros(n, 1, d)
    k[17, 0, 0] = 6.0
    unit = (1.0, 1.0) if fmt == K.FMT_BF16 else (KS, VS)
    pool = torch.zeros(pages + 1, 1, 2, K.part_bytes(fmt, d), dtype=torch.uint8)
    table = (torch.randperm(pages, generator=g) + 1)[None].int()
    at = torch.arange(n)
    slot = (table[0, at // 64] * 64 + at % 64).int()
    K.gqa_pool_write_ref(pool, slot, k * unit[0], v * unit[1], fmt, *unit)
    return pool, table, unit


def dominated(fmt, d, hq, gap, scale, seed):
    """64 pages: token 17 has V = 0 and weight 1, every other token about 2^-gap; V in one scale, mostly positive (an
    E4M3 cache cannot hold the largest scale's codes: the writer's NaN have to come out)."""
    pool, table, unit = dominated_pool(fmt, d, scale, seed)
    n, pages = 4096, 64
    q = torch.zeros(1, hq, d)
    q[0, :, 0] = gap + 0.11 * torch.arange(hq)
    sm = math.log(2.0) / 6.0 / unit[0]                                # the gap in bits is q's only value
    return (q.to(torch.bfloat16), pool, table, torch.tensor([n], dtype=torch.int32),
            torch.arange(pages, dtype=torch.int32).expand(1, 1, pages).contiguous()), sm


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("d,hq", [(128, 1), (128, 4), (128, 8), (128, 16), (256, 4), (256, 16), (512, 2), (512, 8), (512, 16)])
@pytest.mark.parametrize("scale", [2.0 ** -9, 2.0 ** -6, 2.0 ** -2, 256.0])
def test_one_dominating_token(cuda, fmt, d, hq, scale):
    """What the others add up to keeps its precision, however small they and their block scales are."""
    fmt = FMTS[fmt]
    for gap in (15.3, 18.4, 21.4, 25.3):
        args, sm = dominated(fmt, d, hq, gap, scale, d + hq)
        out, lse = S.block_decode(*[x.to(cuda) for x in args], 1, 1, fmt, sm, KS, VS)
        check(out, lse, *args, 1, 1, fmt, sm)


def random_case(fmt, d, hq, hk, n_q, lens, budget, seed, grow=1.0):
    """Requests of the given lengths, FP4 block scales from 2^-9 to 448 side by side, queries `grow` times as large."""
    g = torch.Generator().manual_seed(seed)
    per = [(x + 63) // 64 for x in lens]
    pool = torch.randint(0, 256, (sum(per) + 1, hk, 2, K.part_bytes(fmt, d)), generator=g, dtype=torch.uint8)
    if fmt == K.FMT_BF16:
        pool.view(torch.bfloat16).copy_(torch.randn(sum(per) + 1, hk, 2, K.PAGE * d, generator=g))
    elif fmt == K.FMT_FP8:
        pool &= 0xBF
    else:
        sc = pool[..., K.PAGE * d // 2:]
        sc &= 0x0F
        sc |= 0x28
        pick = torch.tensor([0x01, 0x04, 0x08, 0x20, 0x38, 0x60, 0x7E], dtype=torch.uint8)
        sc[:, :, 1] = pick[torch.randint(0, 7, sc[:, :, 1].shape, generator=g)]
    perm = (torch.randperm(sum(per), generator=g) + 1).int()
    table = torch.zeros(len(lens), max(per), dtype=torch.int32)
    blocks = torch.full((len(lens), hk, budget), -1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(per):
        table[i, :m] = perm[at:at + m]
        at += m
        for h in range(hk):
            pick = torch.randperm(m, generator=g)[:budget].int()
            blocks[i, h, :len(pick)] = pick
    q = (torch.randn(len(lens) * n_q, hq, d, generator=g) * 2 * grow).to(torch.bfloat16)
    return q, pool, table, torch.tensor(lens, dtype=torch.int32), blocks


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("d", [128, 256, 512])
@pytest.mark.parametrize("hq,hk,n_q", [(1, 1, 1), (8, 2, 1), (8, 1, 1), (8, 2, 4)])
@pytest.mark.parametrize("grow", [1.0, 20.0])
def test_every_scale_and_large_queries(cuda, fmt, d, hq, hk, n_q, grow):
    fmt = FMTS[fmt]
    args = random_case(fmt, d, hq, hk, n_q, [448, 300, 77, 1], 7, d + hq + n_q, grow)
    out, lse = S.block_decode(*[x.to(cuda) for x in args], n_q, hk, fmt, d ** -0.5, KS, VS)
    check(out, lse, *args, n_q, hk, fmt, d ** -0.5)


def lone_case(fmt, d, hq, ratio, size, seed):
    """200 tokens whose keys have nothing in dimension 0, where every query has its largest value; the others are about
    `ratio` of it, and the largest is `size`."""
    g = torch.Generator().manual_seed(seed)
    n = 200
    k, v = torch.randn(2, n, 1, d, generator=g)
    k[:, :, 0] = 0
    pool = torch.zeros(5, 1, 2, K.part_bytes(fmt, d), dtype=torch.uint8)
    table = torch.tensor([[3, 1, 4, 2]], dtype=torch.int32)
    at = torch.arange(n)
    K.gqa_pool_write_ref(pool, (table[0, at // 64] * 64 + at % 64).int(), k, v, fmt, KS, VS)
    q = torch.randn(1, hq, d, generator=g) * ratio * size
    q[:, :, 0] = size
    sm = 2.0 / math.sqrt(d) / ratio / size
    return (q.to(torch.bfloat16), pool, table, torch.tensor([n], dtype=torch.int32),
            torch.arange(4, dtype=torch.int32).view(1, 1, 4)), sm


@pytest.mark.parametrize("fmt", ["fp8", "nvfp4"])
@pytest.mark.parametrize("d,hq", [(128, 4), (256, 16), (512, 2), (512, 8)])
@pytest.mark.parametrize("ratio,size", [(2.0 ** -20, 1.0), (2.0 ** -12, 2.0 ** 60), (2.0 ** -3, 2.0 ** 120)])
def test_queries_with_one_large_value(cuda, fmt, d, hq, ratio, size):
    """8-bit and 4-bit caches take queries through f16: the small values of a row keep their bits beside a large one, and
    sizes up to bf16's largest stay finite."""
    fmt = FMTS[fmt]
    args, sm = lone_case(fmt, d, hq, ratio, size, d + hq)
    out, lse = S.block_decode(*[x.to(cuda) for x in args], 1, 1, fmt, sm, KS, VS)
    check(out, lse, *args, 1, 1, fmt, sm)


@pytest.mark.parametrize("d,hq,n_q", [(128, 4, 1), (128, 4, 4), (256, 8, 1), (512, 2, 1), (512, 16, 1)])
def test_an_infinite_value_that_every_row_sees(cuda, d, hq, n_q):
    """Over a bf16 cache: outputs in its dimension are infinite, the others are what they are."""
    q, pool, table, kv, blocks = random_case(K.FMT_BF16, d, hq, 1, n_q, [400, 70], 7, d + hq)
    rb = 2 * d
    for i, (pos, at, bits) in enumerate(((130, 5, 0x7F80), (3, d - 2, 0x7F80 - (1 << 15)))):          # inf, -inf
        part = pool[int(table[i, pos // 64]), 0, 1].view(torch.int16)
        part[pos % 64 * d + int(K.kv_swizzle_perm(rb)[pos % 64][2 * at]) // 2] = bits
    out, lse = S.block_decode(*[x.to(cuda) for x in (q, pool, table, kv, blocks)], n_q, 1, K.FMT_BF16, 0.3, KS, VS)
    want, wlse = S.block_decode_ref(q, pool, table, kv, blocks, n_q, 1, K.FMT_BF16, 0.3, KS, VS, None, torch.float64)
    odd = ~torch.isfinite(want)
    assert odd.sum() == 2 * n_q * hq and torch.equal(out.cpu().double()[odd], want[odd])
    assert torch.equal(torch.isfinite(out.cpu()), ~odd)


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("d,hq,hk,n_q", [(128, 8, 2, 4), (128, 2, 2, 16), (256, 8, 2, 4), (256, 3, 3, 5), (512, 4, 2, 4),
                                         (512, 16, 4, 4)])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(cuda, fmt, d, hq, hk, n_q):
    """A verify group's own tokens, on one page and on two, with infinite or NaN V (over 8-bit and 4-bit caches NaN)."""
    fmt = FMTS[fmt]
    lens = [n_q, 64 + 2, 200, 64 * 5, 64 * 4 + n_q - 1, 64 * 7 + 2]
    q, pool, table, kv, blocks = random_case(fmt, d, hq, hk, n_q, lens, 8, d + n_q)
    for i, n in enumerate(lens):
        for pos, at, kind in ((n - 1, 3, 0x7F80), (n - 2, 3, 0xFF80), (n - 2, d - 1, 0x7FC0), (n - n_q // 2, 40, 0xFF80)):
            page, off = int(table[i, pos // 64]), pos % 64
            part = pool[page, hk - 1, 1]
            rb = K.row_bytes(fmt, d)
            per = 8 if fmt == K.FMT_BF16 else 16
            chunk = int(K.kv_swizzle_perm(rb)[off][at // per * 16]) if fmt != K.FMT_NVFP4 else 0
            if fmt == K.FMT_BF16:
                part[off * rb:(off + 1) * rb].view(torch.int16)[chunk // 2 + at % per] = kind - (1 << 16 if kind >= 1 << 15 else 0)
            elif fmt == K.FMT_FP8:
                part[off * rb + chunk + at % per] = 0x7F if kind != 0xFF80 else 0xFF
            else:
                part[64 * rb + off * (d // 16) + at // 16] = 0x7F
    blocks[5, :, :] = -1
    blocks[5, :, 0] = 6                                               # a list without the group's second page
    out, lse = S.block_decode(*[x.to(cuda) for x in (q, pool, table, kv, blocks)], n_q, hk, fmt, d ** -0.5, KS, VS)
    want, _ = S.block_decode_ref(q, pool, table, kv, blocks, n_q, hk, fmt, d ** -0.5, KS, VS, None, torch.float64)
    assert torch.equal(out.isfinite().cpu(), want.isfinite()) and not want.isfinite().all()
    check(out, lse, q, pool, table, kv, blocks, n_q, hk, fmt, d ** -0.5)

"""Block-sparse attention over the paged GQA cache: a query attends to the pages that a cheap bound of their keys
ranks highest (kernels in csrc/block_sparse.cu and csrc/attn_block_decode.cu; fp32 oracles below).

Three operators, used in this order by a layer of a long-context model:

  block_append   the QKV epilogue (per-head norm, NeoX rotation, cache write) which also keeps, for every page that the
                 call finishes, 8-bit bounds of its 64 keys
  block_select   ranks a request's finished pages for each group of query tokens by those bounds and lists the pages
                 to attend to: the first `sink` pages, the pages around the queries, and the best of the rest
  block_decode   softmax attention over the listed pages, output and log-sum-exp

and `block_summarize`, which recomputes the bounds of pages that something else wrote.

Bounds of one (page, kv head), from its stored keys: lo, hi = min, max over the page's 64 tokens per dimension,
c = (lo + hi) / 2, w = (hi - lo) / 2; codes int8 [pages, Hk, 2 (c, w), D] = clamp(rint(. / 2^e), +-127), scale bf16
[pages, Hk] = 2^e with e = exponent(max(|c|, w)) - 7.  A page with a key that is not finite has scale inf and is always
listed first.  A query row q, coded the same way, scores the page  sum_d q_d c_d + |q_d| w_d , an upper bound of its
dot product with every key of the page; a group's score is the largest over its rows.  Codes, products and sums are
whole numbers below 2^24 and the scales powers of two, so scores are exact and the listed pages do not depend on the
order of any sum; equal scores go to the lower page.

A group is n_q consecutive query tokens of one request (1 for a decode step, the verify length for speculation, a few
for prefill) that share one list; n_q * (Hq / Hk) <= 16.  As in `gqa_decode`, kv_len[b] counts the tokens in the pool,
the group's own included; token t of the group sits at position kv_len[b] - n_q + t and sees positions up to its own.
A group with kv_len 0 (a padding row) lists nothing; a row that sees nothing has output 0 and log-sum-exp -inf.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from .._ext import ext
from . import kvcache as K
from .basic import apply_rope_ref
from .kvcache import PAGE

MAX_LIST = 2048            # pages of one list (kBlockMaxList)
MAX_PAGES = 49152          # page-table width of block_select (kBlockSelectMaxPages)
HEAD_DIMS = (128, 256, 512)


def alloc_bounds(pages: int, hk: int, d: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scale) of a layer pool's pages, zeroed."""
    return (torch.zeros(pages, hk, 2, d, dtype=torch.int8, device=device),
            torch.zeros(pages, hk, dtype=torch.bfloat16, device=device))


def _pow2(amax: torch.Tensor) -> torch.Tensor:
    _, x = torch.frexp(amax)
    return torch.exp2((x.float() - 7).clamp(-100, 100))


def _codes(v: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return (v / scale).round().clamp(-127, 127)


# ------------------------------------------------------------------------------------------------ append
def block_append(qkv: torch.Tensor, q_norm: Optional[torch.Tensor], k_norm: Optional[torch.Tensor],
                 cos_sin: torch.Tensor, pos: torch.Tensor, slot: torch.Tensor, pool: torch.Tensor,
                 codes: torch.Tensor, scale: torch.Tensor, fmt: int, hq: int, hk: int, d: int, eps: float,
                 plus_one: bool, k_scale: float = 1.0, v_scale: float = 1.0,
                 q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """qkv bf16 [T, (Hq + 2 Hk) D]: per-head RMSNorm of q and k (optional), NeoX rotation by cos_sin[pos], q -> bf16
    [T, Hq, D] (returned), k and v -> pool[slot] in the pool's format; everything in fp32 with one rounding at the end
    (`gqa_prep` rounds to bf16 after the norm).  Every page whose last row (slot % 64 == 63) is written gets its key
    bounds.  A row with slot -1, or with a position outside the table, is not written (its q is zero in the latter
    case).  E4M3 values saturate.  Rows of one page are adjacent and ascending in a call, without a row that is not
    written between them, and the page's earlier rows were written by earlier calls on the stream: the order in which a
    request's tokens arrive.  V's bytes are those of `gqa_prep`; K's may differ in the last bit (one rounding, not two)."""
    if qkv.is_cuda:
        return ext().block_append(qkv, q_norm, k_norm, cos_sin, pos, slot, q_out, pool, codes, scale, fmt, k_scale,
                                  v_scale, hq, hk, d, eps, plus_one)
    if q_out is None:
        q_out = torch.empty(qkv.shape[0], hq, d, dtype=torch.bfloat16)
    _check_pool(pool, codes, scale, fmt, hk, d)
    if qkv.dim() != 2 or qkv.shape[1] < (hq + 2 * hk) * d or cos_sin.shape[-1] != d:
        raise RuntimeError("block_append: qkv [T, (Hq + 2 Hk) D], cos_sin [positions, D]")
    if fmt != K.FMT_BF16 and not (k_scale > 0 and v_scale > 0):
        raise RuntimeError("the pool's scales must be positive")
    x = qkv[:, : (hq + 2 * hk) * d].float().unflatten(1, (hq + 2 * hk, d))
    ok = (pos >= 0) & (pos < cos_sin.shape[0])
    at = torch.where(ok, pos, torch.zeros_like(pos))

    def norm(v, w):
        if w is None:
            return v
        return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + eps) * (w.float() + 1.0 if plus_one else w.float())

    q = apply_rope_ref(norm(x[:, :hq], q_norm), at, cos_sin)
    q_out.copy_(torch.where(ok[:, None, None], q, torch.zeros_like(q)))
    k = apply_rope_ref(norm(x[:, hq:hq + hk], k_norm), at, cos_sin)
    wr = torch.where(ok & (slot >= 0) & (slot < pool.shape[0] * PAGE), slot, torch.full_like(slot, -1))
    K.gqa_pool_write_ref(pool, wr, k, x[:, hq + hk:], fmt, k_scale, v_scale)
    done = wr[(wr >= 0) & (wr % PAGE == PAGE - 1)] // PAGE
    block_summarize(pool, done.int(), codes, scale, fmt, hk, d, k_scale)
    return q_out


def block_summarize(pool: torch.Tensor, pages: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, fmt: int,
                    hk: int, d: int, k_scale: float = 1.0) -> None:
    """Key bounds of whole pages (int32 [n]; ids outside the pool are skipped) from what the pool holds."""
    if pool.is_cuda:
        ext().block_summarize(pool, pages, codes, scale, fmt, k_scale, hk, d)
        return
    _check_pool(pool, codes, scale, fmt, hk, d)
    if fmt != K.FMT_BF16 and not k_scale > 0:
        raise RuntimeError("the pool's scale must be positive")
    for p in pages.tolist():
        if not 0 <= p < pool.shape[0]:
            continue
        keys, _ = K.gqa_pool_read_ref(pool, torch.tensor([p]), PAGE, fmt, d, k_scale)          # [64, Hk, D]
        lo, hi = keys.amin(0), keys.amax(0)
        c, w = (lo + hi) * 0.5, (hi - lo) * 0.5
        amax = torch.maximum(c.abs(), w).amax(-1)                                              # [Hk]
        fin = torch.isfinite(keys).all(0).all(-1) & torch.isfinite(amax)
        s = _pow2(torch.where(fin, amax, torch.zeros_like(amax)))
        cw = torch.where(fin[:, None, None], torch.stack([c, w], 1), torch.zeros(()))
        codes[p] = _codes(cw, s[:, None, None]).to(torch.int8)
        scale[p] = torch.where(fin, s, torch.full_like(s, math.inf)).to(torch.bfloat16)


def _check_pool(pool, codes, scale, fmt, hk, d) -> None:
    if d not in HEAD_DIMS or fmt not in (K.FMT_BF16, K.FMT_FP8, K.FMT_NVFP4):
        raise RuntimeError(f"block-sparse attention: head_dim {HEAD_DIMS} and a GQA pool format, got {d}, {fmt}")
    if tuple(pool.shape[1:]) != (hk, 2, K.part_bytes(fmt, d)):
        raise RuntimeError("pool uint8 [pages, Hk, 2, part bytes]")
    if codes is not None and (tuple(codes.shape) != (pool.shape[0], hk, 2, d)
                              or tuple(scale.shape) != (pool.shape[0], hk)):
        raise RuntimeError("codes int8 [pages, Hk, 2, D], scale bf16 [pages, Hk]")


# ------------------------------------------------------------------------------------------------ select
def block_select(q: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, page_table: torch.Tensor,
                 kv_len: torch.Tensor, n_q: int, hk: int, budget: int, sink: int = 1, local: int = 1,
                 req_idx: Optional[torch.Tensor] = None,
                 out: Optional[tuple[torch.Tensor, torch.Tensor]] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """q bf16 [B * n_q, Hq, D] -> (blocks int32 [B, Hk, budget], count int32 [B, Hk]): the logical pages that group b
    attends to, ascending, -1 behind them.  A request of at most `budget` pages lists them all.  Otherwise always in:
    the first `sink` pages and the pages from `local` - 1 before the group's first token on (they need no bounds:
    the last one is unfinished); the rest of the budget goes to the pages with the highest scores.
    budget >= sink + local + 1 (a group may straddle two pages)."""
    if q.is_cuda:
        blocks, count = out if out is not None else (None, None)
        return ext().block_select(q, codes, scale, page_table, req_idx, kv_len, blocks, count, n_q, hk, budget, sink,
                                  local)
    b = kv_len.shape[0]
    blocks, count = out if out is not None else (torch.empty(b, hk, budget, dtype=torch.int32),
                                                 torch.empty(b, hk, dtype=torch.int32))
    _check_groups(q, page_table, kv_len, n_q, hk)
    if sink < 0 or local < 1 or not sink + local + 1 <= budget <= MAX_LIST:
        raise RuntimeError(f"budget must hold sink + local + 1 pages and at most {MAX_LIST}")
    if codes.shape[0] < 1:
        raise RuntimeError("codes of at least one page")
    if page_table.shape[1] > MAX_PAGES:
        raise RuntimeError(f"page_table wider than {MAX_PAGES}")
    blocks.fill_(-1)
    count.zero_()
    g = q.shape[1] // hk
    for i in range(b):
        row = int(req_idx[i]) if req_idx is not None else i
        n = min(int(kv_len[i]), page_table.shape[1] * PAGE) if 0 <= row < page_table.shape[0] else 0
        npages = (max(n, 0) + PAGE - 1) // PAGE
        if npages <= budget:
            blocks[i, :, :npages] = torch.arange(npages, dtype=torch.int32)
            count[i] = npages
            continue
        first_local = max(0, max(0, n - n_q) // PAGE - (local - 1))
        forced = list(range(sink)) + list(range(first_local, npages))
        cand = torch.arange(sink, first_local)
        phys = page_table[row, cand.long()].long()
        inside = (phys >= 0) & (phys < codes.shape[0])
        phys = torch.where(inside, phys, torch.zeros_like(phys))
        for h in range(hk):
            rows = q[i * n_q:(i + 1) * n_q, h * g:(h + 1) * g].reshape(n_q * g, -1).float()
            amax = rows.abs().amax(-1, keepdim=True)
            fin = torch.isfinite(rows).all(-1, keepdim=True)
            sq = _pow2(torch.where(fin, amax, torch.zeros_like(amax)))
            q8 = _codes(torch.where(fin, rows, torch.zeros_like(rows)), sq)
            rec = codes[phys, h].float()                                                 # [N, 2, D]
            val = q8 @ rec[:, 0].t() + q8.abs() @ rec[:, 1].t()
            val = torch.where(fin, val * sq, torch.full_like(val, -math.inf)).amax(0)    # [N]
            sc = scale[phys, h].float()
            val = torch.where(sc == math.inf, torch.full_like(val, math.inf), val * torch.where(sc == math.inf, 1.0, sc))
            val = torch.where(inside, val, torch.full_like(val, -math.inf))
            best = cand[val.sort(descending=True, stable=True).indices[:budget - len(forced)]].tolist()
            blocks[i, h] = torch.tensor(sorted(forced + best), dtype=torch.int32)
            count[i, h] = budget
    return blocks, count


def _check_groups(q, page_table, kv_len, n_q, hk) -> None:
    if q.dim() != 3 or hk < 1 or q.shape[1] % hk or n_q < 1 or n_q * (q.shape[1] // hk) > 16:
        raise RuntimeError("n_q * (Hq / Hk) must be whole and at most 16")
    if q.shape[2] not in HEAD_DIMS:
        raise RuntimeError(f"head_dim {HEAD_DIMS}, got {q.shape[2]}")
    if q.shape[0] != kv_len.shape[0] * n_q or page_table.dim() != 2:
        raise RuntimeError("kv_len [B], q rows B * n_q, page_table [rows, pages]")


# ------------------------------------------------------------------------------------------------ attend
def block_decode(q: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor, kv_len: torch.Tensor,
                 blocks: torch.Tensor, n_q: int, hk: int, fmt: int, sm_scale: float, k_scale: float = 1.0,
                 v_scale: float = 1.0, req_idx: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                 lse: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of q bf16 [B * n_q, Hq, D] over the listed pages -> (out bf16 like q, lse fp32 [B * n_q, Hq], natural
    log).  blocks int32 [B, Hk, budget] from `block_select` or any list of logical pages in any order, each at most
    once; entries < 0, past kv_len or without a page of the pool are skipped.  What the cache holds past kv_len is
    never used, whatever it is.  k_scale / v_scale are ignored on bf16 pools.  status int32 [1]: a copy that did not
    arrive within the wait limit records a code there (and the group's output is NaN).

    Accuracy: scores and sums are fp32; a weight enters the product with V in 11 bits over 8-bit and 4-bit caches (to
    2^-26 of the row's largest, 2^-37 of it below), in 16 bits over bf16 caches; the output is rounded to bf16.  A value of
    V that is not finite reaches the rows that see it and no other."""
    if q.is_cuda:
        return ext().block_decode(q, pool, page_table, req_idx, kv_len, blocks, out, lse, status, n_q, hk, fmt,
                                  sm_scale, k_scale, v_scale)
    if out is None:
        out = torch.empty(q.shape, dtype=torch.bfloat16)
    if lse is None:
        lse = torch.empty(q.shape[0], q.shape[1], dtype=torch.float32)
    _check_groups(q, page_table, kv_len, n_q, hk)
    _check_pool(pool, None, None, fmt, hk, q.shape[2])
    if not (sm_scale > 0 and (fmt == K.FMT_BF16 or k_scale > 0)):
        raise RuntimeError("the softmax scale and the pool's key scale must be positive")
    if tuple(blocks.shape[:2]) != (kv_len.shape[0], hk) or not 1 <= blocks.shape[2] <= MAX_LIST:
        raise RuntimeError(f"blocks [B, Hk, 1 .. {MAX_LIST}]")
    o, z = block_decode_ref(q, pool, page_table, kv_len, blocks, n_q, hk, fmt, sm_scale, k_scale, v_scale, req_idx)
    out.copy_(o)
    lse.copy_(z)
    return out, lse


def block_decode_ref(q, pool, page_table, kv_len, blocks, n_q, hk, fmt, sm_scale, k_scale=1.0, v_scale=1.0,
                     req_idx=None, dtype=torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """Oracle of `block_decode` in `dtype`, not rounded (CPU)."""
    if fmt == K.FMT_BF16:
        k_scale = v_scale = 1.0
    b, (t, hq, d) = kv_len.shape[0], q.shape
    g = hq // hk
    out = torch.zeros(t, hq, d, dtype=dtype)
    lse = torch.full((t, hq), -math.inf, dtype=dtype)
    for i in range(b):
        row = int(req_idx[i]) if req_idx is not None else i
        if not 0 <= row < page_table.shape[0]:
            continue
        n = min(int(kv_len[i]), page_table.shape[1] * PAGE)
        for h in range(hk):
            use = [p for p in blocks[i, h].tolist()
                   if 0 <= p < page_table.shape[1] and p * PAGE < n and 0 <= int(page_table[row, p]) < pool.shape[0]]
            if not use:
                continue
            one = pool[:, h:h + 1]
            kk, vv = K.gqa_pool_read_ref(one, page_table[row, use], len(use) * PAGE, fmt, d, k_scale, v_scale)
            kk, vv = kk[:, 0].to(dtype), vv[:, 0].to(dtype)
            pos = (torch.tensor(use)[:, None] * PAGE + torch.arange(PAGE)).flatten()
            for tt in range(n_q):
                see = pos <= n - n_q + tt
                if not see.any():
                    continue
                r = i * n_q + tt
                s = q[r, h * g:(h + 1) * g].to(dtype) @ kk[see].t() * sm_scale
                lse[r, h * g:(h + 1) * g] = torch.logsumexp(s, -1)
                out[r, h * g:(h + 1) * g] = torch.softmax(s, -1) @ vv[see]
    return out, lse

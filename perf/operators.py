"""Workloads of the block-sparse attention operators over the paged GQA cache, in plain torch form and through
`inference_optimizations_b200.ops.block_sparse`.

  append : per-head norm, rotation and cache write of new tokens; 8-bit key bounds of every page that they finish
  select : the pages that each group of queries attends to, ranked by those bounds
  attend : softmax attention over the selected pages

A cache page holds 64 tokens.  The cache of one layer is uint8 [pages, Hk, 2 (K, V), bytes]: 64 rows of D bf16 or E4M3
values, or of D / 2 bytes of E2M1 pairs followed by 64 x D / 16 E4M3 block scales; the 16-byte chunks of row r are
stored at chunk ^ (r & (n - 1)), n = min(8, chunks per row)."""
import math

import torch

own = False

PAGE = 64
FMT = {"bf16": 0, "fp8": 1, "nvfp4": 2}
K_SCALE, V_SCALE = 0.75, 1.25      # of the 8-bit and 4-bit caches (a bf16 cache has none)
EPS = 1e-6


def listed():
    return [
        # one user's decode step, 8 kv heads of 128: the smallest call, all latency
        dict(name="append decode 1", op="append", fmt="bf16", hq=32, hk=8, d=128, reqs=1, tokens=1, norm=True),
        # a decode step of 64 users on a global layer of the Gemma-class model (32 / 16 heads of 512), FP8 cache
        dict(name="append decode 64 hd512", op="append", fmt="fp8", hq=32, hk=16, d=512, reqs=64, tokens=1, norm=True),
        # a full prefill chunk of one request on that layer, bf16 cache
        dict(name="append prefill 8192 hd512", op="append", fmt="bf16", hq=32, hk=16, d=512, reqs=1, tokens=8192,
             norm=True),
        # a ragged prefill batch on a layer with heads of 256, no q / k norm, FP8 cache
        dict(name="append ragged 7x219 hd256", op="append", fmt="fp8", hq=32, hk=16, d=256, reqs=7, tokens=219,
             norm=False),
        # one user at 204,800 tokens: few rows, a long list
        dict(name="select 1x204800", op="select", hq=32, hk=8, d=128, groups=1, n_q=1, ctx=204800, budget=32,
             shared=False),
        # 32 users at up to 32k on a global layer of the Gemma-class model
        dict(name="select 32x32768 hd512", op="select", hq=32, hk=16, d=512, groups=32, n_q=1, ctx=32768, budget=64,
             shared=False),
        # speculative verify of 8 users: 4 tokens share a list
        dict(name="select verify 8x100001 hd256", op="select", hq=32, hk=8, d=256, groups=8, n_q=4, ctx=100001,
             budget=128, shared=False),
        # a prefill chunk of 2048 tokens of one request, a list for every 4 of them
        dict(name="select prefill 512 groups", op="select", hq=32, hk=8, d=128, groups=512, n_q=4, ctx=34816,
             budget=32, shared=True),
        # one user's decode step over 32 pages: the smallest call
        dict(name="attend 1x32 pages", op="attend", fmt="bf16", hq=32, hk=8, d=128, groups=1, n_q=1, ctx=16384,
             budget=32, shared=False),
        # a decode step of 32 users on a global layer of the Gemma-class model, its default NVFP4 cache
        dict(name="attend 32x64 pages hd512", op="attend", fmt="nvfp4", hq=32, hk=16, d=512, groups=32, n_q=1,
             ctx=8192, budget=64, shared=False),
        # speculative verify of 16 users over an FP8 cache
        dict(name="attend verify 16x45 pages", op="attend", fmt="fp8", hq=32, hk=8, d=128, groups=16, n_q=4,
             ctx=16001, budget=45, shared=False),
        # a prefill chunk of 2048 tokens of one request over a bf16 cache, 4 tokens to a list
        dict(name="attend prefill 512 groups", op="attend", fmt="bf16", hq=32, hk=8, d=128, groups=512, n_q=4,
             ctx=34816, budget=32, shared=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "select", "attend"])
    d = rng.choice([128, 256, 512])
    hk = rng.choice([1, 2, 4, 8, 16])
    g = rng.choice([1, 2, 3, 4, 8, 16])
    c = dict(op=op, hq=hk * g, hk=hk, d=d)
    if op == "append":
        c["fmt"] = rng.choice(["bf16", "fp8"])
        decode = rng.random() < 0.5
        c["reqs"] = _log_int(rng, 1, 200) if decode else rng.randint(1, 9)
        c["tokens"] = rng.choice([1, 1, 3, 4]) if decode else _log_int(rng, 5, 8192 // c["reqs"])
        c["norm"] = rng.random() < 0.5
        return c
    c["n_q"] = rng.choice([n for n in (1, 1, 2, 3, 4, 8, 16) if n * g <= 16])
    c["shared"] = rng.random() < 0.4
    if c["shared"]:
        c["groups"] = _log_int(rng, 2, 300)
        c["ctx"] = _log_int(rng, 200 + c["groups"] * c["n_q"], 30000)
    else:
        c["groups"] = _log_int(rng, 1, 48)
        c["ctx"] = _log_int(rng, 200, 200000 // c["groups"] if op == "attend" else 120000)
    c["budget"] = _log_int(rng, 4, 96)
    if op == "attend":
        c["fmt"] = rng.choice(["bf16", "fp8", "nvfp4"])
        # keep below the largest listed case: listed pages x kv heads x values
        while c["groups"] * c["budget"] * hk * d > 8_000_000:
            c["groups"] = max(1, c["groups"] // 2)
        if c["shared"] and c["groups"] < 2:
            c["shared"] = False
    elif c["shared"]:
        while c["groups"] * hk * d * c["ctx"] > 512 * 8 * 128 * 34816:
            c["groups"] = max(1, c["groups"] // 2)
        c["shared"] = c["groups"] > 1
    return c


def _row_bytes(fmt, d):
    return {"bf16": 2 * d, "fp8": d, "nvfp4": d // 2}[fmt]


def _part_bytes(fmt, d):
    return PAGE * (_row_bytes(fmt, d) + (d // 16 if fmt == "nvfp4" else 0))


def _lengths(case):
    """Tokens in the cache of each group, the group's own included: ragged for users, consecutive for a prefill."""
    n, n_q, ctx = case["groups"], case["n_q"], case["ctx"]
    if case["shared"]:
        return [ctx - (n - 1 - i) * n_q for i in range(n)]
    ln = [max(1, ctx - (i * 7919) % max(1, (2 * ctx) // 3)) for i in range(n)]
    if n >= 8:
        ln[-1] = 0                 # a padding row of a batch: nothing to see
    return ln


def _table(case, lens, gen):
    """Page table with a spare row in front, request rows and the number of pages of the pool (page 0 unused)."""
    per = [(x + PAGE - 1) // PAGE for x in lens]
    rows = [max(per)] if case["shared"] else per
    width = max(rows) + 1
    total = sum(rows) + 1
    perm = torch.randperm(total - 1, generator=gen, device="cuda").to(torch.int32) + 1
    table = torch.zeros(len(rows) + 1, width, dtype=torch.int32, device="cuda")
    at = 0
    for i, m in enumerate(rows):
        table[i + 1, :m] = perm[at:at + m]
        at += m
    req = torch.ones(len(lens), dtype=torch.int32, device="cuda") if case["shared"] else \
        torch.arange(1, len(lens) + 1, dtype=torch.int32, device="cuda")
    return table, req, total


def _fill_pool(total, hk, fmt, d, gen):
    pool = torch.empty(total, hk, 2, _part_bytes(fmt, d), dtype=torch.uint8, device="cuda")
    if fmt == "bf16":
        pool.view(torch.bfloat16).normal_(generator=gen)
        return pool
    pool.random_(0, 256, generator=gen)
    if fmt == "fp8":
        pool.bitwise_and_(0xBF)                              # |x| < 2
    else:
        sc = pool[..., PAGE * d // 2:]
        sc.bitwise_and_(0x0F).bitwise_or_(0x28)              # block scales 0.25 .. 0.47
    return pool


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dev, d, hq, hk = "cuda", case["d"], case["hq"], case["hk"]
    s = dict(case)
    if case["op"] == "append":
        n, m, fmt = case["reqs"], case["tokens"], case["fmt"]
        t = n * m
        start = torch.randint(0, 1000, (n,), generator=gen, device=dev)
        start[0] = 127 if m == 1 else start[0]               # one request finishes a page in a decode step
        pages = (1000 + m) // PAGE + 2
        first = (start // PAGE)[:, None]
        pos = start[:, None] + torch.arange(m, device=dev)[None]
        # the pages from each request's first written one on, in random order in the pool
        per = (m + PAGE - 1) // PAGE + 1
        perm = torch.randperm(n * per, generator=gen, device=dev).view(n, per) + 1
        page = torch.gather(perm, 1, pos // PAGE - first)
        s["pos"] = pos.reshape(-1).to(torch.int32)
        s["slot"] = (page * PAGE + pos % PAGE).reshape(-1).to(torch.int32)
        s["qkv"] = torch.randn(t, (hq + 2 * hk) * d, generator=gen, device=dev).to(torch.bfloat16)
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = (torch.randn(2, d, generator=gen, device=dev) * 0.1).to(torch.bfloat16)
        inv = 1e6 ** (-torch.arange(d // 2, dtype=torch.float64, device=dev) * 2 / d)
        ang = torch.arange(pages * PAGE, dtype=torch.float64, device=dev)[:, None] * inv
        s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], -1).to(torch.float32)
        s["pool"] = _fill_pool(n * per + 1, hk, fmt, d, gen)
        s["codes"] = torch.zeros(n * per + 1, hk, 2, d, dtype=torch.int8, device=dev)
        s["scale"] = torch.zeros(n * per + 1, hk, dtype=torch.bfloat16, device=dev)
        return s
    lens = _lengths(case)
    s["kv_len"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["table"], s["req_idx"], total = _table(case, lens, gen)
    t = case["groups"] * case["n_q"]
    s["q"] = (torch.randn(t, hq, d, generator=gen, device=dev) * 2).to(torch.bfloat16)
    if case["op"] == "select":
        s["codes"] = torch.empty(total, hk, 2, d, dtype=torch.int8, device=dev)
        s["codes"][:, :, 0] = (torch.randn(total, hk, d, generator=gen, device=dev) * 20).round().clamp(-127, 127)
        s["codes"][:, :, 1] = torch.randint(20, 128, (total, hk, d), generator=gen, device=dev)
        s["scale"] = torch.exp2(torch.randint(-7, -3, (total, hk), generator=gen, device=dev).float()).bfloat16()
        return s
    s["pool"] = _fill_pool(total, hk, case["fmt"], d, gen)
    # distinct pages of each group, ascending, its last page among them, -1 behind them
    npg = (s["kv_len"] + PAGE - 1) // PAGE
    width = s["table"].shape[1]
    pick = torch.rand(case["groups"], hk, width, generator=gen, device=dev)
    at = torch.arange(width, device=dev)
    pick = torch.where(at >= npg[:, None, None], 2.0, pick)
    pick = torch.where(at == npg[:, None, None] - 1, -1.0, pick)
    order = pick.argsort(-1)[..., :case["budget"]]
    order = torch.where(order < npg[:, None, None], order, width).sort(-1).values
    order = torch.where(order < width, order, -1).to(torch.int32)
    if order.shape[-1] < case["budget"]:
        order = torch.nn.functional.pad(order, (0, case["budget"] - order.shape[-1]), value=-1)
    s["blocks"] = order.contiguous()
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _chunk_perm(rb, dev):
    """[64, rb / 16]: where chunk j of row r is stored."""
    n = min(8, rb // 16)
    j = torch.arange(rb // 16, device=dev)[None]
    r = torch.arange(PAGE, device=dev)[:, None]
    return (j & ~(n - 1)) | ((j ^ r) & (n - 1))


def _decode_part(part, fmt, d, scale):
    """uint8 [..., part bytes] -> fp32 [..., 64, D]."""
    rb = _row_bytes(fmt, d)
    rows = part[..., :PAGE * rb].unflatten(-1, (PAGE, rb // 16, 16))
    r = torch.arange(PAGE, device=part.device)[:, None]
    rows = rows[..., r, _chunk_perm(rb, part.device), :].flatten(-2)
    if fmt == "bf16":
        return rows.view(torch.bfloat16).float()
    if fmt == "fp8":
        return rows.view(torch.float8_e4m3fn).float() * scale
    lut = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=part.device)
    pair = torch.stack([rows & 15, rows >> 4], -1).flatten(-2)
    sc = part[..., PAGE * rb:].unflatten(-1, (PAGE, d // 16)).view(torch.float8_e4m3fn).float() * scale
    return (lut[pair.int()].unflatten(-1, (d // 16, 16)) * sc[..., None]).flatten(-2)


def _scales(fmt):
    return (1.0, 1.0) if fmt == "bf16" else (K_SCALE, V_SCALE)


def _pow2(amax):
    """2^e of the 8-bit codes of values up to amax: amax 2^-e in [64, 128)."""
    _, x = torch.frexp(amax)
    return torch.exp2((x.float() - 7).clamp(-100, 100))


def _plain_append(s):
    d, hq, hk, fmt = s["d"], s["hq"], s["hk"], s["fmt"]
    x = s["qkv"].float().unflatten(1, (hq + 2 * hk, d))

    def norm(v, w):
        if w is None:
            return v
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * (1.0 + w.float())

    cs = s["cos_sin"][s["pos"].long()][:, None]
    cos, sin = cs[..., :d // 2], cs[..., d // 2:]

    def rope(v):
        a, b = v[..., :d // 2], v[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    q = rope(norm(x[:, :hq], s["q_norm"])).to(torch.bfloat16)
    k, v = rope(norm(x[:, hq:hq + hk], s["k_norm"])), x[:, hq + hk:]
    ks, vs = _scales(fmt)
    kv = torch.stack([k / torch.full((), ks, device=k.device), v / torch.full((), vs, device=k.device)], 2)
    kv = kv.to(torch.bfloat16 if fmt == "bf16" else torch.float8_e4m3fn).view(torch.uint8)      # [T, Hk, 2, rb]
    rb = _row_bytes(fmt, d)
    slot = s["slot"].long()
    page, off = slot // PAGE, slot % PAGE
    rows = s["pool"].view(-1, hk, 2, PAGE, rb // 16, 16)
    perm = _chunk_perm(rb, kv.device)[off]                                                      # [T, chunks]
    rows.permute(0, 3, 4, 1, 2, 5)[page[:, None], off[:, None], perm] = \
        kv.unflatten(-1, (rb // 16, 16)).permute(0, 3, 1, 2, 4)
    done = page[off == PAGE - 1]
    key = _decode_part(s["pool"][done][:, :, 0], fmt, d, ks)                                      # [n, Hk, 64, D]
    lo, hi = key.amin(2), key.amax(2)
    c, w = (lo + hi) * 0.5, (hi - lo) * 0.5
    sc = _pow2(torch.maximum(c.abs(), w).amax(-1, keepdim=True))
    s["codes"][done] = torch.stack([c, w], 2).div(sc[..., None]).round().clamp(-127, 127).to(torch.int8)
    s["scale"][done] = sc[..., 0].to(torch.bfloat16)
    return q


def _plain_select(s):
    d, hk, n_q, budget = s["d"], s["hk"], s["n_q"], s["budget"]
    b = s["kv_len"].shape[0]
    q = s["q"].float().view(b, n_q, hk, -1, d).transpose(1, 2).flatten(2, 3)                     # [B, Hk, R, D]
    sq = _pow2(q.abs().amax(-1, keepdim=True))
    q8 = (q / sq).round().clamp(-127, 127)
    pt = s["table"][s["req_idx"].long()].long()                                                   # [B, N]
    rec = s["codes"][pt].float().permute(0, 2, 1, 3, 4).flatten(3)                                # [B, Hk, N, 2 D]
    score = torch.matmul(torch.cat([q8, q8.abs()], -1), rec.transpose(2, 3))                     # whole numbers
    score = (score * sq).amax(2) * s["scale"][pt].float().transpose(1, 2)                         # [B, Hk, N]
    length = s["kv_len"].long()[:, None, None]
    at = torch.arange(pt.shape[1], device=q.device)
    npg = (length + PAGE - 1) // PAGE
    first_local = (length - n_q).clamp(min=0) // PAGE
    score = torch.where((at < 1) | (at >= first_local), math.inf, score)
    score = torch.where(at >= npg, -math.inf, score)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    order = torch.where(order < npg, order, pt.shape[1]).sort(-1).values
    blocks = torch.where(order < npg, order, -1)
    if blocks.shape[-1] < budget:
        blocks = torch.nn.functional.pad(blocks, (0, budget - blocks.shape[-1]), value=-1)
    return blocks.to(torch.int32), (blocks >= 0).sum(-1).to(torch.int32)


def _plain_attend(s):
    d, hk, n_q, fmt = s["d"], s["hk"], s["n_q"], s["fmt"]
    b = s["kv_len"].shape[0]
    g = s["hq"] // hk
    blocks = s["blocks"].long()
    phys = torch.gather(s["table"][s["req_idx"].long()].long(), 1, blocks.clamp(min=0).flatten(1)).view_as(blocks)
    part = s["pool"][phys, torch.arange(hk, device=phys.device)[None, :, None]]                   # [B, Hk, S, 2, bytes]
    ks, vs = _scales(fmt)
    k = _decode_part(part[..., 0, :], fmt, d, ks).flatten(2, 3)
    v = _decode_part(part[..., 1, :], fmt, d, vs).flatten(2, 3)
    pos = (blocks[..., None] * PAGE + torch.arange(PAGE, device=phys.device)).flatten(2)          # [B, Hk, S * 64]
    listed_ = (blocks >= 0)[..., None].expand(*blocks.shape, PAGE).flatten(2)
    q = s["q"].float().view(b, n_q, hk, g, d).permute(0, 2, 1, 3, 4)                              # [B, Hk, n_q, G, D]
    q_pos = s["kv_len"].long()[:, None] - n_q + torch.arange(n_q, device=phys.device)             # [B, n_q]
    see = listed_[:, :, None] & (pos[:, :, None] <= q_pos[:, None, :, None])                      # [B, Hk, n_q, S * 64]
    x = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)) * d ** -0.5
    x = x.unflatten(2, (n_q, g)).masked_fill(~see[:, :, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (n_q, g)) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total))[..., 0]
    return o.permute(0, 2, 1, 3, 4).reshape(b * n_q, s["hq"], d).to(torch.bfloat16), \
        lse.permute(0, 2, 1, 3).reshape(b * n_q, s["hq"])


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    d, hq, hk = s["d"], s["hq"], s["hk"]
    if own:
        from inference_optimizations_b200.ops import block_sparse as bs
    if s["op"] == "append":
        if own:
            q = bs.block_append(s["qkv"], s["q_norm"], s["k_norm"], s["cos_sin"], s["pos"], s["slot"], s["pool"],
                                s["codes"], s["scale"], FMT[s["fmt"]], hq, hk, d, EPS, True, *_scales(s["fmt"]))
        else:
            q = _plain_append(s)
        kind = torch.bfloat16 if s["fmt"] == "bf16" else torch.float8_e4m3fn
        return q, s["pool"].view(kind), s["codes"] * s["scale"][..., None, None]
    if s["op"] == "select":
        if own:
            return bs.block_select(s["q"], s["codes"], s["scale"], s["table"], s["kv_len"], s["n_q"], hk, s["budget"],
                                   req_idx=s["req_idx"])
        return _plain_select(s)
    if own:
        return bs.block_decode(s["q"], s["pool"], s["table"], s["kv_len"], s["blocks"], s["n_q"], hk, FMT[s["fmt"]],
                               d ** -0.5, *_scales(s["fmt"]), req_idx=s["req_idx"])
    return _plain_attend(s)


def work(case):
    d, hq, hk = case["d"], case["hq"], case["hk"]
    if case["op"] == "append":
        t, eb = case["reqs"] * case["tokens"], 2 if case["fmt"] == "bf16" else 1
        done = t / PAGE
        return {"bytes": t * ((hq + 2 * hk) * d * 2 + hq * d * 2 + 2 * hk * d * eb + 4 * d + 8) + done * hk * (2 * d + 2),
                "flops": t * (hq + 2 * hk) * d * 10}
    lens, n_q = _lengths(case), case["n_q"]
    rows = n_q * hq // hk
    pages = [(x + PAGE - 1) // PAGE for x in lens]
    t = case["groups"] * n_q
    if case["op"] == "select":
        cand = sum(pages)
        read = max(pages) if case["shared"] else cand
        return {"bytes": read * (hk * (2 * d + 2) + 4) + t * hq * d * 2 + case["groups"] * hk * (case["budget"] + 1) * 4,
                "flops": cand * hk * rows * 4 * d}
    per = _part_bytes(case["fmt"], d) * 2 / PAGE
    seen = sum(min(x, case["budget"] * PAGE) for x in lens)
    read = min(seen, max(lens)) if case["shared"] else seen
    return {"bytes": read * hk * per + t * hq * (4 * d + 4) + case["groups"] * hk * case["budget"] * 4,
            "flops": seen * hk * rows * 4 * d}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _stored_row(values, off, chunk):
    """values [T, Hk, D] of rows at offsets off [T], in the order they are stored; chunk = values in 16 bytes."""
    t, hk, d = values.shape
    n = min(8, d // chunk)
    out = torch.empty_like(values)
    for j in range(d // chunk):
        to = (j & ~(n - 1)) | ((j ^ off) & (n - 1))
        src = values[:, :, j * chunk:(j + 1) * chunk]
        idx = (to[:, None] * chunk + torch.arange(chunk, device=values.device))[:, None].expand(t, hk, chunk)
        out.scatter_(2, idx, src)
    return out


def exact(case, seed):
    if case["op"] == "select":
        return None
    s = prepare(case, seed)
    d, hq, hk, fmt = case["d"], case["hq"], case["hk"], case["fmt"]
    g, ks, vs = hq // hk, *_scales(fmt)
    if case["op"] == "append":
        t = s["qkv"].shape[0]
        heads = s["qkv"].double().reshape(t, hq + 2 * hk, d)
        half = d // 2
        ang = s["cos_sin"].double()[s["pos"].long()]
        turn = torch.complex(ang[:, :half], ang[:, half:])[:, None]

        def prepared(h, w):
            if w is not None:
                h = h / torch.sqrt((h * h).sum(-1, keepdim=True) / d + EPS) * (w.double() + 1)
            z = torch.complex(h[..., :half], h[..., half:]) * turn
            return torch.cat([z.real, z.imag], -1)

        q = prepared(heads[:, :hq], s["q_norm"])
        k = prepared(heads[:, hq:hq + hk], s["k_norm"])
        chunk = 8 if fmt == "bf16" else 16
        kind = torch.bfloat16 if fmt == "bf16" else torch.float8_e4m3fn
        pool = s["pool"].view(kind).double().view(-1, hk, 2, PAGE, d)
        slot = s["slot"].long()
        page, off = slot // PAGE, slot % PAGE
        pool[page, :, 0, off] = _stored_row(k / ks, off, chunk)
        pool[page, :, 1, off] = _stored_row(heads[:, hq + hk:] / vs, off, chunk)
        bound = torch.zeros(pool.shape[0], hk, 2, d, dtype=torch.float64, device=pool.device)
        back = torch.arange(PAGE, device=pool.device)
        for p in page[off == PAGE - 1].tolist():
            keys = pool[p, :, 0].transpose(0, 1) * ks                        # [64, Hk, D], in storage order
            n = min(8, d // chunk)
            cols = torch.arange(d, device=pool.device)
            j = cols // chunk
            to = ((j & ~(n - 1))[None] | ((j[None] ^ back[:, None]) & (n - 1))) * chunk + (cols % chunk)[None]
            keys = keys.gather(2, to[:, None].expand(PAGE, hk, d))
            lo, hi = keys.min(0).values, keys.max(0).values
            bound[p, :, 0], bound[p, :, 1] = (hi + lo) / 2, (hi - lo) / 2
        return q, pool.view(pool.shape[0], hk, 2, -1), bound
    b, n_q = case["groups"], case["n_q"]
    out = torch.zeros(b, n_q, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, n_q, hq), -math.inf, dtype=torch.float64, device="cuda")
    table, req, blocks, lens = s["table"].tolist(), s["req_idx"].tolist(), s["blocks"].tolist(), s["kv_len"].tolist()
    q = s["q"].double().view(b, n_q, hk, g, d)
    inside = torch.arange(PAGE, device="cuda")
    for h in range(hk):
        keys = _exact_part(s["pool"][:, h, 0], fmt, d).view(-1, PAGE, d) * ks
        vals = _exact_part(s["pool"][:, h, 1], fmt, d).view(-1, PAGE, d) * vs
        for i in range(b):
            use = [x for x in blocks[i][h] if x >= 0]
            if not use:
                continue
            at = torch.tensor([use, [table[req[i]][x] for x in use]], device="cuda")
            pos = (at[0, :, None] * PAGE + inside).flatten()
            now = lens[i] - n_q + torch.arange(n_q, device="cuda")
            x = torch.einsum("tgd,nd->tgn", q[i, :, h], keys[at[1]].flatten(0, 1)) / math.sqrt(d)
            x = torch.where((pos <= now[:, None])[:, None], x, -math.inf)
            z = torch.logsumexp(x, -1, keepdim=True)
            lse[i, :, h * g:(h + 1) * g] = z[..., 0]
            w = torch.where(z > -math.inf, torch.exp(x - z), 0.0)
            out[i, :, h * g:(h + 1) * g] = torch.einsum("tgn,nd->tgd", w, vals[at[1]].flatten(0, 1))
    return out.view(b * n_q, hq, d), lse.view(b * n_q, hq)


def _exact_part(part, fmt, d):
    """uint8 [pages, bytes] -> float64 [pages * 64, D], one row offset at a time."""
    rb = _row_bytes(fmt, d)
    n = min(8, rb // 16)
    rows = []
    for r in range(PAGE):
        raw = part[:, r * rb:(r + 1) * rb]
        raw = torch.cat([raw[:, 16 * ((j & ~(n - 1)) | ((j ^ r) & (n - 1))):][:, :16] for j in range(rb // 16)], 1)
        if fmt == "bf16":
            rows.append(raw.contiguous().view(torch.bfloat16).double())
        elif fmt == "fp8":
            rows.append(raw.contiguous().view(torch.float8_e4m3fn).double())
        else:
            def value(c):
                e, m = (c >> 1) & 3, (c & 1).double()
                mag = torch.where(e == 0, m / 2, torch.exp2(e.double() - 1) * (1 + m / 2))
                return torch.where(c >= 8, -mag, mag)
            sc = part[:, PAGE * rb + r * (d // 16):][:, :d // 16].contiguous().view(torch.float8_e4m3fn).double()
            v = torch.stack([value(raw & 15), value(raw >> 4)], 2).reshape(-1, d)
            rows.append((v.view(-1, d // 16, 16) * sc[..., None]).reshape(-1, d))
    return torch.stack(rows, 1).reshape(-1, d)

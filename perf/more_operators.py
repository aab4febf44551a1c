"""Operators of a decoding step on device tensors: memories in 8 bits, pages that follow their hypotheses, scores of given tokens.

A case is one pass as a translation or language-model server makes it between its own products: put keys and values into 8-bit pages
(and read them back), attend over such pages, let the pages of all hypotheses follow a beam selection or move to the front of their
pool (and copy what has to be copied), and score given tokens.  ``own = False`` computes the operators in elementary torch
operations, ``own = True`` calls ``linmt_b200.device_ops``.

A page tensor is uint8 [pages, heads, positions / 16, 32 * dim + 16], a block of 16 positions of one head: 16 dim bytes of key codes,
16 dim bytes of value codes, the keys' and the values' scale (float32), 8 bytes of zeros.  A code is a signed byte and stands for
code * scale.  The key code of position t and component c is byte (t / 8) * 8 dim + (c / 16) * 128 + (t % 8) * 16 + c % 16, the value code byte 16 c + t.
A scale is the smallest m * 2^e with m of 4, 5, 6, 7 whose 127-fold reaches the largest component.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
INF = float("inf")


def listed():
    return [
        # every hypothesis of a running batch gets its next position, somewhere in a block that is partly full
        dict(name="write8_step", op="write", seqs=768, grow=1, heads=8, dim=64, page=16, dtype="bf16"),
        # the memory of a few long documents, written at once
        dict(name="write8_job", op="write", seqs=9, grow=11113, heads=8, dim=128, page=64, dtype="bf16"),
        # one sentence's beams over its source
        dict(name="attend8_one", op="attend", n=1, g=5, heads=8, rep=1, dim=64, page=16, lo=23, hi=23, dtype="fp32", cap=0.0, bias=False, windows=False, sinks=0),
        # paragraphs: each beam sees its own part of the text and the first four words; capped scores, a bias that falls with the distance
        dict(name="attend8_64", op="attend", n=64, g=12, heads=8, rep=1, dim=128, page=32, lo=1, hi=4001, dtype="fp16", cap=30.0, bias=True, windows=True, sinks=4),
        # whole documents, several queries on each head of the memory
        dict(name="attend8_long", op="attend", n=8, g=4, heads=8, rep=4, dim=128, page=64, lo=20000, hi=32768, dtype="bf16", cap=0.0, bias=False, windows=False, sinks=0),
        # the hypotheses of a running batch, 12 a sentence, follow their parents behind every step; two layers
        dict(name="fork_64", op="fork", n=64, k=12, page=16, lo=20, hi=90, heads=8, dim=64, layers=2, done=0.05),
        # a large job of long hypotheses
        dict(name="fork_256", op="fork", n=256, k=8, page=32, lo=100, hi=1500, heads=2, dim=64, layers=2, done=0.1),
        # a small pool is made dense again
        dict(name="compact_64", op="compact", n=64, page=16, lo=1, hi=400, live=0.6, heads=8, dim=64),
        # a large one, before part of it is given back
        dict(name="compact_1024", op="compact", n=1024, page=32, lo=1, hi=1500, live=0.5, heads=4, dim=64),
        # the next word of one sentence on the small model
        dict(name="score_one", op="score", n=1, t=1, v=1000, dtype="fp32", top=5, mask="none", pad=0.0),
        # reference translations of a batch on the headline vocabulary, padded to one length
        dict(name="score_64", op="score", n=64, t=60, v=30000, dtype="fp32", top=0, mask="none", pad=0.3),
        # the large vocabulary in 16 bits, alternatives beside each word, every sentence with a word list of its own
        dict(name="score_lists", op="score", n=48, t=41, v=80000, dtype="bf16", top=10, mask="each", pad=0.1),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["write", "attend", "attend", "fork", "compact", "score"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    dim, page = rng.choice([64, 128]), 16 * rng.randint(1, 8)
    if op == "write":
        heads, seqs = rng.randint(1, 16), _spread(rng, 1, 800)
        most = max(1, 100_000 * 1024 // (heads * dim * seqs))
        return dict(op=op, seqs=seqs, grow=rng.choice([1, _spread(rng, 1, most)]), heads=heads, dim=dim, page=page, dtype=dtype)
    if op == "attend":
        heads, rep, g = rng.randint(1, 8), rng.choice([1, 1, 2, 3, 4]), rng.choice([1, rng.randint(1, 14)])
        n = _spread(rng, 1, 400)
        # what a pass reads and multiplies stays below the largest listed case's
        most = max(1, min(32768, 180_000_000 // (n * heads * dim), 3_000_000_000 // (n * heads * rep * g * dim)))
        lo = _spread(rng, 1, most)
        windows = rng.random() < 0.4
        return dict(op=op, n=n, g=g, heads=heads, rep=rep, dim=dim, page=page, lo=lo, hi=rng.randint(lo, most), dtype=dtype, cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                    bias=rng.random() < 0.3, windows=windows, sinks=rng.choice([0, 1, 4, 130]) if windows else 0)
    heads = rng.randint(1, 8)
    if op == "fork":
        k = rng.randint(1, 16)
        n = _spread(rng, 1, 3000 // k)
        layers = rng.randint(1, 3)
        most = max(page, min(2000, 300_000_000 // (n * k * heads * dim * 2 * layers)))
        lo = _spread(rng, 1, most)
        return dict(op=op, n=n, k=k, page=page, lo=lo, hi=rng.randint(lo, most), heads=heads, dim=dim, layers=layers, done=rng.choice([0.0, 0.1, 0.5]))
    if op == "compact":
        n = _spread(rng, 1, 1500)
        most = max(page, min(4000, 200_000_000 // (n * heads * dim * 2)))
        lo = _spread(rng, 1, most)
        return dict(op=op, n=n, page=page, lo=lo, hi=rng.randint(lo, most), live=rng.uniform(0.2, 0.95), heads=heads, dim=dim)
    v = _spread(rng, 500, 130000)
    rows = _spread(rng, 1, min(4000, 310_000_000 // (v * SIZE[dtype])))
    t = rng.randint(1, min(rows, 60))
    return dict(op=op, n=max(1, rows // t), t=t, v=v, dtype=dtype, top=rng.choice([0, 1, 5, 20]), mask=rng.choice(["none", "none", "one", "each"]), pad=rng.choice([0.0, 0.2]))


# ---- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * (seed + 1))
    return g


def _lengths(case, gen):
    """Lengths spread evenly between two bounds, in any order."""
    lens = torch.linspace(case["hi"], case["lo"], case["n"], device="cuda", dtype=torch.float64).round().to(torch.int32)
    return lens[torch.randperm(case["n"], device="cuda", generator=gen)]


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _bytes(gen, *shape):
    return torch.randint(0, 256, shape, device="cuda", generator=gen, dtype=torch.uint8)


def prepare(case, seed):
    gen, op = _gen(seed), case["op"]
    if op == "write":
        seqs, grow, heads, dim, page = (case[x] for x in ("seqs", "grow", "heads", "dim", "page"))
        # a sequence has positions already where it grows by steps; those of its last block have been written
        old = torch.randint(0, 4 * page, (seqs,), device="cuda", generator=gen) if grow <= 64 else torch.zeros(seqs, dtype=torch.int64, device="cuda")
        width = (4 * page + grow + page - 1) // page
        table = torch.randperm(seqs * width, device="cuda", generator=gen).view(seqs, width)
        pos = old[:, None] + torch.arange(grow, device="cuda")
        slots = (torch.gather(table, 1, pos // page) * page + pos % page).flatten()
        before = old[:, None] // 16 * 16 + torch.arange(16, device="cuda")                 # the block that the first new position falls into
        before = torch.where(before < old[:, None], torch.gather(table, 1, before // page) * page + before % page, -1)
        kv = [_normal(gen, seqs * grow, heads, dim).to(TYPES[case["dtype"]]) for _ in range(2)]
        kv[0] = kv[0] + _normal(gen, heads, dim).to(kv[0].dtype)                            # keys have offsets of their own in every component
        past = [_normal(gen, seqs, 16, heads, dim) for _ in range(2)]
        pages = torch.zeros(seqs * width, heads, page // 16, 32 * dim + 16, dtype=torch.uint8, device="cuda")
        at = torch.where(before[:, 0] >= 0, before[:, 0], 0)
        keep = (before >= 0)[:, :, None, None]
        block = _pack(*[torch.where(keep, x, 0.0).transpose(1, 2) for x in past])           # [seqs, heads, 1, bytes]
        pages[at // page, :, at % page // 16] = torch.where((before[:, 0] >= 0)[:, None, None], block[:, :, 0], pages[at // page, :, at % page // 16])
        read = torch.cat([before.flatten(), slots])
        return dict(case, kv=kv, slots=slots, pages=pages, old=old, before=before, read=read)
    if op == "attend":
        n, g, heads, rep, dim, page = (case[x] for x in ("n", "g", "heads", "rep", "dim", "page"))
        lens = _lengths(case, gen)
        width = (case["hi"] + page - 1) // page
        n_pages = n * width + 1
        table = torch.randperm(n_pages, device="cuda", generator=gen)[:n * width].to(torch.int32).view(n, width)
        k, v = _normal(gen, n_pages, heads, page, dim), _normal(gen, n_pages, heads, page, dim)
        k += _normal(gen, heads, 1, dim) * 0.5
        q = _normal(gen, n, g, heads * rep, dim).mul_(1.5).to(TYPES[case["dtype"]])
        s = dict(case, q=q, pages=_pack(k, v), table=table, lens=lens, scale=dim ** -0.5, slope=None, centre=None, first=None, last=None)
        if case["bias"]:
            s["slope"] = 2.0 ** (-8.0 * (torch.arange(heads * rep, device="cuda") + 1) / (heads * rep))
            s["centre"] = torch.rand(n, g, device="cuda", generator=gen) * lens[:, None]
        if case["windows"]:
            a, b = (torch.rand(n, g, device="cuda", generator=gen) * (lens[:, None] + 1) for _ in range(2))
            s["first"], s["last"] = torch.minimum(a, b).to(torch.int32), torch.maximum(a, b).to(torch.int32)
        return s
    if op == "fork":
        n, k, page = case["n"], case["k"], case["page"]
        lens = _lengths(case, gen)[:, None].expand(n, k).contiguous()
        width = (case["hi"] + page - 1) // page
        # hypotheses of a sentence share the pages of their common past and have the later ones for themselves
        common = (torch.rand(n, device="cuda", generator=gen) * (lens[:, 0] // page + 1)).long()
        col = torch.arange(width, device="cuda")
        have = (lens + page - 1) // page
        named = col < have[..., None]
        shared = (col < common[:, None])[:, None, :]
        owner = named & (~shared | (torch.arange(k, device="cuda") == 0)[None, :, None])    # the places that have a page of their own
        count = int(owner.sum())
        n_pages = int(have.sum()) + n * k // 2 + 8
        order = torch.randperm(n_pages, device="cuda", generator=gen)
        number = (owner.flatten().cumsum(0) - 1).view(n, k, width).clamp(min=0)
        number = torch.where(shared, number[:, :1], number)
        table = torch.where(named, order[number], -1).to(torch.int32)
        shares = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        both = shared[:, 0] & named[:, 0]
        shares[table[:, 0][both].long()] = k - 1
        parents = torch.minimum(*(torch.randint(0, k, (n, k), device="cuda", generator=gen, dtype=torch.int32) for _ in range(2)))
        done = torch.rand(n, k, device="cuda", generator=gen) < case["done"]
        pools = [_bytes(gen, n_pages, case["heads"], page // 16, 32 * case["dim"] + 16) for _ in range(case["layers"])]
        return dict(case, table=table, lens=lens, parents=parents, done=done, shares=shares, free=order.to(torch.int32), used=torch.tensor([count], dtype=torch.int32, device="cuda"), pools=pools)
    if op == "compact":
        n, page = case["n"], case["page"]
        lens = _lengths(case, gen)[:, None].contiguous()
        width = (case["hi"] + page - 1) // page
        named = torch.arange(width, device="cuda") < (lens + page - 1)[..., None] // page
        count = int(named.sum())
        n_pages = int(count / case["live"]) + 1
        order = torch.randperm(n_pages, device="cuda", generator=gen)
        table = torch.where(named, order[(named.flatten().cumsum(0) - 1).view(n, 1, width).clamp(min=0)], -1).to(torch.int32)
        shares = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        return dict(case, table=table, lens=lens, shares=shares, pools=[_bytes(gen, n_pages, case["heads"], page // 16, 32 * case["dim"] + 16)])
    n, t, v = case["n"], case["t"], case["v"]
    logits = _normal(gen, n, t, v).mul_(1.5)
    best = torch.randint(0, v, (n, t, 24), device="cuda", generator=gen)                    # the words that a trained model raises
    logits.scatter_add_(2, best, _normal(gen, n, t, 24).abs_().mul_(3.0))
    tokens = torch.where(torch.rand(n, t, device="cuda", generator=gen) < 0.5, best[..., 0], torch.randint(0, v, (n, t), device="cuda", generator=gen))
    length = (t * (1.0 - case["pad"] * torch.rand(n, 1, device="cuda", generator=gen))).ceil()
    tokens = torch.where(torch.arange(t, device="cuda") < length, tokens, -1).to(torch.int32)
    allowed = None
    if case["mask"] != "none":
        bits = torch.randint(0, 2 ** 32, (2, n if case["mask"] == "each" else 1, (v + 31) // 32), device="cuda", generator=gen)
        allowed = (bits[0] | bits[1]).to(torch.int64)                                       # three words of four
        allowed = torch.where(allowed >= 2 ** 31, allowed - 2 ** 32, allowed).to(torch.int32)
    return dict(case, logits=logits.to(TYPES[case["dtype"]]), tokens=tokens, allowed=allowed)


# ---- the 8-bit form

def _scale(big):
    """The smallest 4, 5, 6 or 7 times a power of 2 whose 127-fold reaches `big` (float32), 2^-126 at least; 0 for 0."""
    m, e = torch.frexp(big.double() / 127.0)
    s = torch.ldexp(torch.ceil(m * 8.0) / 8.0, e).clamp(min=2.0 ** -126)
    return torch.where(big > 0, s, 0.0).float()


def _codes(x, scale):
    """Codes of x for a scale."""
    return torch.where(scale == 0, 0.0, torch.round(x / torch.where(scale == 0, 1.0, scale)))


def _clean(x):
    x = x.float()
    return torch.where(torch.isnan(x), 0.0, x).clamp(-2.0 ** 127, 2.0 ** 127)


def _pack(k, v):
    """Blocks [pages, heads, positions / 16, 32 dim + 16] of k, v [pages, heads, positions, dim]."""
    p, h, t, d = k.shape
    parts, scales = [], []
    for x, keys in ((k, True), (v, False)):
        x = _clean(x).view(p, h, t // 16, 16, d)
        s = _scale(x.abs().amax((-1, -2)))
        c = _codes(x, s[..., None, None]).to(torch.int8).view(torch.uint8)
        c = c.view(p, h, t // 16, 2, 8, d // 16, 16).transpose(4, 5) if keys else c.transpose(-1, -2)
        parts.append(c.reshape(p, h, t // 16, 16 * d))
        scales.append(s)
    tail = torch.stack(scales + [torch.zeros_like(scales[0])] * 2, dim=-1).contiguous().view(torch.uint8)
    return torch.cat(parts + [tail], dim=-1)


def _unpack(pages):
    """Keys and values [pages, heads, positions, dim] in float32."""
    p, h, n, b = pages.shape
    d = (b - 16) // 32
    kc, vc, tail = pages.split([16 * d, 16 * d, 16], dim=-1)
    s = tail.contiguous().view(torch.float32)
    kc = kc.contiguous().view(torch.int8).view(p, h, n, 2, d // 16, 8, 16).transpose(4, 5).reshape(p, h, n, 16, d).float()
    vc = vc.contiguous().view(torch.int8).view(p, h, n, d, 16).transpose(3, 4).float()
    return (kc * s[..., 0, None, None]).flatten(2, 3), (vc * s[..., 1, None, None]).flatten(2, 3)


# ---- the operators in plain form

def _write(s):
    """The values that the blocks stand for behind the write: of the positions before, and of those written."""
    seqs, grow, page, before, old = s["seqs"], s["grow"], s["page"], s["before"], s["old"]
    heads, dim = s["heads"], s["dim"]
    lead = before[:, 0].clamp(min=0)
    tile = s["pages"][lead // page, :, lead % page // 16][:, :, None]                       # [seqs, heads, 1, bytes]
    past = [x.transpose(1, 2) for x in _unpack(tile)]                                       # [seqs, 16, heads, dim]
    begun = (before[:, 0] >= 0)[:, None]
    scales = tile[:, :, 0, 32 * dim:].contiguous().view(torch.float32)
    # the new positions in blocks of 16: block and place of each, a sequence's first block may be begun
    blocks = (15 + grow + 15) // 16
    at = old[:, None] % 16 + torch.arange(grow, device="cuda")
    out = []
    for i in range(2):
        x = _clean(s["kv"][i]).view(seqs, grow, heads, dim)
        big = torch.zeros(seqs, blocks, heads, device="cuda").scatter_reduce_(1, (at // 16)[..., None].expand(seqs, grow, heads), x.abs().amax(-1), "amax")
        scale = _scale(big)
        scale[:, 0] = torch.where(begun, torch.maximum(scale[:, 0], scales[..., i]), scale[:, 0])
        mine = torch.gather(scale, 1, (at // 16)[..., None].expand(seqs, grow, heads))[..., None]
        first = scale[:, :1, :, None]
        earlier = torch.where((before >= 0)[:, :, None, None], _codes(past[i], first) * first, 0.0)
        out.append(torch.cat([earlier.flatten(0, 1), (_codes(x, mine) * mine).flatten(0, 1)]).to(s["kv"][i].dtype))
    return tuple(out)


def _attend(s):
    n, g, heads, rep, dim = (s[x] for x in ("n", "g", "heads", "rep", "dim"))
    k, v = _unpack(s["pages"])
    k, v = (x[s["table"].long()].transpose(1, 2).flatten(2, 3) for x in (k, v))             # [n, heads, positions, dim]
    q = s["q"].float().view(n, g, heads, rep, dim).permute(0, 2, 1, 3, 4).reshape(n, heads, g * rep, dim)
    x = (q @ k.transpose(2, 3) * s["scale"]).view(n, heads, g, rep, -1)
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    at = torch.arange(x.shape[-1], device=x.device)
    if s["slope"] is not None:
        x = x - s["slope"].view(1, heads, 1, rep, 1) * (at - s["centre"][..., None]).abs()[:, None, :, None, :]
    seen = (at < s["lens"][:, None])[:, None, :].expand(n, g, -1)
    if s["first"] is not None:
        seen = seen & (((at >= s["first"][..., None]) & (at < s["last"][..., None])) | (at < s["sinks"]))
    x = torch.where(seen[:, None, :, None, :], x, -INF)
    top = x.amax(-1, keepdim=True)
    e = (x - torch.where(top == -INF, 0.0, top)).exp()
    total = e.sum(-1, keepdim=True)
    out = (e / torch.where(total == 0, 1.0, total)).view(n, heads, g * rep, -1) @ v
    lse = torch.where(total == 0, -INF, top + total.log()).squeeze(-1)
    return dict(out=out.view(n, heads, g, rep, dim).permute(0, 2, 1, 3, 4).reshape(n, g, heads * rep, dim).to(s["q"].dtype), lse=lse.permute(0, 2, 1, 3).reshape(n, g, heads * rep))


def _named(s):
    """Of every row: the pages that its table names, and which columns do."""
    n, k, width = s["table"].shape
    table, lens, n_pages = s["table"].view(n * k, width).long(), s["lens"].flatten().long(), s["shares"].numel()
    have = ((lens + s["page"] - 1) // s["page"]).clamp(0, width)
    ok = (torch.arange(width, device=table.device) < have[:, None]) & (table >= 0) & (table < n_pages)
    return torch.where(ok, table, n_pages), ok, have, lens.clamp(0, width * s["page"])


def _listed(values, here, size):
    """values[i] of the places where `here` holds, in order, -1 behind the last."""
    at = torch.where(here, here.cumsum(0) - 1, size)
    return torch.full((size + 1,), -1, dtype=torch.int64, device=values.device).scatter_(0, at, values)[:size]


def _copy(pools, src, dst):
    ok = (src >= 0) & (dst >= 0)
    one = ok.long().argmax(keepdim=True)                     # entries that copy nothing do what another does once more
    some = ok.any()
    src, dst = (torch.where(ok, x, torch.where(some, x[one], 0)) for x in (src, dst))
    for pool in pools:
        pool[dst] = pool[src]


def _fork(s):
    n, k, width = s["table"].shape
    rows, n_pages, n_free = n * k, s["shares"].numel(), s["free"].numel()
    dev = s["table"].device
    table, ok, have, lens = _named(s)
    row = torch.arange(rows, device=dev)
    parents = s["parents"].flatten().long()
    parent = torch.where((parents >= 0) & (parents < k) & ~s["done"].flatten(), row // k * k + parents, rows)
    children = torch.zeros(rows + 1, dtype=torch.int64, device=dev).scatter_add_(0, parent, torch.ones_like(parent))[:rows]
    first = torch.full((rows + 1,), rows, dtype=torch.int64, device=dev).scatter_reduce_(0, parent, row, "amin")
    col = torch.arange(width, device=dev)
    half = (lens % s["page"] != 0)[:, None] & (col == have[:, None] - 1)                     # the place of a page that is not full
    more = torch.where(half, children.clamp(max=1)[:, None], children[:, None]) - 1
    shares = torch.cat([s["shares"].long(), torch.zeros(1, dtype=torch.int64, device=dev)])
    shares = shares.scatter_add_(0, table.flatten(), torch.where(ok, more, 0).flatten())[:n_pages]
    gone = shares < 0
    base = s["used"].long().clamp(0, n_free)
    start = (base - gone.sum()).clamp(min=0)
    at = base - gone.sum() + gone.cumsum(0) - 1
    at = torch.where(gone & (at >= 0), at, n_free)
    free = torch.cat([s["free"].long(), s["free"].new_zeros(1).long()]).scatter_(0, at, torch.arange(n_pages, device=dev))[:n_free]
    # children take their parent's row; all but the first of a parent whose last page is not full get a page for a copy of it
    lives = parent < rows
    up = parent.clamp(max=rows - 1)
    new = torch.where(lives[:, None] & ok[up], table[up], -1)
    last = torch.gather(torch.where(half & ok, table, -1), 1, (have - 1).clamp(min=0)[:, None])[:, 0][up]
    copies = lives & (last >= 0) & (first[parent] != row)
    at = start + copies.cumsum(0) - 1
    fresh = torch.where(at < n_free, free[at.clamp(max=n_free - 1)], -1)
    new = torch.where(copies[:, None] & (col == have[up][:, None] - 1), fresh[:, None], new)
    src, dst = _listed(last, copies, rows), _listed(fresh, copies, rows)
    _copy(s["pools"], src, dst)
    i32 = torch.int32
    return dict(table=new.view(n, k, width).to(i32), lens=torch.where(lives, lens[up], 0).view(n, k).to(i32), shares=shares.clamp(min=0).to(i32), free=free.to(i32),
                used=(start + copies.sum()).to(i32), src=src.to(i32), dst=dst.to(i32), pools=s["pools"])


def _compact(s):
    n, k, width = s["table"].shape
    n_pages = s["shares"].numel()
    table, ok, _, _ = _named(s)
    dev = table.device
    live = torch.zeros(n_pages + 1, dtype=torch.bool, device=dev).scatter_(0, table.flatten(), True)[:n_pages]
    count = live.sum(0, keepdim=True)
    page = torch.arange(n_pages, device=dev)
    goes, hole = live & (page >= count), ~live & (page < count)
    src, dst = _listed(page, goes, n_pages // 2), _listed(page, hole, n_pages // 2)
    to = torch.where(goes, torch.cat([dst, dst.new_full((1,), -1)])[(goes.cumsum(0) - 1).clamp(0, n_pages // 2)], page)
    shares = torch.zeros(n_pages + 1, dtype=torch.int32, device=dev).scatter_(0, torch.where(live, to, n_pages), s["shares"])[:n_pages]
    _copy(s["pools"], src, dst)
    i32 = torch.int32
    return dict(table=torch.where(ok, to[table.clamp(max=n_pages - 1)], -1).view(n, k, width).to(i32), shares=shares, free=page.to(i32), used=count.to(i32),
                src=src.to(i32), dst=dst.to(i32), pools=s["pools"])


def _score(s):
    x = s["logits"].float()
    v = x.shape[-1]
    if s["allowed"] is not None:
        bit = torch.arange(v, device=x.device)
        ok = (s["allowed"][:, bit // 32] >> (bit % 32).to(torch.int32)) & 1
        x = torch.where(ok[:, None, :] != 0, x, -INF)
    top = x.amax(-1, keepdim=True)
    d = x - top
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    entropy = total.log() - torch.where(e == 0, 0.0, e * d).sum(-1, keepdim=True) / total
    lse = total.log()
    tokens = s["tokens"].long()
    there = (tokens >= 0) & (tokens < v)
    logprob = torch.where(there, (torch.gather(d, -1, tokens.clamp(0, v - 1)[..., None]) - lse)[..., 0], 0.0)
    out = dict(logprob=logprob, entropy=entropy[..., 0])
    if s["top"]:
        best, at = torch.sort(x, dim=-1, descending=True, stable=True)
        best, at = best[..., :s["top"]], at[..., :s["top"]]
        out["top_tokens"] = torch.where(best == -INF, -1, at).to(torch.int32)
        out["top_logprobs"] = (best - top) - lse
    return out


def run(state):
    s, op = state, state["op"]
    if own:
        from linmt_b200 import device_ops as ops
        if op == "write":
            ops.write_pages8(s["pages"], s["slots"], s["kv"][0], s["kv"][1])
            return ops.read_pages8(s["pages"], s["read"], dtype=s["kv"][0].dtype)
        if op == "attend":
            out, lse = ops.attend_pages8(s["q"], s["pages"], s["table"], s["lens"], scale=s["scale"], cap=s["cap"], slope=s["slope"], centre=s["centre"],
                                         first=s["first"], last=s["last"], sinks=s["sinks"], want_lse=True)
            return dict(out=out, lse=lse)
        if op == "fork":
            table, lens, shares, free, used, src, dst = ops.fork_pages(s["table"], s["lens"], s["parents"], s["shares"], s["free"], s["used"], page=s["page"], done=s["done"])
            return dict(table=table, lens=lens, shares=shares, free=free, used=used, src=src, dst=dst, pools=ops.copy_pages(s["pools"], src, dst))
        if op == "compact":
            table, shares, free, used, src, dst = ops.compact_pages(s["table"], s["lens"], s["shares"], page=s["page"])
            return dict(table=table, shares=shares, free=free, used=used, src=src, dst=dst, pools=ops.copy_pages(s["pools"], src, dst))
        names = ("logprob", "entropy", "top_tokens", "top_logprobs")
        return dict(zip(names, ops.score_tokens(s["logits"], s["tokens"], allowed=s["allowed"], top=s["top"])))
    return dict(write=_write, attend=_attend, fork=_fork, compact=_compact, score=_score)[op](s)


# ---- what a pass cannot do without

def work(case):
    op, size = case["op"], SIZE.get(case.get("dtype"), 4)
    if op == "write":
        written = case["seqs"] * case["grow"]
        begun = case["seqs"] * 7.5 if case["grow"] <= 64 else 0                              # positions before, in blocks that are begun
        one = 2 * case["heads"] * case["dim"]
        return dict(bytes=written * one * (2 * size + 2) + begun * one * (size + 3) + 16 * written, flops=(written + begun) * one * 4)
    if op == "attend":
        n, g, heads, rep, dim = (case[x] for x in ("n", "g", "heads", "rep", "dim"))
        at = n * (case["lo"] + case["hi"]) / 2
        seen = every = 1.0
        if case["windows"]:                                                                  # two even draws enclose a third of the text, 2 g of them more
            seen, every = 1 / 3, (2 * g - 1) / (2 * g + 1)
        return dict(bytes=at * every * heads * (2 * dim + 1) + n * g * heads * rep * (dim * 2 * size + 4), flops=at * seen * heads * rep * g * dim * 4)
    if op == "score":
        rows, v = case["n"] * case["t"], case["v"]
        lists = {"none": 0, "one": 1, "each": case["n"]}[case["mask"]] * v / 8
        return dict(bytes=rows * v * size + lists + rows * (12 + 8 * case["top"]), flops=rows * v * 5)
    page = case["heads"] * case["page"] * (2 * case["dim"] + 1)
    length = (case["lo"] + case["hi"]) / 2 / case["page"]
    if op == "fork":
        n, k = case["n"], case["k"]
        lives = 1 - case["done"]
        pages = n * k * length * 0.55                                                        # half of a hypothesis' pages are common to its sentence
        copies = n * k * lives * 0.5 * (case["page"] - 1) / case["page"]                     # some half of the children are not their parent's first
        return dict(bytes=2 * copies * case["layers"] * page + 4 * (2 * n * k * length + 3 * n * k + 4 * pages + 2 * n * k), flops=0)
    pages = case["n"] * (length + 0.5)
    return dict(bytes=2 * pages * (1 - case["live"]) * page + 4 * pages * (2 + 4 / case["live"]), flops=0)


# ---- the definitions in 64 bits

def _exact_codes(x, scale):
    return torch.where(scale == 0, 0.0, torch.round(x / torch.where(scale == 0, 1.0, scale)).clamp(-127, 127) * scale)


def _exact_scale(big):
    """By trying: the smallest of the scales around big / 127 that is large enough."""
    e = torch.floor(torch.log2(big.clamp(min=1e-300) / 127.0)) - 1
    found = torch.zeros_like(big)
    for step in range(15, -1, -1):
        s = (4 + step % 4) / 4 * torch.exp2(e + step // 4)
        found = torch.where(127.0 * s >= big, s, found)
    return torch.where(big == 0, 0.0, found.clamp(min=2.0 ** -126))


def _exact_block(block, dim):
    """Keys and values [heads, 16, dim] of one block of each head, each code looked up where the form has it."""
    t, c = torch.arange(16, device="cuda")[:, None], torch.arange(dim, device="cuda")[None, :]
    places = (t // 8 * 8 * dim + c // 16 * 128 + t % 8 * 16 + c % 16, 16 * dim + 16 * c + t)
    scales = block[..., 32 * dim:].contiguous().view(torch.float32).double()
    made = []
    for i, at in enumerate(places):
        code = block[..., at].to(torch.int64)
        made.append(torch.where(code >= 128, code - 256, code).double() * scales[..., i, None, None])
    return made


def _exact_write(s):
    if s["seqs"] > 2000:
        return None
    page, dim, grow, dtype = s["page"], s["dim"], s["grow"], s["kv"][0].dtype
    outs = ([], [])
    new = ([], [])
    for i in range(s["seqs"]):
        old = int(s["old"][i])
        begun = old % 16
        for j in range(2):
            x = s["kv"][j][i * grow:(i + 1) * grow].double()
            earlier = torch.zeros(16, s["heads"], dim, dtype=torch.float64, device="cuda")
            held = torch.zeros(s["heads"], dtype=torch.float64, device="cuda")
            if begun:
                slot = int(s["before"][i, 0])
                block = s["pages"][slot // page, :, slot % page // 16]
                earlier = _exact_block(block, dim)[j].transpose(0, 1)
                held = block[:, 32 * dim:].contiguous().view(torch.float32)[:, j].double()
            head = x[:16 - begun]
            scale = torch.maximum(_exact_scale(head.abs().amax((0, 2))), held)
            earlier = _exact_codes(earlier, scale[:, None])
            earlier[begun:] = 0.0
            made = [_exact_codes(head, scale[:, None])]
            rest = x[16 - begun:]
            if rest.shape[0]:
                full = torch.cat([rest, rest.new_zeros(-rest.shape[0] % 16, *rest.shape[1:])]).view(-1, 16, s["heads"], dim)
                made.append(_exact_codes(full, _exact_scale(full.abs().amax((1, 3)))[:, None, :, None]).flatten(0, 1)[:rest.shape[0]])
            outs[j].append(earlier)
            new[j].extend(made)
    return tuple(torch.cat(outs[j] + new[j]) for j in range(2))


def _exact_attend(s):
    n, g, heads, rep, dim = (s[x] for x in ("n", "g", "heads", "rep", "dim"))
    out = torch.zeros(n, g, heads * rep, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((n, g, heads * rep), -INF, dtype=torch.float64, device="cuda")
    for i in range(n):
        length = int(s["lens"][i])
        blocks = s["pages"][s["table"][i].long()].transpose(0, 1).flatten(1, 2)                # [heads, blocks, bytes]
        k, v = (x.flatten(1, 2)[:, :length].repeat_interleave(rep, 0) for x in _exact_block(blocks, dim))
        z = torch.einsum("ghd,hpd->ghp", s["q"][i].double(), k) * s["scale"]
        if s["cap"]:
            z = torch.tanh(z / s["cap"]) * s["cap"]
        at = torch.arange(length, device="cuda", dtype=torch.float64)
        if s["slope"] is not None:
            z = z - s["slope"].double()[None, :, None] * (at[None, :] - s["centre"][i].double()[:, None]).abs()[:, None, :]
        if s["first"] is not None:
            hidden = ((at[None, :] < s["first"][i][:, None]) | (at[None, :] >= s["last"][i][:, None])) & (at >= s["sinks"])
            z = z.masked_fill(hidden[:, None, :], -INF)
        lse[i] = torch.logsumexp(z, -1)
        out[i] = torch.einsum("ghp,hpd->ghd", torch.softmax(z, -1).nan_to_num(nan=0.0), v)
    return dict(out=out, lse=lse)


def _exact_score(s):
    n, t, v = s["logits"].shape
    words = torch.arange(v, device="cuda")
    out = dict(logprob=torch.zeros(n, t, dtype=torch.float64, device="cuda"), entropy=torch.zeros(n, t, dtype=torch.float64, device="cuda"))
    if s["top"]:
        out.update(top_tokens=None, top_logprobs=torch.zeros(n, t, s["top"], dtype=torch.float64, device="cuda"))
    for i in range(n):
        z = s["logits"][i].double()
        if s["allowed"] is not None:
            row = s["allowed"][min(i, s["allowed"].shape[0] - 1)].long() & 0xFFFFFFFF
            z[:, ((row.repeat_interleave(32)[:v] >> (words % 32)) & 1) == 0] = -INF
        z = torch.log_softmax(z, dim=-1)
        for j in range(t):
            if 0 <= int(s["tokens"][i, j]) < v:
                out["logprob"][i, j] = z[j, int(s["tokens"][i, j])]
        out["entropy"][i] = -(z.exp() * z.masked_fill(z == -INF, 0.0)).sum(-1)
        if s["top"]:
            out["top_logprobs"][i] = torch.topk(z, s["top"]).values
    return out


def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None
    s = prepare(case, seed)
    return dict(write=_exact_write, attend=_exact_attend, score=_exact_score)[case["op"]](s)

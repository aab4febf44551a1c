"""Operators of a decoding step on device tensors: beam selection and reordering, pages of a memory, attention over it in 4 bits.

A case is one call (a write and the read of what it wrote: two) as a translation or language-model server makes it between its own
products: choose the beams that go on, move their states, give a growing memory its pages, put keys and values into them in 4 bits
and attend over them.  ``own = False`` computes the operators in elementary torch operations, ``own = True`` calls
``linmt_b200.device_ops``.

A page tensor is uint8 [pages, heads, positions / 16, 18 * dim]: for 16 positions of one head, 8 dim bytes of key codes, dim bytes of
key scales, 8 dim bytes of value codes, dim bytes of value scales.  A code stands for (code - 8) * scale, a scale (bf16) belongs to 32
neighbouring components.  Keys of a position: the eight codes 32 g + 8 c .. + 7 are 32-bit word c * dim / 32 + g.  Values: unit
(i, g, c) of 16 bytes holds components 64 i + 4 g .. + 3 and the four 32 further, of positions 2 c, 2 c + 1, 2 c + 8 and 2 c + 9, as
16-bit fours of codes in the order pair of positions, four, position.
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
        # the first word of one sentence on the small model: every other beam is empty
        dict(name="select_first", op="select", n=1, k=4, v=1000, dtype="fp32", first=True, done=0.0, mask="none"),
        # a step of the headline decode: 64 sentences, beam 12, 30k words, some beams at their end
        dict(name="select_64", op="select", n=64, k=12, v=30000, dtype="fp32", first=False, done=0.1, mask="none"),
        # the large vocabulary in 16 bits, every sentence with a word list of its own
        dict(name="select_lists", op="select", n=128, k=12, v=80000, dtype="bf16", first=False, done=0.05, mask="each"),
        # states of a handful of sentences on the odd model: three layers of 250, and the words so far
        dict(name="reorder_odd", op="reorder", n=11, k=7, layers=3, hidden=250, dtype="fp32", words=41),
        # h and c of the headline model's four layers behind every step
        dict(name="reorder_64", op="reorder", n=64, k=12, layers=4, hidden=1000, dtype="fp32", words=90),
        # every sentence of a running batch grows by one position
        dict(name="plan_step", op="plan", n=64, page=16, lo=1, hi=400, grow=1),
        # a new job's sentences get their first pages
        dict(name="plan_job", op="plan", n=4096, page=32, lo=1, hi=500, grow=0),
        # the new position of each sentence
        dict(name="write_step", op="write", t=64, heads=8, dim=128, page=16, dtype="bf16"),
        # the memory of long documents, written at once
        dict(name="write_job", op="write", t=100003, heads=8, dim=128, page=64, dtype="bf16"),
        # one sentence's beams over its source
        dict(name="attend_one", op="attend", n=1, g=5, heads=8, rep=1, dim=64, page=16, lo=23, hi=23, dtype="fp32", cap=0.0, bias=False, windows=False),
        # paragraphs: capped scores, a bias that falls with the distance, each beam its own part of the text
        dict(name="attend_64", op="attend", n=64, g=12, heads=8, rep=1, dim=128, page=32, lo=1, hi=4001, dtype="fp16", cap=30.0, bias=True, windows=True),
        # whole documents, several queries on each head of the memory
        dict(name="attend_long", op="attend", n=8, g=4, heads=8, rep=4, dim=128, page=64, lo=20000, hi=32768, dtype="bf16", cap=0.0, bias=False, windows=False),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["select", "reorder", "plan", "write", "attend"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "select":
        k, v = rng.randint(1, 31), _spread(rng, 500, 100000)
        n = _spread(rng, 1, max(1, min(300, 240_000_000 // (k * v * SIZE[dtype]))))
        return dict(op=op, n=n, k=k, v=v, dtype=dtype, first=rng.random() < 0.15, done=rng.choice([0.0, 0.1, 0.5]), mask=rng.choice(["none", "none", "one", "each"]))
    if op == "reorder":
        k, layers, hidden = rng.randint(1, 31), rng.randint(1, 6), _spread(rng, 17, 2100)
        n = _spread(rng, 1, max(1, min(256, 3_000_000 // (k * layers * hidden))))
        return dict(op=op, n=n, k=k, layers=layers, hidden=hidden, dtype=dtype, words=_spread(rng, 1, 200))
    if op == "plan":
        n, page = _spread(rng, 1, 4096), 16 * rng.randint(1, 8)
        lo = _spread(rng, 1, 500)
        hi = _spread(rng, lo, max(lo, min(20000, 1_900_000 // n - lo)))
        return dict(op=op, n=n, page=page, lo=lo, hi=hi, grow=rng.choice([0, 1, 1, rng.randint(2, 40)]))
    dim = rng.choice([64, 128])
    page = 16 * rng.randint(1, 8)
    if op == "write":
        heads = rng.randint(1, 16)
        return dict(op=op, t=_spread(rng, 1, 100_000 * 1024 // (heads * dim)), heads=heads, dim=dim, page=page, dtype=dtype)
    heads, rep, g = rng.randint(1, 8), rng.choice([1, 1, 2, 3, 4]), rng.randint(1, 14)
    n = _spread(rng, 1, 64)
    # what a pass reads and multiplies stays below the largest listed case's
    most = min(32768, 180_000_000 // (n * heads * dim), 3_000_000_000 // (n * heads * rep * g * dim))
    lo = _spread(rng, 1, most)
    return dict(op=op, n=n, g=g, heads=heads, rep=rep, dim=dim, page=page, lo=lo, hi=rng.randint(lo, most), dtype=dtype, cap=rng.choice([0.0, 20.0, 50.0]),
                bias=rng.random() < 0.4, windows=rng.random() < 0.4)


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


def prepare(case, seed):
    gen, op = _gen(seed), case["op"]
    if op == "select":
        n, k, v = case["n"], case["k"], case["v"]
        logits = _normal(gen, n, k, v).mul_(1.5)
        best = torch.randint(0, v, (n, k, 24), device="cuda", generator=gen)      # the words that a trained model raises
        logits.scatter_add_(2, best, _normal(gen, n, k, 24).abs_().mul_(3.0))
        scores = _normal(gen, n, k).mul_(4.0).sub_(12.0)
        if case["first"]:
            scores[:, 1:] = -INF
        done = torch.rand(n, k, device="cuda", generator=gen) < case["done"]
        allowed = None
        if case["mask"] != "none":
            bits = torch.randint(0, 2 ** 32, (2, n if case["mask"] == "each" else 1, (v + 31) // 32), device="cuda", generator=gen)
            allowed = (bits[0] | bits[1]).to(torch.int64)                         # three words of four
            allowed = torch.where(allowed >= 2 ** 31, allowed - 2 ** 32, allowed).to(torch.int32)
        return dict(case, logits=logits.to(TYPES[case["dtype"]]), scores=scores, done=done, allowed=allowed, eos=1)
    if op == "reorder":
        n, k, layers, hidden, t = case["n"], case["k"], case["layers"], case["hidden"], TYPES[case["dtype"]]
        states = [_normal(gen, layers, n, k, hidden).to(t), _normal(gen, layers, n, k, hidden).to(t),
                  torch.randint(0, 30000, (n, k, case["words"]), device="cuda", generator=gen, dtype=torch.int32)]
        parents = torch.randint(0, k, (n, k), device="cuda", generator=gen, dtype=torch.int32)
        return dict(case, states=states, parents=parents, out=[torch.empty_like(s) for s in states])
    if op == "plan":
        n, page = case["n"], case["page"]
        old = _lengths(case, gen) if case["grow"] else torch.zeros(n, dtype=torch.int32, device="cuda")
        new = old + case["grow"] if case["grow"] else _lengths(case, gen)
        width = (case["hi"] + case["grow"] + page - 1) // page
        have = (old + page - 1) // page
        pages = torch.randperm(n * width, device="cuda", generator=gen).to(torch.int32)
        table = torch.where(torch.arange(width, device="cuda") < have[:, None], pages.view(n, width), -1).to(torch.int32).contiguous()
        free = pages.view(n, width)[torch.arange(width, device="cuda") >= have[:, None]].contiguous()
        return dict(case, old=old, new=new, table=table, free=free, used=torch.zeros(1, dtype=torch.int32, device="cuda"), total=int((new - old).sum()))
    if op == "write":
        t, heads, dim, page = case["t"], case["heads"], case["dim"], case["page"]
        kv = [_normal(gen, t, heads, dim).to(TYPES[case["dtype"]]) for _ in range(2)]
        kv[0] = kv[0] + _normal(gen, heads, dim).to(kv[0].dtype)                 # keys have offsets of their own in every component
        n_pages = (t + page - 1) // page + 2
        order = torch.randperm(n_pages, device="cuda", generator=gen)             # whole pages, in any order
        at = torch.arange(t, device="cuda")
        slots = order[at // page] * page + at % page
        return dict(case, kv=kv, slots=slots, pages=torch.zeros(n_pages, heads, page // 16, 18 * dim, dtype=torch.uint8, device="cuda"))
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


# ---- the 4-bit form

def _quantise(x):
    """Codes 0..15 and scales of the last axis, 32 components a scale: the component of largest size (the positive one of two) is -8."""
    x = x.float()
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x).clamp(-3.3895313892515355e38, 3.3895313892515355e38)
    x = x.unflatten(-1, (x.shape[-1] // 32, 32))
    hi, lo = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    scale = (torch.where(hi >= -lo, hi, lo) * -0.125).to(torch.bfloat16)
    s = scale.float()
    code = torch.where(s == 0, torch.zeros_like(x), torch.round(x / torch.where(s == 0, torch.ones_like(s), s))).clamp(-8, 7) + 8
    return code.flatten(-2), scale.squeeze(-1)


def _values(code, scale):
    return ((code.float() - 8).unflatten(-1, (scale.shape[-1], 32)) * scale.float().unsqueeze(-1)).flatten(-2)


def _bytes(nibbles):
    pairs = nibbles.to(torch.uint8).unflatten(-1, (-1, 2))
    return pairs[..., 0] | (pairs[..., 1] << 4)


def _pack(k, v):
    """Pages of k, v [pages, heads, positions, dim]."""
    p, h, t, d = k.shape
    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    kc = kc.view(p, h, t // 16, 16, d // 32, 4, 8).transpose(4, 5).reshape(p, h, t // 16, 16 * d)
    vc = vc.view(p, h, t // 16, 2, 4, 2, d // 64, 2, 8, 4).permute(0, 1, 2, 6, 8, 4, 3, 7, 5, 9).reshape(p, h, t // 16, 16 * d)
    raw = [x.reshape(p, h, t // 16, d // 2).contiguous().view(torch.uint8) for x in (ks, vs)]
    return torch.cat([_bytes(kc), raw[0], _bytes(vc), raw[1]], dim=-1)


def _nibbles(x):
    return torch.stack([x & 15, x >> 4], dim=-1).flatten(-2)


def _unpack(pages):
    """Keys and values [pages, heads, positions, dim] of pages [pages, heads, positions / 16, 18 dim]."""
    p, h, n, b = pages.shape
    d = b // 18
    kc, ks, vc, vs = pages.split([8 * d, d, 8 * d, d], dim=-1)
    kc = _nibbles(kc).view(p, h, n, 16, 4, d // 32, 8).transpose(4, 5).reshape(p, h, n * 16, d)
    vc = _nibbles(vc).view(p, h, n, d // 64, 8, 4, 2, 2, 2, 4).permute(0, 1, 2, 6, 5, 8, 3, 7, 4, 9).reshape(p, h, n * 16, d)
    ks, vs = (x.contiguous().view(torch.bfloat16).view(p, h, n * 16, d // 32) for x in (ks, vs))
    return _values(kc, ks), _values(vc, vs)


# ---- the operators in plain form

def _select(s):
    x = s["logits"].double()                # 64 bits: two beams' candidates may be closer than 32 bits tell apart
    n, k, v = x.shape
    scores, done = s["scores"].double(), s["done"]
    if s["allowed"] is not None:
        bit = torch.arange(v, device=x.device)
        ok = (s["allowed"][:, bit // 32] >> (bit % 32).to(torch.int32)) & 1
        x = torch.where(ok[:, None, :] != 0, x, -INF)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    lse = top + (x - top).exp().sum(-1, keepdim=True).log()
    x = scores[..., None] + (x - lse)
    at_end = torch.where(torch.arange(v, device=x.device) == s["eos"], scores[..., None], -INF)
    x = torch.where(done[..., None], at_end, x)
    x = torch.where(torch.isnan(x), -INF, x).flatten(1)
    best, at = torch.sort(x, dim=-1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    none = best == -INF
    parents = torch.where(none, torch.arange(k, device=x.device), at // v)
    tokens = torch.where(none, s["eos"], at % v)
    done = none | torch.gather(done, 1, parents) | (tokens == s["eos"])
    return dict(tokens=tokens.to(torch.int32), parents=parents.to(torch.int32), scores=best.float(), done=done)


def _plan(s):
    n, page, width = s["n"], s["page"], s["table"].shape[1]
    old, new = s["old"].long(), s["new"].long()
    grown = new - old
    starts = torch.cat([grown.new_zeros(1), grown.cumsum(0)])
    have, want = (old + page - 1) // page, (new + page - 1) // page
    more = want - have
    first = s["used"].long() + more.cumsum(0) - more
    col = torch.arange(width, device=old.device)
    at = first[:, None] + col - have[:, None]
    fresh = (col >= have[:, None]) & (col < want[:, None])
    got = torch.where(at < s["free"].numel(), s["free"][at.clamp(0, max(0, s["free"].numel() - 1))], -1) if s["free"].numel() else torch.full_like(at, -1, dtype=torch.int32)
    table = torch.where(fresh, got, s["table"])
    token = torch.arange(s["total"], device=old.device)
    row = torch.searchsorted(starts, token, right=True) - 1
    pos = token - starts[row] + old[row]
    p = table[row, pos // page].long()
    return dict(slots=torch.where(p >= 0, p * page + pos % page, -1), starts=starts.to(torch.int32), table=table, used=(s["used"] + more.sum()).to(torch.int32))


def _attend(s):
    n, g, heads, rep, dim = (s[x] for x in ("n", "g", "heads", "rep", "dim"))
    k, v = _unpack(s["pages"])
    k, v = (x[s["table"].long()].transpose(1, 2).flatten(2, 3) for x in (k, v))               # [n, heads, positions, dim]
    q = s["q"].float().view(n, g, heads, rep, dim).permute(0, 2, 1, 3, 4).reshape(n, heads, g * rep, dim)
    x = (q @ k.transpose(2, 3) * s["scale"]).view(n, heads, g, rep, -1)
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    at = torch.arange(x.shape[-1], device=x.device)
    if s["slope"] is not None:
        x = x - s["slope"].view(1, heads, 1, rep, 1) * (at - s["centre"][..., None]).abs()[:, None, :, None, :]
    seen = (at < s["lens"][:, None])[:, None, :].expand(n, g, -1)
    if s["first"] is not None:
        seen = seen & (at >= s["first"][..., None]) & (at < s["last"][..., None])
    x = torch.where(seen[:, None, :, None, :], x, -INF)
    top = x.amax(-1, keepdim=True)
    e = (x - torch.where(top == -INF, 0.0, top)).exp()
    total = e.sum(-1, keepdim=True)
    out = (e / torch.where(total == 0, 1.0, total)).view(n, heads, g * rep, -1) @ v
    lse = torch.where(total == 0, -INF, top + total.log()).squeeze(-1)
    return dict(out=out.view(n, heads, g, rep, dim).permute(0, 2, 1, 3, 4).reshape(n, g, heads * rep, dim).to(s["q"].dtype), lse=lse.permute(0, 2, 1, 3).reshape(n, g, heads * rep))


def run(state):
    s, op = state, state["op"]
    if own:
        from linmt_b200 import device_ops as ops
        if op == "select":
            tokens, parents, scores, done = ops.beam_select(s["logits"], s["scores"], done=s["done"], allowed=s["allowed"], eos=s["eos"])
            return dict(tokens=tokens, parents=parents, scores=scores, done=done)
        if op == "reorder":
            return ops.beam_reorder(s["states"], s["parents"], out=s["out"])
        if op == "plan":
            slots, starts, used = ops.plan_pages(s["old"], s["new"], s["table"], s["free"], s["used"], page=s["page"], total=s["total"])
            return dict(slots=slots, starts=starts, table=s["table"], used=used)
        if op == "write":
            ops.write_pages4(s["pages"], s["slots"], s["kv"][0], s["kv"][1])
            return ops.read_pages4(s["pages"], s["slots"], dtype=s["kv"][0].dtype)
        out, lse = ops.attend_pages4(s["q"], s["pages"], s["table"], s["lens"], scale=s["scale"], cap=s["cap"], slope=s["slope"], centre=s["centre"],
                                     first=s["first"], last=s["last"], want_lse=True)
        return dict(out=out, lse=lse)
    if op == "select":
        return _select(s)
    if op == "reorder":
        at = s["parents"].long()
        return [torch.gather(x, x.dim() - 2, at.view((1,) * (x.dim() - 3) + at.shape + (1,)).expand(x.shape)) for x in s["states"]]
    if op == "plan":
        return _plan(s)
    if op == "write":
        return tuple(_values(*_quantise(x)).to(x.dtype) for x in s["kv"])
    return _attend(s)


# ---- what a pass cannot do without

def work(case):
    op, size = case["op"], SIZE.get(case.get("dtype"), 4)
    if op == "select":
        n, k, v = case["n"], case["k"], case["v"]
        rows = n * (1 if case["first"] else k) * (1 - case["done"])               # an empty or finished beam's logits are not needed
        lists = {"none": 0, "one": 1, "each": n}[case["mask"]] * v / 8
        return dict(bytes=rows * v * size + lists + n * k * (5 + 13), flops=rows * v * 4)
    if op == "reorder":
        one = case["n"] * case["k"] * (2 * case["layers"] * case["hidden"] * size + 4 * case["words"])
        return dict(bytes=2 * one + 4 * case["n"] * case["k"], flops=0)
    if op == "plan":
        n, mean = case["n"], (case["lo"] + case["hi"]) / 2
        tokens = n * (case["grow"] or mean)
        return dict(bytes=12 * n + tokens * (8 + 8 / case["page"]), flops=0)
    if op == "write":
        values = 2 * case["t"] * case["heads"] * case["dim"]
        return dict(bytes=values * (2 * size + 2 * 9 / 16) + 16 * case["t"], flops=values * 4)
    n, g, heads, rep, dim = (case[x] for x in ("n", "g", "heads", "rep", "dim"))
    at = n * (case["lo"] + case["hi"]) / 2
    seen = every = 1.0
    if case["windows"]:                                                            # two even draws enclose a third of the text, 2 g of them more
        seen, every = 1 / 3, (2 * g - 1) / (2 * g + 1)
    return dict(bytes=at * every * heads * dim * 18 / 16 + n * g * heads * rep * (dim * 2 * size + 4), flops=at * seen * heads * rep * g * dim * 4)


# ---- the definitions in 64 bits

def _exact_select(s):
    n, k, v = s["logits"].shape
    words = torch.arange(v, device="cuda")
    found = torch.full((n, k), -INF, dtype=torch.float64, device="cuda")
    for i in range(n):
        z = s["logits"][i].double()
        if s["allowed"] is not None:
            row = s["allowed"][min(i, s["allowed"].shape[0] - 1)].long() & 0xFFFFFFFF
            z[:, ((row.repeat_interleave(32)[:v] >> (words % 32)) & 1) == 0] = -INF
        z = torch.log_softmax(z, dim=-1) + s["scores"][i].double()[:, None]
        z[s["done"][i]] = -INF
        z[s["done"][i], s["eos"]] = s["scores"][i].double()[s["done"][i]]
        z = torch.nan_to_num(z, nan=-INF, posinf=INF, neginf=-INF).flatten()
        found[i] = torch.topk(z, k).values
    return dict(tokens=None, parents=None, scores=found, done=None)


def _exact_codes(x):
    """Values of the 4-bit form, from its definition."""
    x = x.double().unflatten(-1, (x.shape[-1] // 32, 32))
    big = x.abs().amax(-1, keepdim=True)
    positive = (x == big).any(-1, keepdim=True)
    scale = (torch.where(positive, -big, big) / 8).to(torch.bfloat16).double()
    code = torch.where(scale == 0, 0.0, torch.round(x / scale)).clamp(-8, 7)
    return (code * scale).flatten(-2)


def _exact_memory(pages):
    """Keys and values of pages, each code looked up where the form has it."""
    p, h, n, b = pages.shape
    d = b // 18
    t, c = torch.arange(16, device="cuda")[:, None], torch.arange(d, device="cuda")[None, :]
    key = t * (d // 2) + 4 * ((c % 32 // 8) * (d // 32) + c // 32) + c % 8 // 2
    unit = (c // 64 * 8 + c % 32 // 4) * 4 + t % 8 // 2
    value = 9 * d + 16 * unit + 8 * (t // 8) + 4 * (c % 64 // 32) + 2 * (t % 2) + c % 4 // 2
    made = []
    for at, scales in ((key, 8 * d), (value, 17 * d)):
        code = (pages[..., at] >> (4 * (c % 2)).to(torch.uint8).expand(16, d)) & 15
        scale = pages[..., scales:scales + d].contiguous().view(torch.bfloat16).view(p, h, n, 16, d // 32).double().repeat_interleave(32, -1)
        made.append(((code.double() - 8) * scale).view(p, h, n * 16, d))
    return made


def _exact_attend(s):
    n, g, heads, rep, dim = (s[x] for x in ("n", "g", "heads", "rep", "dim"))
    out = torch.zeros(n, g, heads * rep, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((n, g, heads * rep), -INF, dtype=torch.float64, device="cuda")
    for i in range(n):
        length = int(s["lens"][i])
        k, v = (x.transpose(0, 1).flatten(1, 2)[:, :length].repeat_interleave(rep, 0) for x in _exact_memory(s["pages"][s["table"][i].long()]))
        z = torch.einsum("ghd,hpd->ghp", s["q"][i].double(), k) * s["scale"]
        if s["cap"]:
            z = torch.tanh(z / s["cap"]) * s["cap"]
        at = torch.arange(length, device="cuda", dtype=torch.float64)
        if s["slope"] is not None:
            z = z - s["slope"].double()[None, :, None] * (at[None, :] - s["centre"][i].double()[:, None]).abs()[:, None, :]
        if s["first"] is not None:
            hidden = (at[None, :] < s["first"][i][:, None]) | (at[None, :] >= s["last"][i][:, None])
            z = z.masked_fill(hidden[:, None, :], -INF)
        lse[i] = torch.logsumexp(z, -1)
        weight = torch.softmax(z, -1).nan_to_num(nan=0.0)
        out[i] = torch.einsum("ghp,hpd->ghd", weight, v)
    return dict(out=out, lse=lse)


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "reorder":
        n, rows = torch.arange(case["n"], device="cuda")[:, None], s["parents"].long()
        return [s["states"][0].double()[:, n, rows], s["states"][1].double()[:, n, rows], None]
    if case["op"] == "select":
        return _exact_select(s)
    if case["op"] == "write":
        return tuple(_exact_codes(x) for x in s["kv"])
    return _exact_attend(s)

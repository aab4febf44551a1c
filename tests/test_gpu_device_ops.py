"""Operators on device tensors against plain implementations in 64 bits."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

INF = float("inf")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}      # largest rounding, relative


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from linmt_b200 import device_ops
    return device_ops


def _rng(*seed):
    return np.random.default_rng(list(seed))


def _cuda(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(dtype)


# ---- selection

def _bits(allowed):
    """Bit lists of a [n, vocab] truth array."""
    n, v = allowed.shape
    b = np.zeros((n, -(-v // 32) * 32), np.uint64)
    b[:, :v] = allowed
    return (b.reshape(n, -1, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)


def select_ref(logits, scores, done=None, allowed=None, eos=1):
    """The definition, candidate by candidate, in 64 bits."""
    x = logits.double().cpu().numpy()
    sc = scores.double().cpu().numpy()
    n, k, v = x.shape
    dn = np.zeros((n, k), bool) if done is None else done.cpu().numpy().astype(bool)
    tok, par, out, fin = np.zeros((n, k), np.int32), np.zeros((n, k), np.int32), np.zeros((n, k)), np.zeros((n, k), bool)
    for i in range(n):
        c = np.full((k, v), -INF)
        for b in range(k):
            if not np.isfinite(sc[i, b]):
                continue
            if dn[i, b]:
                c[b, eos] = sc[i, b]
                continue
            z = x[i, b].copy()
            if allowed is not None:
                z[~allowed[min(i, allowed.shape[0] - 1)]] = -INF
            m = z.max()
            if not np.isfinite(m) or np.isnan(z).any():
                continue
            c[b] = sc[i, b] + ((z - m) - np.log(np.exp(z - m).sum()))
        c = c.ravel()
        order = np.argsort(-c, kind="stable")[:k]
        for j in range(k):
            if j < len(order) and c[order[j]] > -INF:
                at = order[j]
                tok[i, j], par[i, j], out[i, j] = at % v, at // v, c[at]
                fin[i, j] = dn[i, at // v] or at % v == eos
            else:
                tok[i, j], par[i, j], out[i, j], fin[i, j] = eos, j, -INF, True
    return tok, par, out, fin


def select_check(ops, logits, scores, done=None, allowed=None, eos=1):
    got = ops.beam_select(logits, scores, done=done, allowed=None if allowed is None else _cuda(_bits(allowed)), eos=eos)
    tok, par, sc, fin = select_ref(logits, scores, done, allowed, eos)
    assert (got[1].cpu().numpy() == par).all(), "parents"
    assert (got[0].cpu().numpy() == tok).all(), "tokens"
    assert (got[3].cpu().numpy() == fin).all(), "done"
    g = got[2].cpu().numpy().astype(np.float64)
    assert (np.isneginf(g) == np.isneginf(sc)).all()
    ok = np.isfinite(sc)
    # the bound of a 32-bit normaliser: 6e-6 (exponents' arguments 2^-23 log2(vocab), exp2 2^-22 twice, 40 additions of 2^-24, the logarithm 2^-20) and 5.1e-7 (an addition, an
    # exp2 and a product) for each of a lane's steps (at most ceil(vocab / 512) + 2 of them), and the result's own rounding
    tol = 6e-6 + 5.1e-7 * (-(-logits.shape[2] // 512) + 2)
    assert (np.abs(g[ok] - sc[ok]) <= tol + 2.0 ** -24 * np.abs(sc[ok])).all()
    return got


def _logits(rng, n, k, v, dtype):
    x = rng.normal(0, 1.5, (n, k, v))
    for _ in range(6):
        x[np.arange(n)[:, None], np.arange(k)[None, :], rng.integers(0, v, (n, k))] += rng.exponential(3.0, (n, k))
    return _cuda(x.astype(np.float32), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,k,v", [(1, 1, 1), (1, 1, 2), (3, 4, 3), (2, 32, 40), (1, 4, 1000), (3, 31, 517), (5, 12, 30000), (2, 5, 80000), (9, 7, 5003), (1, 13, 250007)])
def test_select(ops, n, k, v, dtype):
    rng = _rng(n, k, v)
    x = _logits(rng, n, k, v, dtype)
    scores = _cuda(rng.normal(-10, 3, (n, k)).astype(np.float32))
    select_check(ops, x, scores, eos=min(1, v - 1))
    first = scores.clone()
    first[:, 1:] = -INF
    select_check(ops, x, first, eos=0)
    done = _cuda(rng.random((n, k)) < 0.4)
    select_check(ops, x, scores, done=done, eos=v - 1)
    select_check(ops, x, scores, done=torch.ones_like(done), eos=v - 1)
    for lists in (1, n):
        allowed = rng.random((lists, v)) < 0.3
        select_check(ops, x, scores, done=done, allowed=allowed, eos=v // 2)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("k,v", [(5, 30000), (12, 4099), (32, 700)])
def test_select_ties_go_to_the_lowest_index(ops, k, v, dtype):
    """All equal; sorted either way in steps; the same row for every beam; groups of equal logits at the end of the row."""
    zeros = torch.zeros(2, k, v, dtype=dtype, device="cuda")
    down = torch.linspace(4, -4, v, device="cuda").to(dtype).expand(2, k, v).contiguous()
    up = down.flip(2).contiguous()
    steps = _cuda(np.repeat(np.arange(-(-v // 700), dtype=np.float32), 700)[:v] * 0.25, dtype).expand(2, k, v).contiguous()
    rng = _rng(k, v)
    row = _logits(rng, 1, 1, v, dtype).expand(2, k, v).contiguous()
    tail = zeros.clone()
    tail[:, :, -3 * k:] = 2
    same = torch.full((2, k), -3.5, device="cuda")
    apart = torch.arange(k, device="cuda", dtype=F32).mul(-0.5).expand(2, k).contiguous()
    for x in (zeros, down, up, steps, row, tail):
        for scores in (same, apart):
            select_check(ops, x, scores)


@pytest.mark.parametrize("n,k,v", [(1, 12, 30000), (80, 5, 9001), (50, 9, 4003), (80, 31, 1500), (160, 12, 3001), (160, 13, 3001), (3, 17, 9000), (140, 24, 2500), (90, 32, 2100)])
def test_select_one_beam_ahead(ops, n, k, v):
    """All that is chosen lies in one row, in few of its places, or in logits too small to tell apart; for one sentence and for so many that each has few CTAs."""
    rng = _rng(n, k, v, 3)
    x = _logits(rng, n, k, v, F16)
    scores = torch.full((n, k), -50.0, device="cuda")
    ahead = _cuda(rng.integers(0, k, (n, 1)))
    scores.scatter_(1, ahead, -1.0)
    select_check(ops, x, scores)
    order = x.sort(dim=2, descending=True).values          # the best words next to each other
    select_check(ops, order, scores)
    select_check(ops, order, torch.zeros_like(scores))
    tiny = _cuda((rng.normal(0, 1, (n, k, v)) * 1e-20).astype(np.float32))
    select_check(ops, tiny, scores)
    select_check(ops, tiny, torch.zeros_like(scores))


@pytest.mark.parametrize("v", [1000, 30000])
def test_select_between_beams_closer_than_32_bits(ops, v):
    """Rows that are permutations of each other under scores one step of 32 bits apart: candidates 1e-6 apart, and 2.4e-7 at smaller scores, which a 32-bit
    normaliser cannot order."""
    rng = _rng(v, 1)
    k = 8
    base = rng.normal(0, 2, v).astype(np.float32)
    for start in (-9.0, -1.5, 0.0):
        s = [np.float32(start)]
        for _ in range(k - 1):
            s.append(np.nextafter(s[-1], np.float32(-100)))
        scores = _cuda(np.stack([np.array(s, np.float32)[rng.permutation(k)] for _ in range(4)]))
        x = _cuda(np.stack([[base[rng.permutation(v)] for _ in range(k)] for _ in range(4)]))
        if start == 0.0:      # next to 0 the steps are 1e-45: rows are told apart by a logit instead
            x += torch.linspace(0, 1e-3, v, device="cuda") * torch.arange(k, device="cuda")[:, None] * 1e-4
        select_check(ops, x, scores)


def test_select_masked_places_may_hold_anything(ops):
    rng = _rng(5)
    n, k, v = 4, 6, 3001
    x = _logits(rng, n, k, v, F32)
    allowed = rng.random((n, v)) < 0.5
    allowed[2] = False                       # nothing is allowed: only finished beams offer
    allowed[3] = False
    allowed[3, 77] = True
    bad = torch.from_numpy(~allowed).cuda()[:, None, :].expand(n, k, v)
    scores = _cuda(rng.normal(-10, 3, (n, k)).astype(np.float32))
    done = _cuda(rng.random((n, k)) < 0.3)
    done[2, 3] = True
    want = select_check(ops, x, scores, done=done, allowed=allowed)
    for value in (INF, -INF, float("nan"), torch.finfo(F32).min, torch.finfo(F32).max):
        got = ops.beam_select(torch.where(bad, value, x), scores, done=done, allowed=_cuda(_bits(allowed)))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), value


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_select_infinities_nan_and_lowest_values(ops, dtype):
    rng = _rng(6)
    n, k, v = 8, 5, 2050
    x = _logits(rng, n, k, v, dtype)
    low = torch.finfo(dtype).min
    x[0, 1, 17] = float("nan")              # these rows offer nothing
    x[0, 2, 2049] = INF
    x[1] = float("nan")
    x[2, :, 100:] = -INF                    # masked by -inf and by the lowest value
    x[3, :, 100:] = low
    x[4, 0] = -INF
    x[4, 1] = low                           # a row of lowest values is an even distribution
    x[5, :, 3:] = -INF                      # fewer words than beams
    x[6] = -INF
    scores = _cuda(rng.normal(-10, 3, (n, k)).astype(np.float32))
    scores[7] = torch.tensor([-INF, float("nan"), INF, -4.0, -INF])
    select_check(ops, x, scores)
    done = torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    done[1, 2] = done[6, 0] = done[7, 1] = done[7, 3] = 255
    select_check(ops, x, scores, done=done, eos=9)


def test_select_reads_any_strides_and_writes_in_place(ops):
    rng = _rng(7)
    n, k, v = 3, 6, 1031
    for dtype in (F32, BF16):
        for shift in (0, 1, 3, 5):
            wide = torch.full((k, n, v + 37), float("nan"), dtype=dtype, device="cuda")
            x = wide.transpose(0, 1)[:, :, shift:shift + v]
            x.copy_(_logits(rng, n, k, v, dtype))
            scores = _cuda(rng.normal(-10, 3, (n, k)).astype(np.float32))
            done = _cuda(rng.random((n, k)) < 0.2)
            want = select_check(ops, x, scores, done=done)
            tokens, parents = torch.empty(n, k, dtype=torch.int32, device="cuda"), torch.empty(n, k, dtype=torch.int32, device="cuda")
            got = ops.beam_select(x, scores, done=done, out=(tokens, parents, scores, done))
            assert got[2] is scores and all(torch.equal(a, b) for a, b in zip(got, want))
    every = x[:, :1].expand(n, k, v)        # one row for all beams of a sentence
    select_check(ops, every, _cuda(rng.normal(-10, 3, (n, k)).astype(np.float32)))


# ---- reordering

def _reordered(x, parents):
    n, k = parents.shape
    p = parents.long()
    p = torch.where((p < 0) | (p >= k), torch.arange(k, device=p.device), p)
    at = torch.arange(n, device=p.device)[:, None]
    return x[:, at, p] if x.dim() == 4 else x[at, p]


@pytest.mark.parametrize("n,k,layers,width,dtype", [(1, 1, 1, 1, F32), (11, 7, 3, 250, F32), (64, 12, 4, 1000, F32), (5, 32, 2, 33, BF16), (3, 17, 1, 1027, F16), (2, 5, 3, 13, torch.uint8), (4, 9, 2, 31, torch.int64)])
def test_reorder(ops, n, k, layers, width, dtype):
    rng = _rng(n, k, width)
    make = lambda *s: _cuda(rng.integers(0, 100, s)).to(dtype)
    parents = _cuda(rng.integers(0, k, (n, k)).astype(np.int32))
    states = [make(layers, n, k, width), make(n, k, width), make(n, k)]
    want = [_reordered(x, parents) for x in states]
    out = [torch.zeros_like(x) for x in states]
    got = ops.beam_reorder(states, parents, out=out)
    assert all(g is o and torch.equal(g, w) for g, o, w in zip(got, out, want))
    got = ops.beam_reorder(states, parents)
    assert all(g is x and torch.equal(g, w) for g, x, w in zip(got, states, want))


def test_reorder_strides_many_states_and_parents_outside(ops):
    rng = _rng(8)
    n, k = 6, 10
    parents = _cuda(rng.integers(-3, k + 3, (n, k)).astype(np.int32))
    parents[0, 0], parents[0, 1] = -2 ** 31, 2 ** 31 - 1
    wide = _cuda(rng.normal(0, 1, (k, n, 3, 45)).astype(np.float32))
    rest = wide.clone()
    view = wide.permute(2, 1, 0, 3)[:, :, :, 3:40]            # layers innermost, rows on 4-byte boundaries
    want = _reordered(view.clone(), parents)
    ops.beam_reorder([view], parents)
    assert torch.equal(view, want)
    assert torch.equal(wide[..., :3], rest[..., :3]) and torch.equal(wide[..., 40:], rest[..., 40:])
    many = [_cuda(rng.normal(0, 1, (n, k, 1 + i)).astype(np.float32)) for i in range(37)]
    want = [_reordered(x, parents) for x in many]
    ops.beam_reorder(many, parents)
    assert all(torch.equal(a, b) for a, b in zip(many, want))
    assert ops.beam_reorder([], parents) == []
    empty = torch.zeros(0, n, k, 4, device="cuda")
    assert ops.beam_reorder([empty, torch.zeros(n, k, 0, device="cuda")], parents)[0] is empty


def test_reorder_columns_of_one_buffer(ops):
    """h and c side by side in one buffer, each a state of its own."""
    rng = _rng(30)
    hc = _cuda(rng.normal(0, 1, (2, 5, 6, 48)).astype(np.float32))
    parents = _cuda(rng.integers(0, 6, (5, 6)).astype(np.int32))
    want = _reordered(hc.clone(), parents)
    ops.beam_reorder([hc[..., :20], hc[..., 20:44], hc[..., 44:]], parents)
    assert torch.equal(hc, want)
    a, b = _cuda(rng.normal(0, 1, (5, 6, 8)).astype(np.float32)), _cuda(rng.normal(0, 1, (5, 6, 8)).astype(np.float32))
    for bad in (lambda: ops.beam_reorder([a, b], parents, out=[b, a]), lambda: ops.beam_reorder([hc[..., :20], hc[..., 19:]], parents), lambda: ops.beam_reorder([a, a], parents, out=[b, b]),
                lambda: ops.beam_reorder([a, b], parents, out=[torch.empty_like(a), a])):
        with pytest.raises(ValueError):
            bad()


def test_reorder_refuses(ops):
    x, parents = torch.zeros(2, 8, 64, device="cuda"), torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    a = x[:, :4]
    for bad in (lambda: ops.beam_reorder([a], parents.long()), lambda: ops.beam_reorder([a], parents, out=[x[:, 2:6]]), lambda: ops.beam_reorder([a, a], parents),
                lambda: ops.beam_reorder([x], parents), lambda: ops.beam_reorder([a.transpose(1, 2)[:, :2].transpose(1, 2)[:, :4, :2].transpose(0, 1)], parents),
                lambda: ops.beam_reorder([x[:, :1].expand(2, 4, 64)], parents), lambda: ops.beam_reorder([a], parents, out=[a.to(F16)]), lambda: ops.beam_reorder([a], parents, out=[]), lambda: ops.beam_reorder([parents], parents),
                lambda: ops.beam_reorder([torch.zeros(2, 40, 4, device="cuda")], torch.zeros(2, 40, dtype=torch.int32, device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            bad()


# ---- pages

def plan_ref(old, new, table, free, used, page, total):
    n, width = table.shape
    table, most = table.copy(), width * page
    slots, starts, q = [], [0], int(used)
    for i in range(n):
        o = min(max(int(old[i]), 0), most) if old is not None else 0
        w = max(min(max(int(new[i]), 0), most), o)
        for p in range(-(-o // page), -(-w // page)):
            table[i, p] = free[q] if 0 <= q < len(free) else -1
            q += 1
        for pos in range(o, w):
            p = int(table[i, pos // page])
            slots.append(p * page + pos % page if p >= 0 else -1)
        starts.append(len(slots))
    slots = (slots + [-1] * max(0, total - len(slots)))[:total]
    return np.array(slots, np.int64), np.array(starts, np.int32), table, q


def plan_check(ops, old, new, table, free, used, page, total):
    want = plan_ref(old, new, table, free, used, page, total)
    t = _cuda(table)
    slots, starts, now = ops.plan_pages(None if old is None else _cuda(old), _cuda(new), t, _cuda(free), torch.tensor([used], dtype=torch.int32, device="cuda"), page=page, total=total)
    assert (slots.cpu().numpy() == want[0]).all() and (starts.cpu().numpy() == want[1]).all() and (t.cpu().numpy() == want[2]).all() and int(now) == want[3]


@pytest.mark.parametrize("n,width,page,lo,hi,grow", [(1, 1, 16, 1, 1, 0), (64, 26, 16, 1, 400, 1), (700, 9, 32, 0, 280, 0), (33, 50, 1, 0, 49, 1), (5, 400, 48, 9000, 19000, 130), (3000, 3, 128, 0, 300, 7), (16384, 2, 16, 0, 31, 1)])
def test_plan(ops, n, width, page, lo, hi, grow):
    rng = _rng(n, width, page)
    old = rng.integers(lo, hi + 1, n).astype(np.int32)
    old[rng.random(n) < 0.1] = 0
    new = old + grow if grow else old.copy()
    if not grow:
        old = None
    pages = rng.permutation(n * width + 5).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    took = 0
    if old is not None:
        for i in range(n):
            have = min(-(-int(old[i]) // page), width)
            table[i, :have] = pages[took:took + have]
            took += have
    free = pages[took:].copy()
    total = int((new - (0 if old is None else old)).sum())
    for used, room in ((0, total), (3, total + 7), (0, max(0, total - 9))):
        plan_check(ops, old, new, table, free, used, page, room)
    plan_check(ops, old, new, table, free[:len(free) // 3], 1, page, total)            # the free list runs out
    plan_check(ops, old, new, table, free[:0], 0, page, total)


def test_plan_clamps_lengths_and_takes_strided_tables(ops):
    old = np.array([-5, 10, 64, 100, 3, 0], np.int32)
    new = np.array([20, 4, 90, 2 ** 31 - 1, -1, 0], np.int32)
    table = np.arange(24, dtype=np.int32).reshape(6, 4)
    free = np.arange(100, 120, dtype=np.int32)
    plan_check(ops, old, new, table, free, 2, 16, 40)
    wide = torch.full((6, 9), 7, dtype=torch.int32, device="cuda")
    wide[:, 2:6] = _cuda(table)
    want = plan_ref(old, new, table, free, 0, 16, 20)
    slots, _, _ = ops.plan_pages(_cuda(old), _cuda(new), wide[:, 2:6], _cuda(free), torch.zeros(1, dtype=torch.int32, device="cuda"), page=16, total=20)
    assert (slots.cpu().numpy() == want[0]).all() and (wide[:, 2:6].cpu().numpy() == want[2]).all()
    assert (wide[:, :2] == 7).all() and (wide[:, 6:] == 7).all()
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    slots, starts, used = ops.plan_pages(None, empty, torch.zeros(0, 3, dtype=torch.int32, device="cuda"), empty, torch.tensor([4], dtype=torch.int32, device="cuda"), page=16, total=3)
    assert slots.tolist() == [-1, -1, -1] and starts.tolist() == [0] and used.tolist() == [4]


# ---- rows in 4 bits

def codes_ref(x):
    """Codes, scales and values of the last axis in the form's own 32-bit arithmetic."""
    x = x.astype(np.float32)
    most = np.float32(3.3895313892515355e38)
    x = np.clip(np.where(np.isnan(x), np.float32(0), x), -most, most)
    g = x.reshape(x.shape[:-1] + (-1, 32))
    hi, lo = g.max(-1), g.min(-1)
    s = torch.from_numpy(np.where(hi >= -lo, hi, lo) * np.float32(-0.125)).to(BF16)
    sf = s.float().numpy()[..., None]
    with np.errstate(all="ignore"):
        c = np.where(sf == 0, np.float32(0), np.clip(np.rint(g / np.where(sf == 0, np.float32(1), sf)), -8, 7)).astype(np.float32)
    return c.astype(np.int64) + 8, s, (c * sf).reshape(x.shape)


def tile_ref(pages, n_pages, heads, page, dim):
    """Key and value codes and scales of a pool as the header describes it: [n_pages, page, heads, dim] and [.., dim / 32]."""
    raw = pages.reshape(n_pages, heads, page // 16, 18 * dim)
    made = [np.zeros((n_pages, page, heads, dim), np.int64) for _ in range(2)]
    scales = [np.zeros((n_pages, page, heads, dim // 32), np.uint16) for _ in range(2)]
    for pos in range(page):
        t, tile = pos % 16, raw[:, :, pos // 16]
        for d in range(dim):
            word = t * dim // 8 + (d % 32 // 8) * dim // 32 + d // 32
            made[0][:, pos, :, d] = (tile[..., 4 * word + d % 8 // 2] >> (4 * (d % 2))) & 15
            i, h, g, a, c, b = d // 64, d % 64 // 32, d % 32 // 4, t // 8, t % 8 // 2, t % 2
            four = 8 * dim + dim + 16 * ((i * 8 + g) * 4 + c) + 2 * (4 * a + 2 * h + b)
            made[1][:, pos, :, d] = (tile[..., four + d % 4 // 2] >> (4 * (d % 2))) & 15
        for s in range(dim // 32):
            for which, start in ((0, 8 * dim), (1, 17 * dim)):
                at = start + 2 * (t * dim // 32 + s)
                scales[which][:, pos, :, s] = tile[..., at].astype(np.uint16) | tile[..., at + 1].astype(np.uint16) << 8
    return made, scales


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,heads,dim,page", [(1, 1, 64, 16), (50, 3, 64, 48), (77, 2, 128, 32), (129, 5, 128, 16)])
def test_write_and_read(ops, t, heads, dim, page, dtype):
    rng = _rng(t, heads, dim)
    n_pages = t // page + 3
    slots = rng.permutation(n_pages * page)[:t].astype(np.int64)
    gone = rng.random(t) < 0.1
    named = np.where(gone, rng.choice(np.array([-1, -2 ** 40, n_pages * page, 2 ** 60], np.int64), t), slots)
    k, v = (rng.normal(0, 1, (t, heads, dim)) * np.exp(rng.normal(0, 2, (t, heads, 1))) for _ in range(2))
    k[0, 0, :32] = 0                          # a scale of 0
    k[-1, -1, 0] = -k[-1, -1].__abs__().max()
    v[0, 0, 3], v[0, 0, 35] = np.nan, np.inf
    v[-1, 0, 40] = -np.inf
    k, v = _cuda(k.astype(np.float32), dtype), _cuda(v.astype(np.float32), dtype)
    pages = ops.new_pages4(n_pages, heads, dim, page)
    pages.fill_(0xA5)
    ops.write_pages4(pages, _cuda(named), k, v)
    (kc, vc), (ks, vs) = tile_ref(pages.cpu().numpy(), n_pages, heads, page, dim)
    for x, got_c, got_s in ((k, kc, ks), (v, vc, vs)):
        c, s, value = codes_ref(x.float().cpu().numpy())
        got_c, got_s = got_c.reshape(-1, heads, dim), got_s.reshape(-1, heads, dim // 32)
        ok = ~gone
        assert (got_c[slots[ok]] == c.reshape(t, heads, dim)[ok]).all()
        assert (got_s[slots[ok]] == s.view(torch.int16).numpy().view(np.uint16)[ok]).all()
        rest = np.ones(n_pages * page, bool)
        rest[slots[ok]] = False
        assert (got_c[rest] == np.tile([5, 10], dim // 2)).all() and (got_s[rest] == 0xA5A5).all()      # all else is as it was
        # a code is the nearest of its 16: within half a step, and a step where the end of the range cuts it off
        f = x.float().cpu().numpy()
        fine = np.isfinite(f) & (np.abs(f) < 1e30)
        step = np.repeat(np.abs(s.float().numpy()), 32, -1)
        assert (np.abs(value - f)[fine] <= 1.04 * step[fine]).all()
    for out in (F32, dtype):
        rk, rv = ops.read_pages4(pages, _cuda(named), dtype=out)
        for x, r in ((k, rk), (v, rv)):
            want = torch.from_numpy(codes_ref(x.float().cpu().numpy())[2])
            want[torch.from_numpy(gone)] = 0
            assert torch.equal(r.cpu(), want.to(out))


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 48)])
def test_write_and_read_of_texts(ops, dim, page):
    """Positions one after the other, as a text's are: whole tiles that begin anywhere among the call's positions, beginnings and ends of tiles, tiles with a gap or two
    places exchanged, and quotients that lie in the middle of two codes."""
    rng = _rng(dim, page)
    heads, n_pages = 3, 40
    runs = [(0, 16), (33, 40), (96, 7), (112, 17), (160, 48), (223, 1), (240, 16), (258, 30), (304, 200)]
    slots = np.concatenate([np.arange(a, a + n) for a, n in runs]).astype(np.int64)
    at = int(np.nonzero(slots == 176)[0][0])
    slots[at + 3], slots[at + 4] = slots[at + 4], slots[at + 3]
    slots[np.nonzero(slots == 245)[0]] = -1
    t = len(slots)
    x = rng.normal(0, 1, (2, t, heads, dim)).astype(np.float32)
    x[:, ::3] = rng.integers(-16, 17, (2, len(x[0, ::3]), heads, dim)) / 2          # halves of a scale of 1, where the largest is 8
    x[:, ::3, :, ::32] = 8
    k, v = _cuda(x[0]), _cuda(x[1])
    pages = ops.new_pages4(n_pages, heads, dim, page)
    pages.fill_(0x5A)
    ops.write_pages4(pages, _cuda(slots), k, v)
    (kc, vc), (ks, vs) = tile_ref(pages.cpu().numpy(), n_pages, heads, page, dim)
    ok = slots >= 0
    rest = np.ones(n_pages * page, bool)
    rest[slots[ok]] = False
    for y, got_c, got_s in ((x[0], kc, ks), (x[1], vc, vs)):
        c, s, value = codes_ref(y)
        got_c, got_s = got_c.reshape(-1, heads, dim), got_s.reshape(-1, heads, dim // 32)
        assert (got_c[slots[ok]] == c.reshape(t, heads, dim)[ok]).all()
        assert (got_s[slots[ok]] == s.view(torch.int16).numpy().view(np.uint16)[ok]).all()
        assert (got_c[rest] == np.tile([10, 5], dim // 2)).all() and (got_s[rest] == 0x5A5A).all()
    rk, rv = ops.read_pages4(pages, _cuda(slots))
    for y, r in ((x[0], rk), (x[1], rv)):
        want = codes_ref(y)[2].reshape(t, heads, dim)
        want[~ok] = 0
        assert torch.equal(r.cpu(), torch.from_numpy(want))


def test_write_extremes_and_strides(ops):
    rng = _rng(9)
    t, heads, dim, page = 6, 2, 64, 16
    wide = _cuda(rng.normal(0, 1, (heads, t, 3 * dim)).astype(np.float32))
    wide[:, 0] *= 1e-42                       # subnormal components: the scale is subnormal or 0
    wide[:, 1] *= 3e37
    wide[:, 2] = 0
    wide[:, 3] *= 1e-38
    k, v = wide[:, :, :dim].transpose(0, 1), wide[:, :, dim:2 * dim].transpose(0, 1)
    pool = torch.zeros(3, 2 * heads, 1, 18 * dim, dtype=torch.uint8, device="cuda")
    mine = pool[:, heads:]                    # a layer's heads in a larger pool
    slots = torch.tensor([3, 40, 17, 18, 0, 47], device="cuda")
    ops.write_pages4(mine, slots, k, v)
    rk, rv = ops.read_pages4(mine, slots)
    for x, r in ((k, rk), (v, rv)):
        assert torch.equal(r.cpu(), torch.from_numpy(codes_ref(x.cpu().numpy())[2]).reshape(t, heads, dim))
    assert not pool[:, :heads].any()


# ---- attention

def attend_ref(q, k, v, table, lens, page, scale, cap, slope, centre, first, last, n_pages):
    """In 64 bits.  k, v [n_pages * page, heads, dim].  Returns out, lse, the sum of w |v|, the largest sum |q||k| scale, and the sum of w times the values' scales."""
    n, g, heads, dim = q.shape
    rep = heads // k.shape[1]
    out, lse, wv, big = np.zeros((n, g, heads, dim)), np.full((n, g, heads), -INF), np.zeros((n, g, heads, dim)), 0.0
    ws = np.zeros((n, g, heads, dim))
    for i in range(n):
        length = min(max(int(lens[i]), 0), table.shape[1] * page)
        at = np.arange(length)
        p = table[i, at // page].astype(np.int64)
        ok = (p >= 0) & (p < n_pages)
        rows = np.where(ok, p, 0) * page + at % page
        for a in range(g):
            seen = ok.copy()
            if first is not None:
                seen &= (at >= first[i, a]) & (at < last[i, a])
            if not seen.any():
                continue
            r, pos = rows[seen], at[seen]
            for h in range(heads):
                kk, vv = k[r, h // rep].astype(np.float64), v[r, h // rep].astype(np.float64)
                s = kk @ q[i, a, h] * scale
                big = max(big, float((np.abs(kk) @ np.abs(q[i, a, h])).max() * scale))
                if cap:
                    s = cap * np.tanh(s / cap)
                if slope is not None:
                    s = s - slope[h] * np.abs(pos - centre[i, a])
                m = s.max()
                e = np.exp(s - m)
                out[i, a, h], wv[i, a, h], lse[i, a, h] = e @ vv / e.sum(), e @ np.abs(vv) / e.sum(), m + np.log(e.sum())
                # a scale is an eighth of the group's largest component, but for its rounding to bf16
                step = np.abs(vv).reshape(len(vv), -1, 32).max(-1).repeat(32, -1) / 8 * (1 + 2.0 ** -7)
                ws[i, a, h] = e @ step / e.sum()
    return out, lse, wv, big, ws


def _memory(ops, rng, lens, heads, dim, page, width=None, spare=2, fill=0xFF):
    """A pool with keys and values of the sentences' positions, the rest of it garbage (scales that are NaN); the values that it stands for."""
    n = len(lens)
    width = max(1, -(-max(max(lens), 1) // page)) if width is None else width
    n_pages = sum(min(-(-x // page), width) for x in lens) + spare
    order = rng.permutation(n_pages)
    table, took = rng.integers(-5, n_pages + 5, (n, width)).astype(np.int32), 0
    slots = []
    for i, x in enumerate(lens):
        have = min(-(-x // page), width)
        table[i, :have] = order[took:took + have]
        took += have
        at = np.arange(min(x, width * page))
        slots.append(table[i, at // page].astype(np.int64) * page + at % page)
    slots = np.concatenate(slots)
    pages = torch.full((n_pages, heads, page // 16, 18 * dim), fill, dtype=torch.uint8, device="cuda")
    k, v = _cuda(rng.normal(0, 1, (len(slots), heads, dim)).astype(np.float32)), _cuda(rng.normal(0, 1, (len(slots), heads, dim)).astype(np.float32))
    k += _cuda(rng.normal(0, 0.5, (heads, dim)).astype(np.float32))
    ops.write_pages4(pages, _cuda(slots), k, v)
    rk, rv = ops.read_pages4(pages, _cuda(slots))
    kk, vv = np.zeros((n_pages * page, heads, dim), np.float32), np.zeros((n_pages * page, heads, dim), np.float32)
    kk[slots], vv[slots] = rk.cpu().numpy(), rv.cpu().numpy()
    return pages, table, kk, vv


def attend_check(ops, q, pages, table, lens, kk, vv, page, scale=None, cap=0.0, slope=None, centre=None, first=None, last=None, out=None):
    dev = lambda x: None if x is None else _cuda(x)
    got, lse = ops.attend_pages4(q, pages, _cuda(table), _cuda(np.asarray(lens, np.int32)), scale=scale, cap=cap, slope=dev(slope), centre=dev(centre), first=dev(first), last=dev(last), want_lse=True, out=out)
    dim = q.shape[3]
    scale = dim ** -0.5 if scale is None else scale
    big_scale = float(np.abs(vv).max()) / 7
    want, wlse, wv, big, ws = attend_ref(q.double().cpu().numpy(), kk, vv, table, lens, page, scale, cap, slope, centre, first, last, pages.shape[0])
    # A score: products of exact values added in 32 bits, at most dim + 8 additions and products; the cap's tanh to 2e-7 of the cap (16-bit queries) and the bias
    # and the change to powers of two a few roundings of their own size.  Queries in 32 bits are exact to 2^-22 in two fp16 terms.
    bias = 0.0 if slope is None else float(np.max(slope)) * (max(lens) + float(np.max(np.abs(centre))))
    lo = np.where(np.isneginf(wlse), 0, wlse)
    score = ((dim + 12) * 2.0 ** -24 + (2.0 ** -22 if q.dtype == F32 else 0)) * big + 4e-7 * cap + 6 * 2.0 ** -24 * (bias + np.abs(lo).max() + 32)
    g = got.double().cpu().numpy()
    # weights: exp2 2^-22 and sums of up to 2^12 additions a lane would be 2^-12 at worst, but each is of positive terms rounded to nearest: 64 warps' and lanes' partial
    # sums of some hundreds, 2^-24 * 300; the rounding of the weight to its terms, the output's own
    # (the product of a weight and a value's scale is rounded to fp16, for 32-bit queries to two terms)
    weight = {BF16: 2.0 ** -11, F16: 2.0 ** -11, F32: 2.0 ** -22}[q.dtype]
    # 16-bit queries: codes go into the products as 0 .. 15 and 8 for each comes off at the end, so that the sums on the way are up to 15 sum(w scale) in size whatever
    # the values are.  A warp adds a product of 16 positions (of the CTA's 64) a time to them; the matrix unit lays its 17 addends side by side and cuts each off below
    # the largest one's 24th bit, 17 * 2^-23 in all, and some 8 additions join the parts: a component whose values cancel, or whose codes are all near 8, is off by that
    # and not by a share of itself.  A weight times its scale is kept in fp16 below 2^4 times the largest scale: 2^-25 / 8 of the largest scale at least.
    steps = max(lens) / 64 + 1
    # 32-bit queries: codes are less 8 already; a weight's second term is kept to 2^-25 below 2^9 times the largest scale, and goes with codes of up to 8.
    shift = 8 * 2.0 ** -34 * big_scale * max(lens) if q.dtype == F32 else (steps * 17 + 8) * 2.0 ** -23 * 15 * ws + 8 * 2.0 ** -28 * big_scale * max(lens)
    tol = HALF_STEP[q.dtype] * np.abs(want) + (weight + 2 * score + 2.0 ** -15) * wv + shift + (2.0 ** -25 if q.dtype == F16 else 0)
    assert np.isfinite(g).all()
    assert (np.abs(g - want) <= tol).all(), float((np.abs(g - want) / np.maximum(tol, 1e-300)).max())
    l = lse.double().cpu().numpy()
    assert (np.isneginf(l) == np.isneginf(wlse)).all()
    ok = np.isfinite(wlse)
    assert (np.abs(l[ok] - wlse[ok]) <= score + 2.0 ** -15 + 2.0 ** -23 * np.abs(wlse[ok])).all()
    return got, lse


def _q(rng, n, g, heads, dim, dtype):
    return _cuda(rng.normal(0, 1.5, (n, g, heads, dim)).astype(np.float32), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim,heads,rep,g,page,lens", [
    (64, 1, 1, 1, 16, [1]), (64, 2, 1, 5, 16, [23, 0, 16, 1]), (128, 1, 4, 4, 32, [17, 64, 65]), (128, 3, 1, 12, 48, [300, 15, 31, 128]), (64, 2, 3, 11, 16, [90, 513]), (128, 2, 1, 1, 128, [1025, 2]),
    (64, 1, 1, 16, 64, [64, 63]), (128, 1, 2, 8, 16, [4100])])
def test_attend(ops, dim, heads, rep, g, page, lens, dtype):
    rng = _rng(dim, heads, rep, g, page, len(lens))
    n, q_heads = len(lens), heads * rep
    pages, table, kk, vv = _memory(ops, rng, lens, heads, dim, page)
    q = _q(rng, n, g, q_heads, dim, dtype)
    attend_check(ops, q, pages, table, lens, kk, vv, page)
    slope, centre = (0.5 ** (1 + np.arange(q_heads) * 0.7)).astype(np.float32), (rng.random((n, g)) * (np.array(lens)[:, None] + 3) - 2).astype(np.float32)
    a, b = rng.integers(-3, max(lens) + 3, (2, n, g)).astype(np.int32)
    first, last = np.minimum(a, b), np.maximum(a, b)
    first[0, 0], last[0, 0] = 5, 5            # a row that sees nothing
    last[-1, -1] = 2 ** 31 - 1
    first[-1, -1] = -2 ** 31
    attend_check(ops, q, pages, table, lens, kk, vv, page, scale=0.3, cap=5.0)
    attend_check(ops, q, pages, table, lens, kk, vv, page, slope=slope, centre=centre)
    attend_check(ops, q, pages, table, lens, kk, vv, page, first=first, last=last)
    attend_check(ops, q, pages, table, lens, kk, vv, page, scale=0.2, cap=20.0, slope=slope, centre=centre, first=first, last=last)
    # one document after the other, each row its own; and what a causal mask leaves of them
    half = np.tile((np.array(lens) // 2).astype(np.int32)[:, None], (1, g))
    attend_check(ops, q, pages, table, lens, kk, vv, page, first=half, last=np.maximum(half, np.array(lens, np.int32)[:, None] - np.arange(g, dtype=np.int32)))


def test_attend_pages_outside_the_pool_and_lengths_outside_the_table(ops):
    rng = _rng(11)
    lens = [100, 70, 64, 33]
    pages, table, kk, vv = _memory(ops, rng, lens, 2, 64, 16)
    q = _q(rng, 4, 3, 2, 64, F16)
    table[0, 2], table[0, 5], table[1, 0], table[1, 4] = -1, pages.shape[0], -2 ** 31, 2 ** 31 - 1
    table[3, :3] = -1                          # no page at all: nothing is seen
    attend_check(ops, q, pages, table, lens, kk, vv, 16)
    attend_check(ops, q, pages, table[:, :4].copy(), [100, -7, 2 ** 31 - 1, 0], kk, vv, 16)
    zero = np.zeros((4, 0), np.int32)
    out, lse = ops.attend_pages4(q, pages, _cuda(zero), _cuda(np.array(lens, np.int32)), want_lse=True)
    assert not out.any() and torch.isneginf(lse).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_attend_long_and_split(ops, dtype):
    rng = _rng(12)
    lens = [9000, 3, 7001]
    pages, table, kk, vv = _memory(ops, rng, lens, 2, 128, 64)
    q = _q(rng, 3, 6, 4, 128, dtype)
    attend_check(ops, q, pages, table, lens, kk, vv, 64)
    first = np.array([[0, 8999, 4000, 10, 16, 2000]] * 3, np.int32)
    last = np.array([[9000, 9000, 4001, 8000, 32, 2048]] * 3, np.int32)
    attend_check(ops, q, pages, table, lens, kk, vv, 64, first=first, last=last)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens", [[5000, 1, 1, 1, 4000, 0, 0, 700], [33] * 150, [3] * 40 + [6000] + [50] * 30, [0, 0, 0], [1] * 700 + [900] + [2] * 300, [129, 130, 8000, 257]])
def test_attend_shares_of_uneven_sentences(ops, lens, dtype):
    """Segments that several CTAs share, that share a CTA, and both: long sentences before, between and behind short ones."""
    rng = _rng(sum(lens), len(lens))
    pages, table, kk, vv = _memory(ops, rng, lens, 2, 64, 16)
    n, g = len(lens), 9
    q = _q(rng, n, g, 4, 64, dtype)                    # 18 rows a head of the pool: two row tiles
    attend_check(ops, q, pages, table, lens, kk, vv, 16)
    a, b = rng.integers(0, max(lens) + 1, (2, n, g)).astype(np.int32)
    attend_check(ops, q, pages, table, lens, kk, vv, 16, first=np.minimum(a, b), last=np.maximum(a, b))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_attend_values_of_all_sizes(ops, dtype):
    """Values that grow and shrink along the positions by 2^16, and values and queries that are small or large throughout: the result is as exact as its largest parts
    allow, whatever came first."""
    rng = _rng(21)
    lens, heads, dim, page = [700, 333, 64], 2, 128, 32
    n_pages, width = 40, 22
    table = rng.permutation(n_pages)[:3 * 13].reshape(3, 13)
    table = np.concatenate([table, np.full((3, width - 13), -1)], 1).astype(np.int32)
    table[0] = rng.permutation(n_pages)[:width]
    lens[1], lens[2] = 333, 64
    table[1:] = np.array([[i for i in range(n_pages) if i not in table[0]][:11] + [-1] * 11, [i for i in range(n_pages) if i not in table[0]][11:13] + [-1] * 20])
    slots = np.concatenate([table[i, np.arange(x) // page].astype(np.int64) * page + np.arange(x) % page for i, x in enumerate(lens)])
    at = np.concatenate([np.arange(x) for x in lens])
    top = {BF16: 1e30, F16: 1e4, F32: 1e20}[dtype]
    for sizes, q_size in ((2.0 ** (at % 17 - 8), 1.0), (2.0 ** -(at / 50), 1.0), (2.0 ** (at / 50), 1.0), (np.full(len(at), 1e-9 if dtype != F16 else 1e-3), 1e-3), (np.full(len(at), top), 1e2)):
        k, v = rng.normal(0, 1, (len(slots), heads, dim)), rng.normal(0, 1, (len(slots), heads, dim)) * sizes[:, None, None]
        pages = ops.new_pages4(n_pages, heads, dim, page)
        ops.write_pages4(pages, _cuda(slots), _cuda(k.astype(np.float32)), _cuda(v.astype(np.float32)))
        rk, rv = ops.read_pages4(pages, _cuda(slots))
        kk, vv = np.zeros((n_pages * page, heads, dim), np.float32), np.zeros((n_pages * page, heads, dim), np.float32)
        kk[slots], vv[slots] = rk.cpu().numpy(), rv.cpu().numpy()
        q = _q(rng, 3, 4, 4, dim, F32).mul_(q_size).to(dtype)
        attend_check(ops, q, pages, table, lens, kk, vv, page, scale=dim ** -0.5 / q_size)


def test_attend_strides(ops):
    rng = _rng(13)
    lens = [50, 200]
    pool = torch.zeros(40, 6, 2, 18 * 64, dtype=torch.uint8, device="cuda")
    pages, table, kk, vv = _memory(ops, rng, lens, 2, 64, 32)
    pool[:pages.shape[0], 3:5] = pages
    for dtype in (BF16, F32):
        wide = torch.zeros(5, 2, 4, 64 + 6, dtype=dtype, device="cuda")
        q = wide.permute(1, 0, 2, 3)[..., 2:66]           # [n, g, heads, dim], 4- or 8-byte aligned
        q.copy_(_q(rng, 2, 5, 4, 64, dtype))
        odd = torch.full((2, 4, 5, 67), 7.0, dtype=dtype, device="cuda")
        out = odd.transpose(1, 2)[..., 1:65]              # and one that is not
        tab = torch.zeros(2, table.shape[1] + 5, dtype=torch.int32, device="cuda")
        tab[:, 2:2 + table.shape[1]] = _cuda(table)
        want, wl = attend_check(ops, q.contiguous(), pages, table, lens, kk, vv, 32)
        got, lse = ops.attend_pages4(q, pool[:pages.shape[0], 3:5], tab[:, 2:2 + table.shape[1]], _cuda(np.array(lens, np.int32)), out=out, want_lse=True)
        assert got is out and torch.equal(got, want) and torch.equal(lse, wl)
        assert (odd[..., 0] == 7).all() and (odd[..., 65:] == 7).all()


def test_far_pages(ops):
    """Pages past 2^31 bytes and positions past 2^31 / dim of a pool."""
    rng = _rng(14)
    heads, dim, page = 2, 128, 128
    n_pages = (5 << 29) // (heads * page // 16 * 18 * dim)              # 2.7 GB
    pool = torch.empty(n_pages, heads, page // 16, 18 * dim, dtype=torch.uint8, device="cuda")
    lens = [200, 129]
    table = np.array([[n_pages - 1, n_pages - 7], [n_pages - 3, n_pages - 2]], np.int32)
    slots = np.concatenate([table[i, np.arange(x) // page].astype(np.int64) * page + np.arange(x) % page for i, x in enumerate(lens)])
    k, v = _cuda(rng.normal(0, 1, (329, heads, dim)).astype(np.float32)), _cuda(rng.normal(0, 1, (329, heads, dim)).astype(np.float32))
    ops.write_pages4(pool, _cuda(slots), k, v)
    rk, rv = ops.read_pages4(pool, _cuda(slots))
    assert torch.equal(rk.cpu(), torch.from_numpy(codes_ref(k.cpu().numpy())[2]).reshape(rk.shape))
    low = int(table.min())
    kk, vv = (np.zeros(((n_pages - low) * page, heads, dim), np.float32) for _ in range(2))
    kk[slots - low * page], vv[slots - low * page] = rk.cpu().numpy(), rv.cpu().numpy()
    q = _q(rng, 2, 3, 2, dim, F16)
    got, _ = ops.attend_pages4(q, pool, _cuda(table), _cuda(np.array(lens, np.int32)), want_lse=True)
    near = pool[low:].clone()
    want, _ = attend_check(ops, q, near, table - low, lens, kk, vv, page)
    assert torch.equal(got, want)


def test_attend_refuses(ops):
    pages, q = ops.new_pages4(4, 2, 64, 16), torch.zeros(1, 2, 4, 64, dtype=BF16, device="cuda")
    table, lens = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    f = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    for bad in (lambda: ops.attend_pages4(q.double(), pages, table, lens), lambda: ops.attend_pages4(q[..., :32], pages, table, lens), lambda: ops.attend_pages4(q[:, :, :3], pages, table, lens),
                lambda: ops.attend_pages4(q, pages.int(), table, lens), lambda: ops.attend_pages4(q, pages, table.long(), lens), lambda: ops.attend_pages4(q, pages, table, lens.long()),
                lambda: ops.attend_pages4(q, pages, table, lens, first=f), lambda: ops.attend_pages4(q, pages, table, lens, slope=torch.zeros(4, device="cuda")), lambda: ops.attend_pages4(q, pages, table, lens, cap=-1.0),
                lambda: ops.attend_pages4(q, pages, table, lens, scale=float("nan")), lambda: ops.attend_pages4(q, pages, table, lens, first=f.float(), last=f),
                lambda: ops.attend_pages4(q, pages, table, lens, out=torch.zeros(1, 2, 4, 64, device="cuda")), lambda: ops.attend_pages4(q.transpose(2, 3), pages, table, lens),
                lambda: ops.attend_pages4(q, pages[:, :, :, :576].reshape(4, 2, 1, 576), table, lens), lambda: ops.attend_pages4(q, pages, table, lens.cpu()), lambda: ops.attend_pages4(q.cpu(), pages, table, lens)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    for bad in (lambda: ops.new_pages4(4, 2, 64, 24), lambda: ops.new_pages4(4, 2, 96, 16), lambda: ops.write_pages4(pages, torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, 2, 64, dtype=BF16, device="cuda")),
                lambda: ops.write_pages4(pages, torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda")),
                lambda: ops.write_pages4(pages, torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(3, 2, 65, device="cuda")[..., 1:], torch.zeros(3, 2, 64, device="cuda")),
                lambda: ops.beam_select(torch.zeros(1, 33, 50, device="cuda"), torch.zeros(1, 33, device="cuda")), lambda: ops.beam_select(torch.zeros(1, 3, 50, device="cuda"), torch.zeros(1, 3, device="cuda"), eos=50),
                lambda: ops.beam_select(torch.zeros(1, 3, 50, device="cuda").transpose(1, 2), torch.zeros(1, 50, device="cuda")), lambda: ops.beam_select(torch.zeros(1, 3, 50, device="cuda"), torch.zeros(1, 3, device="cuda"), done=torch.zeros(1, 3, device="cuda")),
                lambda: ops.beam_select(torch.zeros(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda"), allowed=torch.zeros(2, 1, dtype=torch.int32, device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            bad()


def test_results_that_lie_upon_what_is_read(ops):
    """Results may take the place of scores, finished flags and queries, or lie between the queries; whatever would be written while it is still read is refused."""
    rng = _rng(77)
    n, k, v = 4, 6, 300
    x = _logits(rng, n, k, v, F32)
    pool = torch.zeros(5 * n * k, dtype=torch.int32, device="cuda")
    ints = lambda at: pool[at:at + n * k].view(n, k)
    tokens, parents, scores = ints(0), ints(n * k), pool[2 * n * k:3 * n * k].view(F32).view(n, k)
    scores.copy_(_cuda(rng.normal(-10, 3, (n, k)).astype(np.float32)))
    flags = torch.zeros(2 * n * k, dtype=torch.bool, device="cuda")
    done = flags[:n * k].view(n, k)
    later = pool[2 * n * k + k:3 * n * k + k].view(F32).view(n, k)
    for out in ((tokens, tokens, scores, done), (tokens, ints(k), scores, done), (tokens, parents, later, done), (scores.view(torch.int32), parents, later, done),
                (tokens, parents, scores, flags[k:k + n * k].view(n, k)), (x.view(-1)[:n * k].view(torch.int32).view(n, k), parents, scores, done)):
        with pytest.raises(ValueError, match="overlap"):
            ops.beam_select(x, scores, done=done, out=out)
    want = ops.beam_select(x, scores, done=done)
    got = ops.beam_select(x, scores, done=done, out=(tokens, parents, scores, done))
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    for lens in ([40, 3], [3000, 700]):
        pages, table, kk, vv = _memory(ops, rng, lens, 2, 64, 16)
        fused = torch.zeros(2, 5, 3, 4, 64, dtype=BF16, device="cuda")
        q, beside = fused[:, :, 0], fused[:, :, 1]
        q.copy_(_q(rng, 2, 5, 4, 64, BF16))
        at = lambda **kw: ops.attend_pages4(q, pages, _cuda(table), _cuda(np.asarray(lens, np.int32)), **kw)
        want = at()
        for out in (fused.view(2, 5, 12, 64)[:, :, 2:6], fused.view(-1)[64:64 + 2 * 5 * 12 * 64 - 128].as_strided((2, 5, 4, 64), (5 * 768, 768, 64, 1))):
            with pytest.raises(ValueError, match="overlaps"):
                at(out=out)
        assert torch.equal(at(out=beside), want) and torch.equal(beside, want) and torch.equal(at(out=q), want) and torch.equal(q, want)


def test_gradients_are_refused(ops):
    """No backward pass: a call that would drop a gradient does not go through."""
    x, s = torch.zeros(1, 2, 50, device="cuda", requires_grad=True), torch.zeros(1, 2, device="cuda")
    h, parents = torch.zeros(1, 2, 8, device="cuda", requires_grad=True), torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    for call in (lambda: ops.beam_select(x, s), lambda: ops.beam_reorder([h], parents)):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()


# ---- together

class Toy:
    """A decoder with attention over pages: enough of a model for the operators to be used as they would be.  The source is written once per sentence; a beam's state is a
    vector that attends over it and makes the next word's logits."""

    def __init__(self, rng, n, k, heads=2, dim=64, vocab=500):
        self.n, self.k, self.heads, self.dim, self.vocab = n, k, heads, dim, vocab
        w = heads * dim
        self.emb, self.out, self.mix = (_cuda(rng.normal(0, s, sh).astype(np.float32)) for s, sh in ((1.0, (vocab, w)), (0.6, (w, vocab)), (0.05, (2 * w, w))))

    def step(self, state, word, context):
        n, k, w = self.n, self.k, self.heads * self.dim
        state = torch.tanh(torch.cat([state, context.reshape(n, k, w)], -1) @ self.mix + self.emb[word.long()])
        return state, state @ self.out


def _decode(ops, toy, lens, keys, values, steps, page=16, reference=False):
    n, k = toy.n, toy.k
    dev = "cuda"
    width = -(-max(lens) // page)
    pages = ops.new_pages4(n * width, toy.heads, toy.dim, page)
    pages.fill_(0xFF)
    table = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    free = torch.arange(n * width, dtype=torch.int32, device=dev).flip(0).contiguous()
    used = torch.zeros(1, dtype=torch.int32, device=dev)
    new = _cuda(np.array(lens, np.int32))
    # the source arrives in two parts: all but the last position, then that
    for old, now in ((None, new - 1), (new - 1, new)):
        total = int((now - (0 if old is None else old)).sum())
        slots, starts, used = ops.plan_pages(old, now, table, free, used, page=page, total=total)
        rows = torch.cat([torch.arange(0 if old is None else int(old[i]), int(now[i]), device=dev) + i * max(lens) for i in range(n)])
        ops.write_pages4(pages, slots, keys[rows], values[rows])
    state = torch.zeros(n, k, toy.heads * toy.dim, device=dev)
    scores = torch.full((n, k), -INF, device=dev)
    scores[:, 0] = 0
    done = torch.zeros(n, k, dtype=torch.bool, device=dev)
    word = torch.zeros(n, k, dtype=torch.int32, device=dev)
    words = torch.zeros(n, k, steps, dtype=torch.int32, device=dev)
    for t in range(steps):
        q = state.view(n, k, toy.heads, toy.dim)
        if reference:
            kk, vv = (torch.zeros(pages.shape[0] * page, toy.heads, toy.dim) for _ in range(2))
            for i, x in enumerate(lens):
                at = torch.arange(x, device=dev)
                s = table[i, at // page].long() * page + at % page
                rk, rv = ops.read_pages4(pages, s)
                kk[s.cpu()], vv[s.cpu()] = rk.cpu(), rv.cpu()
            c, _, _, _, _ = attend_ref(q.double().cpu().numpy(), kk.numpy(), vv.numpy(), table.cpu().numpy(), lens, page, toy.dim ** -0.5, 0.0, None, None, None, None, pages.shape[0])
            context = _cuda(c.astype(np.float32))
        else:
            context = ops.attend_pages4(q, pages, table, new)
        state, logits = toy.step(state, word, context)
        if reference:
            tok, par, sc, fin = select_ref(logits, scores, done)
            word, parents, scores, done = _cuda(tok), _cuda(par), _cuda(sc.astype(np.float32)), _cuda(fin)
            state, words = _reordered(state, parents), _reordered(words, parents)
        else:
            word, parents, scores, done = ops.beam_select(logits, scores, done=done)
            ops.beam_reorder([state, words], parents)
        words[:, :, t] = word
    return words, scores, done


def test_together(ops):
    rng = _rng(15)
    lens = [37, 1, 16, 50]
    n, k = len(lens), 5
    toy = Toy(rng, n, k)
    keys, values = (_cuda(rng.normal(0, 1, (n * max(lens), toy.heads, toy.dim)).astype(np.float32)) for _ in range(2))
    words, scores, done = _decode(ops, toy, lens, keys, values, 9)
    w2, s2, d2 = _decode(ops, toy, lens, keys, values, 9, reference=True)
    assert torch.equal(words, w2) and torch.equal(done, d2)
    assert (scores - s2).abs().max() <= 9 * 2e-4      # nine steps' logits, each within 1e-4 for contexts that are 1e-6 apart


def _step_inputs(rng, n=3, k=4, v=700):
    return _logits(rng, n, k, v, F32), _cuda(rng.normal(-5, 1, (n, k)).astype(np.float32))


def test_captured_and_replayed(ops):
    """A step captured into two graphs that are replayed at once on streams of their own, with other inputs than it was captured with."""
    rng = _rng(16)
    lens = [3000, 17, 450]
    pages, table, kk, vv = _memory(ops, rng, lens, 2, 64, 32)
    tab, ln = _cuda(table), _cuda(np.array(lens, np.int32))

    def one():
        x, scores = _step_inputs(rng)
        q = _q(rng, 3, 4, 2, 64, F32)
        state = _cuda(rng.normal(0, 1, (2, 3, 4, 33)).astype(np.float32))
        old = torch.tensor([5, 0, 15], dtype=torch.int32, device="cuda")
        new = old + 3
        free, used, grown = torch.arange(9, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda")

        def step():
            out, lse = ops.attend_pages4(q, pages, tab, ln, want_lse=True)
            tokens, parents, sc, done = ops.beam_select(x, scores)
            moved = ops.beam_reorder([state], parents, out=[torch.empty_like(state)])[0]
            slots, starts, now = ops.plan_pages(old, new, grown, free, used, page=16, total=9)
            return dict(out=out, lse=lse, tokens=tokens, parents=parents, scores=sc, done=done, moved=moved, slots=slots, starts=starts, used=now)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        return graph, res, step, x, q, torch.cuda.Stream()

    runs = [one(), one()]
    for turn in range(3):
        want = []
        for _, _, step, x, q, _ in runs:
            x.copy_(_step_inputs(rng)[0])
            q.copy_(_q(rng, 3, 4, 2, 64, F32))
            want.append({name: y.clone() for name, y in step().items()})
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, _, _, _, _, st in runs:
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, res, *_), w in zip(runs, want):
            assert [name for name in w if not torch.equal(res[name], w[name])] == []


def test_streams(ops):
    """Calls on four streams at once give what they give alone; a call on a stream comes after what that stream holds."""
    rng = _rng(17)
    lens = [2500, 300]
    pages, table, kk, vv = _memory(ops, rng, lens, 2, 128, 16)
    tab, ln = _cuda(table), _cuda(np.array(lens, np.int32))
    work = [(_q(rng, 2, 5, 4, 128, BF16), *_step_inputs(rng, 6, 5, 9000)) for _ in range(4)]
    alone = [(ops.attend_pages4(q, pages, tab, ln), ops.beam_select(x, s)) for q, x, s in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(5):
        got = []
        for st, (q, x, s) in zip(streams, work):
            with torch.cuda.stream(st):
                late = torch.zeros_like(x)
                torch.cuda._sleep(200000)
                late.copy_(x)
                got.append((ops.attend_pages4(q, pages, tab, ln), ops.beam_select(late, s)))
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(alone, got):
            assert torch.equal(a, c) and all(torch.equal(x, y) for x, y in zip(b, d))


def test_a_call_leaves_the_current_device_and_waits_for_nothing(ops):
    assert torch.cuda.current_device() == 0
    x, s = _step_inputs(_rng(18), 64, 12, 30000)
    done = torch.cuda.Event()
    torch.cuda._sleep(50_000_000)
    ops.beam_select(x, s)
    done.record()
    assert not done.query()                # the call came back before the stream did
    torch.cuda.synchronize()
    assert torch.cuda.current_device() == 0

"""Pages that follow their hypotheses, are given back, moved and copied, against plain implementations; and a decoder that uses them with all else."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_device_ops import BF16, F16, F32, HALF_STEP, INF, _cuda, _rng
from test_gpu_pages8 import attend_ref


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from linmt_b200 import device_ops
    return device_ops


def _i32(x):
    return _cuda(np.asarray(x, np.int32))


def fork_ref(table, lens, parents, shares, free, used, page, done=None):
    """The definition, row by row."""
    n, k, width = table.shape
    n_pages, n_free = len(shares), len(free)
    old, length = table.reshape(n * k, width), np.clip(lens.reshape(-1), 0, width * page)
    have = -(-length // page)
    rows = np.arange(n * k)
    up = rows if parents is None else np.where((parents.reshape(-1) >= 0) & (parents.reshape(-1) < k), rows // k * k + parents.reshape(-1), -1)
    if done is not None:
        up = np.where(done.reshape(-1) != 0, -1, up)
    shares, free = shares.copy(), free.copy()
    kept = np.zeros(n * k, bool)
    new, new_len, copies = np.full((n * k, width), -1), np.zeros(n * k, int), []
    for r in rows:
        for c in range(have[r]):
            if 0 <= old[r, c] < n_pages:
                shares[old[r, c]] -= 1
    for r in rows:
        p = up[r]
        if p < 0:
            continue
        new_len[r] = length[p]
        for c in range(have[p]):
            g = old[p, c]
            if not 0 <= g < n_pages:
                continue
            if c == have[p] - 1 and length[p] % page and kept[p]:
                copies.append((r, c, g))
                continue
            new[r, c] = g
            shares[g] += 1
        kept[p] = True
    used = min(max(used, 0), n_free)
    gone = np.flatnonzero(shares < 0)
    for i, g in enumerate(gone):
        at = used - len(gone) + i
        if at >= 0:
            free[at] = g
    shares[gone] = 0
    at = max(used - len(gone), 0)
    src, dst = np.full(n * k, -1), np.full(n * k, -1)
    for i, (r, c, g) in enumerate(copies):
        src[i], dst[i] = g, free[at + i] if at + i < n_free else -1
        new[r, c] = dst[i]
    return new.reshape(table.shape), new_len.reshape(n, k), shares, free, at + len(copies), src, dst


def compact_ref(table, lens, shares, page):
    shape, width, n_pages = table.shape, table.shape[-1], len(shares)
    rows, length = table.reshape(-1, width), np.clip(lens.reshape(-1), 0, width * page)
    named = (np.arange(width) < -(-length // page)[:, None]) & (rows >= 0) & (rows < n_pages)
    live = np.zeros(n_pages, bool)
    live[rows[named]] = True
    u = live.sum()
    src, dst = np.flatnonzero(live & (np.arange(n_pages) >= u)), np.flatnonzero(~live & (np.arange(n_pages) < u))
    to = np.arange(n_pages)
    to[src] = dst
    out = np.zeros(n_pages, int)
    out[to[live]] = shares[live]
    pad = lambda x: np.concatenate([x, np.full(n_pages // 2 - len(x), -1)])
    return np.where(named, to[np.where(named, rows, 0)], -1).reshape(shape), out, np.arange(n_pages), u, pad(src), pad(dst)


def _state(rng, n, k, lens, page, spare, shared=0.5):
    """Hypotheses that share the full pages of a common past; lens [n, k]."""
    width = max(1, -(-int(lens.max()) // page))
    count = int(sum(-(-x // page) for x in lens.reshape(-1)))
    n_pages = count + spare
    order = rng.permutation(n_pages)
    table, shares, used = np.full((n, k, width), -1), np.zeros(n_pages, int), 0
    for i in range(n):
        common = int(rng.random() * (lens[i].min() // page + 1)) if rng.random() < shared * 2 else 0
        for j in range(k):
            for c in range(-(-lens[i, j] // page)):
                if c < common and j:
                    table[i, j, c] = table[i, 0, c]
                    shares[table[i, 0, c]] += 1
                else:
                    table[i, j, c] = order[used]
                    used += 1
    return table, shares, order, used


def fork_check(ops, table, lens, parents, shares, free, used, page, done=None, out=None):
    want = fork_ref(table, lens, parents, shares, free, used, page, done)
    dev = [_i32(x) for x in (table, lens, shares, free, [used])]
    d = None if done is None else _cuda(done)
    if parents is None:
        got = ops.free_pages(dev[0], dev[1], d, *dev[2:], page=page)
        want = want[:5]
    else:
        got = ops.fork_pages(dev[0], dev[1], _i32(parents), *dev[2:], page=page, done=d)
    for name, g, w in zip(("table", "lens", "shares", "free", "used", "src", "dst"), got, want):
        assert (g.cpu().numpy() == w).all(), name
    return got


@pytest.mark.parametrize("n,k,page,lo,hi", [(1, 1, 16, 0, 40), (3, 4, 16, 0, 100), (64, 12, 16, 20, 90), (7, 31, 32, 1, 200), (1, 700, 16, 0, 50), (300, 8, 48, 0, 300), (2, 5, 1, 0, 40), (40, 13, 100, 350, 9000)])
def test_fork(ops, n, k, page, lo, hi):
    rng = _rng(n, k, page, hi)
    for even in (True, False):
        lens = np.repeat(rng.integers(lo, hi + 1, (n, 1)), k, 1) if even else rng.integers(lo, hi + 1, (n, k))
        table, shares, free, used = _state(rng, n, k, lens, page, n * k + 3)
        for parents in (rng.integers(0, k, (n, k)), np.zeros((n, k), int), np.broadcast_to(np.arange(k), (n, k)).copy(), rng.integers(-2, k + 2, (n, k)), np.full((n, k), -1)):
            fork_check(ops, table, lens, parents, shares, free, used, page)
        fork_check(ops, table, lens, rng.integers(0, k, (n, k)), shares, free, used, page, done=rng.random((n, k)) < 0.3)
        fork_check(ops, table, lens, None, shares, free, used, page, done=rng.random((n, k)) < 0.5)
        fork_check(ops, table, lens, None, shares, free, used, page, done=np.ones((n, k), np.uint8))


@pytest.mark.parametrize("n_pages", [40000, 300000])
def test_fork_in_large_pools(ops, n_pages):
    """Pages that are left over all over a pool of more than a warp remembers."""
    rng = _rng(n_pages)
    n, k, page = 200, 6, 16
    lens = rng.integers(1, 300, (n, k))
    table, shares, free, used = _state(rng, n, k, lens, page, 0)
    spread = rng.permutation(n_pages)
    big = np.zeros(n_pages, int)
    big[spread[:len(shares)]] = shares
    fork_check(ops, np.where(table >= 0, spread[table], -1), lens, rng.integers(-1, k, (n, k)), big, spread, used, page)


def test_fork_where_the_free_pages_run_out(ops):
    rng = _rng(2)
    n, k, page = 5, 6, 16
    lens = np.full((n, k), 37)
    table, shares, free, used = _state(rng, n, k, lens, page, 0)
    parents = np.zeros((n, k), int)
    # with no page to spare the copies get what the call gives back; with none of that either, nothing
    got = fork_check(ops, table, lens, parents, shares, free, used, page)
    assert int(got[4]) <= len(free)
    table[:, 1:], lens[:, 1:] = -1, 0
    got = fork_check(ops, table, lens, parents, np.zeros_like(shares), free, len(free) - 3, page)
    assert int(got[4]) == len(free) - 3 + n * (k - 1) and (got[6].cpu().numpy()[:25] == -1).sum() == 22
    for used in (-5, 10 ** 6, 2 ** 31 - 1):
        fork_check(ops, table, lens, parents, np.zeros_like(shares), free, used, page)
    fork_check(ops, table, lens, np.full((n, k), -1), np.zeros_like(shares), free[:2], 1, page)          # more comes back than was taken


def test_fork_lengths_and_entries_outside(ops):
    rng = _rng(3)
    n, k, page, width = 4, 3, 16, 5
    table = rng.permutation(200)[:n * k * width].reshape(n, k, width)
    table[0, 0, 2], table[1, 1, 0], table[2, 2, 4], table[3, 0, 1] = -1, 10 ** 9, -2 ** 31, 200
    lens = np.array([[37, -4, 10 ** 9], [2 ** 31 - 1, 3, 80], [79, 81, 16], [17, 15, 1]])
    for parents in (rng.integers(0, k, (n, k)), np.ones((n, k), int)):
        fork_check(ops, table, lens, parents, np.zeros(200, int), rng.permutation(200), 90, page)


def test_fork_in_place_strided_and_empty(ops):
    rng = _rng(4)
    n, k, page = 9, 4, 16
    lens = rng.integers(1, 60, (n, k))
    table, shares, free, used = _state(rng, n, k, lens, page, 50)
    parents = rng.integers(0, k, (n, k))
    want = fork_ref(table, lens, parents, shares, free, used, page)
    wide = torch.zeros(n, k, table.shape[2] + 3, dtype=torch.int32, device="cuda")[:, :, 2:2 + table.shape[2]]
    wide.copy_(_i32(table))
    s, f, u = _i32(shares), _i32(free), _i32([used])
    out = (torch.zeros(table.shape, dtype=torch.int32, device="cuda"), torch.zeros(n, k, dtype=torch.int32, device="cuda"), s, f, u, torch.zeros(n * k, dtype=torch.int32, device="cuda"), torch.zeros(n * k, dtype=torch.int32, device="cuda"))
    versions = [x._version for x in out]
    assert ops.fork_pages(wide, _i32(lens), _i32(parents), s, f, u, page=page, out=out) is out
    for g, w in zip(out, want):
        assert (g.cpu().numpy() == w).all()
    assert all(x._version > v for x, v in zip(out, versions))
    empty = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")
    for a, b in ((0, 4), (3, 0), (3, 2)):
        got = ops.fork_pages(empty(a, b, 0), empty(a, b), empty(a, b), empty(5), empty(7), empty(1), page=16)
        assert got[0].shape == (a, b, 0) and int(got[4]) == 0
    ops.fork_pages(empty(2, 2, 3), empty(2, 2), empty(2, 2), empty(0), empty(0), empty(1), page=16)
    ops.free_pages(empty(4, 3), empty(4), torch.ones(4, dtype=torch.bool, device="cuda"), empty(5), empty(5), empty(1), page=16)


@pytest.mark.parametrize("n,page,lo,hi,spare", [(1, 16, 0, 5, 0), (5, 16, 0, 300, 30), (64, 16, 1, 400, 700), (700, 32, 0, 900, 20000), (50, 48, 1, 4000, 3), (3, 16, 20, 40, 300000)])
def test_compact(ops, n, page, lo, hi, spare):
    rng = _rng(n, page, hi, spare)
    for k in (1, 3):
        lens = rng.integers(lo, hi + 1, (n, k))
        table, shares, _, _ = _state(rng, n, k, lens, page, spare)
        for drop in (0.0, 0.6):
            gone = rng.random((n, k)) < drop
            length = np.where(gone, 0, lens)
            sh = shares.copy()
            if drop:
                sh[:] = 0
                names = table.reshape(n * k, -1)[~gone.reshape(-1)]
                g, c = np.unique(names[names >= 0], return_counts=True)
                sh[g] = c - 1
            want = compact_ref(table, length, sh, page)
            t, l, s = _i32(table), _i32(length), _i32(sh)
            got = ops.compact_pages(t, l, s, page=page)
            for name, g, w in zip(("table", "shares", "free", "used", "src", "dst"), got, want):
                assert (g.cpu().numpy() == w).all(), name
            again = ops.compact_pages(t, l, s, page=page, out=(t, s) + tuple(torch.empty_like(x) for x in got[2:]))
            assert again[0] is t and (t == got[0]).all() and (s == got[1]).all()
            flat = ops.compact_pages(t.view(n * k, -1), l.view(-1), s, page=page)          # dense already: nothing moves
            assert (flat[4] == -1).all() and (flat[0].view_as(t) == t).all()


@pytest.mark.parametrize("dtype,shape", [(torch.uint8, (3, 2, 2064)), (BF16, (7, 5)), (F32, (129,)), (torch.uint8, (13,)), (torch.int64, ()), (torch.uint8, (40, 4112)), (F16, (2, 8192))])
def test_copy(ops, dtype, shape):
    rng = _rng(len(shape), 6)
    n = 90
    make = lambda: torch.randint(0, 100, (n, *shape), device="cuda").to(dtype)
    pools = [make() for _ in range(18)]
    whole = torch.randint(0, 100, (2 * n, *shape), device="cuda").to(dtype)
    pools.append(whole[::2])
    order = rng.permutation(n)
    src, dst = order[:30], order[30:60].copy()
    src = np.concatenate([src, [-1, 5, n, 7, -2 ** 31, 2 ** 31 - 1, order[60]]])
    dst = np.concatenate([dst, [order[61], -1, order[62], n, order[63], 3, 10 ** 9]])
    want = [p.clone() for p in pools]
    other = whole[1::2].clone()
    for w in want:
        w[order[30:60]] = w[order[:30]]
    versions = [p._version for p in pools]
    got = ops.copy_pages(pools, _i32(src), _i32(dst))
    assert all((g == w).all() for g, w in zip(got, want)) and (whole[1::2] == other).all()
    assert all(p._version > v for p, v in zip(pools, versions))
    ops.copy_pages(pools, _i32([]), _i32([]))
    ops.copy_pages([], _i32([1]), _i32([2]))


def test_copy_far_pages(ops):
    pool = torch.zeros(40, 1 << 27, dtype=torch.uint8, device="cuda")
    pool[39, -1], pool[0, 5] = 9, 4
    ops.copy_pages([pool], _i32([39, 0]), _i32([1, 38]))
    assert pool[1, -1] == 9 and pool[38, 5] == 4 and pool[2:38].count_nonzero() == 0


def test_refusals(ops):
    n, k, w, p = 3, 2, 4, 20
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    args = lambda: [z(n, k, w), z(n, k), z(n, k), z(p), z(p), z(1)]
    ops.fork_pages(*args(), page=16)
    whole = z(400)
    for i, bad, match in [(0, z(n, k), "table"), (0, z(n, k + 1, w), "table"), (0, z(n, k, w).long(), "int32"), (0, z(n, w, k).transpose(1, 2), "contiguous"), (0, z(2 * n, k, w)[::2], "evenly"), (1, z(n), "lens"), (2, z(n, k + 1), "shape"),
                          (3, z(2, p), "shares"), (4, z(p).long(), "Int"), (5, z(2), "shape"), (5, z(1).cpu(), "CUDA")]:
        a = args()
        a[i] = bad
        with pytest.raises(ValueError, match=match):
            ops.fork_pages(*a, page=16)
    with pytest.raises(ValueError, match="page = 0"):
        ops.fork_pages(*args(), page=0)
    with pytest.raises(ValueError, match="16384"):
        ops.fork_pages(z(1, 16385, 1), z(1, 16385), z(1, 16385), z(p), z(p), z(1), page=16)
    with pytest.raises(ValueError, match="tuple of 7"):
        ops.fork_pages(*args(), page=16, out=args())
    a = args()
    out = [z(n, k, w), z(n, k), z(p), z(p), z(1), z(n * k), z(n * k)]
    for i, j, match in [(0, 0, "table"), (1, 1, "lens"), (1, 2, "parents")]:
        o = list(out)
        o[i] = a[j]
        with pytest.raises(ValueError, match="overlaps " + match):
            ops.fork_pages(*a, page=16, out=o)
    o = list(out)
    o[2] = o[3]
    with pytest.raises(ValueError, match="overlaps out"):
        ops.fork_pages(*a, page=16, out=o)
    o = list(out)
    o[3] = a[3]                                             # the free pages into the shares' array
    with pytest.raises(ValueError, match="overlaps shares"):
        ops.fork_pages(*a, page=16, out=o)
    a[3], o = whole[:p], list(out)
    o[2] = whole[1:p + 1]
    with pytest.raises(ValueError, match="overlaps shares"):
        ops.fork_pages(*a, page=16, out=o)
    with pytest.raises(ValueError, match="shape"):
        ops.free_pages(z(n, w), z(n), torch.zeros(n + 1, dtype=torch.bool, device="cuda"), z(p), z(p), z(1), page=16)
    with pytest.raises(ValueError, match="overlaps"):
        t = z(n, w)
        ops.compact_pages(t, z(n), z(p), page=16, out=(z(n, w), z(p), t.view(-1)[:1].expand(p).contiguous(), z(1), z(p // 2), t.view(-1)[:p // 2]))
    pool = torch.zeros(p, 8, device="cuda")
    for pools, src, dst, match in [([pool, pool], z(2), z(2), "another"), ([pool, pool.new_zeros(p + 1, 8)], z(2), z(2), "number of pages"), ([pool.t()], z(2), z(2), "contiguous"), ([pool[:1].expand(p, 8)], z(2), z(2), "share memory"),
                                   ([pool], z(2), z(3), "shape"), ([pool], z(2).long(), z(2), "Int"), ([whole.view(50, 8)], whole[:2], z(2), "src"), ([pool.cpu()], z(2), z(2), "CUDA")]:
        with pytest.raises(ValueError, match=match):
            ops.copy_pages(pools, src, dst)


# ---- together

def test_together(ops):
    """Beam search with a memory of its own for every hypothesis: positions planned and written, attended over, words chosen, pages that follow, the pool made dense.  Every hypothesis'
    attention is that of the keys and values that it has gone through, read back from a copy that is moved whole."""
    rng = _rng(50)
    n, k, heads, dim, page, vocab, steps = 3, 4, 2, 64, 16, 60, 37
    width, n_pages = -(-steps // page), n * k * 3
    pools = [ops.new_pages8(n_pages, heads, dim, page) for _ in range(2)]
    table, lens = torch.full((n, k, width), -1, dtype=torch.int32, device="cuda"), torch.zeros(n, k, dtype=torch.int32, device="cuda")
    shares, free, used = torch.zeros(n_pages, dtype=torch.int32, device="cuda"), torch.randperm(n_pages, device="cuda").to(torch.int32), torch.zeros(1, dtype=torch.int32, device="cuda")
    embed = torch.from_numpy(rng.normal(0, 1, (vocab, 3, heads, dim)).astype(np.float32)).cuda()
    project = torch.from_numpy(rng.normal(0, 0.3, (heads * dim, vocab)).astype(np.float32)).cuda()
    tokens = torch.zeros(n, k, dtype=torch.int32, device="cuda")
    scores = torch.full((n, k), -INF, device="cuda")
    scores[:, 0] = 0
    past = np.zeros((n, k, 0), np.int64)                    # every hypothesis' words
    row = lambda x: x.view(n * k, *x.shape[2:])
    for step in range(steps):
        past = np.concatenate([past, tokens.cpu().numpy()[..., None]], 2)
        x = embed[tokens.view(-1).long()]
        new = lens + 1
        slots, starts, used = ops.plan_pages(row(lens), row(new), row(table), free, used, page=page, total=n * k)
        assert int(used) <= n_pages and (slots >= 0).all()
        for i, pool in enumerate(pools):
            ops.write_pages8(pool, slots, x[:, 1] * (i + 1), x[:, 2])
        lens = new
        out = [ops.attend_pages8(x[:, 0].view(n * k, 1, heads, dim), pool, row(table), row(lens)) for pool in pools]
        # what a hypothesis' pages hold: its own words' keys and values, each within a code of them
        k0, v0 = ops.read_pages8(pools[0], (row(table)[:, torch.arange(step + 1, device="cuda") // page].long() * page + torch.arange(step + 1, device="cuda") % page).view(-1))
        words = torch.from_numpy(past).cuda().view(-1)
        assert ((v0 - embed[words][:, 2]).abs() <= 3 * embed[:, 2].abs().max() / 127).all() and ((k0 - embed[words][:, 1]).abs() <= 3 * embed[:, 1].abs().max() / 127).all()
        kv = torch.stack([k0, v0]).view(2, n * k, step + 1, heads, dim).transpose(2, 3).double().cpu().numpy()
        want, _, tol, _ = attend_ref(x[:, 0].view(n * k, 1, heads, dim), kv, np.arange(n * k)[:, None], [step + 1] * (n * k), dim ** -0.5)
        assert (np.abs(out[0].double().cpu().numpy() - want) <= tol[..., None] + 2.0 ** -24 * np.abs(want)).all()
        logits = (out[0] + out[1]).view(n, k, heads * dim) @ project
        tokens, parents, scores, done = ops.beam_select(logits, scores, eos=vocab - 1, allowed=torch.full((1, 2), -1, dtype=torch.int32, device="cuda"))
        logp, entropy, best, best_logp = ops.score_tokens(torch.gather(logits, 1, parents.long()[..., None].expand(n, k, vocab)), tokens, top=3)
        assert torch.allclose(logp, torch.gather(torch.log_softmax(torch.gather(logits, 1, parents.long()[..., None].expand(n, k, vocab)), -1), 2, tokens.long()[..., None])[..., 0], atol=1e-5)
        table, lens, shares, free, used, src, dst = ops.fork_pages(table, lens, parents, shares, free, used, page=page)
        ops.copy_pages(pools, src, dst)
        past = np.take_along_axis(past, parents.cpu().numpy()[..., None].astype(np.int64), 1)
        names = table.cpu().numpy()[table.cpu().numpy() >= 0]
        g, c = np.unique(names, return_counts=True)
        count = np.zeros(n_pages, int)
        count[g] = c - 1
        assert (shares.cpu().numpy() == count).all() and int(used) == len(g)
        if step % 11 == 10:
            table, shares, free, used, src, dst = ops.compact_pages(table, lens, shares, page=page)
            ops.copy_pages(pools, src, dst)
            assert int(used) == len(g) and int(table.max()) < len(g)
    table, lens, shares, free, used = ops.free_pages(table, lens, torch.ones(n, k, dtype=torch.bool, device="cuda"), shares, free, used, page=page)
    assert int(used) == 0 and (shares == 0).all() and (lens == 0).all() and (table == -1).all() and sorted(free.tolist()) == list(range(n_pages))


def test_captured_and_on_two_streams(ops):
    rng = _rng(51)
    n, k, page = 12, 6, 16
    runs = []
    for i in range(2):
        lens = rng.integers(1, 90, (n, k))
        table, shares, free, used = _state(rng, n, k, lens, page, 80)
        dev = [_i32(x) for x in (table, lens, np.zeros((n, k)), shares, free, [used])]
        pool = torch.randint(0, 256, (len(shares), 64), dtype=torch.uint8, device="cuda")
        step = lambda: (lambda r: r + tuple(ops.copy_pages([pool], r[5], r[6])))(tuple(ops.fork_pages(*dev, page=page)))
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        runs.append((graph, torch.cuda.Stream(), (table, lens, shares, free, used), dev, pool, out))
    for _ in range(5):
        parents = [rng.integers(-1, k, (n, k)) for _ in runs]
        before = []
        for (graph, stream, state, dev, pool, out), p in zip(runs, parents):
            with torch.cuda.stream(stream):
                dev[2].copy_(_i32(p))
                before.append(pool.clone())
                graph.replay()
        torch.cuda.synchronize()
        for (graph, stream, (table, lens, shares, free, used), dev, pool, out), p, b in zip(runs, parents, before):
            want = fork_ref(table, lens, p, shares, free, used, page)
            for g, w in zip(out, want):
                assert (g.cpu().numpy() == w).all()
            src, dst = (x[x >= 0] for x in want[5:7])
            w = b.cpu().numpy()
            w[dst] = b.cpu().numpy()[src]
            assert (pool.cpu().numpy() == w).all()


def test_fork_as_many_rows_as_there_may_be(ops):
    rng = _rng(52)
    for n, k in ((1024, 16), (1, 16384)):
        page = 16
        lens = rng.integers(0, 40, (n, k))
        table, shares, free, used = _state(rng, n, k, lens, page, n * k, shared=0)
        fork_check(ops, table, lens, rng.integers(-1, k, (n, k)), shares, free, used, page)
        fork_check(ops, table, lens, None, shares, free, used, page, done=rng.random((n, k)) < 0.5)

"""Operators on device tensors at the values, overlaps and orders where they can go wrong, against plain implementations in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_device_ops import (BF16, F16, F32, HALF_STEP, INF, _cuda, _logits, _memory, _q, _reordered, _rng, attend_check, attend_ref, plan_ref, select_check)


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from linmt_b200 import device_ops
    return device_ops


NAN = float("nan")


# ---- selection


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,k,v", [(1, 4, 12000), (64, 3, 6100), (200, 12, 5300)])
def test_select_low_values_before_ordinary_ones(ops, n, k, v, dtype):
    """Words masked by a finite value, the first of every row among them, so that a warp's maximum comes from there to the ordinary words."""
    rng = _rng(n, k, v, 40)
    x = _logits(rng, n, k, v, dtype)
    scores = _cuda(rng.normal(-10, 3, (n, k)).astype(np.float32))
    least = torch.finfo(dtype).min
    lows = [-88.7, -266.2, -443.6, -1e9, -1e10, -1e18, -1e30, least] if n < 100 else [-1e9, least]
    for low in [x for x in lows if x >= least]:
        for words in (512, 1024, 5000, v - 100) if n < 100 else (1024,):
            y = x.clone()
            y[:, :, :words] = low
            select_check(ops, y, scores)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,k,v", [(2, 5, 9001), (70, 4, 3000)])
def test_select_logits_far_from_zero(ops, n, k, v, dtype):
    """Logits of 64 and more in size that differ: far up, far down, spread wide, and rows that cross 64."""
    rng = _rng(n, k, v, 41)
    x = _logits(rng, n, k, v, F32)
    scores = _cuda(rng.normal(-10, 3, (n, k)).astype(np.float32))
    ramp = torch.linspace(-150, 150, v, device="cuda")
    for y in (x + 100, x - 100, x * 40, x + ramp, x - ramp, torch.where(ramp < 0, x - 1000, x + 64), torch.where(ramp < 0, x + 70, x)):
        select_check(ops, y.to(dtype), scores)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,k,v", [(1, 4, 1000), (3, 6, 20000), (80, 13, 1500)])
def test_select_nan_beside_ties(ops, n, k, v, dtype):
    """A beam with a NaN offers nothing, whatever ties the others are in: flat rows, a flat row beside a better one with a NaN, and more equal best words than are kept."""
    rng = _rng(n, k, v, 42)
    flat = torch.zeros(n, k, v, dtype=dtype, device="cuda")
    flat[:, 1, v // 3] = NAN
    select_check(ops, flat, torch.full((n, k), -2.0, device="cuda"))
    scores = torch.full((n, k), -10.0, device="cuda")
    scores[:, 1] = -1
    select_check(ops, flat, scores)
    x = _logits(rng, n, k, v, dtype)
    x[:, 0] = 0
    x[:, 2, 5] = x[:, 2, v - 1] = NAN
    scores = torch.full((n, k), -200.0, device="cuda")
    scores[:, 0], scores[:, 2] = -10, -1
    select_check(ops, x, scores)
    x[:, 3, ::7] = 30
    x[:, 3, 1] = INF
    scores[:, 3] = 0
    select_check(ops, x, scores)
    done = torch.zeros(n, k, dtype=torch.bool, device="cuda")
    done[:, 1] = True
    select_check(ops, x, scores, done=done)


def _two_rows(rng, n, k, pattern, dtype, size=8.0, steps=256):
    """Rows 0 and 1 of each sentence are one pattern, moved by a number of each row's own that leaves every difference exact: the definition has them tie, a normaliser in 32
    bits puts either ahead.  The other beams are empty."""
    x = torch.zeros(n, k, len(pattern), device="cuda")
    moved = _cuda(rng.integers(-size * steps, size * steps, (n, 2)).astype(np.float32) / steps)
    x[:, :2] = _cuda(pattern.astype(np.float32)) + moved[..., None]
    assert torch.equal(x.to(dtype).float(), x)
    scores = torch.full((n, k), -INF, device="cuda")
    scores[:, :2] = -3
    return x.to(dtype), scores


@pytest.mark.parametrize("n,k,v", [(64, 4, 1000), (40, 4, 12000), (100, 12, 3000)])
def test_select_ties_above_a_finished_beam(ops, n, k, v):
    """The last candidate that is kept is a finished beam's, far below; what ties with the others is not among them."""
    x, scores = _two_rows(_rng(n, k, v, 43), n, k, np.zeros(v), F32)
    scores[:, 2] = -60
    done = torch.zeros(n, k, dtype=torch.bool, device="cuda")
    done[:, 2] = True
    select_check(ops, x, scores, done=done)


def test_select_ties_of_more_words_than_are_kept_in_one_part(ops):
    """The first words of both rows tie, more of them than a part of the row hands on, but lie in so few places that the parts behind hand on theirs too, which are far below."""
    n, k, v = 148, 12, 9600
    for seed in range(20):
        rng = _rng(seed, 3)
        pattern = rng.integers(-9 * 256, -8 * 256, v) / 256
        for vec in range(200):                 # of the first steps' 16-byte vectors those of three lanes
            if vec % 128 % 32 < 3:
                pattern[4 * vec:4 * vec + 4] = 0
        x, scores = _two_rows(rng, n, k, pattern, F32)
        tokens, parents, _, _ = ops.beam_select(x, scores)
        assert not parents.any() and (tokens.cpu().numpy() == np.nonzero(pattern == 0)[0][:k]).all(), seed      # ties go to the lowest index


@pytest.mark.parametrize("v", [120, 152])
def test_select_ties_where_every_word_is_a_candidate(ops, v):
    """Two flat rows of so few words that all of them are ranked, and more of them tie than are put in order."""
    x, scores = _two_rows(_rng(v, 45), 40, 32, np.zeros(v), F16, size=8.0, steps=64)
    select_check(ops, x, scores)


# ---- attention


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens", [[40, 17], [3000, 700], [20000, 1]])
def test_attend_queries_that_are_not_finite(ops, lens, dtype):
    """A row whose query has a NaN or an infinity gets NaN and says so in its lse, in a sentence that one CTA has and in one that several share; it gets 0 and -inf where it
    sees nothing; the other rows are as they were."""
    rng = _rng(sum(lens), 46)
    pages, table, kk, vv = _memory(ops, rng, lens, 2, 64, 16)
    n, g, heads = 2, 5, 4
    q = _q(rng, n, g, heads, 64, dtype)
    tab, ln = _cuda(table), _cuda(np.array(lens, np.int32))
    first = torch.zeros(n, g, dtype=torch.int32, device="cuda")
    last = torch.full((n, g), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    first[:, 4] = last[:, 4] = 3
    bad = q.clone()
    bad[0, 1, 2, 7] = bad[1, 0, 0, 63] = bad[:, 4] = NAN
    bad[0, 2, 1, 0] = INF
    bad[1, 3, 3, 40] = -INF
    broken = ~torch.isfinite(bad).all(-1)
    broken[:, 4] = False
    centre, slope = torch.zeros(n, g, device="cuda"), torch.full((heads,), 0.01, device="cuda")
    for kw in (dict(), dict(cap=20.0), dict(slope=slope, centre=centre)):
        want, wl = ops.attend_pages4(q, pages, tab, ln, first=first, last=last, want_lse=True, **kw)
        got, lse = ops.attend_pages4(bad, pages, tab, ln, first=first, last=last, want_lse=True, **kw)
        assert torch.isnan(got[broken]).all() and torch.isnan(lse[broken]).all()
        assert torch.equal(got[~broken], want[~broken]) and torch.equal(lse[~broken], wl[~broken])
        assert not got[:, 4].any() and torch.isneginf(lse[:, 4]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cap", [64.0, 65.0, 1e3, 1e4, 1e6, 1e9, 1e20, 3e38])
def test_attend_caps_of_all_sizes(ops, cap, dtype):
    """A large cap leaves the scores nearly as they are: to 2^-20 of a score, however large the cap."""
    rng = _rng(int(np.log2(cap) * 100), 47)
    lens, dim = [33, 500], 64
    pages, table, kk, vv = _memory(ops, rng, lens, 2, dim, 16)
    q = _q(rng, 2, 3, 4, dim, dtype).mul_(4)
    got, lse = ops.attend_pages4(q, pages, _cuda(table), _cuda(np.array(lens, np.int32)), cap=cap, want_lse=True)
    want, wlse, wv, big, ws = attend_ref(q.double().cpu().numpy(), kk, vv, table, lens, 16, dim ** -0.5, cap, None, None, None, None, pages.shape[0])
    # A score as in attend_check, with 3e-7 of a cap of up to 64 and, above that, tanh and its argument's products to 2^-21 of the score (four roundings and tanh's 2^-22).
    score = ((dim + 12) * 2.0 ** -24 + 2.0 ** -21 + (2.0 ** -22 if dtype == F32 else 0)) * big + (4e-7 * cap if cap <= 64 else 0) + 6 * 2.0 ** -24 * (np.abs(wlse).max() + 32)
    weight = {BF16: 2.0 ** -11, F16: 2.0 ** -11, F32: 2.0 ** -22}[dtype]
    steps, big_scale = max(lens) / 64 + 1, float(np.abs(vv).max()) / 7
    shift = 8 * 2.0 ** -34 * big_scale * max(lens) if dtype == F32 else (steps * 17 + 8) * 2.0 ** -23 * 15 * ws + 8 * 2.0 ** -28 * big_scale * max(lens)
    tol = HALF_STEP[dtype] * np.abs(want) + (weight + 2 * score + 2.0 ** -15) * wv + shift + (2.0 ** -25 if dtype == F16 else 0)
    g, l = got.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.isfinite(g).all() and np.isfinite(l).all()
    assert (np.abs(l - wlse) <= score + 2.0 ** -15 + 2.0 ** -23 * np.abs(wlse)).all(), float(np.abs(l - wlse).max())
    assert (np.abs(g - want) <= tol).all(), float((np.abs(g - want) / np.maximum(tol, 1e-300)).max())


# ---- what is written over what is read


def test_plan_refuses_a_table_over_what_it_reads(ops):
    """All of the call's int32 arrays in one buffer: apart, or in the gaps between the table's rows, they are taken; where a table's row has an entry of them they are not."""
    n, width, page = 4, 3, 16
    old, new = np.array([5, 0, 16, 33], np.int32), np.array([20, 3, 40, 34], np.int32)
    free = np.array([7, 3, 9, 1, 12], np.int32)
    total = int((new - old).sum())
    rows = np.full((n, width), -1, np.int32)
    rows[0, 0], rows[2, 0], rows[3] = 20, 21, [22, 23, 24]
    want = plan_ref(old, new, rows, free, 0, page, total)

    def call(table_at, stride, at):
        buf = torch.full((160,), -7, dtype=torch.int32, device="cuda")
        place = lambda x, a: buf[a:a + len(x)].copy_(_cuda(x))
        o, w, f, u = place(old, at[0]), place(new, at[1]), place(free, at[2]), place(np.zeros(1, np.int32), at[3])
        table = buf[table_at:table_at + (n - 1) * stride + width].as_strided((n, width), (stride, 1))
        keep = [x.clone() for x in (o, w, f, u)]
        table.copy_(_cuda(rows))
        for x, y in zip((o, w, f, u), keep):
            x.copy_(y)
        slots, starts, used = ops.plan_pages(o, w, table, f, u, page=page, total=total)
        assert (slots.cpu().numpy() == want[0]).all() and (starts.cpu().numpy() == want[1]).all() and (table.cpu().numpy() == want[2]).all() and int(used) == want[3]
        assert all(torch.equal(x, y) for x, y in zip((o, w, f, u), keep))

    call(0, 3, (12, 16, 20, 25))
    call(0, 12, (3, 7, 15, 11))                # in the gaps
    for bad, name in (((2, 60, 70, 80), "old"), ((60, 11, 70, 80), "new"), ((60, 70, 20, 80), "free"), ((60, 70, 80, 25), "used"), ((60, 70, 33, 80), "free"), ((36, 70, 80, 90), "old")):
        with pytest.raises(ValueError, match="table overlaps " + name):
            call(0, 12, bad)
    with pytest.raises(ValueError, match="overlaps free"):
        call(0, 3, (20, 30, 11, 40))


def test_write_refuses_pages_over_what_it_reads(ops):
    """A pool in the larger of two buffers' halves, beside what is written into it: apart it is taken, over slots, keys or values it is not."""
    rng = _rng(48)
    heads, dim, t = 2, 64, 20
    size = heads * 18 * dim                    # bytes of a page of 16 positions
    buf = torch.zeros(64 * size, dtype=torch.uint8, device="cuda")
    pages = buf[:4 * size].view(4, heads, 1, 18 * dim)
    at = lambda first, dtype, *shape: buf[first:first + int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()].view(dtype).view(shape)
    k, v = (_cuda(rng.normal(0, 1, (t, heads, dim)).astype(np.float32)) for _ in range(2))
    slots = _cuda(rng.permutation(64)[:t].astype(np.int64))
    ops.write_pages4(pages, slots, k, v)
    want = ops.read_pages4(pages, slots)
    pages.zero_()
    far_k, far_v, far_s = at(4 * size, F32, t, heads, dim), at(16 * size, F32, t, heads, dim), at(40 * size, torch.int64, t)
    far_k.copy_(k), far_v.copy_(v), far_s.copy_(slots)
    ops.write_pages4(pages, far_s, far_k, far_v)
    assert all(torch.equal(a, b) for a, b in zip(ops.read_pages4(pages, far_s), want))
    over = at(4 * size - 16, F32, t, heads, dim)
    for args, name in (((at(4 * size - 64, torch.int64, t), k, v), "slots"), ((slots, over, v), "k"), ((slots, k, over), "v")):
        with pytest.raises(ValueError, match="pages overlaps " + name):
            ops.write_pages4(pages, *args)
    layers = buf[:48 * size].view(4, 12, heads, 1, 18 * dim)      # a layer's pages, every twelfth
    pages, far_s = layers[:, 2], layers[1, 5].view(-1)[:8 * t].view(torch.int64)
    far_s.copy_(slots)
    ops.write_pages4(pages, far_s, k, v)       # slots in the gaps between them
    assert all(torch.equal(a, b) for a, b in zip(ops.read_pages4(pages, far_s), want)) and torch.equal(far_s, slots)


def test_attend_refuses_a_result_over_what_it_reads(ops):
    """A result over the table, the lengths, a bias, windows or the pool; beside them in one buffer it is taken."""
    rng = _rng(49)
    lens, heads, dim, g = [40, 21], 2, 64, 3
    pages, table, kk, vv = _memory(ops, rng, lens, heads, dim, 16)
    q = _q(rng, 2, g, heads, dim, F32)
    args = dict(table=_cuda(table), lens=_cuda(np.array(lens, np.int32)), slope=torch.rand(heads, device="cuda"), centre=torch.rand(2, g, device="cuda"),
                first=torch.zeros(2, g, dtype=torch.int32, device="cuda"), last=torch.full((2, g), 30, dtype=torch.int32, device="cuda"), pages=pages)
    size = 2 * g * heads * dim
    buf = torch.zeros(size + 64 + pages.numel() // 4, device="cuda")
    out = buf[:size].view(2, g, heads, dim)
    call = lambda out, a: ops.attend_pages4(q, a["pages"], a["table"], a["lens"], slope=a["slope"], centre=a["centre"], first=a["first"], last=a["last"], out=out)
    want = call(None, args)
    for name, x in args.items():
        def moved(first):                      # the argument's copy in the buffer, behind `first` of its places
            y = buf[first:first + x.numel() * x.element_size() // 4].view(x.dtype).view(x.shape)
            y.copy_(x)
            return dict(args, **{name: y})
        assert torch.equal(call(out, moved(size)), want)
        for first in (size - 4, 4):            # (a pool lies on 16 bytes)
            with pytest.raises(ValueError, match="out overlaps " + name):
                call(out, moved(first))
    wide = torch.zeros(2, g, heads, dim + 8, device="cuda")
    lens_in = wide.view(-1)[dim:dim + 2].view(torch.int32).copy_(args["lens"])      # in the gap behind the first row
    assert torch.equal(call(wide[..., :dim], dict(args, lens=lens_in)), want) and lens_in.tolist() == lens


# ---- beside autograd


def test_tangents_are_refused(ops):
    """No derivative forwards either: a dual tensor's tangent would be dropped."""
    fwd = torch.autograd.forward_ad
    x, s = torch.zeros(1, 2, 50, device="cuda"), torch.zeros(1, 2, device="cuda")
    parents = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    pages, table, lens = ops.new_pages4(2, 1, 64, 16), torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    q, k = torch.zeros(1, 2, 1, 64, device="cuda"), torch.ones(1, 1, 64, device="cuda")
    slots = torch.zeros(1, dtype=torch.int64, device="cuda")
    calls = ((lambda d: ops.beam_select(d, s), x), (lambda d: ops.beam_select(x, d), s), (lambda d: ops.beam_reorder([d], parents), x[..., :8].clone()),
             (lambda d: ops.attend_pages4(d, pages, table, lens), q), (lambda d: ops.write_pages4(pages, slots, k, d), k))
    with fwd.dual_level():
        for call, primal in calls:
            dual = fwd.make_dual(primal, torch.ones_like(primal))
            for guard in (torch.enable_grad(), torch.no_grad()):
                with guard, pytest.raises(ValueError, match="tangent"):
                    call(dual)
            call(fwd.unpack_dual(dual).primal)


def test_writing_in_place_raises_versions(ops):
    """What a call writes into a caller's tensor counts as a change of it, so that autograd refuses a backward pass through a saved tensor that was overwritten; what it only
    reads does not.  Tensors of the inference mode have no count and are written all the same."""
    n, k = 2, 3
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    x, scores, done, tokens, parents = torch.rand(n, k, 40, device="cuda"), torch.zeros(n, k, device="cuda"), torch.zeros(n, k, dtype=torch.bool, device="cuda"), ints(n, k), ints(n, k)
    state, other = torch.rand(2, n, k, 5, device="cuda"), torch.rand(2, n, k, 5, device="cuda")
    pages, table, lens = ops.new_pages4(4, 1, 64, 16), ints(n, 2), torch.full((n,), 20, dtype=torch.int32, device="cuda")
    free, used = torch.arange(4, dtype=torch.int32, device="cuda"), ints(1)
    kv, slots = torch.rand(40, 1, 64, device="cuda"), torch.arange(40, device="cuda")
    q, out = torch.rand(n, k, 1, 64, device="cuda"), torch.zeros(n, k, 1, 64, device="cuda")
    for call, written, read in ((lambda: ops.beam_select(x, scores, done=done, out=(tokens, parents, scores, done)), (tokens, parents, scores, done), (x,)),
                                (lambda: ops.beam_reorder([state[:1], state[1:]], parents), (state,), (parents,)), (lambda: ops.beam_reorder([state], parents, out=[other]), (other,), (state, parents)),
                                (lambda: ops.plan_pages(None, lens, table, free, used, page=16, total=40), (table,), (lens, free, used)),
                                (lambda: ops.write_pages4(pages, slots, kv, kv), (pages,), (slots, kv)), (lambda: ops.read_pages4(pages, slots), (), (pages, slots)),
                                (lambda: ops.attend_pages4(q, pages, table, lens, out=out), (out,), (q, pages, table, lens)), (lambda: ops.attend_pages4(q, pages, table, lens, out=q), (q,), (pages, table, lens))):
        before = [t._version for t in written], [t._version for t in read]
        call()
        assert all(t._version > v for t, v in zip(written, before[0])) and [t._version for t in read] == before[1]
    w = torch.ones_like(state, requires_grad=True)
    y = (w * state).sum()
    ops.beam_reorder([state], parents)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        kept = torch.arange(6., device="cuda").view(1, n, k)[0]
    ops.beam_reorder([kept], torch.tensor([[1, 1, 0], [2, 0, 0]], dtype=torch.int32, device="cuda"))
    assert kept.tolist() == [[1, 1, 0], [5, 3, 3]]


def test_reorder_complex_states(ops):
    """Complex rows are moved as they lie in memory: a conjugate view goes into a conjugate view, or back into itself, and nowhere else."""
    rng = _rng(50)
    parents = _cuda(rng.integers(0, 4, (3, 4)).astype(np.int32))
    x = torch.complex(*(_cuda(rng.normal(0, 1, (3, 4, 5)).astype(np.float32)) for _ in range(2)))
    out = torch.zeros_like(x)
    for state, to in ((x, out), (x.conj(), out.conj())):
        want = _reordered(state.resolve_conj(), parents)
        ops.beam_reorder([state], parents, out=[to])
        assert torch.equal(to.resolve_conj(), want)
    for state, to in ((x.conj(), out), (x, out.conj())):
        with pytest.raises(ValueError, match="conjugate"):
            ops.beam_reorder([state], parents, out=[to])
    view = x.conj()
    want = _reordered(view.resolve_conj(), parents)
    ops.beam_reorder([view], parents)
    assert torch.equal(view.resolve_conj(), want)


def test_reorder_refuses_rows_whose_strides_do_not_nest(ops):
    """Columns 0 and 1, and 4 to 7, of every tenth place in k and every 25th in n: the one's second sentence lies in the other's third beam.  Where the strides nest, in
    any order of the dimensions and with the last row cut short, such columns are states of their own."""
    rng = _rng(51)
    flat = _cuda(rng.normal(0, 1, 200).astype(np.float32))
    cut = lambda first, width, sn, sk: flat[first:].as_strided((2, 3, width), (sn, sk, 1))
    parents = torch.tensor([[2, 0, 1], [1, 1, 0]], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        ops.beam_reorder([cut(0, 2, 25, 10), cut(4, 4, 25, 10)], parents)
    for sn, sk in ((30, 10), (28, 10), (10, 20), (8, 16), (100, 9)):
        a, b = cut(0, 2, sn, sk), cut(4, 4, sn, sk)
        before, (wa, wb) = flat.clone(), [_reordered(x.clone(), parents) for x in (a, b)]
        ops.beam_reorder([a, b], parents)
        assert torch.equal(a, wa) and torch.equal(b, wb)
        a.zero_(), b.zero_()
        touched = flat != before
        before[touched] = 0
        assert torch.equal(flat, before)


# ---- attention to values of very different sizes


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim,lens", [(64, [400, 90]), (128, [1500, 33])])
def test_attend_does_not_feel_what_a_row_does_not_see(ops, dim, lens, dtype):
    """Rows with windows of their own, among positions whose values are of any size: a row's result is the same, bit for bit, whatever the positions hold that it does not see."""
    rng = _rng(dim, 52)
    heads, g, page, n = 2, 6, 16, 2
    pages, table, kk, vv = _memory(ops, rng, lens, heads, dim, page)
    q = _q(rng, n, g, heads, dim, dtype)
    tab, ln = _cuda(table), _cuda(np.array(lens, np.int32))
    first, last = (torch.zeros(n, g, dtype=torch.int32, device="cuda") for _ in range(2))
    for i, x in enumerate(lens):
        cuts = np.linspace(0, x, g + 1).astype(np.int32)
        first[i], last[i] = _cuda(cuts[:-1].copy()), _cuda(cuts[1:].copy())
    call = lambda p: ops.attend_pages4(q, p, tab, ln, first=first, last=last, want_lse=True)
    want, wl = call(pages)
    slots = [_cuda(table[i, np.arange(x) // page].astype(np.int64) * page + np.arange(x) % page) for i, x in enumerate(lens)]
    for row in range(g):
        other = pages.clone()
        for i, x in enumerate(lens):
            at = np.ones(x, bool)
            at[int(first[i, row]):int(last[i, row])] = False
            size = 2.0 ** rng.integers(-40, 41, int(at.sum()))[:, None, None]
            k, v = (_cuda((rng.normal(0, 1, (int(at.sum()), heads, dim)) * s).astype(np.float32)) for s in (1.0, size))
            ops.write_pages4(other, slots[i][_cuda(at)], k, v)
        got, lse = call(other)
        assert torch.equal(got[:, row], want[:, row]) and torch.equal(lse[:, row], wl[:, row])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("where", ["first", "middle", "last", "falling", "rising"])
def test_attend_large_values_of_positions_that_hardly_count(ops, where, dtype):
    """Positions whose values are 2^24 (16-bit results) or 2^50 times the others' and whose weights make nothing of them, before, among and behind the others; and scores that
    rise while values fall, so that the largest values so far no longer count."""
    rng = _rng(len(where), 53)
    heads, dim, page, length = 1, 64, 16, 330
    big = 24 if dtype == F16 else 50
    at = np.arange(length)
    k, v = np.zeros((length, heads, dim), np.float32), rng.normal(0, 1, (length, heads, dim)).astype(np.float32)
    score = rng.normal(0, 1, length)
    if where in ("falling", "rising"):
        step = at // 33                         # ten steps, at each of which values fall by 2^(big / 10) and scores rise by more, or the other way about
        if where == "rising":
            step = step[::-1]
        score += step * 6.0
        v *= (2.0 ** (12 - np.floor(step * big / 10.0))).astype(np.float32)[:, None, None]
    else:
        few = {"first": at < 3, "middle": (at > 150) & (at < 154), "last": at >= length - 3}[where]
        score[few] = -60
        v *= np.float32(2.0 ** -12)
        v[few] *= np.float32(2.0 ** big)
    k[:, 0, 0] = score
    table = rng.permutation(25)[:21].reshape(1, 21).astype(np.int32)
    slots = _cuda(table[0, at // page].astype(np.int64) * page + at % page)
    pages = ops.new_pages4(25, heads, dim, page)
    ops.write_pages4(pages, slots, _cuda(k), _cuda(v))
    rk, rv = ops.read_pages4(pages, slots)
    kk, vv = (np.zeros((25 * page, heads, dim), np.float32) for _ in range(2))
    kk[slots.cpu().numpy()], vv[slots.cpu().numpy()] = rk.cpu().numpy(), rv.cpu().numpy()
    q = torch.zeros(1, 2, 1, dim, device="cuda")
    q[..., 0] = torch.tensor([[[1.0], [0.5]]], device="cuda")
    q = q.to(dtype)
    got = ops.attend_pages4(q, pages, _cuda(table), _cuda(np.array([length], np.int32)), scale=1.0)
    want, wlse, wv, _, ws = attend_ref(q.double().cpu().numpy(), kk, vv, table, [length], page, 1.0, 0.0, None, None, None, None, 25)
    # The score is one product and its change to a power of 2, a few roundings of up to 60 + 32; weights and products as in attend_check.  A weight times its scale is kept to 2^-25 in fp16 where the
    # largest of them is 2^-5 (2^1 in 32-bit queries' second term) at least, so to 2^-20 (2^-26) of that, for each position, and goes with codes of up to 15 (8).
    s = rk.double().cpu().numpy()[:, 0] @ q.double().cpu().numpy()[0, :, 0].T
    w = np.exp(s - wlse[0, :, 0])
    most = (w * np.abs(rv.cpu().numpy()[:, 0]).max(-1)[:, None] / 7).max(0)[None, :, None, None]
    score = 8 * 2.0 ** -24 * 92
    weight = 2.0 ** -22 if dtype == F32 else 2.0 ** -11
    steps = length / 64 + 1
    kept = 8 * 2.0 ** -26 * most * length if dtype == F32 else (steps * 17 + 8) * 2.0 ** -23 * 15 * ws + 15 * 2.0 ** -20 * most * length
    tol = HALF_STEP[dtype] * np.abs(want) + (weight + 2 * score + 2.0 ** -15) * wv + kept + (2.0 ** -25 if dtype == F16 else 0)
    g = got.double().cpu().numpy()
    assert (np.abs(want).max((2, 3)) > 50 * tol.max((2, 3))).all()      # (the test can tell)
    assert (np.abs(g - want) <= tol).all(), float((np.abs(g - want) / tol).max())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cap", [0.0, 3.0, 500.0])
def test_attend_negative_and_zero_scales(ops, cap, dtype):
    """A scale of either sign is that of the queries; one of 0 makes every position alike."""
    rng = _rng(54)
    lens = [77, 1200]
    pages, table, kk, vv = _memory(ops, rng, lens, 2, 64, 16)
    q = _q(rng, 2, 3, 4, 64, dtype)
    tab, ln = _cuda(table), _cuda(np.array(lens, np.int32))
    for scale in (0.11, 2.0):
        want = ops.attend_pages4(-q, pages, tab, ln, scale=scale, cap=cap, want_lse=True)
        got = ops.attend_pages4(q, pages, tab, ln, scale=-scale, cap=cap, want_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for scale in (0.0, -0.0):
        attend_check(ops, q, pages, table, lens, kk, vv, 16, scale=scale, cap=cap)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("length", [1, 2, 16, 64, 256, 512])
def test_attend_means_of_32_bits_are_exact(ops, length, dim):
    """Queries of 0 make the mean of a power of two of values.  A value is an integer of four bits times a scale of eight, scales lie within 2^4 of each other: sums of 512 take 12 + 4 + 9
    bits and a sign, so that nothing is rounded on the way in 32 bits."""
    rng = _rng(length, dim, 55)
    pages, table, kk, vv = _memory(ops, rng, [length, length], 2, dim, 16)
    q = torch.zeros(2, 3, 2, dim, device="cuda")
    got, lse = ops.attend_pages4(q, pages, _cuda(table), _cuda(np.array([length] * 2, np.int32)), want_lse=True)
    at = np.arange(length)
    for i in range(2):
        mean = vv[table[i, at // 16].astype(np.int64) * 16 + at % 16].astype(np.float64).mean(0)
        assert (got[i].double().cpu().numpy() == mean).all()
    assert (np.abs(lse.double().cpu().numpy() - np.log(length)) <= 2.0 ** -22 * (1 + np.log(length))).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_attend_few_positions_in_32_bits(ops, dim):
    """One to three positions and queries of one component each: scores of up to 1 in a handful of roundings, so that what weights and products lose shows."""
    rng = _rng(dim, 56)
    lens, g, heads = [1, 2, 3, 3, 2], 16, 2
    pages, table, kk, vv = _memory(ops, rng, lens, heads, dim, 16)
    q = torch.zeros(5, g, heads, dim, device="cuda")
    q.scatter_(3, _cuda(rng.integers(0, dim, (5, g, heads, 1))), _cuda(rng.uniform(-0.2, 0.2, (5, g, heads, 1)).astype(np.float32)))
    got, lse = ops.attend_pages4(q, pages, _cuda(table), _cuda(np.array(lens, np.int32)), scale=1.0, want_lse=True)
    want, wlse, wv, big, _ = attend_ref(q.double().cpu().numpy(), kk, vv, table, lens, 16, 1.0, 0.0, None, None, None, None, pages.shape[0])
    assert big <= 1
    largest = np.zeros(want.shape)
    for i, x in enumerate(lens):
        largest[i] = np.abs(vv[table[i, 0].astype(np.int64) * 16 + np.arange(x)]).max(0)
    # A score: the query's two terms 2^-22, five roundings of 2^-24.  A weight: twice that (its own and the sum's), exp2 2^-22, its two terms 2^-22; two products of up to four
    # addends, each cut off at 2^-23 of the largest; the sums' and the result's roundings, four of 2^-24.
    score = 2.0 ** -22 + 5 * 2.0 ** -24
    tol = (2 * score + 2 * 2.0 ** -22 + 8 * 2.0 ** -23 + 4 * 2.0 ** -24) * largest
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all(), float((err / np.maximum(tol, 1e-300)).max())
    assert (np.abs(lse.double().cpu().numpy() - wlse) <= 2 * score + 2.0 ** -21).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_attend_small_weights_in_32_bits(ops, dim):
    """A position that has nearly all the weight and components of 0, and others of 2^-17 of its weight, which are all that those components have: a weight times scale is kept to
    2^-34 of the row's largest."""
    rng = _rng(dim, 57)
    length, page, heads = 6, 16, 2
    k, v = np.zeros((length, heads, dim), np.float32), rng.normal(0, 1, (length, heads, dim)).astype(np.float32)
    k[:, :, 0] = -12
    k[3, :, 0] = 0
    zero = rng.random((heads, dim)) < 0.5
    zero[:, ::32] = False
    v[3][zero] = 0
    pages, slots = ops.new_pages4(1, heads, dim, page), torch.arange(length, device="cuda")
    ops.write_pages4(pages, slots, _cuda(k), _cuda(v))
    kk, vv = (np.zeros((page, heads, dim), np.float32) for _ in range(2))
    rk, rv = ops.read_pages4(pages, slots)
    kk[:length], vv[:length] = rk.cpu().numpy(), rv.cpu().numpy()
    q = torch.zeros(1, 5, heads, dim, device="cuda")
    q[..., 0] = torch.linspace(0.9, 1.1, 5, device="cuda")[None, :, None]
    table = np.zeros((1, 1), np.int32)
    got = ops.attend_pages4(q, pages, _cuda(table), _cuda(np.array([length], np.int32)), scale=1.0).double().cpu().numpy()
    want, _, wv, _, _ = attend_ref(q.double().cpu().numpy(), kk, vv, table, [length], page, 1.0, 0.0, None, None, None, None, 1)
    # Scores of up to 13.2 are good to 2^-22 and six roundings of 2^-24, weights to twice that and 2^-21, sums of 12 products to 12 cut-offs of 2^-23: 2^-16 in all.
    scale = np.abs(v[3]).reshape(heads, -1, 32).max(-1).max(-1) / 8 * (1 + 2.0 ** -8)
    tol = 2.0 ** -16 * wv + (length - 1) * 8 * 2.0 ** -34 * scale[None, None, :, None]
    assert (vv[3][zero] == 0).all() and (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / np.maximum(tol, 1e-300)).max())


def test_plan_takes_a_table_without_columns_in_the_midst_of_what_it_reads(ops):
    """A table of no columns has no place that could be written, wherever it points."""
    buf = torch.tensor([0, 0, 0, 0, 11, 12, 13, 14, 15, 16, 17, 18, 0], dtype=torch.int32, device="cuda")
    table = buf[6:].as_strided((4, 0), (1, 1))
    slots, starts, used = ops.plan_pages(None, torch.full((4,), 5, dtype=torch.int32, device="cuda"), table, buf[4:12], buf[12:], page=16, total=2)
    assert slots.tolist() == [-1, -1] and starts.tolist() == [0] * 5 and used.tolist() == [0]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [1e-13, 1e-30, 1e-44])
def test_attend_scores_below_the_smallest_number(ops, scale, dtype):
    """Queries and a scale so small that their product is no number of 32 bits any more: the scores are 0, and positions behind the text stay unseen."""
    rng = _rng(58)
    lens = [23, 700]
    pages, table, kk, vv = _memory(ops, rng, lens, 2, 64, 16)
    q = _q(rng, 2, 3, 2, 64, F32).mul_(1e-30).to(dtype)
    attend_check(ops, q, pages, table, lens, kk, vv, 16, scale=scale)

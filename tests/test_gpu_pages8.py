"""Memories in 8 bits: keys and values in and out, and attention over them, against plain implementations in 64 bits."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_device_ops import BF16, F16, F32, HALF_STEP, INF, _cuda, _rng

NAN = float("nan")
LEAST = 2.0 ** -126


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from linmt_b200 import device_ops
    return device_ops


# ---- keys and values in and out

def scale_ref(big):
    """The smallest of 4, 5, 6, 7 times a power of 2 whose 127-fold reaches `big`, 2^-126 at least: by trying."""
    if big == 0:
        return 0.0
    e = math.floor(math.log2(big / 127)) - 3 if big / 127 > 0 else -200
    while True:
        for m in (4, 5, 6, 7):
            if 127 * m * 2.0 ** e >= big:
                return max(m * 2.0 ** e, LEAST)
        e += 1


def clean(x):
    return np.clip(np.where(np.isnan(x), 0, x), -2.0 ** 127, 2.0 ** 127).astype(np.float32)


def codes_ref(x, s):
    """Quotients in 32 bits, rounded to the nearest integer, to even between two."""
    return np.zeros(x.shape, np.int64) if s == 0 else np.rint((x.astype(np.float32) / np.float32(s))).astype(np.int64)


class Pool8:
    """The definition, run by run: codes and scales of every block."""

    def __init__(self, n_pages, heads, dim, page):
        self.page, self.dim = page, dim
        self.codes = np.zeros((2, n_pages, heads, page, dim), np.int64)
        self.scales = np.zeros((2, n_pages, heads, page // 16))

    def write(self, slots, k, v):
        n, t = self.codes.shape[1] * self.page, 0
        while t < len(slots):
            if not 0 <= slots[t] < n:
                t += 1
                continue
            end = t + 1
            while end < len(slots) and slots[end] == slots[end - 1] + 1 and slots[end] % 16:
                end += 1
            p, at = divmod(int(slots[t]), self.page)
            b, o = at // 16, at % 16
            for j, x in enumerate((k, v)):
                for h in range(self.codes.shape[2]):
                    new = clean(x[t:end, h])
                    old = self.scales[j, p, h, b] if o else 0.0
                    s = max(scale_ref(float(np.abs(new).max())), old)
                    block = self.codes[j, p, h, b * 16:b * 16 + 16]
                    if o and s != old:
                        block[:o] = codes_ref(block[:o] * old, s)
                    block[o:] = 0
                    block[o:o + end - t] = codes_ref(new, s)
                    self.scales[j, p, h, b] = s
            t = end

    def read(self, slots):
        out = np.zeros((2, len(slots), self.codes.shape[2], self.dim))
        for i, s in enumerate(slots):
            if 0 <= s < self.codes.shape[1] * self.page:
                p, at = divmod(int(s), self.page)
                out[:, i] = self.codes[:, p, :, at] * self.scales[:, p, :, at // 16][..., None]
        return out

    def bytes(self):
        return blocks(self.codes, self.scales)


def blocks(codes, scales):
    """uint8 [pages, heads, page / 16, 32 dim + 16] of codes [2, pages, heads, positions, dim] and scales [2, pages, heads, page / 16]."""
    _, p, h, n, d = codes.shape
    c = codes.astype(np.int8).view(np.uint8).reshape(2, p, h, n // 16, 16, d)
    k = c[0].reshape(p, h, n // 16, 2, 8, d // 16, 16).swapaxes(4, 5).reshape(p, h, n // 16, 16 * d)
    v = c[1].swapaxes(3, 4).reshape(p, h, n // 16, 16 * d)
    tail = np.zeros((p, h, n // 16, 4), np.float32)
    tail[..., 0], tail[..., 1] = scales
    return np.concatenate([k, v, tail.view(np.uint8)], -1)


def rows_check(ops, pool, ref, slots, k, v):
    ops.write_pages8(pool, _cuda(np.asarray(slots, np.int64)), k, v)
    ref.write(slots, k.float().cpu().numpy(), v.float().cpu().numpy())
    assert (pool.cpu().numpy() == ref.bytes()).all()
    every = np.arange(-3, ref.codes.shape[1] * ref.page + 5)
    got = ops.read_pages8(pool, _cuda(every))
    want = ref.read(every)
    for g, w in zip(got, want):
        assert (g.cpu().numpy() == w.astype(np.float32)).all()


def _kv(rng, t, heads, dim, dtype, spread=1.0):
    x = rng.normal(0, 1, (2, t, heads, dim)) * np.exp(rng.normal(0, spread, (2, t, 1, 1))) + rng.normal(0, 1, (2, 1, heads, dim))
    return _cuda(x[0].astype(np.float32), dtype), _cuda(x[1].astype(np.float32), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,heads,dim,page", [(1, 1, 64, 16), (5, 3, 128, 16), (16, 2, 64, 32), (47, 5, 128, 48), (130, 9, 64, 64), (300, 1, 128, 128)])
def test_write_and_read(ops, t, heads, dim, page, dtype):
    """A text from any position of a block on, and what it is appended to."""
    rng = _rng(t, heads, dim, page)
    n_pages = t // page + 4
    pool, ref = ops.new_pages8(n_pages, heads, dim, page), Pool8(n_pages, heads, dim, page)
    for start in (0, 3, 21):
        slots = start + np.arange(t)
        rows_check(ops, pool, ref, slots, *_kv(rng, t, heads, dim, dtype))
    few = n_pages * page // 16                      # a position of every block, blocks in any order
    rows_check(ops, pool, ref, rng.permutation(few) * 16 + rng.integers(0, 16), *_kv(rng, few, heads, dim, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
def test_write_step_by_step(ops, dim, dtype):
    """Positions one by one, sizes that grow and fall: scales that have to grow round what was there again."""
    rng = _rng(dim, 1)
    heads, page, seqs = 3, 32, 9
    pool, ref = ops.new_pages8(2 * seqs, heads, dim, page), Pool8(2 * seqs, heads, dim, page)
    table = rng.permutation(2 * seqs).reshape(seqs, 2)
    lens = rng.integers(0, 20, seqs)
    for step in range(30):
        slots = np.array([table[i, lens[i] // page] * page + lens[i] % page if lens[i] < 2 * page else -1 for i in range(seqs)])
        rows_check(ops, pool, ref, slots, *_kv(rng, seqs, heads, dim, dtype, spread=1.5))
        lens += 1


def test_write_many_sequences_by_a_few(ops):
    rng = _rng(77)
    heads, dim, page, seqs = 4, 64, 16, 700
    pool, ref = ops.new_pages8(seqs, heads, dim, page), Pool8(seqs, heads, dim, page)
    start = rng.integers(0, 10, seqs)
    for grow in (3, 1, 2):
        slots = (rng.permutation(seqs)[:, None] * page + 0).repeat(grow, 1)
        slots = slots + (start[slots[:, 0] // page][:, None] + np.arange(grow))
        start[slots[:, 0] // page] += grow
        rows_check(ops, pool, ref, slots.ravel(), *_kv(rng, seqs * grow, heads, dim, BF16))


def test_write_extremes(ops):
    """Zeros, NaN, infinities, the largest and the smallest numbers, sums of ties, each from a block's first position on and appended."""
    rng = _rng(5)
    heads, dim, page = 2, 64, 16
    cases = []
    for dtype in (F32, BF16, F16):
        top = torch.finfo(dtype).max
        for fill in (0.0, NAN, INF, -INF, top, -top, torch.finfo(dtype).tiny, 1e-45 if dtype == F32 else 6e-8):
            x = rng.normal(0, 1, (2, 16, heads, dim))
            x[0, 3] = fill
            x[1, :, 1] = fill
            x[0, 5, 0, ::3] = fill
            cases.append((dtype, x))
        cases.append((dtype, np.full((2, 16, heads, dim), 0.0)))
        cases.append((dtype, rng.integers(-255, 256, (2, 16, heads, dim)) * 0.5))               # ties between codes
        cases.append((dtype, rng.integers(-255, 256, (2, 16, heads, dim)) * 2.0 ** -20 * 7))
        cases.append((dtype, rng.normal(0, 1, (2, 16, heads, dim)) * 2.0 ** -124))
        cases.append((dtype, rng.normal(0, 1, (2, 16, heads, dim)) * 2.0 ** -95))
    pool, ref = ops.new_pages8(3, heads, dim, page), Pool8(3, heads, dim, page)
    for dtype, x in cases:
        k, v = (_cuda(y.astype(np.float32), dtype) for y in x)
        rows_check(ops, pool, ref, np.arange(16, 32), k, v)
        rows_check(ops, pool, ref, np.arange(7), k[:7], v[:7])
        rows_check(ops, pool, ref, np.arange(7, 14), k[:7], v[7:14])
        rows_check(ops, pool, ref, np.array([14]), k[3:4], v[3:4])


def test_write_slots_outside_and_strides(ops):
    """Slots outside the pool among the others, rows with gaps, heads before positions, a pool of which every second page and head is used."""
    rng = _rng(6)
    heads, dim, page, n = 3, 128, 32, 5
    whole = torch.full((2 * n, 2 * heads, page // 16, 32 * dim + 16), 7, dtype=torch.uint8, device="cuda")
    pool, ref = whole[::2, 1::2], Pool8(n, heads, dim, page)
    pool.zero_()
    t = 40
    k = _cuda(rng.normal(0, 1, (heads, t, dim + 8)).astype(np.float32), BF16)[:, :, :dim].transpose(0, 1)
    v = _cuda(rng.normal(0, 1, (t, 2 * heads, dim)).astype(np.float32), BF16)[:, ::2]
    slots = np.concatenate([np.arange(18, 30), [-1, n * page, 2 ** 40, -2 ** 62], np.arange(64, 84), [127, 32, 5, 97]])
    rows_check(ops, pool, ref, slots, k, v)
    left = torch.ones_like(whole, dtype=torch.bool)
    left[::2, 1::2] = False
    assert (whole[left] == 7).all()


def test_write_far_pages(ops):
    """Pages more than 2^32 bytes apart."""
    dim, page = 128, 16
    stride = (1 << 31) // (32 * dim + 16)
    whole = torch.zeros(2 * stride + 5, 1, 1, 32 * dim + 16, dtype=torch.uint8, device="cuda")
    k = torch.randn(32, 1, dim, device="cuda", dtype=F16)
    slots = torch.cat([torch.arange(16), (2 * stride + 3) * 16 + torch.arange(16)]).cuda()
    ops.write_pages8(whole, slots, k, k)
    got, _ = ops.read_pages8(whole, slots, dtype=F32)
    # a code is half a scale off at most, a scale at most 5/4 of a 127th of the largest component
    assert ((got - k.float()).abs() <= k.float().abs().amax() / 127 * 5 / 8).all()
    assert whole[1:-2].count_nonzero() == 0
    out = ops.attend_pages8(torch.zeros(1, 1, 1, dim, device="cuda"), whole, torch.tensor([[0, 2 * stride + 3]], dtype=torch.int32, device="cuda"), torch.tensor([32], dtype=torch.int32, device="cuda"))
    assert torch.allclose(out[0, 0, 0], got[:, 0].mean(0), atol=1e-6)


# ---- attention

def memory8(rng, n, lens, heads, dim, page, sizes=0.0, spare=2):
    """A pool with a table: codes of any size, scales that differ from block to block; what no sentence has is filled with bytes that are no numbers."""
    width = max(1, -(-max([1, *lens]) // page))
    n_pages = n * width + spare
    table = rng.permutation(n_pages)[:n * width].reshape(n, width).astype(np.int32)
    codes = np.clip(np.rint(rng.normal(0, 40, (2, n_pages, heads, page, dim))), -127, 127).astype(np.int64)
    scales = (2.0 ** np.rint(rng.normal(-5.5, sizes, (2, n_pages, heads, page // 16))) * rng.integers(4, 8, (2, n_pages, heads, page // 16)) / 4).astype(np.float32)
    raw = blocks(codes, scales)
    for i, length in enumerate(lens):
        for b in range(-(-length // 16), width * (page // 16)):
            raw[table[i, b * 16 // page], :, b % (page // 16)] = 255
    for p in set(range(n_pages)) - set(table.ravel().tolist()):
        raw[p] = 255
    return _cuda(raw), _cuda(table), codes * scales.astype(np.float64).repeat(16, -1)[..., None]


def attend_ref(q, kv, table, lens, scale, cap=0.0, slope=None, centre=None, first=None, last=None, sinks=0, there=None):
    """out and lse in 64 bits, and bounds of what a kernel that holds its sums in 32 bits may be off (attend_check)."""
    n, g, heads, dim = q.shape
    pool_heads, page = kv.shape[2], kv.shape[3]
    rep = heads // pool_heads
    out, lse = np.zeros((n, g, heads, dim)), np.full((n, g, heads), -INF)
    tol, tol_lse = np.zeros((n, g, heads)), np.zeros((n, g, heads))
    sixteen = q.dtype != F32
    qd = q.double().cpu().numpy()
    for i in range(n):
        length = min(max(lens[i], 0), table.shape[1] * page)
        if length == 0:
            continue
        pos = np.arange(length)
        pages = table[i][pos // page]
        ok = (pages >= 0) & (pages < kv.shape[1])
        k, v = (kv[j][np.where(ok, pages, 0), :, pos % page] for j in range(2))
        for h in range(heads):
            kh, vh = k[:, h // rep], v[:, h // rep]
            for b in range(g):
                x = qd[i, b, h]
                seen = ok.copy()
                if first is not None:
                    seen &= ((pos >= first[i, b]) & (pos < last[i, b])) | (pos < sinks)
                if not seen.any():
                    continue
                if not np.isfinite(x).all():
                    out[i, b, h], lse[i, b, h] = NAN, NAN
                    continue
                s = scale * (kh @ x)
                big = np.abs(s[seen]).max()
                # a component is off by 2^-22 of the largest; a score's integers are added in 32 bits, the low 16 of them off by 2^-22 of a key component's; and six roundings
                d = abs(scale) * np.abs(x).max() * 2.0 ** -22 * (np.abs(kh[seen]).sum(-1).max() + np.abs(kh[seen]).max()) + 6 * 2.0 ** -24 * big
                if cap:
                    s = cap * np.tanh(s / cap)
                    d += 3.6e-7 * cap if sixteen and cap <= 64 else 2.0 ** -21 * cap
                if slope is not None:
                    bias = slope[h] * np.abs(pos - centre[i, b])
                    s = s - bias
                    d += 4 * 2.0 ** -24 * (bias[seen].max() + np.abs(s[seen]).max())
                s = np.where(seen, s, -INF)
                top = s.max()
                w = np.exp(s - top)
                lse[i, b, h] = top + math.log(w.sum())
                out[i, b, h] = (w / w.sum()) @ np.where(seen[:, None], vh, 0)
                # the sums of weights, one of 128 positions a thread, and of their parts; the exponential 2^-22 and what it takes from the rounded difference
                sums = (length / 128 + 40) * 2.0 ** -24 + 2.0 ** -21
                # a weight times its scale to 2^-27 (2^-30) of the row's largest, below which the reference is by a power of 2 at most
                most = np.abs(vh[seen]).max()
                tol[i, b, h] = most * (2 * np.expm1(d) + 2 * sums + length * 2.0 ** (-27 if sixteen else -30))
                tol_lse[i, b, h] = d + sums + 2.0 ** -22 * abs(lse[i, b, h])
    return out, lse, tol, tol_lse


def attend_check(ops, q, pool, table, lens, kv, scale=None, **kw):
    t = lambda x: None if x is None else _cuda(np.asarray(x))
    dev = {k: (t(np.asarray(v, np.float32)) if k in ("slope", "centre") else t(np.asarray(v, np.int32)) if k in ("first", "last") else v) for k, v in kw.items()}
    got, lse = ops.attend_pages8(q, pool, table, t(np.asarray(lens, np.int32)), scale=scale, want_lse=True, **dev)
    ref = {k: (np.asarray(v, np.float32).astype(np.float64) if k in ("slope", "centre") else v) for k, v in kw.items()}
    want, want_lse, tol, tol_lse = attend_ref(q, kv, table.cpu().numpy(), lens, q.shape[-1] ** -0.5 if scale is None else scale, **ref)
    g, l = got.double().cpu().numpy(), lse.double().cpu().numpy()
    assert (np.isneginf(l) == np.isneginf(want_lse)).all() and (np.isnan(l) == np.isnan(want_lse)).all()
    bad = np.isnan(want).any(-1)
    assert (np.isnan(g).all(-1) == bad).all() and not np.isnan(g[~bad]).any()
    off = np.abs(g - want)[~bad] - HALF_STEP[q.dtype] * np.abs(want[~bad])
    assert (off <= tol[~bad][..., None]).all(), (off - tol[~bad][..., None]).max()
    ok = np.isfinite(want_lse)
    assert (np.abs(l - want_lse)[ok] <= tol_lse[ok]).all(), (np.abs(l - want_lse) - tol_lse)[ok].max()
    return got, lse


def _q(rng, n, g, heads, dim, dtype, size=1.5):
    return _cuda((rng.normal(0, size, (n, g, heads, dim))).astype(np.float32), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim,heads,rep,g,page,lens", [
    (64, 1, 1, 1, 16, [1]), (128, 1, 1, 1, 16, [0, 1, 2, 15, 16, 17]), (64, 2, 1, 5, 32, [23, 127, 128, 129]), (128, 3, 4, 1, 48, [300, 1]), (64, 1, 3, 7, 64, [255, 0, 511]),
    (128, 2, 2, 9, 16, [77, 400]), (64, 3, 1, 33, 80, [130, 12]), (128, 1, 8, 1, 112, [1000]), (64, 2, 5, 1, 128, [640, 641])])
def test_attend(ops, dim, heads, rep, g, page, lens, dtype):
    """Every number of rows that go together, and more of them; lengths about a block's, a page's and a product's."""
    rng = _rng(dim, heads, rep, g, page, sum(lens))
    n = len(lens)
    pool, table, kv = memory8(rng, n, lens, heads, dim, page)
    q = _q(rng, n, g, heads * rep, dim, dtype)
    attend_check(ops, q, pool, table, lens, kv)
    attend_check(ops, q, pool, table, lens, kv, scale=-0.03, cap=20.0)
    slope, centre = 2.0 ** -np.arange(1, heads * rep + 1), rng.random((n, g)) * (np.asarray(lens)[:, None] + 1)
    attend_check(ops, q, pool, table, lens, kv, slope=slope, centre=centre)
    a, b = (np.floor(rng.random((n, g)) * (np.asarray(lens)[:, None] + 2)).astype(np.int32) - 1 for _ in range(2))
    for sinks in (0, 1, 20, 200):
        attend_check(ops, q, pool, table, lens, kv, first=np.minimum(a, b), last=np.maximum(a, b), sinks=sinks)
    attend_check(ops, q, pool, table, lens, kv, cap=100.0, slope=slope, centre=centre, first=a, last=b, sinks=3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens", [[5000], [9000, 1, 3000, 0, 40], [700] * 40, [2600] * 12, [16384 * 2 + 5]])
def test_attend_long_and_shared(ops, lens, dtype):
    """Segments that several CTAs share, and CTAs that have several segments."""
    rng = _rng(len(lens), sum(lens))
    n, heads, dim, page = len(lens), 2, 64, 64
    pool, table, kv = memory8(rng, n, lens, heads, dim, page)
    for g, rep in ((1, 1), (3, 2), (2, 8)):
        q = _q(rng, n, g, heads * rep, dim, dtype)
        attend_check(ops, q, pool, table, lens, kv)
    first, last = np.maximum(np.asarray(lens)[:, None] - [[1000, 130]], 0), np.asarray(lens)[:, None] - [[0, 100]]
    attend_check(ops, _q(rng, n, 2, heads, dim, dtype), pool, table, lens, kv, first=first, last=last, sinks=4)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_attend_windows_far_from_the_sinks(ops, dtype):
    """Chunks between the sinks and the windows are left out; sinks that reach into the windows, beyond them, and stand alone; rows that see nothing."""
    rng = _rng(31)
    lens, heads, dim, page, g = [3000, 2500, 64], 1, 128, 32, 4
    pool, table, kv = memory8(rng, 3, lens, heads, dim, page)
    q = _q(rng, 3, g, heads, dim, dtype)
    first = np.array([[2000, 2100, 2900, 5000], [1000, 10, 130, 300], [0, 64, 5, -7]])
    last = np.array([[2050, 2900, 3100, 9000], [1000, 5, 135, 200], [64, 70, 4, 3]])
    for sinks in (0, 4, 128, 129, 1100, 2048, 4000):
        attend_check(ops, q, pool, table, lens, kv, first=first, last=last, sinks=sinks)


def test_attend_more_rows_than_are_looked_at(ops):
    """Windows of more rows than a CTA looks at to find out what to leave out."""
    rng = _rng(32)
    lens, g = [600, 300], 40
    pool, table, kv = memory8(rng, 2, lens, 1, 64, 16)
    a, b = (rng.integers(0, 600, (2, g)) for _ in range(2))
    attend_check(ops, _q(rng, 2, g, 1, 64, BF16), pool, table, lens, kv, first=np.minimum(a, b), last=np.maximum(a, b), sinks=2)


def test_attend_pages_outside_the_pool_and_lengths_outside_the_table(ops):
    rng = _rng(33)
    lens, heads, dim, page = [500, 300, 90], 2, 64, 16
    pool, table, kv = memory8(rng, 3, lens, heads, dim, page)
    table[0, 3:9] = torch.tensor([-1, 10 ** 9, pool.shape[0], -2 ** 31, 2 ** 31 - 1, -1], dtype=torch.int32)
    table[1] = -1
    q = _q(rng, 3, 3, heads, dim, F32)
    attend_check(ops, q, pool, table, lens, kv)
    attend_check(ops, q, pool, table[:, :4], [64, 10 ** 9, 2 ** 31 - 1], kv)
    out, lse = ops.attend_pages8(q, pool, table, torch.tensor([-5, 300, 0], dtype=torch.int32, device="cuda"), want_lse=True)
    assert (out == 0).all() and (lse == -INF).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attend_scales_of_all_sizes(ops, dtype):
    """Scales that differ by many powers of 2 from block to block, and are 0 in some; what a row does not see takes nothing from it."""
    rng = _rng(34)
    lens, heads, dim, page = [400, 130], 2, 64, 16
    pool, table, kv = memory8(rng, 2, lens, heads, dim, page, sizes=6.0)
    q = _q(rng, 2, 3, heads, dim, dtype, size=0.02)
    attend_check(ops, q, pool, table, lens, kv)
    raw = pool.cpu().numpy()
    tail = raw[..., 32 * dim:].copy().view(np.float32)
    at = table.cpu().numpy()
    tail[at[0, 5], :, 0, 1] = 2.0 ** 90          # huge values in a block that the second and third rows do not see
    tail[at[0, 9], :, 0, 1] = 0.0
    tail[at[1, 2], :, 0] = 0.0
    raw[..., 32 * dim:] = tail.view(np.uint8)
    first, last = np.array([[0, 96, 0], [0, 0, 0]]), np.array([[400, 400, 80], [130, 130, 130]])
    base, _ = ops.attend_pages8(q, pool, table, _cuda(np.asarray(lens, np.int32)), first=_cuda(first.astype(np.int32)), last=_cuda(last.astype(np.int32)), want_lse=True)
    kv[1][at[0, 9]] = 0
    for j in range(2):
        kv[j][at[1, 2]] = 0
    changed = _cuda(raw)
    got, _ = ops.attend_pages8(q, changed, table, _cuda(np.asarray(lens, np.int32)), first=_cuda(first.astype(np.int32)), last=_cuda(last.astype(np.int32)), want_lse=True)
    want, _, tol, _ = attend_ref(q, kv, at, lens, dim ** -0.5, first=first, last=last)
    for i, b in ((0, 1), (0, 2), (1, 0), (1, 1), (1, 2)):
        off = np.abs(got[i, b].double().cpu().numpy() - want[i, b]) - HALF_STEP[dtype] * np.abs(want[i, b])
        assert (off <= tol[i, b][:, None]).all(), (i, b)
    assert (got[0, 2] == base[0, 2]).all()       # not a bit


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attend_one_position_far_ahead_of_many(ops, dtype):
    """A first token with nearly all of the weight, 20000 others with equal small ones that count together: none is rounded away."""
    rng = _rng(35)
    length, dim, page = 20001, 64, 64
    width = -(-length // page)
    codes = np.zeros((2, width, 1, page, dim), np.int64)
    codes[0, ..., 0] = 1
    codes[0, 0, 0, 0, 0] = 127
    codes[1] = rng.integers(-127, 128, codes.shape[1:])
    scales = np.full((2, width, 1, page // 16), 0.03125)
    pool, table = _cuda(blocks(codes, scales)), _cuda(np.arange(width, dtype=np.int32)[None])
    q = torch.zeros(1, 1, 1, dim, device="cuda", dtype=dtype)
    for ahead in (8.0, 11.0, 14.0):
        q[..., 0] = ahead / (126 * 0.03125)
        attend_check(ops, q, pool, table, [length], codes * scales.repeat(16, -1)[..., None], scale=1.0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("up", [True, False])
def test_attend_scores_that_rise_and_fall(ops, up, dtype):
    """Every chunk's scores exceed the last one's by far, or none does."""
    rng = _rng(36)
    lens, heads, dim, page = [2000], 1, 64, 16
    pool, table, kv = memory8(rng, 1, lens, heads, dim, page)
    q = _q(rng, 1, 2, heads, dim, dtype)
    for slope in (0.5, 0.05, 8.0):
        attend_check(ops, q, pool, table, lens, kv, slope=[slope], centre=np.array([[2000.0, 1500.5]]) if up else np.array([[0.0, -30.0]]))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attend_queries_that_are_not_finite_zero_and_far(ops, dtype):
    rng = _rng(37)
    lens, heads, dim, page = [200, 0], 2, 128, 16
    pool, table, kv = memory8(rng, 2, lens, heads, dim, page)
    q = _q(rng, 2, 6, heads, dim, dtype)
    q[:, 0, 0, 7], q[:, 1, 1, 0], q[:, 2, 0, 3] = NAN, INF, -INF
    q[:, 3] = 0
    q[:, 4] *= 2.0 ** -14 if dtype == F16 else 2.0 ** -60
    q[:, 5] *= 100
    attend_check(ops, q, pool, table, lens, kv)
    attend_check(ops, q, pool, table, lens, kv, first=np.full((2, 6), 300), last=np.full((2, 6), 400))
    attend_check(ops, q, pool, table, lens, kv, scale=0.0)


def test_attend_strides_and_results_in_place(ops):
    """Rows with gaps, heads before rows, addresses of any alignment, a pool whose pages and heads lie apart, a result that takes the place of the queries."""
    rng = _rng(38)
    lens, heads, rep, g, dim, page = [210, 95], 2, 2, 3, 64, 32
    pool, table, kv = memory8(rng, 2, lens, heads, dim, page)
    base = _q(rng, 2, g, heads * rep, dim, BF16)
    want, lse = attend_check(ops, base, pool, table, lens, kv)
    n = _cuda(np.asarray(lens, np.int32))
    odd = torch.zeros(2, heads * rep, g, dim + 3, device="cuda", dtype=BF16)[..., 1:dim + 1].transpose(1, 2)
    odd.copy_(base)
    assert (ops.attend_pages8(odd, pool, table, n) == want).all()
    wide = torch.full((2, g, 2 * heads * rep, dim), 9.0, device="cuda", dtype=BF16)
    out = wide[:, :, ::2]
    assert ops.attend_pages8(base, pool, table, n, out=out) is out and (out == want).all() and (wide[:, :, 1::2] == 9).all()
    apart = torch.zeros(2 * pool.shape[0], heads + 1, pool.shape[2], pool.shape[3], dtype=torch.uint8, device="cuda")[1::2, 1:]
    apart.copy_(pool)
    assert (ops.attend_pages8(base, apart, table, n) == want).all()
    # strides that are not whole blocks: the pool cannot be looked at as rows of them
    size = pool.shape[2] * pool.shape[3]
    flat = torch.zeros(pool.shape[0] * heads * (size + 32), dtype=torch.uint8, device="cuda").view(pool.shape[0], heads, size + 32)[..., 16:16 + size]
    loose = flat.as_strided((pool.shape[0], heads, pool.shape[2], pool.shape[3]), (flat.stride(0), flat.stride(1), pool.shape[3], 1), flat.storage_offset())
    loose.copy_(pool)
    assert (ops.attend_pages8(base, loose, table, n) == want).all()
    strided = torch.zeros(2, table.shape[1] + 3, dtype=torch.int32, device="cuda")[:, 1:table.shape[1] + 1]
    strided.copy_(table)
    assert (ops.attend_pages8(base, pool, strided, n) == want).all()
    q = base.clone()
    assert ops.attend_pages8(q, pool, table, n, out=q) is q and (q == want).all()
    again, l2 = ops.attend_pages8(base, pool, table, n, want_lse=True)
    assert (again == want).all() and (l2 == lse).all()


def test_attend_loose_pools_of_many_sentences(ops):
    """The same numbers from a pool of rows of blocks and from one that is none."""
    rng = _rng(39)
    lens = list(rng.integers(0, 900, 30))
    pool, table, kv = memory8(rng, 30, lens, 3, 128, 48)
    q = _q(rng, 30, 2, 6, 128, F16)
    n = _cuda(np.asarray(lens, np.int32))
    size = pool.shape[2] * pool.shape[3]
    loose = torch.zeros(pool.shape[0], 3, size + 16, dtype=torch.uint8, device="cuda").as_strided(pool.shape, (3 * (size + 16), size + 16, pool.shape[3], 1))
    loose.copy_(pool)
    a, b = (ops.attend_pages8(q, p, table, n, want_lse=True) for p in (pool, loose))
    assert (a[0] == b[0]).all() and (a[1] == b[1]).all()


def test_refusals(ops):
    pool = ops.new_pages8(4, 2, 64, 32)
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.new_pages8(4, 2, 64, 24)
    with pytest.raises(ValueError, match="64 or 128"):
        ops.new_pages8(4, 2, 96, 32)
    k = torch.zeros(3, 2, 64, device="cuda")
    slots = torch.arange(3, device="cuda")
    for bad, match in [((pool[..., :-16], slots, k, k), "32 \\* dim"), ((pool, slots.int(), k, k), "Long"), ((pool, slots, k[:2], k), "shape"), ((pool, slots, k, k.half()), "alike"),
                       ((pool, slots, k.transpose(1, 2).contiguous().transpose(1, 2), k), "contiguous"), ((pool, slots, torch.zeros(3, 2, 66, device="cuda")[..., 2:], k), "16 bytes"), ((pool.float(), slots, k, k), "uint8")]:
        with pytest.raises(ValueError, match=match):
            ops.write_pages8(*bad)
    with pytest.raises(ValueError, match="overlaps"):
        ops.write_pages8(pool, slots, pool.view(-1)[:6 * 64 * 4].view(F32).view(3, 2, 64), k)
    with pytest.raises(ValueError, match="dtype"):
        ops.read_pages8(pool, slots, dtype=torch.float64)
    q = torch.zeros(2, 3, 4, 64, device="cuda")
    table, lens = torch.zeros(2, 5, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    ops.attend_pages8(q, pool, table, lens)
    row = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for kw, match in [(dict(sinks=-1), "sinks"), (dict(first=row), "first goes"), (dict(slope=torch.zeros(4, device="cuda")), "slope goes"), (dict(cap=-1.0), "finite"), (dict(scale=NAN), "finite"),
                      (dict(first=row[:, :2], last=row), "shape"), (dict(out=q[:, :, :2]), "like q"), (dict(out=q.roll(0, 0)[:, :1].expand(2, 3, 4, 64)), "share memory")]:
        with pytest.raises(ValueError, match=match):
            ops.attend_pages8(q, pool, table, lens, **kw)
    with pytest.raises(ValueError, match="multiple of the pool"):
        ops.attend_pages8(q[:, :, :3], pool, table, lens)
    with pytest.raises(ValueError, match="gradient"):
        ops.attend_pages8(q.clone().requires_grad_(), pool, table, lens)
    whole = torch.zeros(2 * q.numel(), device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        ops.attend_pages8(whole[:q.numel()].view_as(q), pool, table, lens, out=whole[64:64 + q.numel()].view_as(q))
    assert ops.attend_pages8(q[:0], pool, table[:0], lens[:0]).shape == (0, 3, 4, 64)
    assert ops.attend_pages8(q[:, :0], pool, table, lens).shape == (2, 0, 4, 64)


def test_captured_and_replayed(ops):
    """A step of a growing memory, captured: the lengths and slots change between replays; two graphs beside each other on two streams."""
    rng = _rng(40)
    n, heads, dim, page, width = 6, 2, 64, 16, 8
    graphs = []
    for g in range(2):
        pool = ops.new_pages8(n * width, heads, dim, page)
        table = torch.randperm(n * width, device="cuda").to(torch.int32).view(n, width)
        lens, slots = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.full((n,), -1, device="cuda")
        k, v, q = (torch.zeros(n, heads, dim, device="cuda", dtype=BF16) for _ in range(3))
        step = lambda: (ops.write_pages8(pool, slots, k, v), ops.attend_pages8(q.view(n, 1, heads, dim), pool, table, lens, want_lse=True))[1]
        with torch.no_grad():
            step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, torch.cuda.Stream(), pool, table, lens, slots, k, v, q, out, Pool8(n * width, heads, dim, page)))
    for at in range(40):
        for graph, stream, pool, table, lens, slots, k, v, q, out, ref in graphs:
            with torch.cuda.stream(stream):
                for x in (k, v, q):
                    x.copy_(torch.randn_like(x))
                slots.copy_(table[:, at // page].long() * page + at % page)
                lens.fill_(at + 1)
                graph.replay()
        torch.cuda.synchronize()
        for graph, stream, pool, table, lens, slots, k, v, q, out, ref in graphs:
            ref.write(slots.cpu().numpy(), k.float().cpu().numpy(), v.float().cpu().numpy())
            if at % 13 == 0 or at == 39:
                assert (pool.cpu().numpy() == ref.bytes()).all()
                kv = ref.codes * ref.scales.repeat(16, -1)[..., None]
                want, want_lse, tol, tol_lse = attend_ref(q.view(n, 1, heads, dim), kv, table.cpu().numpy(), [at + 1] * n, dim ** -0.5)
                assert (np.abs(out[0].double().cpu().numpy() - want) <= tol[..., None] + HALF_STEP[BF16] * np.abs(want)).all()
                assert (np.abs(out[1].double().cpu().numpy() - want_lse) <= tol_lse).all()


@pytest.mark.parametrize("dtype", [F32, F16])
def test_attend_many_short_sentences(ops, dtype):
    """More sentences than a CTA has threads, empty ones among them; every CTA has many."""
    rng = _rng(41)
    n, dim, page = 3000, 64, 16
    lens = rng.integers(0, 40, n)
    lens[rng.random(n) < 0.3] = 0
    lens[1500] = 800
    pool, table, kv = memory8(rng, n, lens, 1, dim, page)
    attend_check(ops, _q(rng, n, 1, 2, dim, dtype), pool, table, lens, kv)


def test_attend_integers_are_taken_out_before_they_overflow(ops):
    """Eleven million positions of a few pages, named again and again: a CTA has more products than its 32-bit sums hold at the largest codes and equal weights."""
    rng = _rng(42)
    dim, page, pages, columns = 64, 128, 3, 88800
    codes = np.full((2, pages, 1, page, dim), 127, np.int64)
    codes[0] = rng.integers(-3, 4, codes.shape[1:])
    codes[1, ..., 1::2] = -127
    codes[1, 2, :, ::2] = 126
    scales = np.full((2, pages, 1, page // 16), 0.0078125)
    pool = _cuda(blocks(codes, scales))
    names = rng.integers(0, pages, columns)
    length = columns * page - 77
    count = np.zeros((pages, page))
    np.add.at(count, names, 1)
    count[names[-1], page - 77:] -= 1
    kv = codes * 0.0078125
    q = _q(rng, 1, 16, 1, dim, F32, size=0.3)
    out, lse = ops.attend_pages8(q, pool, _cuda(names.astype(np.int32)[None]), torch.tensor([length], dtype=torch.int32, device="cuda"), want_lse=True)
    x = q[0, :, 0].double().cpu().numpy() @ kv[0, :, 0].reshape(-1, dim).T * dim ** -0.5
    w = np.exp(x - x.max(1, keepdims=True)) * count.reshape(-1)
    want = (w / w.sum(1, keepdims=True)) @ kv[1, :, 0].reshape(-1, dim)
    want_lse = x.max(1) + np.log(w.sum(1))
    # a weight is rounded to 2^-30 of the largest; a thread adds up 11e6 / 296 / 128 weights and 300 parts are joined, 2^-24 each; scores are below 2
    tol = np.abs(kv[1]).max() * (length * 2.0 ** -30 + (length / 296 / 128 + 340) * 2.0 ** -23 + 2.0 ** -19)
    assert (np.abs(out[0, :, 0].double().cpu().numpy() - want) <= tol).all()
    assert (np.abs(lse[0, :, 0].double().cpu().numpy() - want_lse) <= (length / 296 / 128 + 340) * 2.0 ** -23 + 2.0 ** -18).all()

"""Logits and scores far from zero, up to the largest numbers of 32 bits, against 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_device_ops import BF16, F16, F32, HALF_STEP, INF, _cuda, _rng
from test_gpu_token_scores import score_ref

FAR = [65530.0, 65600.0, 1e5, 1e6, 4e6, 5e6, 1e9, 3e9, 5e9, 1e10, 1e12, 1e20, 1e30, 1e32, 1e37, 9e37, 1.5e38, 3e38]


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from linmt_b200 import device_ops
    return device_ops


def far_check(ops, x, tokens, top):
    got = [y.cpu().numpy().astype(np.float64) for y in ops.score_tokens(x, tokens, top=top)]
    lp, ent, words, best = score_ref(x, tokens, top)
    lp, best = (np.where(np.abs(y) > torch.finfo(F32).max, np.copysign(INF, y), y) for y in (lp, best))      # beyond 32 bits
    # A term's exponent is a difference to the row's largest logit, rounded to 2^-24 of itself: at most 2^-21 of a term that counts; exp2 is good to 2^-22.  A thread adds up to vocab / 128
    # terms, 2^-24 each, then 10 are joined; logarithms and products 2^-22 of what comes out.
    rel = (x.shape[2] / 128 + 16) * 2.0 ** -24 + 2.0 ** -20
    pairs = [(got[0], lp, rel), (got[1], ent, rel * (2 + 2 * np.log(x.shape[2] + 1)))]
    if top:
        assert (got[2] == words).all()
        pairs.append((got[3], best, rel))
    for g, w, tol in pairs:
        ok = np.isfinite(w)
        assert (g[~ok] == w[~ok]).all()
        off = np.abs(g[ok] - w[ok]) - 2.0 ** -22 * np.abs(w[ok])
        assert (off <= tol).all(), off.max()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v", [(2, 50), (2, 3001), (1, 50003), (300, 5000)])
def test_score_rows_far_from_zero(ops, n, v, dtype):
    """Rows of one far number, alone and beside ordinary words; of neighbouring ones; of numbers on either side of it; of far numbers of all sizes, in threads of their own or before each other."""
    rng = _rng(n, v, 90)
    ordinary = rng.normal(0, 2, v)
    rows = []
    for c in FAR:
        for far in (c, -c):
            one, some = np.full(v, far), np.full(v, far)
            one[v // 3] = 5.0
            some[rng.random(v) < 0.3] = -7.0
            rows += [np.full(v, far), one, some, far * (1 + rng.integers(-3, 4, v) * 2.0 ** -22), far * (1 + rng.integers(-1, 2, v) * 2.0 ** -8), np.where(np.arange(v) < v // 2, far, ordinary), np.where(np.arange(v) < v // 2, ordinary, far)]
    rows += [-np.repeat(FAR, -(-v // len(FAR)))[:v], np.repeat(FAR[::-1], -(-v // len(FAR)))[:v], -np.asarray(FAR)[rng.integers(0, len(FAR), v)], np.where(np.arange(v) % 2, -65530.0, -65545.0)]
    rows += [s * (65536 + rng.normal(0, 3, v)) for s in (1, -1)] + [s * (2.0 ** 22 + rng.normal(0, 3, v)) for s in (1, -1)]
    for at in range(0, len(rows), n) if n < 300 else (0,):
        some = [rows[(at + i) % len(rows)] for i in range(n)]
        x = _cuda(np.stack(some)[:, None].astype(np.float32), dtype)
        tokens = np.full((n, 1), v // 3, np.int32)
        tokens[1::2] = v - 1
        far_check(ops, x, _cuda(tokens), 0 if at % 3 == 0 else 5)


# ---- attention

from test_gpu_pages8 import attend_ref, blocks, memory8


def attend_far_check(ops, q, pool, table, lens, kv, scale, alike=False, slope=None, **window):
    """As attend_ref has it, but where one position has all the weight, or all scores are `alike` to the bit, what a far score is off by does not matter: the result has to be that position's value, or the mean.
    Returns the rows of which that was so."""
    dev = {k: _cuda(np.asarray(v, np.int32)) for k, v in window.items()}
    if slope is not None:
        slope, centre = slope
        dev.update(slope=_cuda(np.asarray(slope, np.float32)), centre=_cuda(np.asarray(centre, np.float32)))
        window.update(slope=np.asarray(slope, np.float32).astype(np.float64), centre=np.asarray(centre, np.float32).astype(np.float64))
    got, lse = ops.attend_pages8(q, pool, table, _cuda(np.asarray(lens, np.int32)), scale=scale, want_lse=True, **dev)
    scale = float(np.float32(scale))
    want, want_lse, tol, _ = attend_ref(q, kv, table.cpu().numpy(), lens, scale, **window)
    n, g, heads, dim = q.shape
    page, rep, clear = kv.shape[3], heads // kv.shape[2], np.zeros((n, g, heads), bool)
    x = q.double().cpu().numpy()
    for i in range(n):
        pos = np.arange(lens[i])
        for b in range(g):
            seen = pos >= 0 if "first" not in window else (pos >= window["first"][i][b]) & (pos < window["last"][i][b])
            if not seen.any():
                continue
            for h in range(heads):
                k, v = (kv[j][table.cpu().numpy()[i][pos // page], h // rep, pos % page][seen] for j in range(2))
                s = scale * (k @ x[i, b, h])
                d = abs(scale) * np.abs(x[i, b, h]).max() * 2.0 ** -22 * (np.abs(k).sum(-1).max() + np.abs(k).max()) + 8 * 2.0 ** -24 * np.abs(s).max()
                if slope is not None:
                    s = s - window["slope"][h] * np.abs(pos[seen] - window["centre"][i, b])
                    d += 8 * 2.0 ** -24 * np.abs(s).max()
                first, second = np.sort(s)[::-1][[0, min(1, len(s) - 1)]]
                clear[i, b, h] = alike or len(s) == 1 or first - second > 2 * d + 60
                if clear[i, b, h]:
                    want[i, b, h] = v.mean(0) if alike else v[s.argmax()]
                    # sums of equal weights and their joins, 2^-24 each, and six roundings; the weight times its scale to 2^-27 or 2^-30 of the row's largest
                    tol[i, b, h] = np.abs(v).max() * ((len(s) / 128 + 40) * 2.0 ** -23 + 2.0 ** -20 + len(s) * 2.0 ** (-30 if q.dtype == F32 else -27)) if alike else \
                        np.abs(want[i, b, h]).max() * (2.0 ** -21 + 2.0 ** (-30 if q.dtype == F32 else -27))
    out, kind = got.double().cpu().numpy(), torch.finfo(q.dtype)
    beyond = np.abs(want) > kind.max * (1 + kind.eps / 4)      # half a step above a type's largest number it has none any more: 65520 in fp16
    assert (out[beyond] == np.sign(want[beyond]) * INF).all()
    off = np.where(beyond, 0, np.abs(np.where(beyond, 0, out) - want) - HALF_STEP[q.dtype] * np.abs(want))
    assert (off <= tol[..., None]).all(), (off - tol[..., None]).max()
    l, seen = lse.double().cpu().numpy(), np.isfinite(want_lse)
    # a score's own roundings, and those of its components (2^-22 of the largest): all of one size here
    assert (l[~seen] == want_lse[~seen]).all() and (np.abs(l - want_lse)[seen] <= 2.0 ** -15 * np.abs(want_lse[seen]) + 2.0 ** -12).all()
    return clear


EXPONENTS = [18, 20, 22, 23, 24, 25, 26, 27, 28, 30, 35, 40, 63, 100]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sign", [1, -1])
def test_attend_one_position_with_a_far_score(ops, sign, dtype):
    """A result is the value of the only position, however far its score."""
    rng = _rng(91)
    lens, heads, dim, page, g = [1, 600], 2, 64, 16, 3
    pool, table, kv = memory8(rng, 2, lens, heads, dim, page, sizes=6.0)
    q = _cuda(np.abs(rng.normal(0, 1, (2, g, heads, dim))).astype(np.float32) + 0.5, dtype)
    first = np.array([[0] * g, [5, 300, 599]])
    for e in EXPONENTS:
        clear = attend_far_check(ops, q, pool, table, lens, kv, sign * 2.0 ** e / 16, first=first, last=first + 1)
        assert clear.all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens", [[300, 77], [20001], [700] * 30])
def test_attend_far_scores_that_are_alike(ops, lens, dtype):
    """All keys and their scales alike, the values' scales differ: the mean of the values, by one CTA or by several."""
    rng = _rng(92, len(lens))
    n, heads, dim, page = len(lens), 1, 64, 64
    pool, table, kv = memory8(rng, n, lens, heads, dim, page, sizes=1.0)
    codes = np.rint(kv / np.maximum(1e-30, np.abs(kv).max((-1), keepdims=True)) * 100).astype(np.int64)
    codes[0] = codes[0, 0, 0, 0]
    scales = (2.0 ** rng.integers(-8, -2, (2, kv.shape[1], heads, page // 16))).astype(np.float32)
    scales[0] = 2.0 ** -5
    pool, kv = _cuda(blocks(codes, scales)), codes * scales.repeat(16, -1)[..., None].astype(np.float64)
    q = _cuda(rng.normal(0, 1, (n, 2, 1, dim)).astype(np.float32), dtype)
    size = np.abs(q.double().cpu().numpy() @ kv[0, 0, 0, 0]).max()
    for e in EXPONENTS:
        for sign in (1, -1):
            attend_far_check(ops, q, pool, table, lens, kv, sign * 2.0 ** e / size, alike=True)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("order", ["rising", "falling", "any"])
def test_attend_far_scores_of_many_positions(ops, order, dtype):
    """The position with the largest score has all the weight, first, last or anywhere; rows with ordinary scores beside them."""
    rng = _rng(93)
    lens, heads, dim, page, g = [4000, 900], 1, 64, 32, 9
    pool, table, kv = memory8(rng, 2, lens, heads, dim, page, sizes=2.0)
    codes = np.clip(np.rint(rng.normal(0, 20, kv.shape)), -60, 60).astype(np.int64)
    scales = (2.0 ** rng.integers(-8, -3, kv.shape[1:3] + (page // 16,))).astype(np.float32)
    scales = np.stack([np.full_like(scales, 2.0 ** -5), scales])
    for i, length in enumerate(lens):
        at = np.arange(length)
        ramp = np.sort(rng.permutation(16129)[:length] - 8064)       # two digits, so that no two are alike
        ramp = {"rising": ramp, "falling": ramp[::-1], "any": rng.permutation(ramp)}[order]
        for c, digit in ((0, np.round(ramp / 127)), (1, ramp - 127 * np.round(ramp / 127))):
            codes[0, table.cpu().numpy()[i][at // page], 0, at % page, c] = digit
    codes[0, ..., 2:] = 0
    pool, kv = _cuda(blocks(codes, scales)), codes * scales.repeat(16, -1)[..., None].astype(np.float64)
    for e in EXPONENTS:
        x = np.zeros((2, g, 1, dim))
        x[..., 0], x[..., 1] = 127, 1
        x[:, 1::3] *= -1
        x[:, ::3] = rng.normal(0, 2.0 ** -12 if dtype == F16 else 2.0 ** -e, x[:, ::3].shape)
        q = _cuda(x.astype(np.float32), dtype)
        clear = attend_far_check(ops, q, pool, table, lens, kv, 2.0 ** (e - 9))
        assert e < 22 or (clear[:, 1::3].all() and clear[:, 2::3].all())      # two scores are 2^(e - 14) apart at least, the bound of what they are off by is 2^(e - 20)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attend_far_biases(ops, dtype):
    """A bias of up to 2^36 a position: the one next to a row's centre, or the last one before it."""
    rng = _rng(94)
    lens, heads, dim, page, g = [3000, 1, 200], 2, 128, 16, 4
    pool, table, kv = memory8(rng, 3, lens, heads, dim, page, sizes=3.0)
    q = _cuda(rng.normal(0, 1, (3, g, heads, dim)).astype(np.float32), dtype)
    centre = np.array([[0.0, 1500.25, 1e5, -7e5], [0.0, 3e4, -3.0, 1.0], [99.75, 0.0, 1e4, 200.0]])
    for e in (14, 20, 28, 36):
        assert attend_far_check(ops, q, pool, table, lens, kv, dim ** -0.5, slope=([2.0 ** e, 2.0 ** (e - 2)], centre)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens", [[700, 90], [6000], [20000]])
@pytest.mark.parametrize("size", [-120, -60, 86, 90, 110, 119])
def test_attend_values_of_all_sizes(ops, size, lens, dtype):
    """Values' scales of 2^size, scores that rise by some 40 powers of 2 behind the first products: by one CTA or by several."""
    from test_gpu_pages8 import attend_check
    rng = _rng(95, len(lens), lens[0])
    n, heads, dim, page, g = len(lens), 2, 64, 64, 3
    pool, table, kv = memory8(rng, n, lens, heads, dim, page)
    codes = rng.integers(-100, 101, kv.shape)
    codes[1, ..., ::3] = np.abs(codes[1, ..., ::3])
    codes[0, ..., 0] = 0
    scales = np.stack([np.full(kv.shape[1:3] + (page // 16,), 2.0 ** -9), 2.0 ** rng.integers(size - 3, size + 1, kv.shape[1:3] + (page // 16,))]).astype(np.float32)
    for i, length in enumerate(lens):
        at = np.arange(length)
        codes[0, table.cpu().numpy()[i][at // page], :, at % page, 0] = np.where(at < 300, 0, 100)[:, None]      # 300 positions: three products
    pool, kv = _cuda(blocks(codes, scales)), codes * scales.repeat(16, -1)[..., None].astype(np.float64)
    q = rng.normal(0, 0.05, (n, g, heads, dim))
    for up in (0.0, 20.0, 27.0, 28.0, 29.0, 30.0, 31.0):      # 2^40 is e^27.7, 2^44 e^30.5
        q[..., 0] = up / (100 * 2.0 ** -9)
        attend_check(ops, _cuda(q.astype(np.float32), dtype), pool, table, lens, kv, scale=1.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v", [(2, 700), (1, 50003), (1, 200003)])
def test_score_one_word_far_from_the_others(ops, n, v, dtype):
    """A single word, so that only one thread and one CTA of a row's meets it, before, among and behind the others; and beside words that are not allowed and hold anything."""
    rng = _rng(n, v, 96)
    ordinary = rng.normal(0, 2, v)
    for at in (0, v // 3, v - 1):
        rows = []
        for c in FAR:
            for far in (c, -c):
                x, y = ordinary.copy(), np.full(v, far)
                x[at], y[at] = far, far * (1 - 2.0 ** -6)
                rows += [x, y]
        for a, b in ((65530.0, 65545.0), (-65545.0, -65530.0), (-4.2e6, -70000.0), (-4.1e6, -60000.0)):
            x = np.full(v, a)
            x[at] = b
            rows.append(x)
        for i in range(0, len(rows) - n + 1, n):
            x = np.stack(rows[i:i + n])[:, None].astype(np.float32)
            far_check(ops, _cuda(x, dtype), _cuda(np.full((n, 1), at if i % 4 else v // 2, np.int32)), 4)
            if i % 5 == 0:
                from test_gpu_token_scores import _bits
                allowed = rng.random((1, v)) < 0.5
                allowed[0, at] = i % 2 == 0
                wild = x.copy()
                wild[:, :, ~allowed[0]] = np.nan
                x[:, :, ~allowed[0]] = -np.inf
                tokens = _cuda(np.full((n, 1), at, np.int32))
                want = ops.score_tokens(_cuda(x, dtype), tokens, top=4)
                got = ops.score_tokens(_cuda(wild, dtype), tokens, top=4, allowed=_cuda(_bits(allowed)))
                far_check(ops, _cuda(x, dtype), tokens, 4)
                assert all((a == b).all() for a, b in zip(got, want))


@pytest.mark.parametrize("lens", [[300, 90], [9000]])
@pytest.mark.parametrize("g", [4, 16])
def test_attend_scores_that_leave_32_bits(ops, g, lens):
    """Rows whose scores leave 32 bits may be NaN; the others of their products are as good as they are alone, and those that see nothing zeros.  (Not the same to the bit: sums are taken out for all
    rows when one asks for it, and are rounded then.)"""
    from test_gpu_pages8 import attend_check
    rng = _rng(97, g)
    n, heads, dim, page = len(lens), 2, 64, 32
    pool, table, kv = memory8(rng, n, lens, heads, dim, page)
    q = _cuda(rng.normal(0, 1, (n, g, heads, dim)).astype(np.float32))
    first, last = np.zeros((n, g), np.int64), np.repeat(np.asarray(lens)[:, None], g, 1)
    first[:, 3] = last[:, 3]                                   # sees nothing
    attend_check(ops, q, pool, table, lens, kv, first=first, last=last)
    want, want_lse, tol, tol_lse = attend_ref(q, kv, table.cpu().numpy(), lens, dim ** -0.5, first=first, last=last)
    wild = q.clone()
    wild[:, 1], wild[:, 2, 0], wild[:, 3] = 3e38, -3e38, 3e38
    dev = dict(first=_cuda(first.astype(np.int32)), last=_cuda(last.astype(np.int32)))
    got, lse = ops.attend_pages8(wild, pool, table, _cuda(np.asarray(lens, np.int32)), want_lse=True, **dev)
    out, l = got.double().cpu().numpy(), lse.double().cpu().numpy()
    ordinary = np.ones((n, g, heads), bool)
    ordinary[:, 1] = ordinary[:, 2, 0] = ordinary[:, 3] = False
    assert (np.abs(out - want)[ordinary] <= tol[ordinary][:, None] + HALF_STEP[F32] * np.abs(want[ordinary])).all() and (np.abs(l - want_lse)[ordinary] <= tol_lse[ordinary]).all()
    assert (got[:, 3] == 0).all() and (lse[:, 3] == -INF).all()
    again, _ = ops.attend_pages8(q, pool, table, _cuda(np.asarray(lens, np.int32)), want_lse=True, scale=1e38, **dev)
    assert (again[:, 3] == 0).all() and again.shape == q.shape

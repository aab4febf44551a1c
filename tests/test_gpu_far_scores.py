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

"""Scores of given tokens against a plain implementation in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_device_ops import BF16, F16, F32, INF, _bits, _cuda, _logits, _rng

NAN = float("nan")


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from linmt_b200 import device_ops
    return device_ops


def score_ref(logits, tokens, top, allowed=None):
    x = logits.double().cpu().numpy()
    tok = tokens.cpu().numpy()
    n, t, v = x.shape
    lp, ent, words, best = np.zeros((n, t)), np.zeros((n, t)), np.full((n, t, top), -1), np.full((n, t, top), -INF)
    for i in range(n):
        for j in range(t):
            z = x[i, j].copy()
            if allowed is not None:
                z[~allowed[min(i, allowed.shape[0] - 1)]] = -INF
            here = 0 <= tok[i, j] < v
            if np.isnan(z).any() or z.max() == INF:
                lp[i, j] = ent[i, j] = NAN
                best[i, j] = NAN
                continue
            if z.max() == -INF:
                lp[i, j] = -INF if here else 0
                continue
            d = z - z.max()
            log_s = np.log(np.exp(d).sum())
            p = np.exp(d) / np.exp(d).sum()
            ent[i, j] = log_s - (p * np.where(p > 0, d, 0)).sum()
            lp[i, j] = d[tok[i, j]] - log_s if here else 0
            order = np.argsort(-z, kind="stable")[:top]
            order = order[z[order] > -INF]
            words[i, j, :len(order)], best[i, j, :len(order)] = order, d[order] - log_s
    return lp, ent, words, best


def score_check(ops, logits, tokens, top=0, allowed=None):
    got = ops.score_tokens(logits, tokens, allowed=None if allowed is None else _cuda(_bits(allowed)), top=top)
    assert len(got) == (4 if top else 2)
    lp, ent, words, best = score_ref(logits, tokens, top, allowed)
    # An exponent is rounded once, to 2^-24 of it (at most 2^-17 where it counts, a term being 2^-150 there; 2^-24 of x log2 e from the constant), exp2 is good to 2^-22; a thread
    # adds up to vocab / 128 terms (256 threads, two sums), which lose 2^-24 each of what is there, then 10 are joined; the logarithm and its products 2^-22 of what comes out.
    big = np.abs(np.nan_to_num(logits.double().cpu().numpy(), nan=0, posinf=0, neginf=0))
    big = np.where(big > 1e5, 0, big).max() if big.size else 0
    rel = (logits.shape[2] / 128 + 16) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -23 * big
    off = lambda g, w: np.abs(g - w) - 2.0 ** -22 * np.abs(w)
    same = lambda g, w: (np.isnan(g) == np.isnan(w)).all() and (np.isneginf(g) == np.isneginf(w)).all()
    g = [x.cpu().numpy().astype(np.float64) for x in got]
    assert same(g[0], lp) and same(g[1], ent)
    ok = np.isfinite(lp)
    assert (off(g[0][ok], lp[ok]) <= rel).all(), off(g[0][ok], lp[ok]).max()
    ok = np.isfinite(ent)
    # T / S is a mean of exponents, each off by its share of the relative error, and by its own
    assert (off(g[1][ok], ent[ok]) <= rel * (2 + 2 * np.log(logits.shape[2] + 1))).all(), off(g[1][ok], ent[ok]).max()
    if top:
        assert (g[2] == words).all() and same(g[3], best)
        ok = np.isfinite(best)
        assert (off(g[3][ok], best[ok]) <= rel).all()
    return got


def _tokens(rng, n, t, v):
    return _cuda(rng.integers(-1, v + 1, (n, t)).astype(np.int32))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,t,v", [(1, 1, 1), (2, 3, 2), (1, 1, 31), (3, 2, 33), (1, 5, 517), (4, 9, 1000), (2, 2, 4099), (1, 3, 8192), (1, 2, 8209), (3, 1, 30000), (1, 1, 80000), (40, 17, 5003), (2, 1, 250007)])
def test_score(ops, n, t, v, dtype):
    rng = _rng(n, t, v, 60)
    x = _logits(rng, n, t, v, dtype)
    for top in (0, 1, 5, 32):
        score_check(ops, x, _tokens(rng, n, t, v), top)
    for lists in (1, n):
        allowed = rng.random((lists, v)) < 0.4
        score_check(ops, x, _tokens(rng, n, t, v), 7, allowed)
        score_check(ops, x, _tokens(rng, n, t, v), 0, allowed)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("n,v", [(3, 700), (2, 5000), (1, 60000), (300, 9001)])
def test_score_ties_go_to_the_lowest_index(ops, n, v, dtype):
    """All equal; sorted either way in steps; more equal best words than a list holds; equal words at the end."""
    zeros = torch.zeros(n, 1, v, dtype=dtype, device="cuda")
    down = torch.linspace(4, -4, v, device="cuda").to(dtype).expand(n, 1, v).contiguous()
    steps = _cuda(np.repeat(np.arange(-(-v // 600), dtype=np.float32), 600)[:v] * 0.25, dtype).expand(n, 1, v).contiguous()
    tail = zeros.clone()
    tail[:, :, -40:] = 2
    some = zeros.clone()
    some[:, :, ::3] = 1
    few = torch.full_like(zeros, -INF)
    few[:, :, v // 2:v // 2 + 3] = 1
    tokens = _cuda(np.full((n, 1), v // 2, np.int32))
    for x in (zeros, down, down.flip(2).contiguous(), steps, tail, some, few):
        for top in (1, 32):
            score_check(ops, x, tokens, top)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("v", [50, 3000, 50000])
def test_score_infinities_nan_and_lowest_values(ops, v, dtype):
    rng = _rng(v, 61)
    x = _logits(rng, 1, 16, v, dtype)
    least, most = torch.finfo(dtype).min, torch.finfo(dtype).max
    x[0, 0, 3] = NAN
    x[0, 1, v - 1] = INF
    x[0, 2] = -INF
    x[0, 3] = least
    x[0, 4, :v // 2] = least
    x[0, 5, :v // 2] = -INF
    x[0, 6] = most
    x[0, 7] = -INF
    x[0, 7, v // 3] = -5
    x[0, 8] = -INF
    x[0, 8, v // 3] = least
    x[0, 9, 7] = most
    x[0, 10] = least
    x[0, 10, 5] = -INF
    x[0, 11, ::2] = NAN
    x[0, 12] = INF
    x[0, 13, v // 2:] = -1e4
    x[0, 14, :v // 2] = 1e4
    tokens = torch.full((1, 16), v // 3, dtype=torch.int32, device="cuda")
    for top in (0, 4, 32):
        score_check(ops, x, tokens, top)
    tokens[0, ::2] = -100
    score_check(ops, x, tokens, 3)
    # words that are not allowed may hold anything
    allowed = rng.random((1, v)) < 0.5
    allowed[0, [3, v - 1, v // 3]] = False
    allowed[0, 5:8] = True
    wild = x.clone()
    wild[:, :, torch.from_numpy(~allowed[0]).cuda()] = NAN
    score_check(ops, wild, tokens, 5, allowed)
    score_check(ops, wild, tokens, 5, np.zeros((1, v), bool))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_score_logits_far_from_zero(ops, dtype):
    rng = _rng(62)
    x = _logits(rng, 2, 3, 9001, F32)
    ramp = torch.linspace(-150, 150, 9001, device="cuda")
    for y in (x + 100, x - 1000, x * 40, x + ramp, torch.where(ramp < 0, x - 1000, x + 64)):
        score_check(ops, y.to(dtype), _tokens(rng, 2, 3, 9001), 9)


def test_score_strides(ops):
    rng = _rng(63)
    for v in (1000, 1001, 33333):
        base = _logits(rng, 3, 4, v, BF16)
        tokens = _tokens(rng, 3, 4, v)
        want = score_check(ops, base, tokens, 6)
        for shift in range(0, 9):
            wide = torch.full((4, 3, v + 17), NAN, dtype=BF16, device="cuda")[:, :, shift:shift + v].transpose(0, 1)
            wide.copy_(base)
            got = ops.score_tokens(wide, tokens, top=6)
            # the words of a row fall to threads by their addresses, so sums are added in another order
            assert (got[2] == want[2]).all() and torch.allclose(got[0], want[0], atol=4e-6) and torch.allclose(got[1], want[1], atol=2e-5)
        assert all((a == b).all() for a, b in zip(want, ops.score_tokens(base, tokens, top=6)))
        same = ops.score_tokens(base[:1].expand(3, 4, v), tokens[:1].expand(3, 4).contiguous(), top=6)
        assert all((a == a[:1]).all() for a in same)


def test_refusals(ops):
    x, t = torch.zeros(2, 3, 50, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for args, kw, match in [((x[0], t), {}, "n, t, vocab"), ((x.double(), t), {}, "n, t, vocab"), ((x, t.long()), {}, "Int"), ((x, t[:1]), {}, "shape"), ((x, t), dict(top=33), "0 .. 32"), ((x, t), dict(top=-1), "0 .. 32"),
                            ((x.transpose(1, 2), torch.zeros(2, 50, dtype=torch.int32, device="cuda")), {}, "contiguous"), ((x, t), dict(allowed=torch.zeros(3, 2, dtype=torch.int32, device="cuda")), "allowed"), ((x, t.cpu()), {}, "CUDA")]:
        with pytest.raises(ValueError, match=match):
            ops.score_tokens(*args, **kw)
    with pytest.raises(ValueError, match="gradient"):
        ops.score_tokens(x.clone().requires_grad_(), t)
    assert ops.score_tokens(x[:0], t[:0], top=2)[2].shape == (0, 3, 2)


def test_captured_and_on_two_streams(ops):
    rng = _rng(64)
    runs = []
    for i in range(2):
        x, t = _logits(rng, 2, 30, 9000 + i, F16), _tokens(rng, 2, 30, 9000)
        ops.score_tokens(x, t, top=4)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.score_tokens(x, t, top=4)
        runs.append((graph, torch.cuda.Stream(), x, t, out))
    for _ in range(4):
        for graph, stream, x, t, out in runs:
            with torch.cuda.stream(stream):
                x.copy_(_logits(rng, *x.shape, F16))
                graph.replay()
        torch.cuda.synchronize()
        for graph, stream, x, t, out in runs:
            for a, b in zip(out, score_check(ops, x, t, 4)):
                assert (a == b).all()

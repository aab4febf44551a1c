"""Tables of pages as a program slices them."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_device_ops import _rng
from test_gpu_page_ops import _i32, _state, compact_ref, fork_ref


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from linmt_b200 import device_ops
    return device_ops


def test_one_hypothesis_of_each_sentence(ops):
    """One of a sentence's hypotheses: its rows lie evenly, further apart than they are long."""
    rng = _rng(70)
    n, k, page = 7, 3, 16
    lens = rng.integers(1, 60, (n, k))
    table, shares, free, used = _state(rng, n, k, lens, page, 20, shared=0)
    dev = _i32(table)
    for j in range(k):
        t, l = dev[:, j:j + 1], _i32(lens[:, j:j + 1])
        want = fork_ref(table[:, j:j + 1], lens[:, j:j + 1], np.zeros((n, 1), int), shares, free, used, page)
        for got in (ops.fork_pages(t, l, _i32(np.zeros((n, 1))), _i32(shares), _i32(free), _i32([used]), page=page), ops.free_pages(t, l, torch.zeros(n, 1, dtype=torch.bool, device="cuda"), _i32(shares), _i32(free), _i32([used]), page=page)):
            for g, w in zip(got, want):
                assert (g.cpu().numpy() == w).all()
        for g, w in zip(ops.compact_pages(t, l, _i32(shares), page=page), compact_ref(table[:, j:j + 1], lens[:, j:j + 1], shares, page)):
            assert (g.cpu().numpy() == w).all()
    # and one in place whose only hypothesis has a stride that says nothing
    one = _i32(table[:, 0])
    odd, s = one.as_strided((n, 1, table.shape[2]), (table.shape[2], 999, 1)), _i32(shares)
    want = compact_ref(table[:, :1], lens[:, :1], shares, page)
    got = ops.compact_pages(odd, _i32(lens[:, :1]), s, page=page, out=(odd, s) + tuple(_i32(np.zeros(m)) for m in (len(shares), 1, len(shares) // 2, len(shares) // 2)))
    for g, w in zip(got, want):
        assert (g.cpu().numpy() == w).all()

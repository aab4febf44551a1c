"""Sizes at the end of what the page plans count in 32 bits: refused before anything reaches a device."""
import pytest

torch = pytest.importorskip("torch")

from test_more_ops_host import ELIMIT, _refused

MOST = 2 ** 31 - 2 ** 17 - 1


@pytest.mark.parametrize("word,kw", [("n_pages", dict(n_pages=2 ** 31 - 1)), ("n_free", dict(n_free=2 ** 31 - 1)), ("n_free", dict(n_free=MOST + 1)), ("width", dict(n=1, k=1, width=2 ** 31 - 1)), ("width", dict(n=1, k=2, width=2 ** 30 - 1))])
def test_fork_refuses_more_than_it_counts(cuda_lib, word, kw):
    _refused(cuda_lib, "linmt_fork_pages", "linmt_fork_pages_args", ELIMIT, word, **kw)


@pytest.mark.parametrize("word,kw", [("n_pages", dict(n_pages=2 ** 31 - 1)), ("n_pages", dict(n_pages=MOST + 1)), ("rows", dict(rows=2 ** 31 - 1, width=1)), ("rows", dict(rows=MOST + 1, width=1)), ("rows", dict(rows=1, width=2 ** 31 - 1))])
def test_compact_refuses_more_than_it_counts(cuda_lib, word, kw):
    _refused(cuda_lib, "linmt_compact_pages", "linmt_compact_pages_args", ELIMIT, word, **kw)

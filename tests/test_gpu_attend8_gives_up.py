"""What attention over 8-bit pages leaves where CTAs have given up a wait: NaN in all rows that they had a part in, and all other rows as they are."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_device_ops import BF16, F16, F32, _cuda, _rng
from test_gpu_pages8 import memory8


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from linmt_b200 import device_ops
    return device_ops


@pytest.mark.parametrize("dtype,heads,rep,g,dim,lens", [(F32, 1, 1, 1, 64, [40]), (BF16, 2, 1, 5, 64, [700] * 40), (F16, 1, 4, 4, 128, [20000, 300, 0, 9000]), (F32, 3, 1, 3, 128, [0, 5, 16, 900] * 200), (BF16, 1, 1, 33, 64, [5000])])
def test_ctas_that_gave_up(ops, cuda_lib, dtype, heads, rep, g, dim, lens):
    rng = _rng(g, dim, len(lens))
    n = len(lens)
    pool, table, _ = memory8(rng, n, lens, heads, dim, 64)
    q, at = _cuda(rng.normal(0, 1, (n, g, heads * rep, dim)).astype(np.float32), dtype), _cuda(np.asarray(lens, np.int32))
    run = lambda: ops.attend_pages8(q, pool, table, at, want_lse=True)
    want, want_lse = run()
    assert not want.isnan().any()
    lost = []
    try:
        for each in (1, 2, 3, 7, 1000):
            assert cuda_lib.linmt_k_attend8_give_up(each) == 0
            out, lse = run()
            nan = lse.isnan()
            assert (out.isnan() == nan[..., None]).all()
            assert (out[~nan] == want[~nan]).all() and (lse[~nan] == want_lse[~nan]).all()
            lost.append(int(nan.sum()))
    finally:
        assert cuda_lib.linmt_k_attend8_give_up(0) == 0
    assert lost[0] == nan.numel() and min(lost) > 0 and (lost[4] < lost[0] or n == 1)      # (the first CTA has the first sentence's rows)
    out, lse = run()
    assert (out == want).all() and (lse == want_lse).all()
    assert cuda_lib.linmt_k_attend8_give_up(-1) != 0

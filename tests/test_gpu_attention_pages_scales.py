""""attention_pages_*" where all of a row's weight lies on values that are 0, beside values under large scales that have next to none."""
import numpy as np
import pytest

import pages_reference as ref
from test_gpu_attention_pages import attend
from test_gpu_pages import Batch

pytestmark = pytest.mark.gpu

# rows of 4 queries to a key head: 16, 32, 64 and 128 columns
FORMS = [(64, 1), (64, 8), (64, 12), (64, 40), (128, 1), (128, 8), (128, 12), (128, 40), (256, 1), (256, 12), (256, 40)]


def far(backend, fmt, d, rows, n, gap, scale):
    """Every query's score of one key, whose page's values are 0, lies `gap` (in powers of two) above all others, about; the others'
    values lie under `scale`."""
    group, block = 4, 16
    b = Batch(backend, d + rows, fmt, 1, block, d, [n])
    sign = np.where(b.rs.rand(d) < 0.5, -1.0, 1.0)
    at, codes = b.table[0, 2], 64.0
    b.pool.kp[:] = ref.encode(fmt, np.zeros(b.pool.kp.shape, np.float32))
    b.pool.kp[at, 0, 5] = ref.encode(fmt, (sign * codes).astype(np.float32))
    q = np.tile(sign, (rows, group)).astype(np.float32) * (1 + 0.01 * b.rs.rand(rows, 1))
    b.pool.ks[:] = np.float32(gap * np.log(2.0) / np.sqrt(d) / codes)
    b.pool.vs[:] = np.float32(scale)
    b.pool.vs[at] = 0.0
    b.upload()
    return b, q.astype(np.float32), group


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
@pytest.mark.parametrize("d,rows", FORMS)
@pytest.mark.parametrize("scale", [1.0, 2.0, 4.0, 300.0, 2.0 ** 60, 2.0 ** 119])
def test_no_weight_beside_zeros(backend, fmt, d, rows, scale):
    """Weights of 2^-300 are 0 in fp32, and so is what they weigh."""
    for n in (100, 1500):
        b, q, group = far(backend, fmt, d, rows, n, 300.0, scale)
        for window, sinks in ((0, 0), (64, 48)):
            got = attend(b, q, [0, rows], group, window, sinks, max_rows=rows)
            assert np.array_equal(got, np.zeros_like(got)), (n, window)


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
@pytest.mark.parametrize("d,rows", FORMS)
@pytest.mark.parametrize("gap,scale", [(40.0, 4.0), (90.0, 2.0 ** 100), (112.0, 2.0 ** 100), (112.0, 2.0 ** 30), (121.0, 2.0 ** 119)])
def test_little_weight_beside_zeros(backend, fmt, d, rows, gap, scale):
    """All that a result has are products of next to no weights: within the bound of any other.  Terms of weights below 2^-116 may lie as if
    those were 2^-116, 2^10 lower than others': the largest at 2^-1 at least, where half of 2^-24 is 2^-24 of it."""
    for n in (100, 1500):
        b, q, group = far(backend, fmt, d, rows, n, gap, scale)
        got = attend(b, q, [0, rows], group, max_rows=rows)
        want, bound = ref.attention(b.pool, b.table[0], n, q.reshape(rows, group, d), group)
        k, v = (x[:, 0].astype(np.float64) for x in b.pool.rows(b.table[0], np.arange(n)))
        s = q.reshape(-1, d).astype(np.float64) @ k.T / np.sqrt(d)
        seen = np.repeat(ref.visible(np.arange(n - rows, n), n, 0, 0), group, 0)
        p = np.where(seen, np.exp(s - s.max(1, keepdims=True)), 0.0)
        assert p[p > 0].min() > 2.0 ** -126 and np.abs(want).max() > 0
        bound += (2.0 ** -24 * (p @ np.abs(v)) / p.sum(1, keepdims=True)).reshape(bound.shape)
        off = np.abs(got - want)
        assert (off <= bound).all(), (n, float((off / bound).max()))


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
@pytest.mark.parametrize("d,rows", FORMS)
def test_a_page_of_nan_stays_one(backend, fmt, d, rows):
    """Values whose scale is NaN make a result NaN, though their weights are 0."""
    b, q, group = far(backend, fmt, d, rows, 1500, 300.0, 4.0)
    b.pool.vs[b.table[0, 70]] = np.nan
    b.upload()
    assert np.isnan(attend(b, q, [0, rows], group, max_rows=rows)).all()

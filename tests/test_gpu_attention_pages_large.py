""""attention_pages_*" of values whose sum over a row's positions is past fp32's range, and of values near its lower end: a mean is in range."""
import numpy as np
import pytest

import pages_shapes as shapes
from test_gpu_attention_pages import check, queries
from test_gpu_pages import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
@pytest.mark.parametrize("how,pairs,d", [x for x in shapes.forms() if x[1] in (1, 16, 32, 33, 65) and x[2] in (64, 128, 256)])
@pytest.mark.parametrize("scale", [2.0 ** 118, 2.0 ** -117])
def test_values_at_the_ends(backend, fmt, how, pairs, d, scale):
    """Scales up to 2^119 (codes of 448: 2^127.8) over hundreds and thousands of positions; scales below 2^-116 (codes of 1: above 2^-118)."""
    group, rows, past, most_rows, most_len = shapes.sizes(how, pairs)
    b = Batch(backend, pairs + d, fmt, shapes.KV, 32, d, [a + n for a, n in zip(past, rows)])
    b.pool.vs[:] = (1.0 + b.rs.rand(*b.pool.vs.shape)) * scale
    if scale > 1.0:     # all of one sign: their sum is as large as can be
        b.pool.vp &= 0x7F
        if fmt == "fp8":
            b.pool.vp[b.pool.vp == 0x7F] = 0x7E
    b.upload()
    check(b, queries(b.rs, sum(rows), shapes.KV * group * d), rows, group, max_rows=most_rows, max_len=most_len)

"""Every form of the kernels of "attention_pages_*" (format, head size, columns of a unit, how positions are shared) against the 64-bit
formula, with the most rows handed over, as decode and drafts are called.  tests/test_page_shapes.py: that each is the form it is for."""
import numpy as np
import pytest

import pages_shapes as shapes
from test_gpu_attention_pages import check, queries
from test_gpu_pages import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
@pytest.mark.parametrize("how,pairs,d", list(shapes.forms()))
def test_form(backend, fmt, how, pairs, d):
    group, rows, past, most_rows, most_len = shapes.sizes(how, pairs)
    block = (16, 32, 64, 128)[(pairs + d // 16) % 4]
    b = Batch(backend, 1000 * pairs + d, fmt, shapes.KV, block, d, [a + n for a, n in zip(past, rows)])
    q = queries(b.rs, sum(rows), shapes.KV * group * d)
    check(b, q, rows, group, max_rows=most_rows, max_len=most_len)
    if how == "short":
        check(b, q, rows, group, 37, 5, max_rows=most_rows, max_len=most_len)


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
@pytest.mark.parametrize("d,rows,group", [(128, 8, 4), (128, 4, 8), (80, 1, 32), (64, 16, 2), (256, 4, 4), (256, 2, 8), (208, 16, 1)])
def test_all_columns_of_a_long_cache(backend, fmt, d, rows, group):
    """As many pairs as a unit has columns, on more positions than a workgroup a head is for, beside a short sequence."""
    past = 40000 if d <= 128 else 30000
    b = Batch(backend, d + rows, fmt, 1, 64, d, [past + rows, 70 + rows])
    q = queries(b.rs, 2 * rows, group * d)
    check(b, q, [rows, rows], group, max_rows=rows)
    check(b, q, [rows, rows], group, 20000, 70, max_rows=rows)

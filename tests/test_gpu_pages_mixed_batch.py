"""A step whose batch has prompts and decoded sequences, its prompts first: in one call of "attention_pages_*", and in two over the same
Starts, Lens and Table, of the prompts alone (fewer `sequences`) and of the others (a `max_rows` that leaves the prompts out)."""
import numpy as np
import pytest

from test_gpu_attention_pages import check, queries
from test_gpu_pages import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,kv,group,block,d", [("q8", 2, 4, 16, 64), ("fp8", 2, 4, 32, 128), ("q8", 1, 6, 64, 256)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 4)])
def test_prompts_and_decoded_sequences(backend, fmt, kv, group, block, d, window, sinks):
    prompts, decoded = [70, 33], [1, 3, 1, 0, 2] * 8
    rows = prompts + decoded
    past = [100, 0] + [(37 * i) % 700 for i in range(len(decoded))]
    b = Batch(backend, d + window, fmt, kv, block, d, [a + n for a, n in zip(past, rows)])
    q = queries(b.rs, sum(rows), kv * group * d)
    check(b, q, rows, group, window, sinks)
    starts, heads, m = np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32), kv * group, sum(rows)
    up = backend.Upload
    out, dq, st = up(np.full(q.shape, 7.0, np.float32)), up(q), up(starts)
    buffers = [dq, *b.dev, b.dev_table, st, b.dev_lens, out]
    _, size, pages, width = b.shape
    for sequences, most in ((len(prompts), max(prompts)), (len(rows), max(decoded))):
        b.go("attention_pages", buffers, [m, heads, kv, d, sequences, size, pages, width, most, 0, window, sinks])
    check(b, q, rows, group, window, sinks, got=backend.CopyD2H(out, dtype=np.float32).reshape(m, heads, d))

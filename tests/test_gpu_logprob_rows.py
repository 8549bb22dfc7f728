"""More rows than a launch of "token_logprobs" takes (16384): each with results at its own place, also behind rows of others."""
import numpy as np
import pytest

from test_gpu_tree import check_logprobs, near, token_logprobs
import tree_reference as ref

pytestmark = pytest.mark.gpu

LAUNCH = 1 << 14


def distinct(rows, vocab, seed):
    return (np.random.RandomState(seed).randn(rows, vocab) * 3).astype(np.float32)


@pytest.mark.parametrize("rows", [LAUNCH, LAUNCH + 1, LAUNCH + 116, 2 * LAUNCH + 3])
@pytest.mark.parametrize("top_k", [0, 5])
def test_rows_around_a_launch(backend, rows, top_k):
    base, vocab = 3, 29
    x = distinct(base + rows, vocab, rows)
    check_logprobs(backend, x, np.random.RandomState(top_k).randint(0, vocab + 1, (rows, 3)), top_k, row_base=base)


def test_rows_of_several_tiles(backend):
    """Rows that no 16 bytes divide; those of both launches that lie next to the border against the formulas, all against one another."""
    base, rows, vocab = 2, LAUNCH + 500, 2301
    x = distinct(base + 300, vocab, 1)
    x = x[np.arange(base + rows) % (base + 300)]                # row r is row r % 302
    tokens = (np.arange(rows)[:, None] * 7 + np.arange(4)) % (vocab + 1)
    got = token_logprobs(backend, x, tokens, 32, base)
    at = np.r_[0:40, LAUNCH - 200:LAUNCH + 200, rows - 40:rows]
    want = ref.logprobs(x[base + at], tokens[at], 32)
    assert np.array_equal(got["top"][at], want["top"])
    for name in ("logprobs", "top_logprobs"):
        size = np.abs(np.where(np.isfinite(want[name]), want[name], 0.0))
        near(got[name][at], want[name], want["bound"][:, None] + 3 * ref.EPS * size)
    near(got["entropy"][at], want["entropy"], want["entropy_bound"])
    same = (base + np.arange(rows)) % 604                       # equal rows that begin alike within 16 bytes: equal bits
    for name in ("entropy", "top", "top_logprobs"):
        first = got[name][np.maximum(same - base, 0)]
        rows_of = same >= base
        assert np.array_equal(got[name][rows_of], first[rows_of])

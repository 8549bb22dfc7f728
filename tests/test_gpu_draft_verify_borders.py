""""draft_verify" where the second random number lies on a border between tokens: sums of halves that are alike, with banned tokens behind
the border.  Which of the border's two tokens it is may hang on a rounding; that it has a probability may not."""
import numpy as np
import pytest

from test_gpu_draft_verify import launch

pytestmark = pytest.mark.gpu

CHUNK = 512      # columns that are summed before chunks are


def halves(rs, full, empty, banned):
    """A row of two halves alike, `full` chunks of which the first `banned` columns have no probability and `empty` ones that have none."""
    half = (rs.randn(full + empty, CHUNK) * 2.5).astype(np.float32)
    half[:, :banned] = -np.inf
    half[full:] = -np.inf
    return np.concatenate([half, half]).reshape(-1)


@pytest.mark.parametrize("full,empty,banned", [(2, 0, 9), (2, 0, 511), (3, 0, 64), (5, 4, 9), (6, 3, 100), (6, 20, 1), (11, 9, 8), (70, 60, 20)])
@pytest.mark.parametrize("kind", ["last", "sampled"])
@pytest.mark.parametrize("alone", [False, True])
def test_a_token_of_the_border(backend, full, empty, banned, kind, alone):
    rs = np.random.RandomState(100 * full + empty + banned)
    n = 48
    rows = np.stack([halves(rs, full, empty, banned) for _ in range(n)])
    vocab = rows.shape[1]
    if kind == "last":
        logits, draft, starts, tokens = rows, None, np.arange(n + 1), np.zeros(n, np.uint32)
    else:       # refused by its random number, with what the draft has taken off a column of each half
        logits = np.repeat(rows, 2, 0)
        draft = np.full_like(logits, -np.inf)
        draft[:, [CHUNK - 1, vocab // 2 + CHUNK - 1]] = logits.max(1, keepdims=True)
        tokens, starts = np.full(2 * n, CHUNK - 1, np.uint32), np.arange(0, 2 * n + 1, 2)
    random = np.ones((len(logits), 2), np.float32)
    random[:, 1] = 0.5
    accepted, after = launch(backend, logits, tokens, random, starts, 1.0, draft, 1.0, alone)
    if kind == "sampled":
        p, q = (np.exp(x.astype(np.float64) - x.max(1, keepdims=True)) for x in (logits, draft))
        left = np.maximum(p / p.sum(1, keepdims=True) - q / q.sum(1, keepdims=True), 0.0)[::2]
    else:
        left = np.isfinite(logits)
    for s in range(n):
        some = np.nonzero(left[s] > 0)[0]
        border = {int(some[some < vocab // 2][-1]), int(some[some >= vocab // 2][0])}
        assert int(accepted[s]) == 0 and int(after[s]) in border, (s, int(after[s]), border)


@pytest.mark.parametrize("alone", [False, True])
def test_no_token_without_a_probability(backend, alone):
    """Quarters alike, most columns banned, and numbers on and beside every border."""
    rs = np.random.RandomState(7)
    half = (rs.randn(24, CHUNK) * 2.5).astype(np.float32)
    half[rs.rand(*half.shape) < 0.9] = -np.inf
    half[:, 0], half[[3, 4, 9, 17]] = -np.inf, -np.inf
    row = np.concatenate([half] * 4).reshape(-1)
    numbers = np.concatenate([[np.nextafter(np.float32(x), np.float32(to)) for to in (0, x, 1)] for x in (0.125, 0.25, 0.375, 0.5, 0.625, 0.75, 0.875)])
    n = len(numbers)
    random = np.stack([np.ones(n), numbers], 1).astype(np.float32)
    _, after = launch(backend, np.tile(row, (n, 1)), np.zeros(n, np.uint32), random, np.arange(n + 1), 1.0, None, 1.0, alone)
    assert np.isfinite(row[after]).all(), after

""""draft_verify" against its statement in 64 bits: the same counts and the same tokens."""
import numpy as np
import pytest

import pages_reference as ref
from tessera_amd import KernelLaunch
from test_gpu_tree import f32_bits

pytestmark = pytest.mark.gpu


def launch(backend, logits, tokens, random, starts, temperature, draft=None, draft_temperature=1.0, alone=False):
    up = backend.Upload
    n = len(starts) - 1
    out = [up(np.full(n, 777, np.uint32)) for _ in range(2)]
    buffers = [up(logits), up(np.asarray(tokens, np.uint32)), up(random.astype(np.float32)), up(np.asarray(starts, np.uint32)), *out]
    if draft is not None:
        buffers.append(up(draft))
    call = KernelLaunch(buffers=buffers, scalars=[*logits.shape, n, f32_bits(temperature), f32_bits(draft_temperature)])
    kernel = backend.LoadKernel("draft_verify")
    if alone:       # the per-thread stream has no scratch block
        backend.Synchronize()
        stream = backend._stream.value or 0
        backend.SetStream(2)
        try:
            backend.LaunchKernel(kernel, call)
            backend.Synchronize()
        finally:
            backend.SetStream(stream)
    else:
        backend.LaunchKernel(kernel, call)
    return [backend.CopyD2H(x, dtype=np.uint32) for x in out]


def check(backend, logits, tokens, random, starts, temperature, draft=None, draft_temperature=1.0):
    want = ref.verify(logits, tokens, random, starts, temperature, draft, draft_temperature)
    for alone in (False, True):
        accepted, after = launch(backend, logits, tokens, random, starts, temperature, draft, draft_temperature, alone)
        for s, w in enumerate(want):
            assert (int(accepted[s]), int(after[s])) == (w or (777, 777)), (s, alone)
    return want


def inputs(rs, rows, vocab, spread=2.5, agree=0.8):
    starts = np.concatenate([[0], np.cumsum(rows)])
    m = int(starts[-1])
    logits = (rs.randn(m, vocab) * spread).astype(np.float32)
    draft = (logits + rs.randn(m, vocab) * 0.5).astype(np.float32)
    tokens = np.where(rs.rand(m) < agree, np.roll(logits.argmax(1), 1), rs.randint(0, vocab, m)).astype(np.uint32)
    return logits, draft, tokens, rs.rand(m, 2).astype(np.float32), starts


ROWS = [1, 5, 3, 1, 8, 2, 4, 17, 5, 5, 6]


@pytest.mark.parametrize("vocab", [1, 2, 63, 500, 511, 513, 1025, 12289, 50001, 131072])
@pytest.mark.parametrize("temperature", [0.0, 0.3, 1.0, 4.0])
@pytest.mark.parametrize("sampled", [False, True])
def test_against_the_statement(backend, vocab, temperature, sampled):
    rs = np.random.RandomState(vocab + int(10 * temperature) + sampled)
    logits, draft, tokens, random, starts = inputs(rs, ROWS, vocab)
    if sampled:     # tokens from the draft's own distribution
        g = -np.log(-np.log(rs.rand(*draft.shape) + 1e-300))
        tokens = np.roll((draft / max(temperature, 0.1) + g).argmax(1), 1).astype(np.uint32)
    want = check(backend, logits, tokens, random, starts, temperature, draft if sampled else None, temperature or 1.0)
    if vocab >= 500 and (sampled or temperature < 1.0):      # (at higher ones the likeliest of many has too little)
        assert sum(w[0] for w in want) > 0


def test_other_temperature_of_the_draft(backend):
    rs = np.random.RandomState(3)
    logits, draft, tokens, random, starts = inputs(rs, ROWS, 5000)
    check(backend, logits, tokens, random, starts, 0.7, draft, 1.3)
    check(backend, logits, tokens, random, starts, 1e-30, draft, 1e30)
    check(backend, logits, tokens, random, starts, 1e30, draft, 1e-30)


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_banned_tokens(backend, temperature):
    """-infinity is a token of probability 0: never drawn, a drafted one never stands; what the draft cannot have drafted does where
    the target has it."""
    rs = np.random.RandomState(5)
    logits, draft, tokens, random, starts = inputs(rs, ROWS, 9000)
    logits[rs.rand(*logits.shape) < 0.9] = -np.inf
    logits[:, 8999] = 0.0
    draft[rs.rand(*draft.shape) < 0.9] = -np.inf
    draft[:, 4100] = 0.0
    for d in (None, draft):
        want = check(backend, logits, tokens, random, starts, temperature, d)
        for s, (at, token) in enumerate(want):
            assert np.isfinite(logits[starts[s] + at, token])
    # a row of one token only; its draft stands
    logits[:] = -np.inf
    logits[:, 77] = -1e30
    tokens[:] = 77
    want = check(backend, logits, tokens, random, starts, temperature)
    assert want == [(n - 1, 77) for n in ROWS]


def test_nothing_left_but_the_target(backend):
    """The draft accounts for all of the target where a token is refused all the same: the next is drawn from the target."""
    rs = np.random.RandomState(7)
    logits, _, tokens, random, starts = inputs(rs, ROWS, 6000)
    tokens[:] = 6000 + np.arange(len(tokens))       # of no vocabulary: never stands, nothing is taken off
    check(backend, logits, tokens, random, starts, 1.0)
    want = check(backend, logits, tokens, random, starts, 1.0, logits)
    assert all(w[0] == 0 for w in want)
    tokens[:] = 0xFFFFFFFF
    check(backend, logits, tokens, random, starts, 1.0, logits)
    check(backend, logits, tokens, random, starts, 0.0)
    # one token has all of the probability and is refused, as its number is not below 1
    logits[:] = -np.inf
    logits[:, 5] = 1.0
    tokens[:] = 5
    random[:, 0] = 1.0
    assert check(backend, logits, tokens, random, starts, 1.0) == [(0, 5)] * len(ROWS)


def test_rows_that_say_nothing(backend):
    """NaN, +infinity or -infinity alone end the draft there with no token."""
    rs = np.random.RandomState(9)
    rows = [4] * 8
    logits, draft, tokens, random, starts = inputs(rs, rows, 5000)
    best = logits.argmax(1)
    tokens = np.roll(best, 1)
    random[:, 0] = 0.0                              # every draft stands
    logits[1, 4500] = np.nan
    logits[4 + 2, 17] = np.inf
    logits[8 + 3] = -np.inf
    draft[12 + 1, 4999] = np.nan
    draft[16 + 3] = np.nan                          # the last row's: not looked at
    draft[20 + 0, 3] = np.inf
    draft[24 + 2] = -np.inf
    want = check(backend, logits, tokens, random, starts, 1.0, draft)
    assert [w[0] for w in want] == [1, 2, 3, 1, 3, 0, 2, 3] and [w[1] == ref.NONE for w in want] == [True, True, True, True, False, True, True, False]
    want = check(backend, logits, tokens, random, starts, 0.0, draft)
    assert [w[0] for w in want] == [1, 2, 3, 3, 3, 3, 3, 3] and [w[1] == ref.NONE for w in want] == [True, True, True] + [False] * 5
    check(backend, logits, tokens, random, starts, 1.0)


def test_equal_logits(backend):
    """The lowest of equals where the likeliest is asked for; all tokens alike where one is drawn; +0 and -0 are equal."""
    vocab = 13000
    logits = np.zeros((6, vocab), np.float32)
    logits[:, ::2] = -0.0
    tokens = np.array([0, 0, 1, 5, 0, 0], np.uint32)
    random = np.array([[0.5, 0.0], [0.99, 0.25], [0.0, 0.5], [0.0, 0.75], [0.0, 0.9999999], [0.0, 0.1]], np.float32)
    assert check(backend, logits, tokens, random, [0, 2, 3, 6], 0.0) == [(1, 0), (0, 0), (2, 0)]
    check(backend, logits, tokens, random, [0, 2, 3, 6], 1.0)
    check(backend, logits, tokens, random, [0, 1, 2, 3, 4, 5, 6], 1.0)
    logits[:, 7000:] = 3.0
    logits[3, 12999] = 3.5
    check(backend, logits, tokens, random, [0, 1, 2, 3, 4, 5, 6], 0.0)


def test_numbers_at_the_ends(backend):
    """0, the largest below 1, and what is no number of [0, 1): no fault, a token of the distribution."""
    rs = np.random.RandomState(13)
    rows = [1] * 6 + [3] * 6
    logits, draft, tokens, random, starts = inputs(rs, rows, 4500)
    logits[:, 4490:] = -np.inf
    odd = np.array([0.0, 1.0 - 2.0 ** -24, 1.0, 5.0, -1.0, np.nan], np.float32)
    random[:6, 1] = odd
    for i in range(6):
        random[6 + 3 * i:9 + 3 * i, 0], random[6 + 3 * i:9 + 3 * i, 1] = odd[i], odd[(i + 3) % 6]
    for d in (None, draft):
        check(backend, logits, tokens, random, starts, 1.0, d)


def test_rows_of_no_sequence_and_sequences_of_no_row(backend):
    rs = np.random.RandomState(17)
    logits, draft, tokens, random, _ = inputs(rs, [12], 800)
    starts = np.array([0, 3, 3, 5, 4, 9, 13, 2], np.uint32)      # 1: none; 3: 5 to 4; 5: 9 to 13 of 12; 6: 13 to 2
    check(backend, logits, tokens, random, starts, 1.0, draft)
    check(backend, logits, tokens, random, starts, 0.0)


def test_large_logits(backend):
    """Differences from the largest are formed in 64 bits: logits of 1e30, of 3e38 and of 1e-30."""
    rs = np.random.RandomState(19)
    logits, draft, tokens, random, starts = inputs(rs, ROWS, 3000)
    for scale, temperature in ((1e30, 1.0), (1e30, 1e29), (2e37, 1e37), (1e-30, 1.0), (1e-30, 1e-30)):
        x, y = (logits * np.float32(scale)), (draft * np.float32(scale))
        check(backend, x, tokens, random, starts, temperature, y, temperature)


def test_the_largest_vocabulary(backend):
    rs = np.random.RandomState(23)
    vocab = 1 << 21
    logits = rs.rand(3, vocab).astype(np.float32)
    tokens = np.array([0, int(logits[0].argmax()), 5], np.uint32)
    random = np.array([[0.0, 0.3], [0.999, 0.7], [0.5, 0.999]], np.float32)
    check(backend, logits, tokens, random, [0, 3], 1.0)
    check(backend, logits, tokens, random, [0, 3], 0.0)


def test_draws_follow_the_target(backend):
    """Verified drafts leave the target's distribution: of 40000 draws over eight tokens each count is within six of its standard
    deviations (a chance of 2e-9 a token)."""
    rs = np.random.RandomState(29)
    n, vocab = 4000, 8
    p, q = ref.softmax(rs.randn(vocab).astype(np.float32), 1.0), ref.softmax(rs.randn(vocab).astype(np.float32), 1.0)
    logits = np.tile(np.log(p).astype(np.float32), (2 * n, 1))
    draft = np.tile(np.log(q).astype(np.float32), (2 * n, 1))
    counts = np.zeros(vocab)
    for _ in range(10):
        tokens = np.zeros(2 * n, np.uint32)
        tokens[1::2] = rs.choice(vocab, n, p=q)
        accepted, after = launch(backend, logits, tokens, rs.rand(2 * n, 2).astype(np.float32), np.arange(0, 2 * n + 1, 2), 1.0, draft)
        counts += np.bincount(np.where(accepted == 1, tokens[1::2], after), minlength=vocab)
    assert (np.abs(counts - 10 * n * p) <= 6 * np.sqrt(10 * n * p * (1 - p))).all()

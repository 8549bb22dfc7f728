""""attention_pages_q8", "attention_pages_fp8" against the 64-bit formula over the numbers that the pages hold (pages_reference.py: how far
fp32 sums may be from it)."""
import numpy as np
import pytest
import torch

import pages_reference as ref
from test_gpu_pages import Batch

pytestmark = pytest.mark.gpu


def attend(b, q, starts, heads, window=0, sinks=0, max_rows=0, max_len=0, fill=7.0, m=None):
    m = m or q.shape[0]
    up = b.backend.Upload
    out, dq, st = up(np.full((m, q.shape[1]), fill, np.float32)), up(q), up(np.asarray(starts, np.uint32))
    b.go("attention_pages", [dq, *b.dev, b.dev_table, st, b.dev_lens, out], [m, heads, b.pool.kv, b.pool.d, *b.shape, max_rows, max_len, window, sinks])
    return b.backend.CopyD2H(out, dtype=np.float32).reshape(m, heads, b.pool.d)


def check(b, q, rows, group, window=0, sinks=0, got=None, only=None, **how):
    heads, d = b.pool.kv * group, b.pool.d
    starts = np.concatenate([[0], np.cumsum(rows)])
    if got is None:
        got = attend(b, q, starts, heads, window, sinks, **how)
    for s, n in enumerate(rows):
        if n == 0 or (only is not None and s not in only):
            continue
        want, bound = ref.attention(b.pool, b.table[s], int(b.lens[s]), q[starts[s]:starts[s + 1]].reshape(n, heads, d), group, window, sinks)
        off = np.abs(got[starts[s]:starts[s + 1]] - want)
        assert (off <= bound).all(), (s, n, float((off / np.maximum(bound, 1e-300)).max()))
    return got


def queries(rs, m, wide):
    return rs.randn(m, wide).astype(np.float32)


SHAPES = [  # format, key heads, queries to each, block, head size
    ("q8", 2, 1, 16, 64), ("fp8", 1, 4, 32, 64), ("q8", 1, 6, 16, 128), ("fp8", 2, 8, 128, 128), ("q8", 4, 6, 32, 256), ("fp8", 1, 3, 64, 256),
    ("q8", 1, 2, 64, 80), ("fp8", 2, 4, 16, 96), ("q8", 1, 16, 16, 48), ("q8", 1, 33, 32, 16), ("fp8", 3, 5, 16, 208)]


@pytest.mark.parametrize("fmt,kv,group,block,d", SHAPES)
def test_decode_and_verify(backend, fmt, kv, group, block, d):
    """One row and a few, from the first position on, lengths around pages and tiles."""
    rows = [1, 1, 2, 5, 1, 3, 0, 1, 16, 1, 4]
    past = [0, 1, 0, 14, 15, 62, 33, 63, 64, 127, 1000]
    b = Batch(backend, d + group, fmt, kv, block, d, [a + n for a, n in zip(past, rows)])
    check(b, queries(b.rs, sum(rows), kv * group * d), rows, group)


@pytest.mark.parametrize("fmt,kv,group,block,d", SHAPES)
def test_windows_and_sinks(backend, fmt, kv, group, block, d):
    rows = [1, 3, 1, 7, 2, 1]
    past = [0, 10, 500, 777, 4, 1300]
    b = Batch(backend, 3 * d + group, fmt, kv, block, d, [a + n for a, n in zip(past, rows)])
    q = queries(b.rs, sum(rows), kv * group * d)
    for window, sinks in ((1, 0), (1, 1), (7, 4), (64, 4), (100, 0), (130, 70), (300, 513), (1299, 1), (5000, 3), (1 << 48, 1 << 48)):
        check(b, q, rows, group, window, sinks)


@pytest.mark.parametrize("fmt,kv,group,block,d", SHAPES)
def test_prefill(backend, fmt, kv, group, block, d):
    """Chunks of many rows, of several sequences, with rows of decode among them."""
    rows = [150, 1, 67, 0, 20]
    past = [0, 300, 211, 5, 1]
    b = Batch(backend, 5 * d + group, fmt, kv, block, d, [a + n for a, n in zip(past, rows)])
    q = queries(b.rs, sum(rows), kv * group * d)
    check(b, q, rows, group)
    check(b, q, rows, group, 90, 4)
    check(b, q, rows, group, 17, 0, max_rows=150, max_len=301)


@pytest.mark.parametrize("fmt,d,group,rows,past", [("q8", 256, 6, 1, 20000), ("fp8", 128, 4, 5, 33333), ("q8", 64, 4, 2, 9000), ("fp8", 256, 1, 16, 8191), ("q8", 128, 8, 9, 12345)])
def test_long(backend, fmt, d, group, rows, past):
    """Positions in parts, of one sequence and beside a short one."""
    kv = 2
    b = Batch(backend, d + rows, fmt, kv, 32, d, [past + rows, 40 + rows])
    q = queries(b.rs, 2 * rows, kv * group * d)
    check(b, q, [rows, rows], group)
    check(b, q, [rows, rows], group, 4096, 100)


@pytest.mark.parametrize("fmt,d,kv,group,most_rows,sequences,most", [("q8", 64, 2, 4, 1, 70, 2600), ("fp8", 128, 4, 4, 5, 66, 3000), ("q8", 256, 2, 6, 2, 70, 2600),
                                                                     ("fp8", 80, 1, 16, 1, 90, 3500)])
def test_many_sequences_of_all_lengths(backend, fmt, d, kv, group, most_rows, sequences, most):
    """More tiles than the chip takes at once, of sequences of one position to many, some without rows, one that does not hold."""
    rs = np.random.RandomState(sequences)
    rows = rs.randint(0, most_rows + 1, sequences) if most_rows > 1 else (rs.rand(sequences) < 0.9).astype(int)
    lens = np.maximum(rs.randint(1, most, sequences), rows)
    lens[3], lens[4], lens[-1], rows[3], rows[-1] = rows[4] or 1, most, most, most_rows, most_rows
    rows[7], lens[7] = most_rows, most_rows - 1             # more rows than positions
    b = Batch(backend, 59, fmt, kv, 32, d, [int(n) for n in np.maximum(lens, 1)])
    b.lens[7] = most_rows - 1
    b.upload()
    q = queries(b.rs, int(rows.sum()), kv * group * d)
    holds = [s for s in range(sequences) if rows[s] <= b.lens[s]]
    assert 7 not in holds
    for window, sinks in ((0, 0), (2200, 70)):
        got = check(b, q, [int(n) for n in rows], group, window, sinks, only=holds, max_rows=most_rows)
        at = int(rows[:7].sum())
        assert np.all(got[at:at + rows[7]] == 7.0)


@pytest.mark.parametrize("fmt,sequences,most", [("q8", 4096, 40), ("fp8", 257, 300), ("q8", 256, 70), ("fp8", 129, 4000)])
def test_the_most_sequences(backend, fmt, sequences, most):
    """Up to as many sequences as a call takes, with rows and without, written, read and attended."""
    kv, group, d, block = 1, 2, 16, 16
    rs = np.random.RandomState(sequences + most)
    rows = (rs.rand(sequences) < 0.7).astype(int)
    rows[[0, -1]] = 0, 1
    b = Batch(backend, 61, fmt, kv, block, d, [int(n) for n in rs.randint(1, most, sequences)])
    m = int(rows.sum())
    k, v = queries(b.rs, m, kv * d), queries(b.rs, m, kv * d)
    want = b.want_write([int(n) for n in rows], k, v)
    b.write([int(n) for n in rows], k, v)
    b.same_as(want)
    b.pool = want
    check(b, queries(b.rs, m, kv * group * d), [int(n) for n in rows], group, max_rows=1)
    got = b.read(np.concatenate([[0], np.cumsum(rows)]), m)
    wanted = [want.rows(b.table[s], np.array([int(b.lens[s]) - 1])) for s in range(sequences) if rows[s]]
    for g, w in zip(got, zip(*wanted)):
        assert np.array_equal(g, np.concatenate([x.reshape(1, -1) for x in w]))


def test_rows_behind_the_last_and_what_does_not_hold(backend):
    """Rows of no sequence stay as they were; so do those of sequences that do not hold, or exceed what the launch was made for."""
    kv, group, d, block = 2, 3, 64, 16
    rows = [2, 3, 40, 4, 5]
    b = Batch(backend, 41, "q8", kv, block, d, [50, 3, 100, 2, 400])      # 3: four rows of two positions
    q = queries(b.rs, sum(rows) + 7, kv * group * d)
    starts = np.concatenate([[0], np.cumsum(rows)])
    got = attend(b, q, starts, kv * group)
    check(b, q, rows, group, got=got, only=(0, 1, 2, 4))
    assert np.all(got[45:49] == 7.0) and np.all(got[54:] == 7.0)
    got = attend(b, q, starts, kv * group, max_rows=5)
    check(b, q, rows, group, got=got, only=(0, 1, 4))
    assert np.all(got[5:49] == 7.0) and np.all(got[54:] == 7.0)
    got = attend(b, q, starts, kv * group, max_len=100)
    check(b, q, rows, group, got=got, only=(0, 1, 2))
    assert np.all(got[45:] == 7.0)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("rows", [1, 30])
def test_unknown_pages(backend, window, sinks, rows):
    """Positions of unknown pages are not seen; a row that sees none becomes zeros."""
    kv, group, d, block = 1, 4, 64, 16
    b = Batch(backend, 43, "q8", kv, block, d, [200, 190, 64])
    b.table[0, [0, 3, 7]] = [b.pool.pages, 0xFFFFFFFF, 0x80000000]
    b.table[1, :] = b.pool.pages + 5
    b.upload()
    q = queries(b.rs, 3 * rows, kv * group * d)
    got = check(b, q, [rows] * 3, group, window, sinks)
    assert np.all(got[rows:2 * rows] == 0.0)


@pytest.mark.parametrize("rows,past,d", [(1, 160, 64), (1, 5000, 128), (5, 900, 256), (40, 200, 96)])
def test_unknown_pages_beside_codes_of_nan(backend, rows, past, d):
    """What is walked in place of an unknown page is no page of the pool: there may be anything in those that no table names."""
    kv, group, block = 2, 4, 16
    b = Batch(backend, 44, "fp8", kv, block, d, [past + rows, 70 + rows])
    unused = np.setdiff1d(np.arange(b.pool.pages), np.concatenate([b.table[s, :-(-int(n) // block)] for s, n in enumerate(b.lens)]))
    assert len(unused)
    b.table[b.table == 0], b.pool.kp[0], b.pool.vp[0] = unused[0], 0x7F, 0xFF
    b.table[0, [0, 3, -(-past // block) - 1]] = [b.pool.pages, 0xFFFFFFFF, 0x80000000]
    b.table[1, 2] = b.pool.pages + 5
    b.upload()
    check(b, queries(b.rs, 2 * rows, kv * group * d), [rows] * 2, group)


@pytest.mark.parametrize("rows", [1, 4, 40])
def test_not_finite_where_hidden(backend, rows):
    """Pages that are NaN, where no row sees them, or some: others' results are as if they were zeros."""
    kv, group, d, block, n = 2, 4, 64, 16, 300
    b = Batch(backend, 47, "q8", kv, block, d, [n])
    hidden = b.table[0, [3, 4]]                         # positions 48 .. 79
    b.pool.ks[hidden[0], 0], b.pool.vs[hidden[1], 1] = np.nan, np.nan
    b.upload()
    q = queries(b.rs, rows, kv * group * d)
    check(b, q, [rows], group, 100, 4)                  # (the rows' windows begin behind position 80)
    heads = kv * group
    got = attend(b, q, [0, rows], heads)                # all see them
    assert np.isnan(got).all()
    # rows around the NaN: only those at or behind it are NaN
    b.lens = np.array([64], np.uint32)
    b.dev_lens = backend.Upload(b.lens)
    got = attend(b, q, [0, rows], heads)
    at = 64 - rows + np.arange(rows)
    assert np.isnan(got[at >= 48][:, :group]).all() and np.isfinite(got[:, group:]).all() and np.isfinite(got[at < 48]).all()


def test_queries_not_finite(backend):
    kv, group, d = 1, 4, 64
    b = Batch(backend, 53, "fp8", kv, 16, d, [500])
    q = queries(b.rs, 9, kv * group * d)
    q[2, 5], q[4, 70] = np.nan, np.inf
    got = attend(b, q, [0, 9], kv * group)
    bad = np.zeros((9, group), bool)
    bad[2, 0] = bad[4, 1] = True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
@pytest.mark.parametrize("rows", [1, 40])
def test_scales_far_apart(backend, fmt, rows):
    """Pages whose values' scales lie 2^40 apart, the large ones hardly weighed; queries of all sizes; zeros."""
    kv, group, d, block, n = 1, 4, 64, 16, 260
    b = Batch(backend, 59, fmt, kv, block, d, [n])
    b.pool.vs[b.table[0, 3], 0] *= np.float32(2.0 ** 20)
    b.pool.vs[b.table[0, 5], 0] *= np.float32(2.0 ** -20)
    b.pool.vs[b.table[0, 9], 0] = 0.0
    b.pool.ks[b.table[0, 2], 0] *= np.float32(30.0)
    b.pool.ks[b.table[0, 7], 0] = 0.0
    b.upload()
    q = queries(b.rs, rows, kv * group * d)
    q[0] *= 1e-20
    q[-1, :32] *= 20.0
    q[rows // 2, 64:128] = 0.0
    check(b, q, [rows], group)


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
def test_one_key_far_above(backend, fmt):
    """The last position's weight is all but everything, or next to nothing."""
    kv, group, d, n = 1, 2, 128, 700
    b = Batch(backend, 61, fmt, kv, 16, d, [n])
    page, at = b.table[0, (n - 1) // 16], (n - 1) % 16
    for sign in (1.0, -1.0):
        q = queries(b.rs, 1, group * d)
        b.pool.kp[page, 0, at] = ref.encode(fmt, (sign * np.sign(q[0, :d]) * 120).astype(np.float32))
        b.upload()
        check(b, q, [1], group)


def test_many_sequences(backend):
    """More sequences than lanes, and rows of no or any number."""
    rs = np.random.RandomState(67)
    lens = rs.randint(1, 90, 200)
    rows = [int(rs.randint(1, min(n, 6) + 1)) if rs.rand() < 0.6 else 0 for n in lens]
    b = Batch(backend, 71, "fp8", 2, 16, 64, lens)
    check(b, queries(b.rs, sum(rows), 2 * 3 * 64), rows, 3)


def test_pages_past_four_gigabytes(backend):
    """Page numbers whose bytes lie past 2^32 and 2^33."""
    kv, d, block, group = 4, 256, 128, 4
    pages = (5 << 30) // (kv * d * block)
    dev = torch.device("cuda:0")
    pool = [torch.zeros(pages, kv, block * d, dtype=torch.uint8, device=dev) for _ in range(2)] + [torch.zeros(pages, kv, device=dev) for _ in range(2)]
    small = Batch(backend, 73, "q8", kv, block, d, [300, 140])
    host = small.pool
    place = np.array([pages - 1, 1 + (1 << 32) // (kv * d * block), 5, pages - 2, (1 << 31) // (kv * d * block), 7, 9, 11])[:host.pages]
    assert len(set(place)) == host.pages
    for t, x in zip(pool, (host.kp, host.vp, host.ks, host.vs)):
        t[torch.from_numpy(place).to(dev)] = torch.from_numpy(x.reshape(host.pages, *t.shape[1:])).to(dev)
    torch.cuda.synchronize()
    wrap = lambda t: backend.WrapBuffer(t.data_ptr(), t.numel() * t.element_size())     # noqa: E731
    far = object.__new__(Batch)
    far.__dict__.update(small.__dict__)
    far.dev, far.dev_table = [wrap(t) for t in pool], backend.Upload(place[small.table % host.pages].astype(np.uint32))
    far.shape = [2, block, pages, small.width]
    q = queries(small.rs, 5, kv * group * d)
    near = attend(small, q, [0, 3, 5], kv * group)
    assert np.array_equal(attend(far, q, [0, 3, 5], kv * group), near)
    rows = [200, 9]
    k, v = (small.rs.randn(209, kv * d).astype(np.float32) * 9 for _ in range(2))
    for b in (small, far):
        b.write(rows, k, v)
    for x, y in zip(small.read([0, 300, 440], 440), far.read([0, 300, 440], 440)):
        assert np.array_equal(x, y)
    assert np.array_equal(attend(far, q, [0, 3, 5], kv * group), attend(small, q, [0, 3, 5], kv * group))

""""pages_write_q8", "pages_write_fp8", "pages_read_q8", "pages_read_fp8" against their plain statement: the same codes, scales and rows."""
import numpy as np
import pytest

import pages_reference as ref
from tessera_amd import KernelLaunch

pytestmark = pytest.mark.gpu

f32 = np.float32


class Batch:
    """A pool on the device and on the host, and the metadata of a batch in it."""

    def __init__(self, backend, seed, fmt, kv, block, d, lens, width=None, spare=3):
        self.backend, self.rs = backend, np.random.RandomState(seed)
        self.lens = np.asarray(lens, np.uint32)
        slots = [-(-int(n) // block) for n in lens]
        self.width = width or max(slots + [1]) + 1
        pages = sum(slots) + spare
        self.pool = ref.Pool(self.rs, fmt, pages, kv, block, d)
        order = self.rs.permutation(pages)
        self.table = self.rs.randint(0, pages, (len(lens), self.width)).astype(np.uint32)       # (past a sequence's pages anything)
        at = 0
        for s, n in enumerate(slots):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.shape = [len(lens), block, pages, self.width]
        self.upload()

    def upload(self):
        p, up = self.pool, self.backend.Upload
        self.dev = [up(x) for x in (p.kp, p.vp, p.ks, p.vs)]
        self.dev_table, self.dev_lens = up(self.table), up(self.lens)

    def go(self, name, buffers, scalars, **how):
        self.backend.LaunchKernel(self.backend.LoadKernel(name + "_" + self.pool.fmt), KernelLaunch(buffers=buffers, scalars=scalars), **how)

    def write(self, rows, k, v, starts=None, m=None, strides=(0, 0)):
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32) if starts is None else starts
        up = self.backend.Upload
        held = [up(np.ascontiguousarray(x)) for x in (k, v)] + [up(starts)]
        self.go("pages_write", [held[0], held[1], self.dev_table, held[2], self.dev_lens, *self.dev],
                [m or int(starts[-1]), self.pool.kv, self.pool.d, *self.shape, *strides])
        self.backend.Synchronize()

    def read(self, starts, m, f16=False, fill=7.0):
        wide = self.pool.kv * self.pool.d
        t = np.float16 if f16 else f32
        out = [self.backend.Upload(np.full((m, wide), fill, t)) for _ in range(2)]
        st = self.backend.Upload(np.asarray(starts, np.uint32))
        self.go("pages_read", [*self.dev, self.dev_table, st, self.dev_lens, *out], [m, self.pool.kv, self.pool.d, *self.shape, int(f16)])
        return [self.backend.CopyD2H(x, dtype=t).reshape(m, wide) for x in out]

    def device_pool(self):
        other = self.pool.copy()
        shapes = [x.shape for x in (other.kp, other.vp, other.ks, other.vs)]
        other.kp, other.vp, other.ks, other.vs = (self.backend.CopyD2H(b, dtype=t).reshape(s) for b, t, s in
                                                  zip(self.dev, (np.uint8, np.uint8, f32, f32), shapes))
        return other

    def same_as(self, want):
        got = self.device_pool()
        for name in ("kp", "vp"):
            assert np.array_equal(getattr(got, name), getattr(want, name)), name
        for name in ("ks", "vs"):
            a, b = getattr(got, name), getattr(want, name)
            assert np.array_equal(a.view(np.uint32)[~np.isnan(b)], b.view(np.uint32)[~np.isnan(b)]) and np.isnan(a[np.isnan(b)]).all(), name

    def want_write(self, rows, k, v):
        want, at = self.pool.copy(), 0
        kv, d = want.kv, want.d
        for s, n in enumerate(rows):
            if n:
                want.write(self.table[s], int(self.lens[s]), k[at:at + n].reshape(n, kv, d), v[at:at + n].reshape(n, kv, d))
            at += n
        return want


def numbers(rs, rows, wide, spread=1.0):
    return (rs.randn(rows, wide) * np.exp(rs.randn(rows, 1) * spread)).astype(f32)


SHAPES = [("q8", 1, 16, 16), ("q8", 2, 16, 64), ("fp8", 3, 32, 48), ("q8", 4, 64, 128), ("fp8", 1, 128, 256), ("q8", 1, 128, 80), ("fp8", 8, 16, 128), ("q8", 2, 32, 240)]


@pytest.mark.parametrize("fmt,kv,block,d", SHAPES)
def test_rows_into_pages_and_back(backend, fmt, kv, block, d):
    """Prompts and decoded rows that begin, end and cross anywhere in a page; what no row goes to stays as it was."""
    rows = [1, block, block - 1, 1, 2 * block + 3, 2, 1, block + 1, 0, 5]
    past = [0, 0, 1, block - 1, block + block // 2, 3 * block - 1, 2 * block, block - 1, 9, 200]
    lens = [a + b for a, b in zip(rows, past)]
    b = Batch(backend, d + block, fmt, kv, block, d, lens)
    m = sum(rows)
    k, v = numbers(b.rs, m, kv * d), numbers(b.rs, m, kv * d, 0.3)
    want = b.want_write(rows, k, v)
    b.write(rows, k, v)
    b.same_as(want)
    # back: the last positions of every sequence, older ones among them
    back = [min(n, block + 5) for n in lens]
    starts = np.concatenate([[0], np.cumsum(back)])
    for f16 in (False, True):
        got = b.read(starts, int(starts[-1]), f16)
        for s, n in enumerate(back):
            for g, w in zip(got, want.rows(b.table[s], np.arange(lens[s] - n, lens[s]))):
                w = w.reshape(n, -1)
                assert np.array_equal(g[starts[s]:starts[s + 1]], w.astype(np.float16) if f16 else w), (s, f16)


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
def test_token_by_token(backend, fmt):
    """Each token grows its page's scale or not; a number is off by half a step for itself and for every time that its page was
    quantized again, in steps of the last scale (an E4M3 step is at most 2^-3 of the number; its codes end in steps of 2^-9)."""
    kv, block, d, tokens = 2, 16, 64, 37
    b = Batch(backend, 5, fmt, kv, block, d, [tokens])
    x = [numbers(b.rs, tokens, kv * d, 0.7) for _ in range(2)]
    pool, grown = b.pool.copy(), np.zeros((2, tokens, kv))
    for n in range(1, tokens + 1):
        b.lens = np.array([n], np.uint32)
        b.dev_lens = b.backend.Upload(b.lens)
        b.write([1], x[0][n - 1:n], x[1][n - 1:n])
        page = int(b.table[0, (n - 1) // block])
        before = (pool.ks[page].copy(), pool.vs[page].copy())
        pool.write(b.table[0], n, x[0][n - 1:n].reshape(1, kv, d), x[1][n - 1:n].reshape(1, kv, d))
        first = (n - 1) // block * block
        for i, now in enumerate((pool.ks[page], pool.vs[page])):
            grown[i, first:n - 1] += now != before[i]
    b.same_as(pool)
    for i, rows in enumerate(pool.rows(b.table[0], np.arange(tokens))):
        page = b.table[0, np.arange(tokens) // block]
        step = (pool.ks if i == 0 else pool.vs)[page][:, :, None].astype(np.float64)
        true = x[i].reshape(tokens, kv, d).astype(np.float64)
        half = 0.5 if fmt == "q8" else np.maximum(np.abs(true) / step * 2.0 ** -4 * 1.2, 2.0 ** -10)
        # (1.2: a number that was rounded up by an eighth lies in the next, wider steps)
        assert (np.abs(rows - true) <= (1 + grown[i][:, :, None]) * half * step * (1 + 1e-5)).all()


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
def test_strides_and_rows_behind_the_last(backend, fmt):
    """A fused projection's rows; rows of the call behind the last sequence are no one's."""
    kv, block, d, rows = 2, 32, 96, [3, 0, 40, 1]
    b = Batch(backend, 11, fmt, kv, block, d, [9, 0, 64, 33])
    m, wide = sum(rows), kv * d
    fused = numbers(b.rs, m + 5, 3 * wide)
    k, v = fused[:, wide:2 * wide], fused[:, 2 * wide:]
    dev = backend.Upload(fused)
    want = b.want_write(rows, k[:m], v[:m])
    starts = backend.Upload(np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32))
    span = 4 * ((m + 4) * 3 * wide + wide)
    b.go("pages_write", [backend.WrapBuffer(dev.Handle() + 4 * wide, span), backend.WrapBuffer(dev.Handle() + 8 * wide, span), b.dev_table, starts, b.dev_lens, *b.dev],
         [m + 5, kv, d, *b.shape, 3 * wide, 3 * wide])
    backend.Synchronize()
    b.same_as(want)
    got = b.read(np.concatenate([[0], np.cumsum(rows)]), m + 5)
    for g in got:
        assert np.all(g[m:] == 7.0) and not np.any(np.all(g[:m] == 7.0, 1))


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
def test_what_does_not_hold_is_left_out(backend, fmt):
    """Unknown pages, rows that the call or the sequence has not, lengths past the table: nothing of them is written or read."""
    kv, block, d = 2, 16, 64
    b = Batch(backend, 13, fmt, kv, block, d, [20, 20, 20, 3, 20, 20], width=2)
    b.lens[5] = 40
    b.table[1, 1] = b.pool.pages                       # an unknown page: its positions are lost, the others not
    b.table[4, :] = 0xFFFFFFFF
    b.upload()
    starts = np.array([0, 6, 12, 10, 16, 22, 28], np.uint32)     # 2: its rows end before they begin; 3: six rows of three positions; 5: past the table
    k, v = numbers(b.rs, 28, kv * d), numbers(b.rs, 28, kv * d)
    want = b.pool.copy()
    for s, (first, end) in enumerate(zip(starts[:-1], starts[1:])):
        if s in (0, 1, 4):
            want.write(b.table[s], 20, k[first:end].reshape(-1, kv, d), v[first:end].reshape(-1, kv, d))
    b.write(None, k, v, starts)
    b.same_as(want)
    got = b.read(starts, 28)
    for i in range(2):
        for s in (0, 1, 4):
            assert np.array_equal(got[i][starts[s]:starts[s + 1]], want.rows(b.table[s], np.arange(20 - int(starts[s + 1] - starts[s]), 20))[i].reshape(-1, kv * d)), s
        assert np.all(got[i][12:16] == 7.0) and np.all(got[i][22:] == 7.0)
    # the last sequence's rows end past the call's: they are no one's, the others' are written again
    b.pool = want
    starts = np.array([0, 6, 12, 12, 12, 12, 29], np.uint32)
    want = want.copy()
    for s in (0, 1):
        want.write(b.table[s], 20, k[starts[s]:starts[s + 1]].reshape(-1, kv, d), v[starts[s]:starts[s + 1]].reshape(-1, kv, d))
    b.lens[5] = 20
    b.dev_lens = backend.Upload(b.lens)
    b.write(None, k, v, starts, m=28)
    b.same_as(want)


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
def test_zero_tiny_huge_and_not_finite(backend, fmt):
    """All zeros; numbers whose scale is subnormal; the largest; infinities and NaN, which make their page and head NaN until it is
    begun anew, and no other."""
    kv, block, d = 2, 16, 32
    rows = [4, 4, 4, 4, 4, 4, 4]
    b = Batch(backend, 17, fmt, kv, block, d, [20, 16, 4, 12, 9, 4, 19])
    m = sum(rows)
    k, v = numbers(b.rs, m, kv * d), numbers(b.rs, m, kv * d)
    k[0:4], v[0:4] = 0.0, 1e-42
    k[4:8], v[4:8] = 3e38, -3.4e38
    k[8:12], v[8:12] = 0.0, 0.0
    k[12, 5], v[13, d + 3] = np.inf, np.nan
    v[17, 0], k[18, d] = -np.inf, np.nan
    k[20:24], v[20:24] = 1e-44, 2e-45
    want = b.want_write(rows, k, v)
    b.write(rows, k, v)
    b.same_as(want)
    assert np.isnan(want.ks).sum() == 2 and np.isnan(want.vs).sum() == 2
    # more of the same pages: those that are NaN stay it, one that is begun anew does not
    b.pool = want
    used = {int(p) for s, n in enumerate(b.lens) for p in b.table[s, :-(-int(n) // block)]}
    b.table[1, 1] = [p for p in range(want.pages) if p not in used][0]      # (the second sequence's next page)
    b.dev_table = backend.Upload(b.table)
    b.lens = np.array([23, 19, 7, 15, 3, 7, 22], np.uint32)
    b.dev_lens = backend.Upload(b.lens)
    rows = [3] * 7
    k, v = numbers(b.rs, 21, kv * d), numbers(b.rs, 21, kv * d)
    after = b.want_write(rows, k, v)
    b.write(rows, k, v)
    b.same_as(after)
    assert np.isnan(after.ks).sum() == 1 and np.isnan(after.vs).sum() == 1


def test_every_e4m3_rounding(backend):
    """Numbers at, between and next to all E4M3 numbers, under a scale of 1 (the page's largest is 448)."""
    kv, block, d = 1, 16, 256
    mags = ref.E4M3[:127].astype(np.float64)
    mid = (mags[1:] + mags[:-1]) / 2
    probe = np.concatenate([mags, mid, np.nextafter(mid.astype(f32), f32(0)), np.nextafter(mid.astype(f32), f32(1e9)), [1e-30, 2.0 ** -11]]).astype(f32)
    x = np.zeros(4 * d, f32)
    x[:len(probe)] = probe
    x[4 * d - 1] = 448.0
    x = np.concatenate([x, -x]).reshape(8, d)
    b = Batch(backend, 19, "fp8", kv, block, d, [8])
    want = b.want_write([8], x, x)
    b.write([8], x, x)
    b.same_as(want)
    assert want.ks[b.table[0, 0], 0] == 1.0


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
def test_a_sequence_cut_short_goes_on(backend, fmt):
    """Drafted rows are refused: the next call has fewer positions, its rows replace them under a scale that knows them still."""
    kv, block, d = 2, 16, 64
    b = Batch(backend, 23, fmt, kv, block, d, [21])
    want = b.pool
    for length, rows in ((21, 5), (18, 1), (23, 6), (17, 1), (16, 3), (33, 17)):
        if length > 32:
            b.table[0, 2] = [p for p in range(b.pool.pages) if p not in b.table[0, :2]][0]
            b.dev_table = backend.Upload(b.table)
        b.pool = want
        b.lens = np.array([length], np.uint32)
        b.dev_lens = backend.Upload(b.lens)
        k, v = numbers(b.rs, rows, kv * d), numbers(b.rs, rows, kv * d)
        want = b.want_write([rows], k, v)
        b.write([rows], k, v)
        b.same_as(want)


def test_many_sequences(backend):
    """More sequences than a wavefront's lanes, many of them without rows."""
    kv, block, d = 1, 16, 64
    rs = np.random.RandomState(29)
    lens = rs.randint(1, 60, 300)
    rows = [int(rs.randint(1, n + 1)) if rs.rand() < 0.4 else 0 for n in lens]
    b = Batch(backend, 31, "q8", kv, block, d, lens)
    m = sum(rows)
    k, v = numbers(b.rs, m, d), numbers(b.rs, m, d)
    want = b.want_write(rows, k, v)
    b.write(rows, k, v)
    b.same_as(want)
    starts = np.concatenate([[0], np.cumsum(rows)])
    got = b.read(starts, m)
    for s, n in enumerate(rows):
        for i in range(2):
            assert np.array_equal(got[i][starts[s]:starts[s + 1]], want.rows(b.table[s], np.arange(lens[s] - n, lens[s]))[i].reshape(n, kv * d)), s

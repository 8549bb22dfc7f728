"""A tree of drafted tokens: its masks, its queries and keys, its attention and its tokens' log probabilities, each against
the plain 64-bit statements of tree_reference.py and a whole verification step through all of them."""
import numpy as np
import pytest

import tree_reference as ref
from tree_reference import EPS, ROOT
from test_gpu_attention import cache
from util import run

pytestmark = pytest.mark.gpu


def f32_bits(x):
    return int(np.float32(x).view(np.uint32))


# ---- tree_mask -----------------------------------------------------------------------------------

def tree_mask(backend, parents, base):
    n = len(parents)
    words = (n + 31) // 32
    mask, pos = backend.Upload(np.full(n * words + 8, 0xAAAAAAAA, np.uint32)), backend.Upload(np.full(n * 3 + 4, 77, np.uint64))
    run(backend, "tree_mask", [backend.Upload(np.asarray(parents, np.uint32)), mask, pos], [n, base])
    backend.Synchronize()
    got, where = backend.CopyD2H(mask, dtype=np.uint32), backend.CopyD2H(pos, dtype=np.uint64)
    assert np.all(got[n * words:] == 0xAAAAAAAA) and np.all(where[n * 3:] == 77)      # nothing past the rows
    return got[:n * words].reshape(n, words), where[:n * 3].reshape(n, 3)


def check_tree(backend, parents, base=0):
    seen = ref.seen_of(parents)
    mask, pos = tree_mask(backend, parents, base)
    assert np.array_equal(mask, ref.words_of(seen))
    assert np.array_equal(pos, ref.positions_of(seen, base))


@pytest.mark.parametrize("nodes", [1, 2, 16, 31, 32, 33, 63, 64, 65, 100, 257, 1000, 1024])
@pytest.mark.parametrize("reach", [0, 1, 7, 1000])
def test_tree_mask(backend, nodes, reach):
    """Chains (reach 0), bushes (every node may follow any earlier one), sizes around words and workgroups."""
    check_tree(backend, ref.random_parents(np.random.RandomState(nodes + reach), nodes, min(reach, nodes)), base=5000)


def test_tree_mask_roots_and_padding(backend):
    check_tree(backend, [ROOT] * 70)
    check_tree(backend, [0])                                   # its own parent: padding
    check_tree(backend, [ROOT, 5, 1, 0, 3, 4, 0xFFFFFFFE, 6])  # a later parent, its followers, one far out of range and its follower
    check_tree(backend, ref.random_parents(np.random.RandomState(3), 90, 9, padding=30), base=1 << 48)
    chain = np.arange(-1, 1023).astype(np.int64)
    chain[0], chain[500] = ROOT, 500                           # everything behind node 500 follows padding
    check_tree(backend, chain)


# ---- qk_norm_rope --------------------------------------------------------------------------------

ROPE = [
    # rows, heads, kv_heads, head_dim, rope_dim
    (1, 1, 1, 64, 64), (1, 24, 4, 256, 64), (3, 5, 1, 128, 128), (17, 16, 4, 64, 32), (33, 32, 8, 128, 64),
    (2, 3, 3, 80, 80), (2, 3, 1, 96, 48), (5, 4, 2, 72, 40), (1, 2, 1, 256, 256), (300, 6, 2, 256, 256),
    (2, 3, 1, 2, 2), (3, 2, 2, 34, 34), (2, 2, 1, 128, 100), (4, 2, 1, 250, 6),          # a wavefront a head
]


def qk_norm(backend, shape, axes, gated, f16, q_more=0, k_more=0, k_row=0, base=4000, theta=1e6, eps=1e-6, seed=0, gain=1.0):
    rows, heads, kv, d, rope_dim = shape
    rs = np.random.RandomState(seed + rows + d)
    wide = heads * d * (2 if gated else 1)
    q = (rs.randn(rows, wide + q_more) * gain).astype(np.float32)
    k = (rs.randn(rows, kv * d + k_more) * gain).astype(np.float32)
    wq, wk = rs.rand(d).astype(np.float32) + 0.5, rs.rand(d).astype(np.float32) + 0.5
    sections = (rope_dim // 2 - 2 * (rope_dim // 6), rope_dim // 6, rope_dim // 6) if axes else (rope_dim // 2, 0, 0)
    pos = base + rs.randint(0, 1000, (rows, 3)).astype(np.uint64) if axes else np.repeat(base + np.arange(rows)[:, None], 3, 1).astype(np.uint64)
    elem = np.float16 if f16 else np.float32
    dq_out = backend.Upload(np.full(rows * heads * d + 4, 7.0, np.float32))
    dk_out = backend.Upload(np.full((k_row + rows + 1) * kv * d, 7.0, elem))
    dgate = backend.Upload(np.full(rows * heads * d + 4, 7.0, np.float32))
    up = backend.Upload
    buffers = [up(q), up(k), up(wq), up(wk)] + ([up(pos)] if axes else []) + [dq_out, dk_out] + ([dgate] if gated else [])
    scalars = [rows, heads, kv, d, rope_dim] + ([] if axes else [base]) + [f32_bits(theta), f32_bits(eps), q.shape[1], k.shape[1], int(f16), k_row]
    run(backend, "qk_norm_mrope" if axes else "qk_norm_rope", buffers, scalars + (list(sections) if axes else []))
    backend.Synchronize()
    size = rows * heads * d
    got_q, got_gate = backend.CopyD2H(dq_out, dtype=np.float32), backend.CopyD2H(dgate, dtype=np.float32)
    got_k = backend.CopyD2H(dk_out, dtype=elem).reshape(-1, kv * d)
    assert np.all(got_q[size:] == 7.0) and np.all(got_k[:k_row] == 7.0) and np.all(got_k[k_row + rows:] == 7.0)
    fused = q[:, :wide].reshape(rows, heads, -1)
    eps32 = float(np.float32(eps))
    want, mags = ref.rotate(fused[..., :d], wq, pos, rope_dim, np.float32(theta), eps32, sections)
    assert np.all(np.abs(got_q[:size].reshape(want.shape) - want) <= ref.ROTATE_ROUNDINGS * EPS * mags)
    want, mags = ref.rotate(k[:, :kv * d].reshape(rows, kv, d), wk, pos, rope_dim, np.float32(theta), eps32, sections)
    bound = ref.ROTATE_ROUNDINGS * EPS * mags + (2.0 ** -11 * np.abs(want) * 1.001 + 2.0 ** -25 if f16 else 0.0)   # (rounds to fp16 once)
    assert np.all(np.abs(got_k[k_row:k_row + rows].reshape(want.shape).astype(np.float64) - want) <= bound)
    if gated:
        assert np.array_equal(got_gate[:size].reshape(rows, heads, d), fused[..., d:])
    assert np.all(got_gate[size if gated else 0:] == 7.0)


@pytest.mark.parametrize("shape", ROPE)
@pytest.mark.parametrize("axes", [False, True])
def test_qk_norm_rope(backend, shape, axes):
    qk_norm(backend, shape, axes, gated=False, f16=False)
    qk_norm(backend, shape, axes, gated=True, f16=True, k_row=3)


@pytest.mark.parametrize("more", [(8, 4), (3, 5), (4, 1)])
def test_qk_norm_rope_strides(backend, more):
    """Rows of a fused projection, also ones that no vector load fits."""
    for shape in [(5, 4, 2, 64, 64), (9, 3, 1, 256, 32)]:
        qk_norm(backend, shape, False, gated=False, f16=True, q_more=more[0], k_more=more[1], k_row=1)
        qk_norm(backend, shape, True, gated=True, f16=False, q_more=more[0], k_more=more[1])


@pytest.mark.parametrize("base", [0, 1, (1 << 20) + 3, (1 << 31) + 1, 1 << 40])
def test_qk_norm_rope_far_positions(backend, base):
    qk_norm(backend, (4, 2, 1, 128, 128), False, gated=False, f16=False, base=base)
    qk_norm(backend, (4, 2, 1, 34, 34), True, gated=False, f16=False, base=base, theta=10000.0)


@pytest.mark.parametrize("dim", [128, 34])
def test_qk_norm_mrope_positions_past_2_to_50(backend, dim):
    """They count as 2^50: bounded results whatever the positions' buffer holds."""
    rows, heads, kv = 6, 2, 1
    rs = np.random.RandomState(dim)
    up = backend.Upload
    q, k, w = up(rs.randn(rows, heads * dim).astype(np.float32)), up(rs.randn(rows, kv * dim).astype(np.float32)), up(np.ones(dim, np.float32))
    outs = []
    for far in ([1 << 50] * 3, [(1 << 50) + 1, 1 << 63, (1 << 64) - 1]):
        out = [backend.AllocateBuffer(rows * n * dim * 4) for n in (heads, kv)]
        pos = up(np.array([far] * rows, np.uint64))
        run(backend, "qk_norm_mrope", [q, k, w, w, pos, *out], [rows, heads, kv, dim, dim, f32_bits(1e6), f32_bits(1e-6), 0, 0, 0, 0, dim // 2 - 10, 5, 5])
        backend.Synchronize()
        outs.append([backend.CopyD2H(x, dtype=np.float32) for x in out])
    assert all(np.array_equal(x, y) for x, y in zip(*outs))


@pytest.mark.parametrize("gain", [0.0, 1e-12, 1e12])
def test_qk_norm_rope_magnitudes(backend, gain):
    qk_norm(backend, (3, 4, 2, 128, 64), False, gated=False, f16=False, gain=gain, eps=1e-5)


def test_qk_norm_rope_in_place(backend):
    rows, heads, kv, d = 21, 6, 2, 128
    rs = np.random.RandomState(5)
    q, k = rs.randn(rows, heads * d).astype(np.float32), rs.randn(rows, kv * d).astype(np.float32)
    w = backend.Upload(np.ones(d, np.float32))
    outs = []
    for same in (False, True):
        dq, dk = backend.Upload(q), backend.Upload(k)
        oq, ok = (dq, dk) if same else (backend.AllocateBuffer(q.nbytes), backend.AllocateBuffer(k.nbytes))
        run(backend, "qk_norm_rope", [dq, dk, w, w, oq, ok], [rows, heads, kv, d, 64, 9, f32_bits(1e4), f32_bits(1e-6), 0, 0, 0, 0])
        backend.Synchronize()
        outs.append((backend.CopyD2H(oq, dtype=np.float32), backend.CopyD2H(ok, dtype=np.float32)))
    assert np.array_equal(outs[0][0], outs[1][0]) and np.array_equal(outs[0][1], outs[1][1])


# ---- attention_tree ------------------------------------------------------------------------------

def elements(kind, codes, scale, width):
    if kind in ("f32", "f16"):
        return np.asarray(codes, np.float64).reshape(-1, width)
    if kind == "q8":
        x = np.asarray(codes).view(np.int8).reshape(-1, width).astype(np.float64)
    elif kind == "q4":
        b = np.asarray(codes).view(np.uint8).reshape(-1, width // 2)
        x = np.stack([b & 15, b >> 4], 2).reshape(-1, width).astype(np.float64)
        x = np.where(x > 7, x - 16, x)
    else:
        c = np.asarray(codes).view(np.uint8).reshape(-1, width).astype(np.int64)
        e, f = (c >> 3) & 15, c & 7
        x = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
        x = np.where((c & 127) == 127, np.nan, x) * np.where(c >> 7, -1.0, 1.0)
    return x * np.asarray(scale, np.float64).reshape(-1, 1)


def attend_tree(backend, kind, q, k, v, ks, vs, words, tree, m, n, heads, kv_heads, head_dim, window, no_alloc=False):
    dout = backend.Upload(np.full(m * heads * head_dim + 4, 7.0, np.float32))
    scales = [] if ks is None else [backend.Upload(ks), backend.Upload(vs)]
    scalars = [m, n, heads, kv_heads, head_dim, tree, window] + ([int(kind == "f16")] if ks is None else [])
    run(backend, "attention_tree" if ks is None else "attention_tree_" + kind,
        [backend.Upload(q), backend.Upload(k), backend.Upload(v), *scales, backend.Upload(words), dout], scalars)
    backend.Synchronize()
    got = backend.CopyD2H(dout, dtype=np.float32)
    assert np.all(got[m * heads * head_dim:] == 7.0)
    return got[:m * heads * head_dim].reshape(m, heads * head_dim)


def check_attention(backend, kind, m, n, heads, kv_heads, head_dim, tree, window, seen=None, seed=0, spoil=False):
    rs = np.random.RandomState(seed + n + head_dim)
    g = np.random.default_rng(seed + n * 3 + head_dim)
    width = kv_heads * head_dim
    q = rs.randn(m, heads * head_dim).astype(np.float32)
    k, ks = cache(g, kind, n, width)
    v, vs = cache(g, kind, n, width)
    if seen is None:
        seen = rs.rand(m, tree) < 0.5
    see = ref.visible(seen, n - tree, window)
    if spoil:       # what no row sees may hold anything
        hidden = ~see.any(0)
        assert hidden.any()
        if ks is None:
            k[hidden], v[hidden] = np.nan, np.inf
        else:
            ks, vs = np.where(hidden, np.float32(np.nan), ks), np.where(hidden, np.float32(np.inf), vs)
            if kind == "fp8":
                k, v = (np.where(hidden[:, None], np.uint8(0x7F), x.reshape(n, width)) for x in (k, v))
    words = ref.words_of(seen)
    if tree % 32:   # bits past the tree say nothing
        words[:, -1] |= np.uint32(0xFFFFFFFF << (tree % 32) & 0xFFFFFFFF)
    ke, ve = (np.where(see.any(0)[:, None], elements(kind, x, s, width), 0.0) for x, s in ((k, ks), (v, vs)))
    want = ref.attention(q, ke, ve, see, heads, kv_heads, head_dim)
    got = attend_tree(backend, kind, q, k, v, ks, vs, words, tree, m, n, heads, kv_heads, head_dim, window)
    bound = ref.attention_bound(q, ke, ve, see, heads, kv_heads, head_dim)
    err = np.max(np.abs(got - want))
    assert err <= bound, (err, bound)
    assert np.all(got[~see.any(1)] == 0.0)
    return got


ATTEND = [
    # m, n, heads, kv_heads, head_dim, tree, window
    (1, 1, 1, 1, 64, 1, 0),
    (2, 2, 2, 1, 64, 2, 0),
    (5, 37, 4, 4, 64, 5, 0),
    (7, 64, 8, 1, 128, 7, 0),
    (16, 129, 9, 1, 128, 16, 0),
    (16, 577, 24, 4, 256, 16, 0),
    (33, 300, 16, 4, 64, 33, 0),
    (64, 700, 6, 2, 256, 64, 0),
    (64, 64, 6, 2, 128, 64, 0),              # nothing before the tree
    (3, 517, 8, 2, 96, 70, 0),               # more of the cache under masks than rows
    (70, 1100, 4, 2, 128, 70, 0),
    (12, 400, 6, 2, 80, 12, 0),
    (12, 400, 4, 2, 160, 12, 0),
    (5, 90, 2, 1, 16, 5, 0),
    (6, 150, 8, 4, 34, 6, 0),                # no kind's runs
    (20, 333, 17, 1, 64, 20, 0),
    (9, 2100, 24, 4, 256, 9, 0),
    (9, 300, 6, 2, 128, 9, 250),             # windows: into the prefix, across it, within the tree
    (9, 300, 6, 2, 256, 9, 12),
    (40, 300, 4, 2, 64, 40, 3),
    (40, 300, 8, 4, 34, 40, 25),
    (33, 900, 8, 2, 128, 33, 1),
    (33, 900, 8, 2, 128, 33, 5000),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "q8", "q4", "fp8"])
@pytest.mark.parametrize("case", ATTEND)
def test_attention_tree(backend, kind, case):
    """Random bits, so that rows see nodes in no order, some of them none."""
    check_attention(backend, kind, *case)


@pytest.mark.parametrize("kind", ["f32", "f16", "q8", "fp8"])
@pytest.mark.parametrize("case", [(5, 3001, 4, 2, 128, 2500, 700), (40, 3001, 8, 2, 256, 2100, 0), (40, 2600, 8, 2, 64, 2600, 900), (3, 2600, 8, 4, 34, 1500, 40)])
def test_attention_tree_of_many_words(backend, kind, case):
    """More keys under masks than "tree_mask" writes, windows that begin between them."""
    check_attention(backend, kind, *case)


@pytest.mark.parametrize("kind", ["f32", "f16", "q8", "q4", "fp8"])
@pytest.mark.parametrize("case", [(3, 900, 4, 2, 128, 900, 0), (40, 900, 12, 2, 64, 900, 30), (33, 70, 6, 2, 256, 70, 0), (3, 900, 8, 4, 34, 900, 5), (1, 1, 8, 4, 34, 1, 0)])
@pytest.mark.parametrize("which", ["none", "one", "last"])
def test_attention_tree_of_rows_that_see_nothing(backend, kind, case, which):
    """No row sees a key, one row does, the last key alone is seen: whatever else the cache holds."""
    m, n = case[:2]
    seen = np.zeros((m, n), bool)
    if which == "one":
        seen[m // 2, n // 3:n // 3 + 5] = True
    elif which == "last":
        seen[:, n - 1] = True
    check_attention(backend, kind, *case, seen=seen, spoil=n > 1)


@pytest.mark.parametrize("kind", ["f32", "f16", "q8", "q4", "fp8"])
@pytest.mark.parametrize("case", [c for c in ATTEND if c[0] == c[5]])
def test_attention_tree_of_drafts(backend, kind, case):
    m = case[0]
    seen = ref.seen_of(ref.random_parents(np.random.RandomState(m), m, 5, padding=min(2, m - 1)))
    check_attention(backend, kind, *case, seen=seen, seed=1)


@pytest.mark.parametrize("kind", ["f32", "f16", "q8", "q4", "fp8"])
@pytest.mark.parametrize("case", [(5, 40, 6, 2, 64, 20, 0), (17, 600, 24, 4, 256, 40, 0), (33, 300, 8, 2, 128, 64, 100), (20, 130, 8, 4, 34, 20, 0)])
def test_attention_tree_hidden_keys_may_hold_anything(backend, kind, case):
    m, tree = case[0], case[5]
    rs = np.random.RandomState(tree)
    seen = rs.rand(m, tree) < 0.4
    seen[:, rs.rand(tree) < 0.5] = False
    seen[:, 0], seen[:, tree - 1] = True, False
    check_attention(backend, kind, *case, seen=seen, spoil=True)


@pytest.mark.parametrize("kind", ["f32", "f16", "q8", "q4", "fp8"])
@pytest.mark.parametrize("head_dim", [64, 128, 256, 34])
def test_attention_tree_spoiled_for_others(backend, kind, head_dim):
    """A key that is not finite reaches the rows that see it and no other."""
    m, n, heads, kv_heads = 18, 150, 8, 4
    rs, g = np.random.RandomState(1), np.random.default_rng(head_dim)
    width = kv_heads * head_dim
    q = rs.randn(m, heads * head_dim).astype(np.float32)
    k, ks = cache(g, kind, n, width)
    v, vs = cache(g, kind, n, width)
    seen = np.ones((m, m), bool)
    seen[::2, 4] = False
    if ks is None:
        v = v.copy()
        v[n - m + 4] = np.nan
    else:
        vs = vs.copy()
        vs[n - m + 4] = np.nan
    got = attend_tree(backend, kind, q, k, v, ks, vs, ref.words_of(seen), m, m, n, heads, kv_heads, head_dim, 0)
    assert np.all(np.isnan(got[1::2]))
    see = ref.visible(seen, n - m, 0)[::2]
    ke, ve = (np.where(np.arange(n)[:, None] == n - m + 4, 0.0, elements(kind, x, s, width)) for x, s in ((k, ks), (v, vs)))
    want = ref.attention(q[::2], ke, ve, see, heads, kv_heads, head_dim)
    assert np.max(np.abs(got[::2] - want)) <= ref.attention_bound(q[::2], ke, ve, see, heads, kv_heads, head_dim)


@pytest.mark.parametrize("kind,what", [("f32", np.inf), ("f32", -np.inf), ("f32", np.nan), ("f16", np.inf), ("f16", -np.inf), ("f16", np.nan), ("q8", np.nan), ("q4", np.nan), ("fp8", np.nan)])
@pytest.mark.parametrize("case", [(18, 150, 8, 4, 64), (18, 1500, 8, 4, 128), (40, 1500, 24, 4, 256), (5, 150, 8, 4, 34), (2, 90, 4, 2, 256)])
def test_attention_tree_of_a_key_not_finite(backend, kind, what, case):
    """One element of a key (a quantized one's scale): the rows that see it become what the formula makes of them, no other."""
    m, n, heads, kv_heads, head_dim = case
    rs, g = np.random.RandomState(2), np.random.default_rng(head_dim)
    width, at = kv_heads * head_dim, n - m + 1
    q = rs.randn(m, heads * head_dim).astype(np.float32)
    k, ks = cache(g, kind, n, width)
    v, vs = cache(g, kind, n, width)
    seen = np.ones((m, m), bool)
    seen[::2, 1] = False
    if ks is None:
        k = k.copy().reshape(n, width)
        k[at, 3::head_dim] = what
    else:
        ks = ks.copy()
        ks[at] = what
    got = attend_tree(backend, kind, q, k, v, ks, vs, ref.words_of(seen), m, m, n, heads, kv_heads, head_dim, 0)
    see = ref.visible(seen, n - m, 0)
    ke, ve = elements(kind, k, ks, width).astype(np.float64), elements(kind, v, vs, width)
    want = np.zeros((m, heads, head_dim))
    with np.errstate(invalid="ignore"):
        for i in range(m):
            for h in range(heads):
                on = slice(h // (heads // kv_heads) * head_dim, (h // (heads // kv_heads) + 1) * head_dim)
                x = ke[see[i], on] @ q[i, h * head_dim:(h + 1) * head_dim].astype(np.float64) / np.sqrt(head_dim)
                w = np.exp(x - x.max())
                want[i, h] = w @ ve[see[i], on] / w.sum()
    want = want.reshape(m, -1)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(want).any() and not np.isnan(want).all()
    finite = np.where(np.isfinite(ke), ke, 0.0)
    bound = ref.attention_bound(q, finite, ve, see, heads, kv_heads, head_dim)
    assert np.nanmax(np.abs(got - want)) <= bound


@pytest.mark.parametrize("case", [(1, 700, 4, 4, 64), (40, 2000, 8, 2, 64), (40, 2000, 8, 2, 128), (40, 2000, 6, 1, 256), (40, 1500, 4, 2, 72)])
def test_attention_tree_f32_of_many_magnitudes(backend, case):
    """Keys and values from 2^-115 to 2^100, elements of one key apart by 2^30, some below the least normal number, some keys 0."""
    m, n, heads, kv_heads, head_dim = case
    rs = np.random.RandomState(n + head_dim)
    width = kv_heads * head_dim
    scale = lambda low, high: np.exp2(rs.randint(low, high, (n, kv_heads, 1)).astype(np.float64))
    q = (rs.randn(m, heads * head_dim) * 2.0 ** 50).astype(np.float32)
    k = (rs.randn(n, kv_heads, head_dim) * scale(-115, -49) * np.exp2(-rs.randint(0, 31, (1, 1, head_dim)))).reshape(n, width).astype(np.float32)
    v = (rs.randn(n, kv_heads, head_dim) * scale(-115, 100) * np.exp2(-rs.randint(0, 31, (n, 1, head_dim)))).reshape(n, width).astype(np.float32)
    k[::50], v[25::50], k[7] = 0.0, 0.0, np.float32(3e-42)
    seen = rs.rand(m, m) < 0.5
    see = ref.visible(seen, n - m, 0)
    got = attend_tree(backend, "f32", q, k, v, None, None, ref.words_of(seen), m, m, n, heads, kv_heads, head_dim, 0)
    want = ref.attention(q, k, v, see, heads, kv_heads, head_dim)
    assert np.max(np.abs(got - want)) <= ref.attention_bound(q, k, v, see, heads, kv_heads, head_dim)


@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_attention_tree_past_4_gib(backend, kind):
    """A window at the end of a cache of more than 2^32 bytes, which is keys and values in one."""
    heads, kv_heads, head_dim, window = 16, 8, 256, 500
    width, elem = kv_heads * head_dim, np.float16 if kind == "f16" else np.float32
    n = (1 << 32) // (width * elem().itemsize) + 5000
    rs = np.random.RandomState(3)
    rows = rs.randn(997, width).astype(elem)                 # row j of the cache: row j % 997 of these
    kv = backend.Upload(np.take(rows, np.arange(n) % 997, axis=0))
    tail = rows[np.arange(n - 1000, n) % 997]
    for m in (1, 40):
        q = rs.randn(m, heads * head_dim).astype(np.float32)
        seen = np.tril(np.ones((m, m), bool))
        out = backend.AllocateBuffer(q.nbytes)
        run(backend, "attention_tree", [backend.Upload(q), kv, kv, backend.Upload(ref.words_of(seen)), out],
            [m, n, heads, kv_heads, head_dim, m, window, int(kind == "f16")])
        backend.Synchronize()
        see = ref.visible(seen, 1000 - m, window)
        want = ref.attention(q, tail, tail, see, heads, kv_heads, head_dim)
        got = backend.CopyD2H(out, dtype=np.float32).reshape(want.shape)
        assert np.max(np.abs(got - want)) <= ref.attention_bound(q, tail, tail, see, heads, kv_heads, head_dim)


@pytest.mark.parametrize("kind", ["f16", "q8"])
@pytest.mark.parametrize("m", [1, 8, 40])
def test_attention_tree_of_a_chain_is_causal_attention(backend, kind, m):
    """A chain's rows see what causal rows see."""
    from test_gpu_attention import attend
    n, heads, kv_heads, head_dim, window = 700, 12, 2, 128, 300
    g = np.random.default_rng(m)
    q = g.standard_normal((m, heads * head_dim)).astype(np.float32)
    k, ks = cache(g, kind, n, kv_heads * head_dim)
    v, vs = cache(g, kind, n, kv_heads * head_dim)
    for w in (0, window):
        got = attend_tree(backend, kind, q, k, v, ks, vs, ref.words_of(np.tril(np.ones((m, m), bool))), m, m, n, heads, kv_heads, head_dim, w)
        want = attend(backend, kind, q, k, v, ks, vs, m, n, heads, kv_heads, head_dim, n - m, w)
        ke, ve = elements(kind, k, ks, kv_heads * head_dim), elements(kind, v, vs, kv_heads * head_dim)
        see = ref.visible(np.tril(np.ones((m, m), bool)), n - m, w)
        assert np.max(np.abs(got - want)) <= 2 * ref.attention_bound(q, ke, ve, see, heads, kv_heads, head_dim)


# ---- token_logprobs ------------------------------------------------------------------------------

def token_logprobs(backend, x, tokens, top_k, row_base=0, no_alloc=False):
    rows, count = tokens.shape
    vocab = x.shape[1]
    up = backend.Upload
    outs = [up(np.full(rows * count + 4, 7.0, np.float32)), up(np.full(rows + 4, 7.0, np.float32))]
    if top_k:
        outs += [up(np.full(rows * top_k + 4, 7, np.uint32)), up(np.full(rows * top_k + 4, 7.0, np.float32))]
    run(backend, "token_logprobs", [up(x), up(tokens.astype(np.uint32)), *outs], [rows, vocab, count, top_k, row_base])
    backend.Synchronize()
    logp, entropy = backend.CopyD2H(outs[0], dtype=np.float32), backend.CopyD2H(outs[1], dtype=np.float32)
    assert np.all(logp[rows * count:] == 7.0) and np.all(entropy[rows:] == 7.0)
    got = {"logprobs": logp[:rows * count].reshape(rows, count), "entropy": entropy[:rows]}
    if top_k:
        ids, vals = backend.CopyD2H(outs[2], dtype=np.uint32), backend.CopyD2H(outs[3], dtype=np.float32)
        assert np.all(ids[rows * top_k:] == 7) and np.all(vals[rows * top_k:] == 7.0)
        got.update(top=ids[:rows * top_k].reshape(rows, top_k), top_logprobs=vals[:rows * top_k].reshape(rows, top_k))
    return got


def check_logprobs(backend, x, tokens, top_k, row_base=0):
    want = ref.logprobs(x[row_base:], tokens, top_k)
    got = token_logprobs(backend, x, tokens, top_k, row_base)
    if top_k:
        assert np.array_equal(got["top"], want["top"])
    for name in ("logprobs", "top_logprobs"):
        if name in got:
            near(got[name], want[name], want["bound"][:, None] + 3 * EPS * np.abs(np.where(np.isfinite(want[name]), want[name], 0.0)))
    near(got["entropy"], want["entropy"], want["entropy_bound"])


def near(got, want, bound):
    finite = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~finite & ~np.isnan(want)], want[~finite & ~np.isnan(want)].astype(np.float32))
    err = np.abs(np.where(finite, got, 0.0) - np.where(finite, want, 0.0))
    assert np.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 8189, 8190, 8192, 8193, 16384, 50001, 131072])
@pytest.mark.parametrize("rows,top_k", [(1, 1), (3, 8), (5, 32), (2, 0)])
def test_token_logprobs(backend, vocab, rows, top_k):
    rs = np.random.RandomState(vocab + rows)
    x = (rs.randn(rows + 2, vocab) * 3).astype(np.float32)
    tokens = rs.randint(0, vocab, (rows, 3))
    tokens[:, 1] = x[2:].argmax(1)
    tokens[0, 2] = vocab                       # no token
    check_logprobs(backend, x, tokens, min(top_k, vocab), row_base=2)


@pytest.mark.parametrize("rows", [1, 40])
def test_token_logprobs_past_4_gib(backend, rows):
    """Rows behind 2^32 bytes of others."""
    vocab = 131072
    base = (1 << 32) // (vocab * 4) + 3
    rs = np.random.RandomState(rows)
    x = np.zeros((base + rows, vocab), np.float32)
    x[base:] = rs.randn(rows, vocab)
    check_logprobs(backend, x, rs.randint(0, vocab, (rows, 3)), 5, row_base=base)


@pytest.mark.parametrize("vocab", [700, 9000, 40003])
@pytest.mark.parametrize("shape", ["equal", "rising", "falling", "few", "one", "steps", "zeros", "huge", "flat"])
def test_token_logprobs_orders_and_ties(backend, vocab, shape):
    """Rows whose largest entries hide from a bound: all alike, sorted, almost all banned."""
    rs = np.random.RandomState(vocab)
    i = np.arange(vocab)
    row = {"equal": np.full(vocab, 1.5), "rising": i * 0.01, "falling": -i * 0.01, "few": np.where(rs.rand(vocab) < 0.0005, 2.0, -np.inf),
           "one": np.where(i == vocab // 2, 0.25, -np.inf), "steps": np.floor(rs.randn(vocab)), "zeros": np.where(i % 2 == 0, -0.0, 0.0),
           "huge": np.where(rs.rand(vocab) < 0.3, -3.4028235e38, rs.randn(vocab) * 1e4), "flat": rs.randn(vocab) * 1e-6 + 100}[shape].astype(np.float32)
    if shape == "few":
        row[7] = 1.0
    x = np.stack([row, row[::-1].copy()])
    check_logprobs(backend, x, np.array([[0, vocab - 1], [1, vocab // 2]]) % vocab, 32)


def test_token_logprobs_not_finite(backend):
    rs = np.random.RandomState(9)
    for vocab in (50, 20000):
        x = rs.randn(6, vocab).astype(np.float32)
        x[0, 3] = np.nan
        x[1, 40] = np.inf
        x[2, :] = -np.inf
        x[3, :] = np.nan
        x[4, 5:] = np.nan
        x[5, 9:] = -np.inf
        x[5, 30:] = np.nan
        check_logprobs(backend, x, rs.randint(0, 50, (6, 2)), 20)


def test_token_logprobs_many_rows(backend):
    """More rows than shares of which fit the scratch block at once."""
    rs = np.random.RandomState(11)
    rows, vocab = 5000, 65000
    x = rs.randn(8, vocab).astype(np.float32)
    tokens = rs.randint(0, vocab, (rows, 1))
    import torch
    dx = torch.from_numpy(x).cuda().repeat(rows // 8, 1)
    logits = backend.WrapBuffer(dx.data_ptr(), dx.numel() * 4)
    torch.cuda.synchronize()
    up = backend.Upload
    outs = [backend.AllocateBuffer(rows * 4), backend.AllocateBuffer(rows * 4), backend.AllocateBuffer(rows * 128), backend.AllocateBuffer(rows * 128)]
    run(backend, "token_logprobs", [logits, up(tokens.astype(np.uint32)), *outs], [rows, vocab, 1, 32, 0])
    backend.Synchronize()
    want = ref.logprobs(x, tokens[:8], 32)
    ids = backend.CopyD2H(outs[2], dtype=np.uint32).reshape(rows, 32)
    assert np.array_equal(ids, np.tile(want["top"], (rows // 8, 1)))
    entropy = backend.CopyD2H(outs[1], dtype=np.float32)
    near(entropy, np.tile(want["entropy"], rows // 8), np.tile(want["entropy_bound"], rows // 8))
    logp = backend.CopyD2H(outs[0], dtype=np.float32)
    x64 = x.astype(np.float64)
    lse = np.log(np.exp(x64).sum(1))
    near(logp, x64[np.arange(rows) % 8, tokens[:, 0]] - lse[np.arange(rows) % 8], np.tile(want["bound"], rows // 8) + 40 * EPS)


# ---- a verification step -------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16", "q8"])
def test_verify_step(backend, kind):
    """Masks and positions from the parents, queries and keys from a fused projection, keys and values into the cache,
    attention of the tree and the tokens' log probabilities: each id on what the one before it left on the device."""
    m, past, heads, kv, d, vocab, theta = 21, 90, 6, 2, 64, 3001, 1e5
    rs = np.random.RandomState(2)
    parents = ref.random_parents(rs, m, 4, padding=2)
    seen = ref.seen_of(parents)
    rows = rs.randn(m, 2 * heads * d + 2 * kv * d).astype(np.float32)
    w = (rs.rand(d) + 0.5).astype(np.float32)
    g = np.random.default_rng(4)
    old = [cache(g, kind, past, kv * d) for _ in range(2)]
    head = (rs.randn(heads * d, vocab) * 0.2).astype(np.float32)
    n, up, new = past + m, backend.Upload, backend.AllocateBuffer
    mask, pos = new(m * 4), new(m * 24)
    run(backend, "tree_mask", [up(parents), mask, pos], [m, past])
    fused = up(rows)
    wide = 2 * heads * d
    part = lambda at: backend.WrapBuffer(fused.Handle() + 4 * at, fused.Size() - 4 * at)   # noqa: E731
    row = kv * d * {"f32": 4, "f16": 2, "q8": 1}[kind]
    stores = [new(n * row), new(n * row)]
    scales = [new(n * 4), new(n * 4)] if kind == "q8" else []
    for i, (codes, s) in enumerate(old):
        backend.CopyH2D(stores[i], codes)
        if scales:
            backend.CopyH2D(scales[i], s)
    q, gate = new(m * heads * d * 4), new(m * heads * d * 4)
    keys = stores[0] if kind != "q8" else new(m * kv * d * 4)
    run(backend, "qk_norm_mrope", [part(0), part(wide), up(w), up(w), pos, q, keys, gate],
        [m, heads, kv, d, d, f32_bits(theta), f32_bits(1e-6), rows.shape[1], rows.shape[1], int(kind == "f16"), 0 if kind == "q8" else past, 16, 8, 8])
    values = np.ascontiguousarray(rows[:, wide + kv * d:])
    dv = up(values)
    if kind == "q8":
        codes, s = new(m * row), new(m * 4)
        for i, x in enumerate((keys, dv)):
            run(backend, "quantize_q8", [x, codes, s], [m, kv * d])
            backend.CopyD2D(stores[i], past * row, codes, 0, m * row)
            backend.CopyD2D(scales[i], past * 4, s, 0, m * 4)
    elif kind == "f16":
        half = new(m * row)
        run(backend, "cast_f32_f16", [dv, half], [m * kv * d])
        backend.CopyD2D(stores[1], past * row, half, 0, m * row)
    else:
        backend.CopyD2D(stores[1], past * row, dv, 0, m * row)
    out = new(m * heads * d * 4)
    scalars = [m, n, heads, kv, d, m, 0] + ([] if scales else [int(kind == "f16")])
    run(backend, "attention_tree" + ("_q8" if scales else ""), [q, *stores, *scales, mask, out], scalars)
    backend.Synchronize()
    got = backend.CopyD2H(out, dtype=np.float32).reshape(m, heads * d)
    logits = (got.astype(np.float64) @ head).astype(np.float32)
    tokens = rs.randint(0, vocab, (m, 2)).astype(np.uint32)
    check_logprobs(backend, logits, tokens, 4)

    # the same step in 64 bits over the cache as it stands
    position = ref.positions_of(seen, past)
    x = rows[:, :wide].reshape(m, heads, 2 * d)
    want_q, _ = ref.rotate(x[..., :d], w, position, d, np.float32(theta), float(np.float32(1e-6)), (16, 8, 8))
    assert np.array_equal(backend.CopyD2H(gate, dtype=np.float32).reshape(m, heads, d), x[..., d:])
    dtype = {"f32": np.float32, "f16": np.float16, "q8": np.uint8}[kind]
    held = [backend.CopyD2H(s, dtype=dtype).reshape(n, -1) for s in stores]
    factors = [backend.CopyD2H(s, dtype=np.float32) for s in scales] or [None, None]
    ke, ve = (elements(kind, c, s, kv * d) for c, s in zip(held, factors))
    want_k, mags = ref.rotate(rows[:, wide:wide + kv * d].reshape(m, kv, d), w, position, d, np.float32(theta), float(np.float32(1e-6)), (16, 8, 8))
    step = {"f32": 0.0, "f16": 2.0 ** -11 * 1.001, "q8": 0.5 / 127 * 1.001}[kind]
    largest = np.abs(want_k).reshape(m, -1).max(1)[:, None, None] if kind == "q8" else np.abs(want_k)
    assert np.all(np.abs(ke[past:].reshape(m, kv, d) - want_k) <= ref.ROTATE_ROUNDINGS * EPS * mags + step * largest + 2.0 ** -25)
    see = ref.visible(seen, past, 0)
    want = ref.attention(want_q.reshape(m, -1), ke, ve, see, heads, kv, d)
    # the queries' own 16 roundings move a score by at most 16 EPS of what its products sum to, as its own sum's do
    assert np.max(np.abs(got - want)) <= 3 * ref.attention_bound(want_q, ke, ve, see, heads, kv, d)

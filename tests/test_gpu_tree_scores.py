"""Scores of any size that fp32 holds: "attention_tree" over whole caches and in parts, by rows and with shared keys."""
import numpy as np
import pytest

import tree_reference as ref
from tree_reference import EPS
from test_gpu_attention import cache
from test_gpu_tree import attend_tree, elements

pytestmark = pytest.mark.gpu

# few rows and many, keys in one part and in several (launch_rules.hpp: tree_rule), head sizes of the matrix kernels and not
CASES = [(1, 40, 4, 2, 64), (3, 3000, 4, 2, 128), (2, 5000, 8, 2, 256), (40, 120, 8, 2, 64), (40, 130, 8, 2, 256),
         (40, 3000, 8, 2, 64), (40, 3000, 8, 2, 128), (40, 2500, 12, 2, 256), (5, 100, 8, 4, 34), (3, 2000, 4, 2, 34)]


def one_key_leads(backend, kind, case, size, lead):
    """Scores of about `size`, negative or positive, that are alike but for one key of the cache and one of the tree, which lie
    above the others by a hundredth of it, the tree's by twice that: a row becomes the values of the tree's where it sees that key,
    and of the cache's otherwise.  A weight is 1 and the others 0, so the result is the value as it is carried: an fp32 or
    quantized one as two terms, 2 EPS each, its scales and the division 4 more."""
    m, n, heads, kv_heads, head_dim = case
    rs, g = np.random.RandomState(n + head_dim), np.random.default_rng(n)
    width, tree = kv_heads * head_dim, min(m, 8)
    q = (np.abs(rs.randn(m, heads * head_dim)) + 1).astype(np.float32)
    row = np.abs(rs.randn(1, width)) + 1
    factor = np.ones((n, 1))
    prefix_best, tree_best = (n - tree) * 2 // 3, n - tree + tree // 2
    step = 0.01 if lead else -0.01
    factor[prefix_best], factor[tree_best] = 1 + step, 1 + 2 * step
    x = (row * factor).astype(np.float32)
    if kind == "f32":       # the size lies in both, in the keys' power of two and the queries'
        q, k, ks = q * np.float32(np.sqrt(abs(size))) * np.sign(size), x * np.float32(np.sqrt(abs(size))), None
    elif kind == "f16":
        q, k, ks = q * np.float32(size), x.astype(np.float16), None
    else:                   # the codes of one row for all, the sizes in the scales
        code, s = cache(g, "q8", 1, width)
        k = np.repeat(np.abs(code.view(np.int8).astype(np.int32)).clip(1, 127).astype(np.int8).view(np.uint8).reshape(1, width), n, 0)
        q, ks = q * np.float32(size), (factor[:, 0] / 64).astype(np.float32)
    q = q.astype(np.float32)
    v, vs = cache(g, kind, n, width)
    seen = rs.rand(m, tree) < 0.7
    seen[::2, tree // 2] = False
    seen[1::2, tree // 2] = True
    got = attend_tree(backend, kind, q, k, v, ks, vs, ref.words_of(seen), tree, m, n, heads, kv_heads, head_dim, 0)
    ve = elements(kind, v, vs, width).reshape(n, kv_heads, head_dim)
    best = np.where(seen[:, tree // 2], tree_best, prefix_best)
    want = np.repeat(ve[best], heads // kv_heads, 1).reshape(m, -1)
    assert np.isfinite(got).all()
    assert np.all(np.abs(got - want) <= 8 * EPS * np.abs(want) + 2.0 ** -25 * EPS * np.abs(ve).max())


@pytest.mark.parametrize("kind", ["f32", "f16", "q8"])
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("size", [1e6, 1e9, 1e12, 1e25, 2e31, 1e34])
def test_large_scores(backend, kind, case, size):
    """Positive ones, of which the greatest leads, and negative ones, of which the least far from 0 does."""
    one_key_leads(backend, kind, case, size, True)
    one_key_leads(backend, kind, case, -size, False)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("case", CASES)
def test_no_score_above_minus_infinity(backend, kind, case):
    """Rows that see keys, but none with a score above -infinity, are zeros as rows that see none are."""
    m, n, heads, kv_heads, head_dim = case
    rs, g = np.random.RandomState(n), np.random.default_rng(n + 1)
    width = kv_heads * head_dim
    q = (np.abs(rs.randn(m, heads * head_dim)) + 1).astype(np.float32)
    k, _ = cache(g, kind, n, width)
    v, _ = cache(g, kind, n, width)
    k = k.reshape(n, width).copy()
    k[:, ::head_dim] = -np.inf
    got = attend_tree(backend, kind, q, k, v, None, None, ref.words_of(np.tril(np.ones((m, m), bool))), m, m, n, heads, kv_heads, head_dim, 0)
    assert np.all(got == 0.0)

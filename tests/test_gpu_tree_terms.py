"""How far "attention_tree" carries what is small beside something large: query elements, fp32 keys' and values' elements and weights
beside the largest of their head, key or row, by rows and where many rows share their keys (test_tree_rules.py: which)."""
import numpy as np
import pytest

import tree_reference as ref
from tree_reference import EPS
from test_gpu_attention import cache
from test_gpu_tree import attend_tree, elements

pytestmark = pytest.mark.gpu

CASES = [(2, 300, 8, 2, 64), (3, 900, 8, 2, 256), (40, 700, 8, 2, 64), (40, 2000, 8, 2, 128), (40, 2000, 12, 2, 256), (4, 200, 8, 4, 34)]


def one_element(kind, n, kv_heads, head_dim, at, size):
    """Keys of one element each, `size` (n x kv_heads, positive; the quantized kinds take the first head's for all)."""
    width = kv_heads * head_dim
    x = np.zeros((n, kv_heads, head_dim), np.float32)
    if kind in ("f32", "f16"):
        x[:, :, at] = size
        return x.reshape(n, width).astype(np.float32 if kind == "f32" else np.float16), None
    x[:, :, at] = 1
    codes = x.reshape(n, width).astype(np.uint8) * {"q8": 1, "q4": 1, "fp8": 0x38}[kind]
    if kind == "q4":
        codes = codes[:, 0::2] | codes[:, 1::2] << 4
    return np.ascontiguousarray(codes), size[:, 0].astype(np.float32)


@pytest.mark.parametrize("kind", ["f32", "f16", "q8", "q4", "fp8"])
@pytest.mark.parametrize("case", CASES)
def test_query_elements_beside_a_large_one(backend, kind, case):
    """A query's first element is 2^27 times the one that meets the keys, and meets zeros."""
    m, n, heads, kv_heads, head_dim = case
    rs, g = np.random.RandomState(n + head_dim), np.random.default_rng(n)
    q = np.zeros((m, heads, head_dim), np.float32)
    q[:, :, 0], q[:, :, 5] = 2.0 ** 27, 1 + rs.rand(m, heads)
    k, ks = one_element(kind, n, kv_heads, head_dim, 5, np.abs(rs.randn(n, kv_heads)) * 16)
    v, vs = cache(g, kind, n, kv_heads * head_dim)
    q = q.reshape(m, -1)
    seen = rs.rand(m, m) < 0.5
    see = ref.visible(seen, n - m, 0)
    ke, ve = elements(kind, k, ks, kv_heads * head_dim), elements(kind, v, vs, kv_heads * head_dim)
    got = attend_tree(backend, kind, q, k, v, ks, vs, ref.words_of(seen), m, m, n, heads, kv_heads, head_dim, 0)
    err = np.abs(got - ref.attention(q, ke, ve, see, heads, kv_heads, head_dim)).max()
    bound = ref.attention_bound(q, ke, ve, see, heads, kv_heads, head_dim)
    assert err <= bound, (err, bound)


@pytest.mark.parametrize("case", CASES)
def test_fp32_key_elements_beside_a_large_one(backend, case):
    """A key's first element is some 2^27 times the one that meets the queries, and meets zeros.  Below 2^-28 of the largest an element
    is off by 2^-50 of it, here 2^-23, times queries of at most 64: 6 EPS a score and sqrt(head_dim), less than a score's bound."""
    m, n, heads, kv_heads, head_dim = case
    rs = np.random.RandomState(n + head_dim)
    width = kv_heads * head_dim
    q, k = np.zeros((m, heads, head_dim), np.float32), np.zeros((n, kv_heads, head_dim), np.float32)
    q[:, :, 5] = 32 * (1 + rs.rand(m, heads))
    k[:, :, 0], k[:, :, 5] = 2.0 ** 27, rs.randn(n, kv_heads)
    v = rs.randn(n, width).astype(np.float32)
    q, k = q.reshape(m, -1), k.reshape(n, width)
    seen = rs.rand(m, m) < 0.5
    see = ref.visible(seen, n - m, 0)
    got = attend_tree(backend, "f32", q, k, v, None, None, ref.words_of(seen), m, m, n, heads, kv_heads, head_dim, 0)
    err = np.abs(got - ref.attention(q, k, v, see, heads, kv_heads, head_dim)).max()
    bound = ref.attention_bound(q, k, v, see, heads, kv_heads, head_dim)
    assert err <= bound, (err, bound)


@pytest.mark.parametrize("case", CASES)
def test_fp32_value_elements_beside_a_large_one(backend, case):
    """Each row becomes the values of one key, whose elements lie up to 2^27 apart: a weight of 1, so each is off by 2 EPS of itself or
    2^-50 of the key's largest, by a rounding of the sum and by the scales, the merges and the division, 5 more."""
    m, n, heads, kv_heads, head_dim = case
    rs = np.random.RandomState(n + head_dim)
    width = kv_heads * head_dim
    q, k = np.zeros((m, heads, head_dim), np.float32), np.zeros((n, kv_heads, head_dim), np.float32)
    q[:, :, 5], k[:, :, 5] = 64.0, -64.0
    best = rs.randint(0, n - m, kv_heads)
    k[best, np.arange(kv_heads), 5] = 64.0                  # scores 1024 apart
    v = (rs.randn(n, kv_heads, head_dim) * np.exp2(-rs.randint(0, 28, (n, kv_heads, head_dim)))).astype(np.float32)
    got = attend_tree(backend, "f32", q.reshape(m, -1), k.reshape(n, width), v.reshape(n, width), None, None,
                      ref.words_of(rs.rand(m, m) < 0.5), m, m, n, heads, kv_heads, head_dim, 0)
    want = np.repeat(v[best, np.arange(kv_heads)].astype(np.float64), heads // kv_heads, 0)
    bound = 8 * EPS * np.abs(want) + 2.0 ** -49 * np.abs(want).max(1, keepdims=True)
    err = np.abs(got.reshape(m, heads, head_dim) - want)
    assert np.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("kind", ["f32", "f16", "q8", "q4", "fp8"])
@pytest.mark.parametrize("case", CASES)
def test_small_weights_of_large_values(backend, kind, case):
    """The values are the larger the smaller the weight that they meet, up to 2^12.  A weight misses as attention_bound says, and (times
    its value's scale over fp32 and quantized keys) by 2^-34 of the row's largest; each such error counts with the value's element."""
    m, n, heads, kv_heads, head_dim = case
    rs, g = np.random.RandomState(n + head_dim), np.random.default_rng(n)
    width, group = kv_heads * head_dim, heads // kv_heads
    q = np.zeros((m, heads, head_dim), np.float32)
    q[:, :, 5] = 1 + rs.rand(m, heads) / 8
    k, ks = one_element(kind, n, kv_heads, head_dim, 5, rs.rand(n, 1).repeat(kv_heads, 1) * 20 * np.sqrt(head_dim))
    ke = elements(kind, k, ks, width).reshape(n, kv_heads, head_dim)
    v, vs = cache(g, kind, n, width, gain=np.exp2(12 * (1 - ke[:, 0, 5] / ke[:, 0, 5].max())))
    ve = elements(kind, v, vs, width).reshape(n, kv_heads, head_dim)
    seen = rs.rand(m, m) < 0.5
    see = ref.visible(seen, n - m, 0)
    got = attend_tree(backend, kind, q.reshape(m, -1), k, v, ks, vs, ref.words_of(seen), m, m, n, heads, kv_heads, head_dim, 0).reshape(m, heads, head_dim)
    for i in range(m):
        for h in range(heads):
            kv = h // group
            s = ke[see[i], kv] @ q[i, h].astype(np.float64) / np.sqrt(head_dim)
            w, x = np.exp(s - s.max()), ve[see[i], kv]
            scale = np.ones(len(w)) if kind == "f16" else np.abs(x).max(1) if vs is None else vs[see[i]]
            rel = (2 * (head_dim / 16 + 14) * s.max() + 4 * s.max() + 8) * EPS
            want = w @ x / w.sum()
            each = w * rel + (w * scale).max() * 2.0 ** -34 / scale
            bound = (each @ np.abs(x) + (rel + (n / 16 + 32) * EPS) * (w @ np.abs(x))) / w.sum()
            assert np.all(np.abs(got[i, h] - want) <= bound), (i, h, (np.abs(got[i, h] - want) / bound).max())

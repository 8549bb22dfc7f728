"""The shared-key kernel of "attention_tree" in parts: windows that begin before the tree, inside it and across it, rows that see little,
head sizes between its tiles', every kind of cache (tree_shapes.py)."""
import numpy as np
import pytest

from test_gpu_tree import check_attention
from tree_shapes import KINDS, calls

pytestmark = pytest.mark.gpu

ALL = [(kind, call) for kind in KINDS for call in calls(kind)]


def uneven(m, tree, seed):
    """Bits of rows that see much of the tree, little of it, one key, none; no row sees what its neighbour does."""
    rs = np.random.RandomState(seed)
    seen = rs.rand(m, tree) < np.array([0.95, 0.5, 0.1, 0.7])[np.arange(m) % 4, None]
    seen[5], seen[6] = False, False
    seen[6, tree // 2] = True
    seen[7] = True
    return seen


@pytest.mark.parametrize("kind,call", ALL)
def test_shared_keys(backend, kind, call):
    m, tree = call[0], call[5]
    check_attention(backend, kind, *call, seen=uneven(m, tree, m + tree), seed=3)


@pytest.mark.parametrize("kind,call", [(k, c) for k, c in ALL if c[6]])
def test_shared_keys_of_which_some_are_hidden_from_all(backend, kind, call):
    """They may hold anything, the last one and every third of the tree's too."""
    m, tree = call[0], call[5]
    seen = uneven(m, tree, m)
    seen[:, ::3], seen[:, -1] = False, False
    check_attention(backend, kind, *call, seen=seen, seed=4, spoil=True)


@pytest.mark.parametrize("kind", KINDS)
def test_shared_keys_behind_a_window_of_the_tree(backend, kind):
    """Nothing before the tree; windows that begin at any of its words, rows that see less than the window."""
    for d in (64, 128, 256):
        heads, kv_heads = (32, 8) if d == 64 else (8, 2)
        m, n = 40, 4100
        check_attention(backend, kind, m, n, heads, kv_heads, d, n, 3000, seen=uneven(m, n, d), seed=5)

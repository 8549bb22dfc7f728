"""Calls of "attention_tree" whose rows share their keys on the shared-key kernel, in parts: by a window, at head sizes between those that
its tiles are made for, and with many words of bits.  test_tree_rules_shared.py holds the rule to it, test_gpu_tree_shared.py runs them."""

KINDS = ["f32", "f16", "q8", "q4", "fp8"]
SIZES = [64, 80, 96, 128, 160, 256]


def calls(kind):
    """m, n, heads, kv_heads, head_dim, tree, window."""
    shapes = []
    for d in SIZES:
        heads, kv_heads = (32, 8) if kind == "f32" and d == 64 else (8, 2)
        n = 9000 if heads == 32 else 4200
        shapes += [(33, n, heads, kv_heads, d, 33, n // 2 - 100), (40, n, heads, kv_heads, d, 2600, n // 2 - 300), (40, n, heads, kv_heads, d, 40, 0)]
    return shapes

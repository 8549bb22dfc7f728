"""Calls of "attention_pages_*" that reach every form of its kernels on a chip of 256 CUs: which, tests/test_page_shapes.py says."""

# (row, head) pairs of the longest sequence to a key head: queries to each key head, rows
PAIRS = {1: (1, 1), 16: (4, 4), 17: (17, 1), 32: (8, 4), 33: (3, 11), 64: (4, 16), 65: (5, 13), 90: (6, 15), 128: (8, 16), 129: (3, 43)}
HEAD_DIMS = (64, 80, 128, 208, 256)
KV = 2


def batch(how, rows):
    """Rows and earlier positions of the sequences of a batch, the first with `rows` of them."""
    if how == "short":          # a workgroup a unit
        return [rows, 1, 0, max(1, rows // 2), rows], [300, 0, 70, 129, 17]
    if how == "many":           # more units than CUs
        return [rows] + [1 + i % rows for i in range(129)], [30] + [i % 37 for i in range(129)]
    if how == "parts":          # parts of the positions
        return [rows, max(1, rows - 1)], [2300, 300]
    assert how == "even"        # even runs of all tiles
    return [rows] + [1 + i % rows for i in range(40)], [2600, 1500] + [7 * i % 90 for i in range(39)]


def sizes(how, pairs):
    """queries to each key head, rows, earlier positions, the most rows, the most positions"""
    group, rows = PAIRS[pairs]
    each, past = batch(how, rows)
    return group, each, past, rows, max(a + b for a, b in zip(each, past))


def columns(pairs, d):
    return 16 if pairs <= 16 else 32 if pairs <= 32 and d <= 128 else None


def forms():
    """(how, pairs, head_dim) with `how` one that these sizes have."""
    for d in HEAD_DIMS:
        for pairs in PAIRS:
            few = columns(pairs, d) is not None
            for how in ("short", "many", "parts", "even") if few else ("short", "parts"):
                if how == "short" or few or pairs in (33, 64, 65, 129):
                    yield how, pairs, d

"""Plain 64-bit statements of the ids around a tree of drafted tokens, and how far an fp32 kernel may be from them."""
import numpy as np

EPS = 2.0 ** -24
ROOT = 0xFFFFFFFF


def seen_of(parents):
    """seen[i][j]: node i sees node j."""
    n = len(parents)
    seen = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if p == ROOT:
            seen[i, i] = True
        elif p < i and seen[p, p]:
            seen[i] = seen[p]
            seen[i, i] = True
    return seen


def words_of(seen):
    """Bit j % 32 of word j / 32."""
    n, t = seen.shape
    bits = np.zeros((n, (t + 31) // 32 * 32), np.uint8)
    bits[:, :t] = seen
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32)


def positions_of(seen, base):
    depth = np.maximum(seen.sum(1).astype(np.int64), 1) - 1
    return np.repeat((base + depth)[:, None], 3, 1).astype(np.uint64)


def random_parents(rs, nodes, reach, padding=0):
    parents = np.empty(nodes, np.uint32)
    for i in range(nodes):
        p = i - 1 - rs.randint(0, reach + 1)
        parents[i] = ROOT if i == 0 or p < 0 else p
        if i >= nodes - padding:
            parents[i] = i
    return parents


def visible(seen, prefix, window):
    """Rows x keys of the cache, of which the last are the tree's."""
    m = seen.shape[0]
    all_keys = np.concatenate([np.ones((m, prefix), bool), seen], 1)
    if window:
        order = np.cumsum(all_keys, 1)
        all_keys &= order[:, -1:] - order < window
    return all_keys


def attention(q, k, v, see, heads, kv_heads, head_dim):
    """q: rows x heads*head_dim; k, v: keys x kv_heads*head_dim (their elements); hidden keys take no part whatever they hold."""
    m, n = see.shape
    group = heads // kv_heads
    out = np.zeros((m, heads, head_dim))
    q = q.reshape(m, heads, head_dim).astype(np.float64)
    k, v = k.reshape(n, kv_heads, head_dim).astype(np.float64), v.reshape(n, kv_heads, head_dim).astype(np.float64)
    for i in range(m):
        at = np.nonzero(see[i])[0]
        if not len(at):
            continue
        for h in range(heads):
            with np.errstate(invalid="ignore"):
                s = k[at, h // group] @ q[i, h] / np.sqrt(head_dim)
                top = s.max()
                p = np.exp(s - (0.0 if top == -np.inf else top))
                out[i, h] = (p @ v[at, h // group]) / p.sum() if p.sum() != 0 else 0.0
    return out.reshape(m, heads * head_dim)


def attention_bound(q, k, v, see, heads, kv_heads, head_dim):
    """A score is a sum of head_dim products: an element is carried to 2 EPS, the products are added in chains of at most
    head_dim / 16 + 8 roundings, a quantized key's scale and the division by sqrt(head_dim) are 4 more, each of at most A =
    max sum |q k| / sqrt(head_dim).  A weight exp(s - max) then misses by twice that, by its argument's rounding (at most 2
    A of its size) and by 8 EPS for the exponential and its own two terms.  The result misses by twice the weights' (they enter the
    sum and the total), and by one rounding of the running sums a tile of 16 keys or more: of at most max |v| each."""
    m, n = see.shape
    group = heads // kv_heads
    q, k = np.abs(q).reshape(m, heads, head_dim).astype(np.float64), np.abs(k).reshape(n, kv_heads, head_dim).astype(np.float64)
    most = 0.0
    for h in range(heads):
        a = np.where(see, (q[:, h] @ k[:, h // group].T) / np.sqrt(head_dim), 0.0)
        most = max(most, a.max())
    values = np.abs(np.where(see.any(0)[:, None], v, 0.0)).max()
    weight = (2 * (head_dim / 16 + 14) * most + 4 * most + 8) * EPS
    return (2 * weight + (n / 16 + 32) * EPS) * values


def rotate(x, w, pos, rope_dim, theta, eps, sections):
    """Rows x heads x head_dim; pos: rows x 3.  The result and the sum of the magnitudes that each element is made of."""
    rows, _, d = x.shape
    pairs = rope_dim // 2
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(2, keepdims=True) + eps) * w
    j = np.arange(pairs)
    axis = np.where(j < sections[0], 0, np.where(j < sections[0] + sections[1], 1, 2))
    turn = float(theta) ** (-2.0 * j / rope_dim)
    angle = np.asarray(pos, np.float64)[:, axis] * turn
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = y[..., :pairs], y[..., pairs:rope_dim]
    out = np.concatenate([a * c - b * s, b * c + a * s, y[..., rope_dim:]], 2)
    # the angle itself misses by a few roundings of 64 bits
    far = 1 + angle[:, None] * (8 * 2.0 ** -53 / EPS)
    size = np.concatenate([(np.abs(a) + np.abs(b)) * far, (np.abs(a) + np.abs(b)) * far, np.abs(y[..., rope_dim:])], 2)
    return out, size


# A head's mean square is a sum of positive terms in at most 10 roundings (5 of its root), the gain 3 more, its products with the
# element and the weight 2, the rotation's cosine, products and sum 4.
ROTATE_ROUNDINGS = 16


def logprobs(x, tokens, top_k):
    x = x.astype(np.float64)
    rows, vocab = x.shape
    out = {"logprobs": np.full(tokens.shape, np.nan), "entropy": np.full(rows, np.nan), "top": np.zeros((rows, top_k), np.int64),
           "top_logprobs": np.full((rows, top_k), np.nan), "bound": np.zeros(rows), "entropy_bound": np.zeros(rows)}
    for r in range(rows):
        v = x[r]
        order = np.where(np.isnan(v), -np.inf, v)
        rank = np.lexsort((np.arange(vocab), -order, np.isnan(v)))[:top_k]
        out["top"][r] = rank
        m = order.max()
        if np.isnan(v).any() or np.isinf(m):
            continue
        d = v - m
        e = np.exp(d)
        total = e.sum()
        p = e / total
        ds = np.where(e > 0, d, 0.0)
        logp = d - np.log(total)
        ok = tokens[r] < vocab
        out["logprobs"][r] = np.where(ok, logp[np.where(ok, tokens[r], 0)], -np.inf)
        out["entropy"][r] = np.log(total) - (p * ds).sum()
        out["top_logprobs"][r] = logp[rank]
        # e^d misses by (|d| + 3) EPS of itself; a thread adds at most `adds` of them, then wavefronts, workgroup, shares
        adds = vocab / 1024 + 100
        first, second = (p * np.abs(ds)).sum(), (p * ds * ds).sum()
        in_total = (first + 3 + adds) * EPS
        out["bound"][r] = in_total + 4 * EPS * (np.log(total) + 1)
        out["entropy_bound"][r] = in_total * (1 + first) + (second + (4 + adds) * first) * EPS + 8 * EPS * (np.log(total) + first + 1)
    return out

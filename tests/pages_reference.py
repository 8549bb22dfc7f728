"""Plain statements of the ids around a paged cache and of the verification of drafts, on the host: codes, scales and tokens exact,
attention in 64 bits with a bound of what an fp32 kernel may be off by."""
import numpy as np

EPS = 2.0 ** -24        # half a step of fp32
NONE = 0xFFFFFFFF
LARGEST = {"q8": np.float32(127.0), "fp8": np.float32(448.0)}
E4M3 = np.array([(-1.0) ** (b >> 7) * ((b & 7) * 2.0 ** -9 if (b >> 3 & 15) == 0 else (8 + (b & 7)) * 2.0 ** ((b >> 3 & 15) - 10)) for b in range(256)],
                np.float32)
E4M3[[0x7F, 0xFF]] = np.nan
_MAGNITUDES = E4M3[:127].astype(np.float64)      # of codes 0 .. 126, ascending


def encode(fmt, x):
    """fp32 numbers to the nearest code, ties to the even one."""
    x = np.clip(x.astype(np.float64), -float(LARGEST[fmt]), float(LARGEST[fmt]))
    if fmt == "q8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    mag = np.abs(x)
    up = np.clip(np.searchsorted(_MAGNITUDES, mag), 1, 126)
    below, above = mag - _MAGNITUDES[up - 1], _MAGNITUDES[up] - mag
    code = np.where((above < below) | ((above == below) & (up % 2 == 0)), up, up - 1)
    return (code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def decode(fmt, codes):
    return codes.view(np.int8).astype(np.float32) if fmt == "q8" else E4M3[codes]


class Pool:
    """Kp [page][kv][position][element], Vp [page][kv][element][position], Ks, Vs [page][kv]."""

    def __init__(self, rs, fmt, pages, kv, block, d):
        self.fmt, self.pages, self.kv, self.block, self.d = fmt, pages, kv, block, d
        self.kp, self.vp = (encode(fmt, rs.randn(*shape).astype(np.float32) * (LARGEST[fmt] / 4)) for shape in ((pages, kv, block, d), (pages, kv, d, block)))
        self.ks, self.vs = ((rs.rand(pages, kv) + 0.5).astype(np.float32) * spread / LARGEST[fmt] for spread in (np.float32(4), np.float32(3)))

    def copy(self):
        other = object.__new__(Pool)
        other.__dict__.update({k: v.copy() if isinstance(v, np.ndarray) else v for k, v in self.__dict__.items()})
        return other

    def rows(self, table, positions):
        """Keys and values (positions x kv x d, fp32) of a sequence; those of unknown pages 0."""
        page = np.asarray(table)[positions // self.block].astype(np.int64)
        at, known = positions % self.block, (page < self.pages)
        page = np.where(known, page, 0)
        with np.errstate(invalid="ignore"):
            k = decode(self.fmt, self.kp[page, :, at]) * self.ks[page][:, :, None]
            v = decode(self.fmt, self.vp[page, :, :, at]) * self.vs[page][:, :, None]
        return np.where(known[:, None, None], k, np.float32(0)), np.where(known[:, None, None], v, np.float32(0))

    def write(self, table, length, k, v):
        """The last len(k) positions of a sequence (rows x kv x d, fp32)."""
        rows, block = len(k), self.block
        for slot in range((length - rows) // block, (length - 1) // block + 1):
            page, base = int(table[slot]), slot * block
            if page >= self.pages:
                continue
            first, end = max(length - rows - base, 0), min(length - base, block)
            new = slice(base + first - (length - rows), base + end - (length - rows))
            for x, codes, scales in ((k, self.kp, self.ks), (v, self.vp.transpose(0, 1, 3, 2), self.vs)):
                for h in range(self.kv):
                    rows_of = x[new, h].astype(np.float32)
                    before = scales[page, h] if first else np.float32(0)
                    with np.errstate(all="ignore"):
                        own = np.float32(np.abs(rows_of).max() / LARGEST[self.fmt])
                        after = max(before, own) if np.isfinite(rows_of).all() and 0 <= before < np.inf else np.float32(np.nan)
                        held = codes[page, h, :first].copy()
                        fresh = np.zeros((block, self.d), np.uint8)
                        if after > 0:
                            if after != before:
                                held = encode(self.fmt, (decode(self.fmt, held) * before).astype(np.float32) / after)
                            fresh[:first], fresh[first:end] = held, encode(self.fmt, rows_of / after)
                    codes[page, h], scales[page, h] = fresh, after


def visible(positions, length, window, sinks):
    """rows x positions: what rows at these positions see."""
    j = np.arange(length)[None]
    p = np.asarray(positions)[:, None]
    see = j <= p
    if window:
        see &= (p - j < window) | (j < sinks)
    return see


def attention(pool, table, length, q, group, window=0, sinks=0):
    """q: rows x heads x d, the last rows of a sequence.  Returns the result in 64 bits and how far fp32 sums may be from it.

    A score is a sum of d products: an element enters to 2^-22 of itself (two fp16 terms) or, where the second is subnormal, to half
    of 2^-24 under a power of two that brings the row's largest to 2^13 at least; over int8 pages to half a step of an integer whose
    largest is 8355584 (2^-23 of the row's largest: 2^-24 and the rounding of what it is multiplied by); the products are exact, each
    addition rounds to 2^-24 of at most the sum of their magnitudes; then a few roundings (scales, log2 e, the reference) of the score.  A weight is
    off by that, relatively, and by the exponential's and its own two terms' 2^-21 or, where the second is subnormal, by half of
    2^-24 under a power of two that brings the row's largest weight times value scale to 2^9 at least: 2^-34 of that, times each
    value's code.  Sums of n weights and products are off by n + 64 roundings."""
    rows, heads, d = q.shape
    k, v = (x.astype(np.float64) for x in pool.rows(table, np.arange(length)))
    page = np.asarray(table)[np.arange(length) // pool.block].astype(np.int64)
    v_scale = pool.vs[np.where(page < pool.pages, page, 0)].astype(np.float64)
    see = visible(np.arange(length - rows, length), length, window, sinks) & (page < pool.pages)[None]
    out, bound = np.zeros((rows, heads, d)), np.zeros((rows, heads, d))
    for i in range(rows):
        at = np.nonzero(see[i])[0]
        if not len(at):
            continue
        for h in range(heads):
            kk, vv, x = k[at, h // group], v[at, h // group], q[i, h].astype(np.float64)
            with np.errstate(invalid="ignore"):
                s, mass = kk @ x / np.sqrt(d), np.abs(kk) @ np.abs(x) / np.sqrt(d)
                p = np.exp(s - s.max())
                out[i, h] = p @ vv / p.sum()
                low = 2.0 ** (-23 if pool.fmt == "q8" else -38) * np.abs(x).max() * np.abs(kk).sum(1).max() / np.sqrt(d)
                off = mass.max() * (2.0 ** -22 + (d + 8) * EPS) + low + np.abs(s).max() * 8 * EPS
                bound[i, h] = (np.expm1(2 * off) + 2.0 ** -20 + (len(at) + 64) * 2 * EPS) * (p @ np.abs(vv) / p.sum())
                vs = v_scale[at, h // group]
                codes = np.abs(vv) / np.where(vs > 0, vs, 1.0)[:, None]
                bound[i, h] += 2.0 ** -34 * (p * vs).max() * codes.sum(0) / p.sum()
    return out, bound


def weights(logits, temperature):
    """What softmax divides by its sum, in 64 bits; None where a row says nothing (NaN, +infinity, or -infinity alone)."""
    x = logits.astype(np.float64)
    if np.isnan(x).any() or x.max() == np.inf or x.max() == -np.inf:
        return None
    return np.exp((x - x.max()) / float(np.float32(temperature)))


def softmax(logits, temperature):
    e = weights(logits, temperature)
    return e / e.sum()


def verify(logits, tokens, random, starts, temperature, draft=None, draft_temperature=1.0):
    """(accepted, next) of each sequence; None for one without rows."""
    out = []
    vocab = logits.shape[1]
    for first, end in zip(starts[:-1], starts[1:]):
        if not first < end <= len(logits):
            out.append(None)
            continue
        for row in range(first, end):
            at, last = row - first, row == end - 1
            token = None if last else int(tokens[row + 1])
            if temperature == 0.0:
                x = logits[row]
                bad = np.isnan(x).any() or x.max() in (np.inf, -np.inf)
                best = NONE if bad else int(np.argmax(x))
                if bad or last or best != token:
                    out.append((at, best))
                    break
                continue
            # (weights relative to the target's largest, so that equal logits have sums without rounding)
            p = weights(logits[row], temperature)
            q = weights(draft[row], draft_temperature) if draft is not None and not last else None
            if p is not None and q is not None:
                q = q * (p.sum() / q.sum())
            if p is None or (draft is not None and not last and q is None):
                out.append((at, NONE))
                break
            if not last:
                px = p[token] if token < vocab else 0.0
                qx = q[token] if q is not None and token < vocab else p.sum()
                if float(random[row, 0]) * qx < px:
                    continue
                if q is not None:
                    rest = np.maximum(p - q, 0.0)
                else:
                    rest = p.copy()
                    if token < vocab:
                        rest[token] = 0.0
                p = rest if rest.sum() > 0 else p
            run = np.cumsum(p)
            u = float(random[row, 1])
            over = np.nonzero(run > (min(u, 1.0 - 2.0 ** -24) if u >= 0 else 0.0) * run[-1])[0]     # (outside [0, 1): the nearest in it)
            out.append((at, int(over[0]) if len(over) else int(np.nonzero(p > 0)[0][-1])))
            break
    return out

"""The verification of a tree of drafted tokens, as measurable cases.

A draft of several continuations is a tree: node i follows node parents[i], or the last token that the cache
holds.  One pass over the model then scores all nodes at once.  What that pass needs beyond the projections:

  mask     "tree_mask": from the parents, which nodes each node sees (itself and its ancestors) and its position
  rope     "qk_norm_rope", "qk_norm_mrope": RMS norm of each query and key head and its rotary embedding, from the
           (fused) projection's rows, the keys as fp32 or as the fp16 cache's rows, a query gate set apart
  attend   "attention_tree" and its forms over quantized caches: the nodes' rows against all keys before the tree
           and the nodes that their masks name, a window of the last keys that a row sees
  logprob  "token_logprobs": log probabilities of given tokens, the distribution's entropy and its top tokens

With ``own`` false, run() computes them in elementary operations in 32 bits (angles in 64); with ``own`` true
it makes the launches that a program makes through ``tessera_amd.Backend``.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

NONE = 0xFFFFFFFF     # parent of a node that follows the cache's last token
#: bytes of one key or value element in the cache
BYTES_KV = {"f32": 4.0, "f16": 2.0, "q8": 1.0, "q4": 0.5, "fp8": 1.0}


def listed():
    return [
        # the largest draft of a verify batch: sixteen nodes, where the launch is all there is
        {"name": "mask_16", "kind": "mask", "nodes": 16, "reach": 4, "base": 1187},
        # a wide and deep tree of a draft model that is sampled many times, its nodes no multiple of a word
        {"name": "mask_1000", "kind": "mask", "nodes": 1000, "reach": 24, "base": 32768},
        # one decoded token of a gated layer, keys into the fp16 cache
        {"name": "rope_decode", "kind": "rope", "rows": 1, "heads": 24, "kv_heads": 4, "head_dim": 256, "rope_dim": 64, "base": 9300,
         "axes": False, "gated": True, "keys": "f16", "fused": True},
        # a tree's rows, each at its own position, keys for a quantized cache
        {"name": "rope_tree", "kind": "rope", "rows": 33, "heads": 32, "kv_heads": 8, "head_dim": 128, "rope_dim": 128, "base": 32768,
         "axes": True, "gated": False, "keys": "f32", "fused": True},
        # a prefill chunk
        {"name": "rope_prefill", "kind": "rope", "rows": 2048, "heads": 24, "kv_heads": 4, "head_dim": 256, "rope_dim": 256, "base": 2000,
         "axes": False, "gated": False, "keys": "f16", "fused": True},
        # a draft of five tokens in two branches on a short conversation
        {"name": "attend_short", "kind": "attend", "rows": 5, "reach": 2, "context": 301, "heads": 16, "kv_heads": 4, "head_dim": 64, "cache": "f16",
         "window": 0, "padding": 0},
        # a verify batch against a long conversation in an int8 cache
        {"name": "attend_long_q8", "kind": "attend", "rows": 16, "reach": 5, "context": 9300, "heads": 24, "kv_heads": 4, "head_dim": 256, "cache": "q8",
         "window": 0, "padding": 0},
        # a padded batch under a window over E4M3 keys
        {"name": "attend_window_fp8", "kind": "attend", "rows": 33, "reach": 8, "context": 5000, "heads": 32, "kv_heads": 8, "head_dim": 128, "cache": "fp8",
         "window": 4096, "padding": 3},
        # a large tree against a very long context
        {"name": "attend_wide_f16", "kind": "attend", "rows": 64, "reach": 16, "context": 32768, "heads": 24, "kv_heads": 4, "head_dim": 256, "cache": "f16",
         "window": 0, "padding": 0},
        # one decoded token's logits: the sampled token and eight alternatives
        {"name": "logprob_decode", "kind": "logprob", "rows": 1, "vocab": 131072, "tokens": 1, "top_k": 8, "banned": 0.0},
        # a tree's rows under a grammar that bans most tokens, the children's tokens of each node
        {"name": "logprob_tree", "kind": "logprob", "rows": 33, "vocab": 50001, "tokens": 4, "top_k": 5, "banned": 0.7},
        # the scores of a prompt
        {"name": "logprob_prompt", "kind": "logprob", "rows": 512, "vocab": 131072, "tokens": 1, "top_k": 20, "banned": 0.0},
    ]


def draw(rng):
    def between(lo, hi, step=1):
        """A multiple of `step`, evenly over the logarithm of the range."""
        v = lo * (hi / lo) ** rng.random()
        return max(lo, min(hi, int(round(v / step)) * step))

    kind = rng.choice(["mask", "rope", "rope", "attend", "attend", "attend", "attend", "logprob", "logprob"])
    case = {"kind": kind}
    if kind == "mask":
        nodes = between(1, 1024)
        case.update(nodes=nodes, reach=between(1, nodes), base=rng.choice([0, between(1, 1 << 20)]))
        return case
    if kind == "logprob":
        vocab = between(500, 131072)
        case.update(rows=between(1, 512), vocab=vocab, tokens=between(1, 16), top_k=rng.choice([0, 1, between(2, 32), 20]), banned=rng.choice([0.0, 0.0, 0.5, 0.99]))
        return case
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256, 256])
    group, kv_heads = rng.choice([1, 2, 3, 4, 6, 8]), rng.choice([1, 2, 4, 8])
    while group * kv_heads * head_dim > 6144:
        group, kv_heads = rng.choice([1, 2, 3, 4, 6]), rng.choice([1, 2, 4])
    case.update(heads=group * kv_heads, kv_heads=kv_heads, head_dim=head_dim)
    if kind == "rope":
        case.update(rows=rng.choice([1, between(2, 64), between(65, 2048)]), rope_dim=rng.choice([head_dim, head_dim, head_dim // 2, 32]), base=between(1, 1 << 20),
                    axes=rng.random() < 0.5, gated=rng.random() < 0.5, keys=rng.choice(["f32", "f16"]), fused=rng.random() < 0.7)
    else:
        rows = rng.choice([1, between(2, 16), between(2, 64)])
        context = between(1, 32768) if rng.random() < 0.95 else 0
        case.update(rows=rows, reach=between(1, rows), context=context, cache=rng.choice(["f16", "f16", "f16", "q8", "q8", "fp8", "q4", "f32"]),
                    window=between(8, 8192) if rng.random() < 0.25 else 0, padding=rng.choice([0, 0, 0, min(2, rows - 1)]))
        if case["cache"] == "f32":
            case["context"] = min(context, 8192)
    return case


# ---- inputs --------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _parents(seed, nodes, reach, padding=0):
    """A random tree: each node follows one of the `reach` nodes before it or the cache; the last `padding` nodes are none."""
    rs = np.random.RandomState(seed % (1 << 31))
    parents = np.empty(nodes, np.int64)
    for i in range(nodes):
        p = i - 1 - rs.randint(0, reach + 1)
        parents[i] = NONE if i == 0 or p < 0 else p
        if i >= nodes - padding:
            parents[i] = i      # a parent that is no earlier node: padding
    return parents


def _seen(parents):
    """seen[i][j]: node i sees node j."""
    n = len(parents)
    seen = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if p == NONE:
            seen[i, i] = True
        elif p < i and seen[p, p]:
            seen[i] = seen[p]
            seen[i, i] = True
    return seen


def _words(seen):
    """Bits as the operators hold them: bit j % 32 of word j / 32."""
    n, t = seen.shape
    bits = np.zeros((n, (t + 31) // 32 * 32), np.uint8)
    bits[:, :t] = seen
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32)


def _sections(rope_dim):
    """Pairs that take the temporal, the height and the width position."""
    h = rope_dim // 6
    return rope_dim // 2 - 2 * h, h, h


def _cache(g, kind, positions, width):
    """Keys or values as the cache holds them: (elements or codes, one scale a position)."""
    v = torch.randn(positions, width, device="cuda", generator=g)
    if kind == "f32":
        return v, None
    if kind == "f16":
        return v.half(), None
    amax = v.abs().amax(1)
    if kind == "fp8":
        s = amax / 448.0
        return (v / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), s
    s = amax / (127.0 if kind == "q8" else 7.0)
    q = (v / s[:, None]).round().to(torch.int8)
    if kind == "q8":
        return q.view(torch.uint8), s
    q = q.view(torch.uint8) & 15
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), s


def prepare(case, seed):
    c, kind = case, case["kind"]
    s = {"case": dict(c)}
    if kind == "mask":
        s["parents"] = torch.from_numpy(_parents(seed, c["nodes"], c["reach"]).astype(np.uint32).view(np.int32)).cuda()
        return s
    g = _gen(seed)
    if kind == "rope":
        rows, heads, kv, d = c["rows"], c["heads"], c["kv_heads"], c["head_dim"]
        wide = heads * d * (2 if c["gated"] else 1)
        if c["fused"]:      # one projection's rows: queries (and gates), keys, values
            s["rows"] = torch.randn(rows, wide + 2 * kv * d, device="cuda", generator=g) * 1.7
            s["q"], s["k"] = s["rows"][:, :wide], s["rows"][:, wide:wide + kv * d]
        else:
            s["q"] = torch.randn(rows, wide, device="cuda", generator=g) * 1.7
            s["k"] = torch.randn(rows, kv * d, device="cuda", generator=g) * 0.6
        s["wq"] = torch.rand(d, device="cuda", generator=g) + 0.5
        s["wk"] = torch.rand(d, device="cuda", generator=g) + 0.5
        if c["axes"]:
            rs = np.random.RandomState(seed % (1 << 31))
            pos = c["base"] + rs.randint(0, max(2, rows), (rows, 3))
            s["pos"] = torch.from_numpy(pos.astype(np.int64)).cuda()
        # the keys' place: rows of the cache behind those of earlier positions
        s["first"] = 7 if c["keys"] == "f16" else 0
        s["cache"] = torch.zeros(s["first"] + rows, kv * d, device="cuda", dtype=torch.float16 if c["keys"] == "f16" else torch.float32)
    elif kind == "attend":
        m, heads, kv, d, n = c["rows"], c["heads"], c["kv_heads"], c["head_dim"], c["context"] + c["rows"]
        s["q"] = torch.randn(m, heads * d, device="cuda", generator=g)
        s["k"], s["ks"] = _cache(g, c["cache"], n, kv * d)
        s["v"], s["vs"] = _cache(g, c["cache"], n, kv * d)
        s["mask"] = torch.from_numpy(_words(_seen(_parents(seed, m, c["reach"], c["padding"]))).view(np.int32)).cuda()
    else:
        rows, vocab = c["rows"], c["vocab"]
        x = torch.randn(rows, vocab, device="cuda", generator=g) * 2.5
        if c["banned"]:
            x.masked_fill_(torch.rand(rows, vocab, device="cuda", generator=g) < c["banned"], -math.inf)
            x[:, 3] = 1.0   # (the grammar allows something)
        s["logits"] = x
        s["tokens"] = torch.randint(0, vocab, (rows, c["tokens"]), device="cuda", dtype=torch.int32, generator=g)
        s["tokens"][:, 0] = x.argmax(1)
    return s


# ---- the plain forms ------------------------------------------------------------------------------

def _bit_words(seen):
    """The words of a matrix of truth values, as int32."""
    n, t = seen.shape
    words = (t + 31) // 32
    bits = torch.zeros(n, words * 32, dtype=torch.int64, device=seen.device)
    bits[:, :t] = seen
    return (bits.view(n, words, 32) << torch.arange(32, device=seen.device)).sum(2).to(torch.int32)


def _plain_mask(s):
    base, parents = s["case"]["base"], s["parents"]
    n = parents.numel()
    index = torch.arange(n, device="cuda")
    # whom a node sees in one step, then in two, four, ...: squares of the matrix of steps
    steps = ((parents[:, None] == index[None, :]) | (index[:, None] == index[None, :])).float()
    for _ in range((n - 1).bit_length()):
        steps = (steps @ steps > 0).float()
    position = base - 1 + steps.sum(1).to(torch.int64)
    return {"mask": _bit_words(steps > 0), "positions": position[:, None].expand(n, 3).contiguous()}


def _rotate(x, w, angle, eps):
    """Rows x heads x head_dim, normed a head and rotated by a row's angles."""
    pairs = angle.shape[1]
    y = x * torch.rsqrt(x.square().mean(2, keepdim=True) + eps) * w
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = y[:, :, :pairs], y[:, :, pairs:2 * pairs]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[:, :, 2 * pairs:]], 2)


def _angles(c, pos, base):
    """Rows x pairs, in 64 bits."""
    pairs = c["rope_dim"] // 2
    turn = torch.pow(torch.tensor(1e6, dtype=torch.float64, device="cuda"), torch.arange(pairs, device="cuda", dtype=torch.float64) * (-2.0 / c["rope_dim"]))
    if pos is None:
        return (base + torch.arange(c["rows"], device="cuda", dtype=torch.float64))[:, None] * turn
    sec_t, sec_h, _ = _sections(c["rope_dim"])
    j = torch.arange(pairs, device="cuda")
    axis = (j >= sec_t).long() + (j >= sec_t + sec_h).long()
    return pos.double()[:, axis] * turn


def _plain_rope(s):
    c = s["case"]
    rows, heads, kv, d = c["rows"], c["heads"], c["kv_heads"], c["head_dim"]
    angle = _angles(c, s.get("pos"), c["base"])
    fused = s["q"].reshape(rows, heads, -1)
    out = {"q": _rotate(fused[:, :, :d], s["wq"], angle, 1e-6).reshape(rows, heads * d)}
    if c["gated"]:
        out["gate"] = fused[:, :, d:].reshape(rows, heads * d).contiguous()
    s["cache"][s["first"]:] = _rotate(s["k"].reshape(rows, kv, d), s["wk"], angle, 1e-6).reshape(rows, kv * d)
    out["keys"] = s["cache"][s["first"]:]
    return out


def _values(kind, codes, scale, dtype=torch.float32):
    """The elements that a cache's rows stand for."""
    if kind in ("f32", "f16"):
        return codes.to(dtype)
    if kind == "fp8":
        return codes.view(torch.float8_e4m3fn).to(dtype) * scale.to(dtype)[:, None]
    if kind == "q8":
        return codes.view(torch.int8).to(dtype) * scale.to(dtype)[:, None]
    low, high = (codes & 15).to(torch.int8), (codes >> 4).to(torch.int8)
    pairs = torch.stack([low, high], 2).reshape(codes.shape[0], -1)
    return (pairs - 16 * (pairs > 7)).to(dtype) * scale.to(dtype)[:, None]


def _visible(c, mask):
    """Rows x keys: what a row sees."""
    m, t = c["rows"], c["rows"]
    bits = (mask.to(torch.int64)[:, :, None] >> torch.arange(32, device="cuda")) & 1
    seen = torch.cat([torch.ones(m, c["context"], dtype=torch.bool, device="cuda"), bits.reshape(m, -1)[:, :t] > 0], 1)
    if c["window"]:
        order = seen.to(torch.int32).cumsum(1)
        seen = seen & (order[:, -1:] - order < c["window"])
    return seen


def _plain_attend(s):
    c = s["case"]
    m, heads, kv, d = c["rows"], c["heads"], c["kv_heads"], c["head_dim"]
    group = heads // kv
    k = _values(c["cache"], s["k"], s["ks"]).view(-1, kv, d).permute(1, 2, 0).contiguous()
    v = _values(c["cache"], s["v"], s["vs"]).view(-1, kv, d).permute(1, 0, 2).contiguous()
    q = s["q"].view(m, kv, group, d).permute(1, 0, 2, 3).reshape(kv, m * group, d)
    score = torch.matmul(q, k).view(kv, m, group, -1) * (1.0 / math.sqrt(d))
    score = score.masked_fill(~_visible(c, s["mask"])[None, :, None, :], -math.inf)
    most = score.amax(3, keepdim=True)
    weight = torch.exp(score - most.masked_fill(most == -math.inf, 0.0))
    total = weight.sum(3, keepdim=True)
    weight = weight / total.masked_fill(total == 0, 1.0)
    out = torch.matmul(weight.view(kv, m * group, -1), v)
    return {"attended": out.view(kv, m, group, d).permute(1, 0, 2, 3).reshape(m, heads * d)}


def _top(x, k):
    """Columns of the k largest values of each row, equal ones by their column."""
    bits = (x + 0.0).contiguous().view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    key = (order << 32) - torch.arange(x.shape[1], device="cuda")
    return key.topk(k, dim=1).indices


def _plain_logprob(s):
    c, x = s["case"], s["logits"]
    most = x.amax(1, keepdim=True)
    e = torch.exp(x - most)
    total = e.sum(1, keepdim=True)
    logp = (x - most) - torch.log(total)
    out = {"logprobs": logp.gather(1, s["tokens"].long()),
           "entropy": -(e / total * logp.masked_fill(e == 0, 0.0)).sum(1)}
    if c["top_k"]:
        top = _top(x, c["top_k"])
        out["top_tokens"], out["top_logprobs"] = top.to(torch.int32), logp.gather(1, top)
    return out


# ---- the framework's calls ------------------------------------------------------------------------

def _f32_bits(x):
    return int(np.float32(x).view(np.uint32))


def _program(s):
    """The launch of a state and the tensors it fills: what a program keeps beside its buffers."""
    from tessera_amd import CreateBackend, KernelLaunch

    backend, c = CreateBackend(), s["case"]

    def wrap(t, more=0):
        return backend.WrapBuffer(t.data_ptr(), t.numel() * t.element_size() + more)

    def span(t):        # a block of columns of wider rows
        return backend.WrapBuffer(t.data_ptr(), 4 * ((t.shape[0] - 1) * t.stride(0) + t.shape[1]))

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda")

    kind = c["kind"]
    if kind == "mask":
        n = c["nodes"]
        out = {"mask": empty(n, (n + 31) // 32, dtype=torch.int32), "positions": empty(n, 3, dtype=torch.int64)}
        name, buffers, scalars, grid = "tree_mask", [wrap(s["parents"]), wrap(out["mask"]), wrap(out["positions"])], [n, c["base"]], 1
    elif kind == "rope":
        rows, heads, kv, d = c["rows"], c["heads"], c["kv_heads"], c["head_dim"]
        out = {"q": empty(rows, heads * d)}
        if c["gated"]:
            out["gate"] = empty(rows, heads * d)
        out["keys"] = s["cache"][s["first"]:]
        buffers = [span(s["q"]), span(s["k"]), wrap(s["wq"]), wrap(s["wk"])] + ([wrap(s["pos"])] if c["axes"] else [])
        buffers += [wrap(out["q"]), wrap(s["cache"])] + ([wrap(out["gate"])] if c["gated"] else [])
        scalars = [rows, heads, kv, d, c["rope_dim"]] + ([] if c["axes"] else [c["base"]])
        scalars += [_f32_bits(1e6), _f32_bits(1e-6), s["q"].stride(0), s["k"].stride(0), int(c["keys"] == "f16"), s["first"]]
        scalars += list(_sections(c["rope_dim"])) if c["axes"] else []
        name, grid = "qk_norm_mrope" if c["axes"] else "qk_norm_rope", rows
    elif kind == "attend":
        m, heads, kv, d, n = c["rows"], c["heads"], c["kv_heads"], c["head_dim"], c["context"] + c["rows"]
        out = {"attended": empty(m, heads * d)}
        plain = c["cache"] in ("f32", "f16")
        buffers = [wrap(s["q"]), wrap(s["k"]), wrap(s["v"])] + ([] if plain else [wrap(s["ks"]), wrap(s["vs"])])
        buffers += [wrap(s["mask"]), wrap(out["attended"])]
        scalars = [m, n, heads, kv, d, m, c["window"]] + ([int(c["cache"] == "f16")] if plain else [])
        name, grid = "attention_tree" if plain else "attention_tree_" + c["cache"], m * heads
    else:
        rows, k = c["rows"], c["top_k"]
        out = {"logprobs": empty(rows, c["tokens"]), "entropy": empty(rows)}
        if k:
            out.update(top_tokens=empty(rows, k, dtype=torch.int32), top_logprobs=empty(rows, k))
        buffers = [wrap(s["logits"]), wrap(s["tokens"])] + [wrap(t) for t in out.values()]
        name, scalars, grid = "token_logprobs", [rows, c["vocab"], c["tokens"], k, 0], rows
    launch = KernelLaunch(grid_x=grid, buffers=buffers, scalars=scalars)
    return backend.LaunchKernel, backend.LoadKernel(name), launch, out


def run(state):
    if own:
        if "program" not in state:
            state["program"] = _program(state)
        call, kernel, launch, out = state["program"]
        call(kernel, launch)
        return out
    kind = state["case"]["kind"]
    if kind == "mask":
        return _plain_mask(state)
    if kind == "rope":
        return _plain_rope(state)
    if kind == "attend":
        return _plain_attend(state)
    return _plain_logprob(state)


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    c, kind = case, case["kind"]
    if kind == "mask":
        n = c["nodes"]
        return {"bytes": 4 * n + 4 * n * ((n + 31) // 32) + 24 * n, "flops": 0}
    if kind == "rope":
        rows, q, k = c["rows"], c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
        wide = 2 * q if c["gated"] else q
        return {"bytes": rows * (8 * wide + k * (4 + (2 if c["keys"] == "f16" else 4)) + (24 if c["axes"] else 0)) + 8 * c["head_dim"],
                "flops": 6 * rows * (q + k)}
    if kind == "attend":
        m, heads, kv, d, past = c["rows"], c["heads"], c["kv_heads"], c["head_dim"], c["context"]
        keys = min(past, c["window"]) + m if c["window"] else past + m
        each = min(past + (m + 1) // 2, c["window"]) if c["window"] else past + (m + 1) // 2
        scales = 8 if c["cache"] in ("q8", "q4", "fp8") else 0
        return {"bytes": int(keys * (2 * kv * d * BYTES_KV[c["cache"]] + scales)) + 8 * m * heads * d + 4 * m * ((m + 31) // 32),
                "flops": 4 * m * each * heads * d}
    rows, vocab, k = c["rows"], c["vocab"], c["top_k"]
    return {"bytes": 4 * rows * vocab + rows * (8 * c["tokens"] + 4 + 8 * k), "flops": 5 * rows * vocab}


# ---- the definitions in 64 bits -------------------------------------------------------------------

def _exact_rope(c, s):
    rows, heads, kv, d, rd = c["rows"], c["heads"], c["kv_heads"], c["head_dim"], c["rope_dim"]
    pairs = rd // 2
    sec_t, sec_h, _ = _sections(rd)
    j = np.arange(pairs)
    freq = 1e6 ** (-2.0 * j / rd)
    if c["axes"]:
        pos = s["pos"].cpu().numpy()[:, np.where(j < sec_t, 0, np.where(j < sec_t + sec_h, 1, 2))]
    else:
        pos = (c["base"] + np.arange(rows))[:, None]
    z = torch.from_numpy(np.exp(1j * (pos * freq))).cuda()[:, None, :]

    def of(x, w):
        x = x.double()
        y = x / torch.sqrt((x * x).sum(2, keepdim=True) / d + 1e-6) * w.double()
        turned = torch.complex(y[..., :pairs].contiguous(), y[..., pairs:rd].contiguous()) * z
        return torch.cat([turned.real, turned.imag, y[..., rd:]], 2)

    fused = s["q"].reshape(rows, heads, -1)
    out = {"q": of(fused[..., :d], s["wq"]).reshape(rows, heads * d)}
    if c["gated"]:
        out["gate"] = fused[..., d:].reshape(rows, heads * d).double()
    out["keys"] = of(s["k"].reshape(rows, kv, d), s["wk"]).reshape(rows, kv * d)
    return out


def _exact_attend(c, s, seed):
    m, heads, kv, d, past = c["rows"], c["heads"], c["kv_heads"], c["head_dim"], c["context"]
    k = _values(c["cache"], s["k"], s["ks"], torch.float64).view(-1, kv, d)
    v = _values(c["cache"], s["v"], s["vs"], torch.float64).view(-1, kv, d)
    seen = _seen(_parents(seed, m, c["reach"], c["padding"]))
    out = torch.zeros(m, heads, d, dtype=torch.float64, device="cuda")
    for i in range(m):
        keys = np.concatenate([np.arange(past), past + np.nonzero(seen[i])[0]])
        if c["window"]:
            keys = keys[-c["window"]:]
        if not len(keys):
            continue
        at = torch.from_numpy(keys).cuda()
        for h in range(kv):
            q = s["q"][i].view(kv, -1, d)[h].double()
            p = torch.softmax(q @ k[at, h].t().contiguous() / math.sqrt(d), 1)
            out[i].view(kv, -1, d)[h] = p @ v[at, h]
    return {"attended": out.view(m, heads * d)}


def _exact_logprob(c, s):
    x = s["logits"].double()
    logp = x - torch.logsumexp(x, 1, keepdim=True)
    p = logp.exp()
    out = {"logprobs": logp.gather(1, s["tokens"].long()), "entropy": -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)}
    if c["top_k"]:
        out["top_tokens"] = None
        out["top_logprobs"] = torch.topk(logp, c["top_k"], dim=1).values
    return out


def exact(case, seed):
    c = case
    if c["kind"] == "mask":
        return None     # whole numbers
    s = prepare(c, seed)
    if c["kind"] == "rope":
        return _exact_rope(c, s)
    return _exact_attend(c, s, seed) if c["kind"] == "attend" else _exact_logprob(c, s)

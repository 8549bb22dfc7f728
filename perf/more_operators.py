"""A batch of sequences served from a paged cache of 8-bit keys and values, as measurable cases.

The cache is a pool of pages.  A page holds `block` positions of one sequence, keys [kv_head][position][element] and
values [kv_head][element][position], 8 bits each, under one fp32 scale for each page and key head.  A sequence's
row of the table names its pages in order.  Rows Starts[s] .. Starts[s + 1] - 1 of a call are the last positions of
sequence s, which then has Lens[s] of them: one row in decode, a few where drafted tokens are verified, many in
prefill.

  cache    "pages_write_q8", "pages_write_fp8" quantize a call's keys and values as they go into the pages (a page
           that grows past its scale is quantized again), "pages_read_q8", "pages_read_fp8" give rows back
  read     the reading alone
  attend   "attention_pages_q8", "attention_pages_fp8": each row against the positions up to its own, of those the
           last `window` and the first `sinks`
  verify   "draft_verify": how many of each sequence's drafted tokens stand, by the target's probabilities, the
           draft's and given random numbers, and the token that follows them

With ``own`` false, run() computes them in elementary operations in 32 bits (the verification, whose tokens hang on
sums next to a border, in 64); with ``own`` true it makes the launches that a program makes through
``tessera_amd.Backend``.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False


def listed():
    return [
        # one decoded token of one conversation: its key and value are written, nothing else; the launch is all there is
        {"name": "cache_one", "kind": "cache", "sequences": 1, "rows": 1, "past": 1186, "mix": 0, "kv_heads": 4, "head_dim": 64, "block": 16, "format": "q8",
         "back": 1, "f16": False, "fused": True},
        # a decode step of a full batch: each sequence's row joins a page that holds earlier ones
        {"name": "cache_batch", "kind": "cache", "sequences": 48, "rows": 1, "past": 8000, "mix": 1, "kv_heads": 4, "head_dim": 256, "block": 32, "format": "fp8",
         "back": 16, "f16": False, "fused": True},
        # a prefill chunk of three prompts that continue
        {"name": "cache_prefill", "kind": "cache", "sequences": 3, "rows": 1100, "past": 2000, "mix": 2, "kv_heads": 8, "head_dim": 128, "block": 64, "format": "q8",
         "back": 1100, "f16": True, "fused": True},
        # a long conversation leaves the pages for a contiguous fp16 cache
        {"name": "read_long", "kind": "read", "sequences": 1, "rows": 32768, "past": 0, "mix": 0, "kv_heads": 4, "head_dim": 256, "block": 16, "format": "fp8", "f16": True},
        # one decoded token of a small model
        {"name": "attend_one", "kind": "attend", "sequences": 1, "rows": 1, "past": 1186, "mix": 0, "heads": 16, "kv_heads": 4, "head_dim": 64, "block": 16, "format": "q8",
         "window": 0, "sinks": 0},
        # a decode step of a batch of conversations of all lengths
        {"name": "attend_batch", "kind": "attend", "sequences": 48, "rows": 1, "past": 8000, "mix": 1, "heads": 24, "kv_heads": 4, "head_dim": 256, "block": 32,
         "format": "q8", "window": 0, "sinks": 0},
        # drafts of four tokens against one very long context
        {"name": "attend_verify_long", "kind": "attend", "sequences": 1, "rows": 5, "past": 65000, "mix": 0, "heads": 32, "kv_heads": 8, "head_dim": 128, "block": 16,
         "format": "fp8", "window": 0, "sinks": 0},
        # streams that run for ever: the last 4096 positions and the first four, a few drafted rows a sequence
        {"name": "attend_stream", "kind": "attend", "sequences": 8, "rows": 5, "past": 130000, "mix": 3, "heads": 32, "kv_heads": 8, "head_dim": 128, "block": 64,
         "format": "q8", "window": 4096, "sinks": 4},
        # a prefill chunk of two prompts that continue
        {"name": "attend_prefill", "kind": "attend", "sequences": 2, "rows": 1500, "past": 2000, "mix": 4, "heads": 24, "kv_heads": 4, "head_dim": 256, "block": 32,
         "format": "q8", "window": 0, "sinks": 0},
        # one conversation's draft without probabilities (looked up, not sampled)
        {"name": "verify_one", "kind": "verify", "sequences": 1, "rows": 5, "mix": 0, "vocab": 131072, "draft": False, "temperature": 0.8, "banned": 0.0},
        # a batch's greedy drafts under a grammar that bans most tokens
        {"name": "verify_greedy", "kind": "verify", "sequences": 8, "rows": 5, "mix": 5, "vocab": 50001, "draft": False, "temperature": 0.0, "banned": 0.7},
        # a batch's drafts that were sampled from a draft model
        {"name": "verify_batch", "kind": "verify", "sequences": 32, "rows": 5, "mix": 6, "vocab": 131072, "draft": True, "temperature": 1.0, "banned": 0.0},
    ]


def draw(rng):
    def between(lo, hi, step=1):
        """A multiple of `step`, evenly over the logarithm of the range."""
        v = lo * (hi / lo) ** rng.random()
        return max(lo, min(hi, int(round(v / step)) * step))

    kind = rng.choice(["cache", "cache", "read", "attend", "attend", "attend", "attend", "verify", "verify"])
    sequences = rng.choice([1, between(1, 64)])
    case = {"kind": kind, "sequences": sequences, "mix": rng.randint(0, 1 << 20)}
    if kind == "verify":
        case.update(sequences=min(sequences, 32), rows=rng.choice([1, 2, 3, 4, 5]), vocab=between(500, 131072), draft=rng.random() < 0.5,
                    temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]), banned=rng.choice([0.0, 0.0, 0.5, 0.99]))
        return case
    head_dim, kv_heads = rng.choice([64, 64, 80, 96, 128, 128, 128, 256, 256]), rng.choice([1, 2, 4, 8])
    case.update(kv_heads=kv_heads, head_dim=head_dim, block=rng.choice([16, 16, 32, 64, 128]), format=rng.choice(["q8", "q8", "fp8"]))
    if kind == "read":
        case.update(sequences=min(sequences, 16), past=0, f16=rng.random() < 0.5)
        case.update(rows=between(1, 32768 * 1024 // max(1024, kv_heads * head_dim) // case["sequences"]))
        return case
    if kind == "cache":
        if rng.random() < 0.5:
            case.update(rows=rng.randint(1, 5))
        else:
            case.update(sequences=min(sequences, 4), rows=between(1, 2048 // min(sequences, 4)))
        case.update(past=rng.choice([0, between(1, 8192)]), back=rng.choice([1, between(1, 64)]), f16=rng.random() < 0.5, fused=rng.random() < 0.7)
        return case
    group = rng.choice([1, 2, 3, 4, 6, 8])
    while group * kv_heads * head_dim > 6144:
        group = rng.choice([1, 2, 3, 4, 6])
    window = between(8, 8192) if rng.random() < 0.4 else 0
    case.update(heads=group * kv_heads, window=window, sinks=rng.choice([0, 1, 4, 4, between(2, 300)]) if window else 0)
    regime = rng.choice(["decode", "decode", "verify", "prefill"])
    if regime == "prefill":
        case.update(sequences=min(sequences, 3), past=rng.choice([0, between(1, 2048)]))
        case.update(rows=between(1, 2048 // case["sequences"]))
    else:
        rows = 1 if regime == "decode" else rng.randint(1, 16 if sequences == 1 else 5)
        case.update(rows=rows, past=between(1, min(65536, 400000 // sequences)) if rng.random() < 0.95 else 0)
    return case


def _mixed(case):
    """Rows and earlier positions of each sequence: of a batch the first as the case says, the others fewer."""
    rs = np.random.RandomState(case["mix"])
    rows, past = [case["rows"]], [case.get("past", 0)]
    for _ in range(case["sequences"] - 1):
        rows.append(int(rs.randint(1, case["rows"] + 1)) if case["rows"] <= 16 else max(1, int(case["rows"] ** rs.uniform(0.5, 1.0))))
        past.append(int(rs.randint(0, past[0] + 1)))
    return rows, past


# ---- inputs --------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _ints(values):
    return torch.tensor(np.asarray(values, np.int64).astype(np.uint32).view(np.int32), device="cuda")


def _codes(fmt, x):
    """Numbers under their scale to codes: to nearest, ties to even."""
    if fmt == "q8":
        return x.clamp(-127, 127).round().to(torch.int8).view(torch.uint8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _numbers(fmt, codes, dtype=torch.float32):
    """What codes stand for, but for the scale."""
    return codes.view(torch.int8 if fmt == "q8" else torch.float8_e4m3fn).to(dtype)


def _most(fmt):
    return 127.0 if fmt == "q8" else 448.0


def _scale(fmt, largest):
    """A true quotient: by a number of the host it would be a product with the reciprocal."""
    return largest / torch.full_like(largest, _most(fmt))


def _pool(g, c, lens, width):
    """A pool with every sequence's pages written, in no order and with a few pages of nobody between them."""
    kv, d, block, fmt = c["kv_heads"], c["head_dim"], c["block"], c["format"]
    used = [-(-n // block) for n in lens]
    pages = sum(used) + 3 + sum(used) // 16
    order = torch.randperm(pages, device="cuda", generator=g)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n].to(torch.int32)
        at += n

    def plane(shape, spread):
        scale = (torch.rand(pages, kv, device="cuda", generator=g) * 0.5 + 0.75) * spread / _most(fmt)
        codes = torch.empty(pages, *shape, dtype=torch.uint8, device="cuda")
        for a in range(0, pages, 4096):      # (a piece at a time)
            part = codes[a:a + 4096]
            part.copy_(_codes(fmt, torch.randn(part.shape, device="cuda", generator=g) * (_most(fmt) / 4.0)))
        return codes, scale

    kp, ks = plane((kv, block, d), 4.0)
    vp, vs = plane((kv, d, block), 3.0)
    return {"table": table, "kp": kp, "ks": ks, "vp": vp, "vs": vs, "pages": pages, "width": width}


def prepare(case, seed):
    c, kind = case, case["kind"]
    s, g = {"case": dict(c)}, _gen(seed)
    rows, past = s["rows"], s["past"] = _mixed(c)
    starts = np.concatenate([[0], np.cumsum(rows)])
    s["m"], s["sequences"], s["starts"] = int(starts[-1]), len(rows), _ints(starts)
    if kind == "verify":
        m, vocab = s["m"], c["vocab"]
        x = torch.randn(m, vocab, device="cuda", generator=g) * 2.5
        if c["banned"]:
            x.masked_fill_(torch.rand(m, vocab, device="cuda", generator=g) < c["banned"], -math.inf)
            x[:, 3] = 1.0   # (the grammar allows something)
        s["logits"], s["random"] = x, torch.rand(m, 2, device="cuda", generator=g)
        if c["draft"]:      # a draft model's opinion, and tokens sampled from it
            s["draft"] = x + torch.randn(m, vocab, device="cuda", generator=g) * 0.5
            pick = torch.multinomial(torch.softmax(s["draft"] / (c["temperature"] or 1.0), 1), 1, generator=g)[:, 0]
        else:               # mostly the likeliest token
            pick = torch.where(torch.rand(m, device="cuda", generator=g) < 0.8, x.argmax(1), torch.randint(0, vocab, (m,), device="cuda", generator=g))
        s["tokens"] = torch.roll(pick, 1).to(torch.int32)
        return s
    lens = [a + b for a, b in zip(past, rows)]
    s["lens"], s["most_rows"], s["most_len"] = _ints(lens), max(rows), max(lens)
    s.update(_pool(g, c, lens, -(-max(lens) // c["block"]) + 1))
    wide = c["kv_heads"] * c["head_dim"]
    if kind == "cache":
        size = 3 * wide if c["fused"] else wide      # one projection's rows: queries (here as wide), keys, values
        x = torch.randn(s["m"], size, device="cuda", generator=g)
        x *= torch.exp(torch.randn(s["m"], 1, device="cuda", generator=g) * 0.5)     # (so that pages grow past their scale)
        s["k"] = x[:, wide:2 * wide] if c["fused"] else x
        s["v"] = x[:, 2 * wide:] if c["fused"] else torch.randn(s["m"], size, device="cuda", generator=g) * 0.7
        s["back"] = [min(c["back"], n) for n in lens]
        s["back_starts"] = _ints(np.concatenate([[0], np.cumsum(s["back"])]))
    elif kind == "attend":
        s["q"] = torch.randn(s["m"], c["heads"] * c["head_dim"], device="cuda", generator=g)
    return s


# ---- the plain forms ------------------------------------------------------------------------------

def _places(starts, lens, table, block, m):
    """Sequence, position, page and place in it of each row of a call."""
    starts, lens = starts.long(), lens.long()
    row = torch.arange(m, device="cuda")
    seq = (row[:, None] >= starts[None, 1:]).sum(1)
    pos = lens[seq] - starts[seq + 1] + row
    return seq, pos, table.long()[seq, pos // block], pos % block


def _plain_write(s):
    c = s["case"]
    kv, d, block, fmt, m = c["kv_heads"], c["head_dim"], c["block"], c["format"], s["m"]
    _, _, page, place = _places(s["starts"], s["lens"], s["table"], block, m)
    touched, of = torch.unique(page, return_inverse=True)
    n = touched.numel()
    first = torch.full((n,), block, device="cuda").scatter_reduce(0, of, place, "amin")
    held = (torch.arange(block, device="cuda")[None] < first[:, None])
    for rows, codes, scales, turned in ((s["k"], s["kp"], s["ks"], False), (s["v"], s["vp"], s["vs"], True)):
        x = rows.reshape(m, kv, d)
        most = _scale(fmt, torch.zeros(n, kv, device="cuda").scatter_reduce(0, of[:, None].expand(m, kv), x.abs().amax(2), "amax"))
        before = torch.where(first[:, None] > 0, scales[touched], torch.zeros(n, kv, device="cuda"))
        after = torch.maximum(before, most)
        under = torch.where(after > 0, after, torch.ones_like(after))[:, :, None, None]
        old = codes[touched].transpose(2, 3) if turned else codes[touched]       # [page][kv_head][position][element]
        old = _codes(fmt, _numbers(fmt, old.contiguous()) * before[:, :, None, None] / under)
        new = torch.where(held[:, None, :, None], old, torch.zeros_like(old))
        new[of, :, place] = _codes(fmt, x / under[of][:, :, 0])
        codes[touched] = new.transpose(2, 3) if turned else new
        scales[touched] = after


def _plain_read(s, starts, m, f16):
    c = s["case"]
    fmt, kv, d = c["format"], c["kv_heads"], c["head_dim"]
    _, _, page, place = _places(starts, s["lens"], s["table"], c["block"], m)
    k = _numbers(fmt, s["kp"][page, :, place]) * s["ks"][page][:, :, None]
    v = _numbers(fmt, s["vp"][page, :, :, place]) * s["vs"][page][:, :, None]
    out = [x.reshape(m, kv * d) for x in (k, v)]
    return {"k": out[0].half(), "v": out[1].half()} if f16 else {"k": out[0], "v": out[1]}


def _plain_attend(s):
    c = s["case"]
    heads, kv, d, block, fmt = c["heads"], c["kv_heads"], c["head_dim"], c["block"], c["format"]
    group, out, at = heads // kv, torch.empty(s["m"], heads * d, device="cuda"), 0
    for i, (rows, past) in enumerate(zip(s["rows"], s["past"])):
        n = past + rows
        low = max(0, past + 1 - c["window"]) if c["window"] else 0       # the first position of a row's window
        slot = torch.arange(-(-n // block), device="cuda")
        slot = slot[(slot * block < c["sinks"]) | (slot >= low // block)]
        pages, key = s["table"][i].long()[slot], (slot[:, None] * block + torch.arange(block, device="cuda")).view(1, -1)
        k = (_numbers(fmt, s["kp"][pages]) * s["ks"][pages][:, :, None, None]).permute(1, 3, 0, 2).reshape(kv, d, -1)
        v = (_numbers(fmt, s["vp"][pages]) * s["vs"][pages][:, :, None, None]).permute(1, 0, 3, 2).reshape(kv, -1, d)
        q = s["q"][at:at + rows].view(rows, kv, group, d).permute(1, 0, 2, 3).reshape(kv, rows * group, d)
        score = torch.matmul(q, k.contiguous()).view(kv, rows, group, -1) * (1.0 / math.sqrt(d))
        pos = past + torch.arange(rows, device="cuda")[:, None]
        seen = key <= pos
        if c["window"]:
            seen &= (key > pos - c["window"]) | (key < c["sinks"])
        score.masked_fill_(~seen[None, :, None, :], -math.inf)
        weight = torch.exp(score - score.amax(3, keepdim=True))
        weight /= weight.sum(3, keepdim=True)
        o = torch.matmul(weight.view(kv, rows * group, -1), v.contiguous())
        out[at:at + rows] = o.view(kv, rows, group, d).permute(1, 0, 2, 3).reshape(rows, heads * d)
        at += rows
    return {"attended": out}


def _plain_verify(s):
    c, m, dev = s["case"], s["m"], "cuda"
    starts, tokens, x = s["starts"].long(), s["tokens"].long(), s["logits"]
    row = torch.arange(m, device=dev)
    seq = (row[:, None] >= starts[None, 1:]).sum(1)
    last = starts[seq + 1] - 1
    drafted = tokens[torch.minimum(row + 1, last)]          # (of a sequence's last row none)
    if c["temperature"] == 0.0:
        best = torch.where(x == x.amax(1, keepdim=True), torch.arange(x.shape[1], device=dev), x.shape[1]).amin(1)
        stands = best == drafted
    else:
        p = torch.softmax(x.double() / c["temperature"], 1)
        q = torch.softmax(s["draft"].double() / c["temperature"], 1) if c["draft"] else None
        px = p.gather(1, drafted[:, None])[:, 0]
        qx = q.gather(1, drafted[:, None])[:, 0] if c["draft"] else 1.0
        stands = s["random"][:, 0].double() * qx < px
    stands &= row < last
    stop = torch.full((s["sequences"],), m, device=dev).scatter_reduce(0, seq, torch.where(stands, m, row), "amin")
    accepted = stop - starts[:-1]
    if c["temperature"] == 0.0:
        return {"accepted": accepted.to(torch.int32), "next": best[stop].to(torch.int32)}
    rest = p[stop]
    fails = (stop < starts[1:] - 1)[:, None]                # the draft's token was refused there: what the draft does not account for
    if c["draft"]:
        less = (rest - q[stop]).clamp_min(0.0)
    else:
        less = rest.scatter(1, drafted[stop][:, None], 0.0)
    rest = torch.where(fails & (less.sum(1, keepdim=True) > 0), less, rest)
    running = rest.cumsum(1)
    goal = s["random"][stop, 1].double()[:, None] * running[:, -1:]
    return {"accepted": accepted.to(torch.int32), "next": (running <= goal).sum(1).to(torch.int32)}


# ---- the framework's calls ------------------------------------------------------------------------

def _f32_bits(x):
    return int(np.float32(x).view(np.uint32))


def _program(s):
    """The launches of a state and the tensors they fill: what a program keeps beside its buffers."""
    from tessera_amd import CreateBackend, KernelLaunch

    backend, c = CreateBackend(), s["case"]

    def wrap(t):
        return backend.WrapBuffer(t.data_ptr(), t.numel() * t.element_size())

    def span(t):        # a block of columns of wider rows
        return backend.WrapBuffer(t.data_ptr(), 4 * ((t.shape[0] - 1) * t.stride(0) + t.shape[1]))

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda")

    kind, m, sequences = c["kind"], s["m"], s["sequences"]
    if kind == "verify":
        out = {"accepted": empty(sequences, dtype=torch.int32), "next": empty(sequences, dtype=torch.int32)}
        buffers = [wrap(s["logits"]), wrap(s["tokens"]), wrap(s["random"]), wrap(s["starts"])] + [wrap(t) for t in out.values()]
        buffers += [wrap(s["draft"])] if c["draft"] else []
        launches = [("draft_verify", buffers, [m, c["vocab"], sequences, _f32_bits(c["temperature"]), _f32_bits(c["temperature"])])]
    else:
        pool = [wrap(s["kp"]), wrap(s["vp"]), wrap(s["ks"]), wrap(s["vs"])]
        kv, d = c["kv_heads"], c["head_dim"]
        shape = [sequences, c["block"], s["pages"], s["width"]]
        launches = []
        if kind == "attend":
            out = {"attended": empty(m, c["heads"] * d)}
            buffers = [wrap(s["q"])] + pool + [wrap(s["table"]), wrap(s["starts"]), wrap(s["lens"]), wrap(out["attended"])]
            launches.append(("attention_pages_" + c["format"], buffers, [m, c["heads"], kv, d] + shape + [s["most_rows"], s["most_len"], c["window"], c["sinks"]]))
        else:
            starts, back = (s["back_starts"], sum(s["back"])) if kind == "cache" else (s["starts"], m)
            if kind == "cache":
                buffers = [span(s["k"]), span(s["v"]), wrap(s["table"]), wrap(s["starts"]), wrap(s["lens"])] + pool
                launches.append(("pages_write_" + c["format"], buffers, [m, kv, d] + shape + [s["k"].stride(0), s["v"].stride(0)]))
            out = {n: empty(back, kv * d, dtype=torch.float16 if c["f16"] else torch.float32) for n in ("k", "v")}
            buffers = pool + [wrap(s["table"]), wrap(starts), wrap(s["lens"]), wrap(out["k"]), wrap(out["v"])]
            launches.append(("pages_read_" + c["format"], buffers, [back, kv, d] + shape + [int(c["f16"])]))
    return backend.LaunchKernel, [(backend.LoadKernel(n), KernelLaunch(buffers=b, scalars=x)) for n, b, x in launches], out


def run(state):
    if own:
        if "program" not in state:
            state["program"] = _program(state)
        call, launches, out = state["program"]
        for kernel, launch in launches:
            call(kernel, launch)
        return out
    c = state["case"]
    if c["kind"] == "cache":
        _plain_write(state)
        return _plain_read(state, state["back_starts"], sum(state["back"]), c["f16"])
    if c["kind"] == "read":
        return _plain_read(state, state["starts"], state["m"], c["f16"])
    return _plain_attend(state) if c["kind"] == "attend" else _plain_verify(state)


# ---- what a pass cannot do without ----------------------------------------------------------------

def _visible(c):
    """(row, position) pairs that are seen, and positions that some row of their sequence sees."""
    pairs = keys = 0
    for rows, past in zip(*_mixed(c)):
        w, sinks, n = c["window"], c["sinks"], past + rows
        if not w:
            pairs, keys = pairs + rows * past + rows * (rows + 1) // 2, keys + n
            continue
        for p in range(past, n):
            low = max(0, p + 1 - w)
            pairs += p + 1 - low + min(sinks, low)
        low = max(0, past + 1 - w)
        keys += n - low + min(sinks, low)
    return pairs, keys


def work(case):
    c, kind = case, case["kind"]
    rows, past = _mixed(c)
    m = sum(rows)
    if kind == "verify":
        planes = 2 if c["draft"] and c["temperature"] else 1
        return {"bytes": 4 * m * c["vocab"] * planes + 12 * m + 8 * len(rows), "flops": 5 * m * c["vocab"] * planes}
    wide = c["kv_heads"] * c["head_dim"]
    if kind == "attend":
        pairs, keys = _visible(c)
        return {"bytes": 2 * keys * wide + 8 * c["kv_heads"] * (keys // c["block"] + 1) + 8 * m * c["heads"] * c["head_dim"], "flops": 4 * pairs * c["heads"] * c["head_dim"]}
    out = 2 * (2 if c["f16"] else 4)
    if kind == "read":
        return {"bytes": m * wide * (2 + out), "flops": 2 * m * wide}
    back = sum(min(c["back"], a + b) for a, b in zip(rows, past))
    old = sum(p % c["block"] for p in past)     # rows of pages that are continued
    return {"bytes": wide * (m * (8 + 2) + old * (2 + 2) + back * (2 + out)), "flops": 4 * m * wide + 2 * back * wide}


# ---- the definitions in 64 bits -------------------------------------------------------------------

_E4M3 = np.array([(-1.0) ** (b >> 7) * ((b & 7) * 2.0 ** -9 if b >> 3 & 15 == 0 else (8 + (b & 7)) * 2.0 ** ((b >> 3 & 15) - 10)) for b in range(256)])


def _decoded(fmt, codes):
    """Codes as 64-bit numbers, on the host."""
    b = codes.cpu().numpy()
    return b.view(np.int8).astype(np.float64) if fmt == "q8" else _E4M3[b]


def _nearest(fmt, x):
    """The number that a code can stand for nearest to x; ties to the even code."""
    x = np.clip(x, -_most(fmt), _most(fmt))
    if fmt == "q8":
        return np.rint(x)
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -20))), -6) - 3)
    return np.rint(x / step) * step


def _f32(x):
    return x.astype(np.float32).astype(np.float64)


def _exact_rows(c, s, back):
    """The rows that are read: the scale is the fp32 number nearest to largest / 127 (448), a code the nearest to
    the fp32 quotient, a row the fp32 (then fp16) number nearest to their product."""
    fmt, block, kv, d = c["format"], c["block"], c["kv_heads"], c["head_dim"]
    out, at = {"k": [], "v": []}, 0
    table = s["table"].cpu().numpy()
    with np.errstate(divide="ignore", invalid="ignore"):
        for i, (rows, past) in enumerate(zip(s["rows"], s["past"])):
            n = past + rows
            first = (n - back[i]) // block
            if c["kind"] == "cache":
                first = min(first, past // block)
            pages = table[i, first:-(-n // block)].astype(np.int64)
            index = torch.from_numpy(pages).cuda()
            for name, codes, scales in (("k", s["kp"], s["ks"]), ("v", s["vp"], s["vs"])):
                number = _decoded(fmt, codes[index])
                if name == "v":
                    number = number.transpose(0, 1, 3, 2)
                number, scale = number.copy(), scales[index].cpu().numpy().astype(np.float64)
                if c["kind"] == "cache":
                    new = s[name][at:at + rows].cpu().numpy().astype(np.float64).reshape(rows, kv, d)
                    for j in range(len(pages)):
                        lo, hi = (first + j) * block, (first + j + 1) * block
                        a, b = max(lo, past), min(hi, n)
                        if a >= b:
                            continue
                        x = new[a - past:b - past].transpose(1, 0, 2)
                        was = scale[j] if a > lo else np.zeros(kv)
                        now = np.maximum(was, _f32(np.abs(x).max((1, 2)) / _most(fmt)))
                        number[j, :, :a - lo] = _nearest(fmt, _f32(_f32(number[j, :, :a - lo] * was[:, None, None]) / now[:, None, None]))
                        number[j, :, a - lo:b - lo] = _nearest(fmt, _f32(x / now[:, None, None]))
                        scale[j] = now
                value = _f32(number * scale[:, :, None, None]).transpose(0, 2, 1, 3).reshape(len(pages) * block, kv * d)
                out[name].append(value[n - back[i] - first * block:n - first * block])
            at += rows
    made = {k: torch.from_numpy(np.concatenate(v)) for k, v in out.items()}
    return {k: v.half().double() for k, v in made.items()} if c["f16"] else made


def _exact_attend(c, s):
    heads, kv, d, fmt, block = c["heads"], c["kv_heads"], c["head_dim"], c["format"], c["block"]
    level = torch.from_numpy(_E4M3 if fmt == "fp8" else np.arange(256, dtype=np.uint8).view(np.int8).astype(np.float64)).cuda()
    out, at = torch.empty(s["m"], kv, heads // kv, d, dtype=torch.float64, device="cuda"), 0
    for i, (rows, past) in enumerate(zip(s["rows"], s["past"])):
        n = past + rows
        pages = s["table"][i].long()[:(n + block - 1) // block]
        for h in range(kv):
            k = level[s["kp"][pages, h].long()].mul_(s["ks"][pages, h].double()[:, None, None]).reshape(-1, d)[:n]
            v = level[s["vp"][pages, h].long()].mul_(s["vs"][pages, h].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:n]
            for a in range(0, rows, 256):
                b = min(rows, a + 256)
                q = s["q"][at + a:at + b].view(b - a, kv, -1, d)[:, h].double()
                score = torch.matmul(q.reshape(-1, d), k.t().contiguous()).view(b - a, -1, n) / math.sqrt(d)
                age = (past + torch.arange(a, b, device="cuda"))[:, None] - torch.arange(n, device="cuda")[None]
                hidden = age < 0
                if c["window"]:
                    hidden |= (age >= c["window"]) & (torch.arange(n, device="cuda") >= c["sinks"])[None]
                weight = torch.softmax(score.masked_fill(hidden[:, None], -math.inf), 2)
                out[at + a:at + b, h] = torch.matmul(weight.view(-1, n), v).view(b - a, -1, d)
        at += rows
    return {"attended": out.view(s["m"], heads * d)}


def exact(case, seed):
    c = case
    if c["kind"] == "verify":
        return None     # whole numbers
    s = prepare(c, seed)
    if c["kind"] == "attend":
        return _exact_attend(c, s)
    return _exact_rows(c, s, s["back"] if c["kind"] == "cache" else s["rows"])

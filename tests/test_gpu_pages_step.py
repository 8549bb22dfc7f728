"""The paged cache's ids together, as a program that decodes a batch with drafts uses them: norm and rotation, rows into pages, attention,
log probabilities that stand for a model's head, the verification, and on from the tokens that stand."""
import numpy as np
import pytest

import pages_reference as ref
from tessera_amd import KernelLaunch
from test_gpu_pages import Batch
from test_gpu_tree import f32_bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["q8", "fp8"])
def test_decoding_with_drafts(backend, fmt):
    rs = np.random.RandomState(3)
    sequences, kv, group, d, block, vocab = 5, 2, 4, 64, 16, 700
    heads = kv * group
    lens = rs.randint(10, 40, sequences)                                            # prompts
    b = Batch(backend, 5, fmt, kv, block, d, lens + 64)                             # room for what is decoded
    wide_q, wide_k = heads * d, kv * d
    embed = rs.randn(vocab, wide_q + 2 * wide_k).astype(np.float32)                 # a layer's fused projection, by token
    head = (rs.randn(wide_q, vocab) * 0.5).astype(np.float32)
    up = backend.Upload
    weights = [up(np.ones(d, np.float32)) for _ in range(2)]

    def launch(name, buffers, scalars):
        backend.LaunchKernel(backend.LoadKernel(name), KernelLaunch(buffers=buffers, scalars=scalars))

    def rotated(x, n_heads, positions):
        """RMS norm and rotary embedding in fp64: tests/test_gpu_tree.py holds the id to it; here it says what the pages should hold."""
        y = x.reshape(len(x), n_heads, d).astype(np.float64)
        y = y / np.sqrt((y * y).mean(2, keepdims=True) + 1e-6)
        angle = positions[:, None] * 1e4 ** (-2.0 * np.arange(d // 2) / d)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        return np.concatenate([y[..., :d // 2] * c - y[..., d // 2:] * s, y[..., d // 2:] * c + y[..., :d // 2] * s], 2)

    def step(tokens, rows, lengths):
        """One pass over `rows` tokens of each sequence; logits of every row."""
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32)
        m = int(starts[-1])
        fused = embed[tokens]
        positions = np.concatenate([np.arange(n - r, n) for n, r in zip(lengths, rows)])
        dev = up(fused)
        span = lambda at, n: backend.WrapBuffer(dev.Handle() + 4 * at, 4 * ((m - 1) * fused.shape[1] + n))      # noqa: E731
        q, k, out = (backend.AllocateBuffer(4 * m * n) for n in (wide_q, wide_k, wide_q))
        pos = up(np.repeat(positions[:, None], 3, 1).astype(np.uint64))
        launch("qk_norm_mrope", [span(0, wide_q), span(wide_q, wide_k), *weights, pos, q, k],
               [m, heads, kv, d, d, f32_bits(1e4), f32_bits(1e-6), fused.shape[1], fused.shape[1], 0, 0, d // 2, 0, 0])
        dev_starts, dev_lens = up(starts), up(np.asarray(lengths, np.uint32))
        b.go("pages_write", [k, span(wide_q + wide_k, wide_k), b.dev_table, dev_starts, dev_lens, *b.dev], [m, kv, d, *b.shape, 0, fused.shape[1]])
        b.go("attention_pages", [q, *b.dev, b.dev_table, dev_starts, dev_lens, out], [m, heads, kv, d, *b.shape, int(max(rows)), int(max(lengths)), 0, 0])
        attended = backend.CopyD2H(out, dtype=np.float32).reshape(m, heads, d)
        # what the pages should hold and the rows see
        b.lens = np.asarray(lengths, np.uint32)
        dq, dk = backend.CopyD2H(q, dtype=np.float32).reshape(m, -1), backend.CopyD2H(k, dtype=np.float32).reshape(m, -1)
        for got, want in ((dq, rotated(fused[:, :wide_q], heads, positions)), (dk, rotated(fused[:, wide_q:wide_q + wide_k], kv, positions))):
            assert np.abs(got.reshape(want.shape) - want).max() <= 1e-5
        b.pool = b.want_write(rows, dk, np.ascontiguousarray(fused[:, wide_q + wide_k:]))
        b.same_as(b.pool)
        for s, n in enumerate(rows):
            want, bound = ref.attention(b.pool, b.table[s], int(lengths[s]), dq[starts[s]:starts[s + 1]].reshape(n, heads, d), group)
            assert (np.abs(attended[starts[s]:starts[s + 1]] - want) <= bound).all()
        return (attended.reshape(m, -1) @ head).astype(np.float32), starts

    tokens = rs.randint(0, vocab, int(lens.sum()))
    logits, starts = step(tokens, lens, lens)
    now = logits[starts[1:] - 1].argmax(1)                                          # the first token of each sequence
    lengths, standing = lens.copy(), 0
    for turn in range(6):
        drafted = rs.randint(0, 4, sequences)                                       # some sequences have no draft
        rows = drafted + 1
        batch = np.concatenate([[t, *rs.randint(0, vocab, n)] for t, n in zip(now, drafted)]).astype(np.int64)
        if turn % 2 == 0:                                                           # drafts that stand: what greedy decoding says, a token at a time, on a copy
            for i in range(int(drafted.max(initial=0))):
                keep = b.device_pool()
                look, at = step(batch, rows, lengths + rows)
                for s in range(sequences):
                    if i < drafted[s]:
                        batch[at[s] + i + 1] = look[at[s] + i].argmax()
                b.pool = keep
                b.upload()
        logits, starts = step(batch, rows, lengths + rows)
        draft = (logits + rs.randn(*logits.shape)).astype(np.float32)
        random = rs.rand(len(batch), 2).astype(np.float32)
        for temperature, of in ((0.0, None), (0.8, draft), (0.8, None)):
            out = [up(np.zeros(sequences, np.uint32)) for _ in range(2)]
            launch("draft_verify", [up(logits), up(batch.astype(np.uint32)), up(random), up(starts), *out] + ([up(of)] if of is not None else []),
                   [*logits.shape, sequences, f32_bits(temperature), f32_bits(temperature)])
            got = [backend.CopyD2H(x, dtype=np.uint32) for x in out]
            assert list(zip(*got)) == ref.verify(logits, batch, random, starts, temperature, of, temperature)
            if temperature == 0.0:
                accepted, now = got[0].astype(np.int64), got[1].astype(np.int64)
        # (on even turns nearly all stand: a later draft's rows change the scale that earlier rows of its page are quantized under)
        standing += int(accepted.sum())
        lengths = lengths + accepted + 1                                            # refused rows' positions are written over
    assert standing > 0

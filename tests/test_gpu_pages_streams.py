"""The paged cache's ids and "draft_verify" on several streams at once, recorded beside eager ones and replayed with other lengths,
through the entry point that allocates nothing, with a caller's workspace set, and without a scratch block."""
import numpy as np
import pytest
import torch

from tessera_amd import KernelLaunch
from test_gpu_streams import Call, home, record     # noqa: F401 (a fixture)
from test_gpu_tree import f32_bits

pytestmark = pytest.mark.gpu


class Pages(Call):
    """Call with its buffers made here; `y` holds all its results.  `rows` of each of `lens` positions."""

    def __init__(self, backend, kind, rows, lens, seed, most_len=0):
        dev = torch.device("cuda:0")
        g = torch.Generator(device="cuda").manual_seed(seed)
        randn = lambda *s: torch.randn(*s, device=dev, generator=g)                      # noqa: E731
        ints = lambda x: torch.from_numpy(np.asarray(x, np.int32)).to(dev)               # noqa: E731
        wrap = lambda t: backend.WrapBuffer(t.data_ptr(), t.numel() * t.element_size())  # noqa: E731
        self.backend, self.k, self.m, self.n = backend, kind, sum(rows), 0
        starts, sequences, m = ints(np.concatenate([[0], np.cumsum(rows)])), len(rows), sum(rows)
        if kind == "draft_verify":
            vocab = lens[0]
            logits = randn(m, vocab) * 3
            self.held = [logits, (logits.argmax(1).roll(1)).to(torch.int32), torch.rand(m, 2, device=dev, generator=g), starts, logits + randn(m, vocab) * 0.3]
            half = (sequences + 3) // 4 * 4
            self.y = torch.zeros(2 * half, device=dev)
            buffers, scalars = [*self.held[:4], self.y[:sequences], self.y[half:half + sequences], self.held[4]], [m, vocab, sequences, f32_bits(1.0), f32_bits(1.0)]
            self.used = np.concatenate([np.arange(sequences), half + np.arange(sequences)])
        else:
            heads, kv, d, block = 12, 2, 128, 32
            width = max(-(-n // block) for n in lens) + 1
            pages = sum(-(-n // block) for n in lens) + 2
            order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
            table, at = torch.zeros(sequences, width, dtype=torch.int32, device=dev), 0
            for s, n in enumerate(lens):
                table[s, :-(-n // block)] = order[at:at + -(-n // block)]
                at += -(-n // block)
            self.lens = ints(lens)
            codes = [torch.randint(-100, 101, (pages, kv, block * d), device=dev, generator=g).to(torch.int8) for _ in range(2)]
            if kind.endswith("fp8"):
                codes = [(c.float() * 0.5).to(torch.float8_e4m3fn) for c in codes]
            scales = [(torch.rand(pages, kv, device=dev, generator=g) + 0.5) / 100 for _ in range(2)]
            pool, shape = [*codes, *scales], [sequences, block, pages, width]
            if kind.startswith("attention"):
                q = randn(m, heads * d)
                self.y = torch.zeros(m * heads * d, device=dev)
                buffers = [q, *pool, table, starts, self.lens, self.y]
                scalars = [m, heads, kv, d, *shape, max(rows), most_len, 0, 0]
            elif kind.startswith("pages_read"):
                self.y = torch.zeros(2 * m * kv * d, device=dev)
                buffers, scalars = [*pool, table, starts, self.lens, self.y[:m * kv * d], self.y[m * kv * d:]], [m, kv, d, *shape, 0]
            else:       # the pool is the result
                sizes = [pages * kv * block * d // 4] * 2 + [pages * kv] * 2
                ends = np.cumsum([(s + 3) // 4 * 4 for s in sizes])
                self.y = torch.zeros(int(ends[-1]), device=dev)
                pool = [self.y[e - (s + 3) // 4 * 4:e - (s + 3) // 4 * 4 + s] for s, e in zip(sizes, ends)]
                buffers, scalars = [randn(m, kv * d), randn(m, kv * d), table, starts, self.lens, *pool], [m, kv, d, *shape, 0, 0]
            self.held, self.used = buffers, np.arange(self.y.numel())
        self.kernel = backend.LoadKernel(kind)
        self.launch = KernelLaunch(buffers=[wrap(t) for t in buffers], scalars=scalars)

    def bits(self):
        return super().bits()[self.used]

    def alone(self, stream):
        self.y.zero_()
        torch.cuda.synchronize()
        self.go(stream)
        torch.cuda.synchronize()
        return self.bits()


# (each writes whole pages, from their first position: a pool that was cleared gives the same bits again)
CALLS = [("pages_write_q8", [64, 7], [64, 7]), ("pages_write_fp8", [33], [65]), ("pages_read_q8", [90, 3], [200, 35]), ("pages_read_fp8", [5], [70]),
         ("attention_pages_q8", [1] * 5, [1900, 33, 700, 64, 5000]), ("attention_pages_fp8", [2], [20000]), ("attention_pages_q8", [200, 1, 30], [260, 900, 30]),
         ("attention_pages_q8", [1] * 6, [12000, 300, 9000, 64, 12000, 5000]), ("attention_pages_fp8", [5, 3, 4], [16000, 9000, 500]),
         ("draft_verify", [5, 1, 4], [40001]), ("draft_verify", [3] * 9, [3000])]


@pytest.mark.parametrize("spec", CALLS)
def test_two_streams_at_once(backend, home, spec):      # noqa: F811
    one, two = Pages(backend, *spec, 1), Pages(backend, *spec, 2)
    want = one.alone(home), two.alone(home)
    assert not np.array_equal(*want)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        one.y.zero_(), two.y.zero_()
        torch.cuda.synchronize()
        for _ in range(30):
            one.go(s)
            two.go(t)
        torch.cuda.synchronize()
        assert np.array_equal(one.bits(), want[0]) and np.array_equal(two.bits(), want[1])


def test_recorded_calls_beside_eager_ones(backend, home):       # noqa: F811
    first, second, eager = ([Pages(backend, *s, seed + i) for i, s in enumerate(CALLS)] for seed in (10, 20, 30))
    want = [[c.alone(home) for c in group] for group in (first, second, eager)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = record(first, side), record(second, side)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        for c in (*first, *second, *eager):
            c.y.zero_()
        torch.cuda.synchronize()
        for _ in range(10):
            with torch.cuda.stream(s):
                graphs[0].replay()
            with torch.cuda.stream(t):
                graphs[1].replay()
            for c in eager:
                c.go(side)
        torch.cuda.synchronize()
        for group, bits in zip((first, second, eager), want):
            for c, b in zip(group, bits):
                assert np.array_equal(c.bits(), b), (c.k, c.m)


@pytest.mark.parametrize("spec", CALLS)
def test_same_kernels_whatever_ran_before(backend, home, spec):     # noqa: F811
    call = Pages(backend, *spec, 40)
    assert backend.WorkspaceBytes(call.kernel, call.launch.scalars) == 0
    graph = record([call])
    for _ in range(3):
        call.y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        recorded = call.bits()
        eager = call.alone(home)
        assert np.array_equal(recorded, eager)
    small = torch.empty(256, dtype=torch.uint8, device="cuda")
    backend.SetWorkspace(backend.WrapBuffer(small.data_ptr(), 256))
    assert np.array_equal(call.alone(home), eager)
    backend.SetWorkspace(None)
    call.y.zero_()
    call.go(home, no_alloc=True)
    torch.cuda.synchronize()
    assert np.array_equal(call.bits(), eager)
    # without a block (the per-thread stream): attention the same to fp32 rounding, the others the same bits
    call.y.zero_()
    torch.cuda.synchronize()
    backend.SetStream(2)
    backend.LaunchKernel(call.kernel, call.launch)
    torch.cuda.synchronize()
    plain = call.bits()
    if not call.k.startswith("attention"):
        assert np.array_equal(plain, eager)
        return
    plain, eager = (b.view(np.float32).astype(np.float64) for b in (plain, eager))
    assert np.isfinite(eager).all() and np.linalg.norm(plain - eager) <= 1e-6 * np.linalg.norm(plain)


def test_a_recorded_step_goes_on(backend, home):        # noqa: F811
    """One recording for every later length: the lengths and the tables are the device's."""
    call = Pages(backend, "attention_pages_q8", [1, 1, 1], [3000, 3000, 3000], 50, most_len=3000)
    graph = record([call])
    rs = np.random.RandomState(0)
    for _ in range(5):
        lens = rs.randint(1, 3001, 3)
        call.lens.copy_(torch.from_numpy(lens.astype(np.int32)))
        call.y.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        recorded = call.bits()
        assert np.array_equal(call.alone(home), recorded) and np.isfinite(recorded.view(np.float32)).all()

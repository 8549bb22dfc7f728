"""The tree's ids, whose parts of keys and shares of rows lie in a stream's scratch block, on several streams at once, recorded
beside eager ones, through the entry point that allocates nothing, with a caller's workspace set, and without a block."""
import numpy as np
import pytest
import torch

import tree_reference as ref
from tessera_amd import KernelLaunch
from test_gpu_streams import Call, home, record     # noqa: F401 (a fixture)
from test_gpu_tree import f32_bits

pytestmark = pytest.mark.gpu


class Tree(Call):
    """Call with its buffers made here; `y` holds all its results."""

    def __init__(self, backend, kind, m, n, seed):
        dev = torch.device("cuda:0")
        g = torch.Generator(device="cuda").manual_seed(seed)
        rs = np.random.RandomState(seed)
        randn = lambda *s: torch.randn(*s, device=dev, generator=g)                      # noqa: E731
        put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)                # noqa: E731
        wrap = lambda t: backend.WrapBuffer(t.data_ptr(), t.numel() * t.element_size())  # noqa: E731
        self.backend, self.k, self.m, self.n = backend, kind, m, n
        parents = ref.random_parents(rs, min(m, 1024), 5)
        heads, kv, d = 24, 4, 128
        sizes = []      # of the results, in floats, each from a multiple of four on
        if kind == "tree_mask":
            self.held, scalars, sizes = [put(parents.view(np.int32))], [m, n], [m * ((m + 31) // 32), m * 6]
        elif kind == "qk_norm_rope":
            self.held = [randn(m, heads * d), randn(m, kv * d), randn(d), randn(d)]
            scalars, sizes = [m, heads, kv, d, d, n, f32_bits(1e6), f32_bits(1e-6), 0, 0, 0, 0], [m * heads * d, m * kv * d]
        elif kind.startswith("attention_tree"):
            q, k, v = randn(m, heads * d), randn(n, kv * d), randn(n, kv * d)
            words = put(ref.words_of(ref.seen_of(parents)).view(np.int32))
            if kind == "attention_tree":
                self.held, tail = [q, k.half(), v.half(), words], [1]
            else:
                codes = [(x * 40).round().clamp(-127, 127).to(torch.int8) for x in (k, v)]
                self.held, tail = [q, *codes, *((torch.rand(n, device=dev, generator=g) + 0.5) / 40 for _ in range(2)), words], []
            scalars, sizes = [m, n, heads, kv, d, m, 0, *tail], [m * heads * d]
        else:
            self.held = [randn(m, n) * 3, put(rs.randint(0, n, (m, 2)).astype(np.int32))]
            scalars, sizes = [m, n, 2, 7, 0], [m * 2, m, m * 7, m * 7]
        starts = np.concatenate([[0], np.cumsum([(s + 3) // 4 * 4 for s in sizes])])
        self.y = torch.zeros(int(starts[-1]), device=dev)
        results = [self.y[a:a + s] for a, s in zip(starts, sizes)]
        self.kernel = backend.LoadKernel(kind)
        self.launch = KernelLaunch(grid_x=m, buffers=[wrap(t) for t in (*self.held, *results)], scalars=scalars)
        self.used = np.concatenate([np.arange(a, a + s) for a, s in zip(starts, sizes)])

    def bits(self):
        return super().bits()[self.used]


CALLS = [("tree_mask", 200, 77), ("qk_norm_rope", 40, 5000), ("attention_tree", 33, 2100), ("attention_tree_q8", 5, 3000),
         ("attention_tree", 2, 900), ("token_logprobs", 1, 131072), ("token_logprobs", 40, 40001)]


@pytest.mark.parametrize("spec", CALLS)
def test_two_streams_at_once(backend, home, spec):      # noqa: F811
    one, two = Tree(backend, *spec, 1), Tree(backend, *spec, 2)
    want = one.alone(home), two.alone(home)
    assert not np.array_equal(*want)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        one.y.fill_(float("nan")), two.y.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(30):
            one.go(s)
            two.go(t)
        torch.cuda.synchronize()
        assert np.array_equal(one.bits(), want[0]) and np.array_equal(two.bits(), want[1])


def test_recorded_calls_beside_eager_ones(backend, home):       # noqa: F811
    first, second, eager = ([Tree(backend, *s, seed + i) for i, s in enumerate(CALLS)] for seed in (10, 20, 30))
    want = [[c.alone(home) for c in group] for group in (first, second, eager)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = record(first, side), record(second, side)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        for c in (*first, *second, *eager):
            c.y.fill_(float("nan"))
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
                assert np.array_equal(c.bits(), b), (c.k, c.m, c.n)


@pytest.mark.parametrize("spec", CALLS)
def test_same_kernels_whatever_ran_before(backend, home, spec):     # noqa: F811
    call = Tree(backend, *spec, 40)
    assert backend.WorkspaceBytes(call.kernel, call.launch.scalars) == 0
    graph = record([call])
    for _ in range(3):
        call.y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        recorded = call.bits()
        eager = call.alone(home)
        assert np.array_equal(recorded, eager)
    small = torch.empty(256, dtype=torch.uint8, device="cuda")
    backend.SetWorkspace(backend.WrapBuffer(small.data_ptr(), 256))
    assert np.array_equal(call.alone(home), eager)
    backend.SetWorkspace(None)
    call.y.fill_(float("nan"))
    call.go(home, no_alloc=True)
    torch.cuda.synchronize()
    assert np.array_equal(call.bits(), eager)
    # without a block (the per-thread stream): the same to fp32 rounding, the same tokens
    call.y.fill_(float("nan"))
    torch.cuda.synchronize()
    backend.SetStream(2)
    backend.LaunchKernel(call.kernel, call.launch)
    torch.cuda.synchronize()
    plain = call.bits()
    if call.k in ("tree_mask", "qk_norm_rope"):
        assert np.array_equal(plain, eager)
        return
    if call.k == "token_logprobs":
        m = call.m
        assert np.array_equal(plain[3 * m:10 * m], eager[3 * m:10 * m])       # the tokens
        plain, eager = (np.concatenate([b[:3 * m], b[10 * m:]]) for b in (plain, eager))
    plain, eager = (b.view(np.float32).astype(np.float64) for b in (plain, eager))
    assert np.isfinite(eager).all() and np.linalg.norm(plain - eager) <= 1e-6 * np.linalg.norm(plain)

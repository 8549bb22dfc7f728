"""Launches of the tree's ids that are refused, before any device work: one of every kind that test_tree_args.py goes
through without a device."""
import numpy as np
import pytest

from tessera_amd import KernelLaunch, StatusCode, StatusError
from test_gpu_tree import f32_bits

pytestmark = pytest.mark.gpu


def test_refusals_leave_everything_as_it_was(backend):
    up = lambda n: backend.Upload(np.full(n, 7.0, np.float32))    # noqa: E731
    a, b, c, d, e, f, g = (up(4096) for _ in range(7))

    def refused(name, buffers, scalars):
        with pytest.raises(StatusError) as error:
            backend.LaunchKernel(backend.LoadKernel(name), KernelLaunch(buffers=buffers, scalars=scalars))
        assert error.value.code == StatusCode.InvalidArgument, (name, scalars)
        assert name.split("_")[0] in str(error.value)

    theta, eps = f32_bits(1e4), f32_bits(1e-6)
    refused("tree_mask", [a, b, c], [1025, 0])
    refused("tree_mask", [a, a, c], [4, 0])
    refused("qk_norm_rope", [a, b, c, d, e, f], [2, 4, 2, 64, 64, 0, theta, eps, 0, 0, 0, 40])
    refused("qk_norm_rope", [a, b, c, d, e, e], [2, 4, 2, 64, 64, 0, theta, eps, 0, 0, 0, 0])
    refused("qk_norm_rope", [a, b, c, d, a, f], [2, 4, 2, 64, 64, 0, theta, eps, 300, 0, 0, 0])
    refused("qk_norm_mrope", [a, b, c, d, e, f, g], [2, 4, 2, 64, 64, theta, eps, 0, 0, 0, 0, 20, 10, 10])
    refused("qk_norm_mrope", [a, b, c, d, e, f, g], [2, 4, 2, 257, 64, theta, eps, 0, 0, 0, 0, 0, 0, 0])
    refused("attention_tree", [a, b, c, d, e], [2, 8, 4, 2, 64, 9, 0, 0])
    refused("attention_tree", [a, b, c, d, a], [2, 8, 4, 2, 64, 2, 0, 0])
    refused("attention_tree", [a, b, c, d, e], [2, 800, 4, 2, 64, 2, 0, 0])
    for kind in ("q8", "q4", "fp8"):
        refused("attention_tree_" + kind, [a, b, c, d, e, f, g], [2, 8, 4, 2, 64, 0, 0])
        refused("attention_tree_" + kind, [a, b, c, d, e, f], [2, 8, 4, 2, 64, 2, 0])
    refused("token_logprobs", [a, b, c, d, e, f], [2, 100, 1, 33, 0])
    refused("token_logprobs", [a, b, c, d], [2, 100, 1, 4, 0])
    refused("token_logprobs", [a, b, c, c], [2, 100, 1, 0, 0])
    off = backend.WrapBuffer(a.Handle() + 4, a.Size() - 4)
    with pytest.raises(StatusError):
        backend.LaunchKernel(backend.LoadKernel("token_logprobs"), KernelLaunch(buffers=[off, b, c, d], scalars=[2, 100, 1, 0, 0]))
    backend.Synchronize()
    assert all(np.all(backend.CopyD2H(x, dtype=np.float32) == 7.0) for x in (a, b, c, d, e, f, g))

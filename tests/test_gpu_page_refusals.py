"""Launches of the paged cache's ids and of "draft_verify" that are refused, before any device work: one of every kind that
test_page_args.py goes through without a device."""
import numpy as np
import pytest

from tessera_amd import KernelLaunch, StatusCode, StatusError
from test_gpu_tree import f32_bits

pytestmark = pytest.mark.gpu


def test_refusals_leave_everything_as_it_was(backend):
    x = [backend.Upload(np.full(4096, 7.0, np.float32)) for _ in range(9)]

    def refused(name, buffers, scalars):
        with pytest.raises(StatusError) as error:
            backend.LaunchKernel(backend.LoadKernel(name), KernelLaunch(buffers=buffers, scalars=scalars))
        assert error.value.code == StatusCode.InvalidArgument, (name, scalars)
        assert name.rsplit("_", 1)[0] in str(error.value) or name in str(error.value)

    one = f32_bits(1.0)
    for fmt in ("q8", "fp8"):
        refused("pages_write_" + fmt, x, [2, 2, 60, 1, 16, 4, 2, 0, 0])
        refused("pages_write_" + fmt, x, [2, 2, 64, 1, 20, 4, 2, 0, 0])
        refused("pages_write_" + fmt, x, [2, 2, 64, 1, 16, 40, 2, 0, 0])       # a pool that does not fit
        refused("pages_write_" + fmt, x, [2, 2, 64, 1, 16, 4, 2, 64, 0])
        refused("pages_write_" + fmt, x[:8] + x[:1], [2, 2, 64, 1, 16, 4, 2, 0, 0])
        refused("pages_read_" + fmt, x, [2, 2, 64, 1, 16, 4, 2, 3])
        refused("pages_read_" + fmt, x[:8] + x[:1], [2, 2, 64, 1, 16, 4, 2, 0])
        refused("attention_pages_" + fmt, x, [2, 3, 2, 64, 1, 16, 4, 2, 0, 0, 0, 0])
        refused("attention_pages_" + fmt, x, [2, 4, 2, 64, 1, 16, 4, 2, 3, 0, 0, 0])
        refused("attention_pages_" + fmt, x, [2, 4, 2, 64, 1, 16, 4, 2, 0, 33, 0, 0])
        refused("attention_pages_" + fmt, x, [2, 4, 2, 64, 1, 16, 4, 2, 0, 0, 0, 4])
        refused("attention_pages_" + fmt, x[:8] + x[:1], [2, 4, 2, 64, 1, 16, 4, 2, 0, 0, 0, 0])
    refused("draft_verify", x[:6], [2, 100, 1, f32_bits(-1.0), one])
    refused("draft_verify", x[:7], [2, 100, 1, one, 0])
    refused("draft_verify", x[:7], [2, 4096, 1, one, one])
    refused("draft_verify", x[:5] + x[:1], [2, 100, 1, one, one])
    refused("draft_verify", x[:5], [2, 100, 1, one, one])
    backend.Synchronize()
    assert all(np.all(backend.CopyD2H(b, dtype=np.float32) == 7.0) for b in x)

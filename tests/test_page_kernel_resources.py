"""The attention over pages was sized against a register limit: no scratch memory (as test_kernel_resources.py)."""
import shutil

import pytest

from test_kernel_resources import HIPCC, resource_remarks


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason="hipcc not found")
@pytest.mark.parametrize("src,wanted", [("attention_pages.hip", ["attention_pages_few_kernel", "attention_pages_tile_kernel", "attention_pages_merge_kernel"]),
                                        ("pages.hip", ["pages_write_kernel", "pages_read_kernel"]),
                                        ("draft_verify.hip", ["draft_stats_kernel", "draft_rest_kernel"])])
def test_no_scratch_memory(src, wanted):
    kernels = resource_remarks(src)
    for want in wanted:
        hits = {k: v for k, v in kernels.items() if want in k}
        assert hits
        for name, res in hits.items():
            assert res.get("ScratchSize [bytes/lane]", 0) == 0, (name, res)
            assert res.get("VGPR Spill", 0) == 0, (name, res)

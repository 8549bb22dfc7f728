"""The tree's attention was sized against a register limit: no scratch memory (as test_kernel_resources.py)."""
import shutil

import pytest

from test_kernel_resources import HIPCC, resource_remarks


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason="hipcc not found")
def test_no_scratch_memory():
    kernels = resource_remarks("attention_tree.hip")
    for want in ("attention_pairs_kernel", "attention_tree_kernel"):
        hits = {k: v for k, v in kernels.items() if want in k}
        assert hits
        for name, res in hits.items():
            assert res.get("ScratchSize [bytes/lane]", 0) == 0, (name, res)
            assert res.get("VGPR Spill", 0) == 0, (name, res)

"""The calls that test_gpu_tree_shared.py means for the shared-key kernel go there, in several parts (launch_rules.hpp: tree_rule)."""
import pytest

from test_launch_rules import run_program
from tree_shapes import KINDS, calls


@pytest.mark.parametrize("kind", KINDS)
def test_shared_calls(tmp_path, kind):
    lines = []
    for m, n, heads, kv_heads, d, _, window in calls(kind):
        padded = 64 if d <= 64 else 128 if d <= 128 else 256
        # (whether the rows' kernels take a head size decides for more calls, never for fewer, that keys are shared)
        lines.append(f"  {{ const TreeShape s = tree_rule(TreeCall{{{m}, {window or n}, {heads}, {kv_heads}, {d}, {padded}, {str(kind == 'f32').lower()}, "
                     f"{str(kind in ('q8', 'q4', 'fp8')).lower()}, true, true}}, 256, 64, size_t{{16}} << 20);"
                     f" CHECK(s.tile && s.parts > 1, \"%d of %d: %zu parts\", {m}, {d}, static_cast<size_t>(s.parts)); }}")
    run_program(tmp_path, "\n".join(lines))

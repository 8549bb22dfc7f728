"""Long caches are shared among many workgroups whatever number of columns a call has (tessera_amd/csrc/launch_rules.hpp: pages_rule)."""
from test_launch_rules import run_program


def test_no_long_cache_in_a_workgroup_a_head(tmp_path):
    """Few heads of long sequences fill the chip, also where a unit has all of its columns, and what the parts leave fits the scratch memory."""
    run_program(tmp_path, r"""
  int full = 0, all = 0;
  for (uint64_t d : {16, 64, 80, 128, 208, 256}) for (uint64_t kv : {1, 2, 4, 8}) for (uint64_t sequences : {1, 2, 5, 8}) for (uint64_t group : {1, 2, 4, 5, 8, 16, 32})
  for (uint64_t rows = 1; rows * group <= (d <= 128 ? 32u : 16u); ++rows) for (uint64_t len : {20000, 32000, 65000, 131072, 1 << 20}) {
    const PagesCall c{rows * sequences, sequences, group, kv, d, rows, len, 0, 0};
    const size_t most = size_t{16} << 20;
    const PagesShape s = pages_rule(c, 256, most);
    const uint64_t groups = pages_units(c, s.columns) * kv, workgroups = s.even != 0 ? s.even : groups * s.parts;
    CHECK(s.columns <= 32, "%zu columns", static_cast<size_t>(s.columns));
    CHECK(workgroups <= 512 && (workgroups > 256 || (s.parts > 1 && s.part_tiles == 4)), "%zu rows of %zu, %zu x %zu heads of %zu, %zu positions: %zu workgroups", static_cast<size_t>(rows), static_cast<size_t>(group),
          static_cast<size_t>(sequences), static_cast<size_t>(kv), static_cast<size_t>(d), static_cast<size_t>(len), static_cast<size_t>(workgroups));
    CHECK(pages_bytes(c, s) <= most, "%zu bytes", pages_bytes(c, s));
    full += pages_stored(c, s.columns) == s.columns, ++all;
  }
  CHECK(full > 500 && all > 2000, "%d %d", full, all);
""")

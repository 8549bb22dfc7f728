"""How "attention_pages_*" run a call (tessera_amd/csrc/launch_rules.hpp: pages_rule), over the sizes that they take."""
from test_launch_rules import run_program


def test_pages_rule(tmp_path):
    """The parts cover every position, their sums fit the scratch memory that there is, the merge takes them, and every launch is a grid."""
    run_program(tmp_path, r"""
  int one = 0, parted = 0, even = 0, tall = 0;
  for (uint64_t sequences : {1, 2, 7, 48, 300, 4096}) for (uint64_t each : {1, 2, 5, 40, 3000}) for (uint64_t kv : {1, 4, 8, 512})
  for (uint64_t group : {1, 4, 6, 16, 33, 128}) for (uint64_t d : {16, 64, 80, 128, 208, 256}) for (uint64_t len : {1, 63, 400, 1200, 3000, 8000, 65000, 1 << 30})
  for (uint64_t window : {0, 1, 100, 4096, 1 << 20}) for (uint64_t cus : {8, 256}) {
    const uint64_t rows = sequences * each;
    if (rows * kv * group > 0xFFFFFF || sequences * kv > (1u << 21)) continue;
    const uint64_t sinks = window == 0 ? 0 : len % 70;
    for (const PagesCall& c : {PagesCall{rows, sequences, group, kv, d, each, len, window, sinks}, PagesCall{rows, sequences, group, kv, d, rows, len, window, sinks}}) {
      const size_t most = size_t{16} << 20;
      const PagesShape s = pages_rule(c, cus, most);
      const uint64_t units = pages_units(c, s.columns), groups = units * kv, tiles = pages_tiles(c, s.columns), stored = pages_stored(c, s.columns);
      CHECK(s.columns == 16 || s.columns == 64 || s.columns == 128 || (s.columns == 32 && d <= 128), "%zu columns", static_cast<size_t>(s.columns));
      CHECK(s.columns >= 64 || c.max_rows * group <= s.columns, "a sequence is one unit");
      CHECK(units >= sequences * ((each * group + s.columns - 1) / s.columns), "%zu units", static_cast<size_t>(units));      // (all have as many rows)
      CHECK(stored >= 1 && stored <= s.columns, "stored");
      CHECK(s.parts >= 1 && s.part_tiles >= 1 && s.parts * s.part_tiles >= tiles, "%zu parts", static_cast<size_t>(s.parts));
      CHECK(pages_bytes(c, s) <= most, "%zu bytes", pages_bytes(c, s));
      CHECK(s.parts <= kPagePartsMost && s.even <= kPagePartsMost && (s.even == 0 || s.parts == 1), "merge");
      CHECK(s.even == 0 || (s.columns < 64 && sequences * kv * (tiles + begin_tiles(5)) < (1u << 30)), "sums in 32 bits");
      CHECK(s.even != 0 || groups * s.parts * 512 < uint64_t{1} << 32, "grid");
      CHECK((s.even == 0 && s.parts == 1) || groups * stored * 256 < uint64_t{1} << 32, "merge's grid");
      CHECK(s.waves == 4 || (s.waves == 8 && s.parts == 1 && s.even == 0 && s.columns < 64), "waves");
      const PagesShape without = pages_rule(c, cus, 0);
      CHECK(without.parts == 1 && without.even == 0 && pages_bytes(c, without) == 0 && without.columns == s.columns, "without scratch");
      one += s.parts == 1 && s.even == 0, parted += s.parts > 1, even += s.even != 0, tall += s.waves == 8;
    }
  }
  CHECK(one > 1000 && parted > 1000 && even > 1000 && tall > 1000, "%d %d %d %d", one, parted, even, tall);
""")

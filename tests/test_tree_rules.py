"""How "attention_tree" runs a call (tessera_amd/csrc/launch_rules.hpp: tree_rule), over the sizes that it takes."""
from test_launch_rules import run_program


def test_tree_rule(tmp_path):
    run_program(tmp_path, r"""
  int tiles = 0, parted = 0, calls = 0;
  for (uint64_t rows : {1, 2, 5, 16, 33, 64, 1000, 16777216}) for (uint64_t keys : {1, 47, 48, 96, 300, 9300, 32832, 2147483647})
  for (uint64_t kv : {1, 4, 8}) for (uint64_t group : {1, 3, 6, 17}) for (uint64_t d : {34, 64, 80, 128, 256}) for (int kind = 0; kind < 3; ++kind)
  for (int ways = 1; ways < 4; ++ways) for (uint64_t most : {1, 64}) for (uint64_t cus : {8, 256}) {
    if (rows * kv * group > 0xFFFFFF) continue;
    const TreeCall call{rows, keys, kv * group, kv, d, d <= 64 ? 64u : d <= 128 ? 128u : 256u, kind == 0, kind == 2, (ways & 1) != 0, (ways & 2) != 0};
    const size_t bytes = size_t{16} << 20;
    const TreeShape s = tree_rule(call, cus, most, bytes);
    ++calls, tiles += s.tile, parted += s.parts > 1;
    CHECK(s.tile ? call.shared : call.by_rows, "%zu rows", static_cast<size_t>(rows));
    CHECK(s.parts >= 1 && s.parts <= most, "%zu parts", static_cast<size_t>(s.parts));
    CHECK(s.parts == 1 || (keys / s.parts >= 48 && attention_parts_size(rows, kv * group, d, s.parts) <= bytes), "%zu parts", static_cast<size_t>(s.parts));
    CHECK(s.tile ? s.pairs == 64 : s.pairs >= 1 && s.pairs <= (call.fp32 ? 16 : 8), "%zu pairs", static_cast<size_t>(s.pairs));
    CHECK(tree_units(call, s.pairs) >= 1 && tree_units(call, s.pairs) * s.pairs >= rows * kv * group, "units");
  }
  CHECK(tiles > calls / 4 && tiles < calls * 3 / 4 && parted > calls / 8, "%d of %d, %d", tiles, calls, parted);
""")

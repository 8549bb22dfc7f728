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


def test_logprob_plan(tmp_path):
    """The tiles of a row cover its columns wherever it begins, its shares fit the scratch memory that there is, and every launch is a grid."""
    run_program(tmp_path, r"""
  int shared = 0, apart = 0, limited = 0;
  for (uint64_t rows : {1, 2, 33, 128, 512, 5000, 16384, 16385, 31488, 1 << 30})
  for (uint64_t vocab : {1, 2, 3, 1000, 2045, 2046, 2048, 2049, 4096, 4097, 50001, 131072, 1048576, 0x7FFFFFFF})
  for (uint64_t top_k : {0, 1, 32}) for (uint64_t cus : {8, 256}) for (size_t most : {size_t{0}, size_t{1} << 16, size_t{16} << 20}) {
    const LogprobPlan p = logprob_plan(rows, vocab, top_k, cus, most);
    const uint64_t tiles = uint64_t{p.tiles} * p.shares, here = rows < kLogprobRows ? rows : kLogprobRows;
    CHECK(p.threads == 256 || p.threads == 512 || p.threads == 1024, "%u threads", p.threads);
    CHECK(p.width % 4 == 0 && p.width > 0 && p.width <= p.threads * kLogprobEach, "width %u", p.width);
    for (uint64_t shift = 0; shift < 4; ++shift) {            // entries between 16 bytes and the row's first
      if (vocab % 4 != 0 || shift == 0) CHECK(tiles * p.width >= vocab + shift, "%zu tiles of %u", static_cast<size_t>(tiles), p.width);
    }
    CHECK(p.shares >= 1 && p.shares <= kLogprobShares && p.tiles >= 1, "%u shares", p.shares);
    CHECK(logprob_bytes(p, rows, top_k) <= most && (p.shares == 1 || rows <= kLogprobRows), "%zu bytes", logprob_bytes(p, rows, top_k));
    CHECK(here * p.shares * p.threads <= uint64_t{1} << 30, "%zu rows", static_cast<size_t>(here));
    shared += p.shares > 1, apart += p.shares == 1, limited += p.shares < logprob_plan(rows, vocab, top_k, cus, ~size_t{0}).shares;
  }
  CHECK(shared > 100 && apart > 100 && limited > 20, "%d %d %d", shared, apart, limited);
  CHECK(logprob_plan(5000, 65000, 32, 256, size_t{16} << 20).shares == 1, "rows that fill the chip");
""")

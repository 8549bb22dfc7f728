"""The largest calls of the ids around a tree of drafted tokens are a grid that a launch can have: fewer than 2^32 threads."""
from test_tree_args import run_program


def test_qk_norm_rows_and_heads(tmp_path):
    """A head size that takes a wavefront a row and head: four to a workgroup of 256."""
    run_program(tmp_path, r"""
  const uint64_t theta = 0x461C4000, eps = 0x358637BD;
  const std::vector<size_t> big(6, size_t{1} << 40);
  QkNormCall call;
  auto grid = [&](uint64_t rows, uint64_t heads, uint64_t kv) {
    return !check_qk_norm(Launch(big, {rows, heads, kv, 2, 2, 0, theta, eps, 0, 0, 0, 0}).args(), false, &call);
  };
  CHECK(grid((1 << 24) - 1, 3, 1));                                     // 2^26 - 4
  CHECK(!grid(1 << 24, 3, 1));
  CHECK(!grid(8191, 8192, 1));                                          // 2^26 - 1
  for (uint64_t rows : {1ull, 8190ull, 8191ull, 13421772ull, (1ull << 24) - 1, 1ull << 24}) for (uint64_t heads : {1, 3, 4, 8191, 8192, 65536}) {
    if (grid(rows, heads, 1)) CHECK((rows * (heads + 1) + 3) / 4 * 256 < uint64_t{1} << 32);
  }
""")

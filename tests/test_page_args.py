"""What the ids around a paged cache and the verification of drafts refuse (tessera_amd/csrc/page_args.hpp): host logic without
HIP, run here as a small C++ program; a launch raises the same before any device work (test_gpu_page_refusals.py)."""
import os
import shutil
import subprocess

import pytest

from test_tree_args import HEAD, ROOT

POOL = r"""
// rows 3, 2 key heads of 64, 2 sequences, pages of 16, 5 of them, a table of 4
const size_t codes = 5 * 2 * 16 * 64, scales = 40, row = 512;
std::vector<uint64_t> with(std::vector<uint64_t> shape, std::vector<uint64_t> more) {
  shape.insert(shape.end(), more.begin(), more.end());
  return shape;
}
const std::vector<uint64_t> shape = {3, 2, 64, 2, 16, 5, 4};
// the shape with one scalar changed
std::vector<uint64_t> but(size_t i, uint64_t v) {
  auto s = shape;
  s[i] = v;
  return s;
}
"""


def run_program(tmp_path, body):
    if shutil.which("g++") is None:
        pytest.skip("g++ not found")
    src, exe = tmp_path / "args.cpp", tmp_path / "args"
    src.write_text("#include <string>\n" + HEAD.replace("tree_args.hpp", "page_args.hpp") + POOL + "int main() {\n" + body + "\n}\n")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Wextra", "-I" + os.path.join(ROOT, "tessera_amd", "csrc"), "-o", str(exe), str(src)],
                   check=True, timeout=120)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout


def test_pages_write(tmp_path):
    run_program(tmp_path, r"""
  PageWriteCall call;
  auto why = [&](std::vector<size_t> b, std::vector<uint64_t> s) { return check_pages_write(Launch(b, s).args(), &call); };
  const std::vector<size_t> fits = {3 * row, 3 * row, 32, 12, 8, codes, codes, scales, scales}, big(9, size_t{1} << 46);
  CHECK(!why(fits, with(shape, {0, 0})));
  CHECK(call.k_stride == 128 && call.v_stride == 128 && call.page.touched() == 3);
  for (size_t i = 0; i < 9; ++i) {
    auto less = fits;
    less[i] -= 4;
    CHECK(why(less, with(shape, {0, 0})));
  }
  for (size_t i = 0; i < 7; ++i) CHECK(why(big, with(but(i, 0), {0, 0})));
  for (uint64_t d : {8, 63, 72, 272, 512}) CHECK(why(big, with(but(2, d), {0, 0})));
  for (uint64_t d : {16, 80, 128, 256}) CHECK(!why(big, with(but(2, d), {0, 0})));
  for (uint64_t b : {1, 8, 15, 24, 48, 256}) CHECK(why(big, with(but(4, b), {0, 0})));
  for (uint64_t b : {16, 32, 64, 128}) CHECK(!why(big, with(but(4, b), {0, 0})));
  CHECK(why(big, with(but(0, (1 << 24) + 1), {0, 0})));
  CHECK(why(big, with(but(1, 4097), {0, 0})));
  CHECK(why(big, with(but(3, 4097), {0, 0})) && !why(big, with(but(3, 4096), {0, 0})));
  CHECK(why(big, with(but(5, uint64_t{1} << 31), {0, 0})));
  CHECK(why(big, with(but(6, (1 << 26) + 1), {0, 0})) && !why(big, with(but(6, 1 << 26), {0, 0})));   // 2^30 positions
  CHECK(why(big, with(but(6, ~uint64_t{0} / 8), {0, 0})));                                            // (no overflow)
  CHECK(why(big, with(shape, {127, 0})) && why(big, with(shape, {0, 124})) && why(big, with(shape, {130, 0})));
  CHECK(!why(big, with(shape, {384, 132})));
  CHECK(!why({2 * 1536 + row, 3 * row, 32, 12, 8, codes, codes, scales, scales}, with(shape, {384, 0})));
  CHECK(why({2 * 1536 + row - 4, 3 * row, 32, 12, 8, codes, codes, scales, scales}, with(shape, {384, 0})));
  CHECK(why(fits, with(shape, {0})) && why(fits, with(shape, {0, 0, 0})));
  CHECK(why({3 * row, 3 * row, 32, 12, 8, codes, codes, scales}, with(shape, {0, 0})));
  // the pool apart from everything
  for (size_t i = 5; i < 9; ++i) for (size_t j = 0; j < 9; ++j) {
    if (i == j) continue;
    Launch l(fits, with(shape, {0, 0}));
    l.buf[i] = l.buf[j];
    CHECK(check_pages_write(l.args(), &call));
  }
  Launch l(fits, with(shape, {0, 0}));
  l.buf[1] = l.buf[0];                                       // keys and values may be the same rows
  CHECK(!check_pages_write(l.args(), &call));
  // sizes unknown: only the scalars are checked
  CHECK(!check_pages_write(Launch(fits, with(shape, {0, 0})).args(false), &call));
  // pages and heads of a grid
  CHECK(why(big, with({1 << 24, 64, 16, 1, 16, 1 << 20, 1 << 20}, {0, 0})));
  for (uint64_t rows : {1ull, 17ull, 1ull << 20, 1ull << 24}) for (uint64_t kv : {1, 2, 7, 64, 4096}) for (uint64_t seq : {1, 4096}) {
    if (!why(std::vector<size_t>(9, size_t{1} << 60), with({rows, kv, 16, seq, 16, 1, 1}, {0, 0}))) {
      CHECK(static_cast<unsigned __int128>(call.page.touched()) * kv * 2 * 256 < (static_cast<unsigned __int128>(1) << 32));
    }
  }
""")


def test_pages_read(tmp_path):
    run_program(tmp_path, r"""
  PageReadCall call;
  auto why = [&](std::vector<size_t> b, std::vector<uint64_t> s) { return check_pages_read(Launch(b, s).args(), &call); };
  const std::vector<size_t> fits = {codes, codes, scales, scales, 32, 12, 8, 3 * row, 3 * row}, big(9, size_t{1} << 46);
  CHECK(!why(fits, with(shape, {0})) && !call.f16);
  for (size_t i = 0; i < 9; ++i) {
    auto less = fits;
    less[i] -= 2;
    CHECK(why(less, with(shape, {0})));
  }
  auto half = fits;
  half[7] /= 2, half[8] /= 2;
  CHECK(!why(half, with(shape, {1})) && call.f16 && why(half, with(shape, {0})));
  CHECK(why(big, with(shape, {2})) && why(big, shape) && why(big, with(shape, {0, 0})));
  for (size_t i = 0; i < 7; ++i) CHECK(why(big, with(but(i, 0), {0})));
  for (size_t i = 7; i < 9; ++i) for (size_t j = 0; j < 9; ++j) {
    if (i == j) continue;
    Launch l(fits, with(shape, {0}));
    l.buf[i] = l.buf[j];
    CHECK(check_pages_read(l.args(), &call));
  }
""")


def test_attention_pages(tmp_path):
    run_program(tmp_path, r"""
  PageAttentionCall call;
  auto why = [&](std::vector<size_t> b, std::vector<uint64_t> s) { return check_attention_pages(Launch(b, s).args(), &call); };
  // rows, heads, kv_heads, ...
  auto full = [&](std::vector<uint64_t> page, uint64_t heads, std::vector<uint64_t> tail) {
    page.insert(page.begin() + 1, heads);
    return with(page, tail);
  };
  const size_t q = 3 * 6 * 64 * 4;
  const std::vector<size_t> fits = {q, codes, codes, scales, scales, 32, 12, 8, q}, big(9, size_t{1} << 46);
  CHECK(!why(fits, full(shape, 6, {0, 0, 0, 0})));
  CHECK(call.max_rows == 3 && call.max_len == 64);
  CHECK(!why(fits, full(shape, 6, {2, 63, 5, 4})) && call.max_rows == 2 && call.max_len == 63 && call.window == 5 && call.sinks == 4);
  for (size_t i = 0; i < 9; ++i) {
    auto less = fits;
    less[i] -= 4;
    CHECK(why(less, full(shape, 6, {0, 0, 0, 0})));
  }
  for (size_t i = 0; i < 7; ++i) CHECK(why(big, full(but(i, 0), 6, {0, 0, 0, 0})));
  CHECK(why(big, full(shape, 0, {0, 0, 0, 0})) && why(big, full(shape, 5, {0, 0, 0, 0})) && why(big, full(shape, 65538, {0, 0, 0, 0})));
  CHECK(why(big, full(shape, 6, {4, 0, 0, 0})) && why(big, full(shape, 6, {0, 65, 0, 0})));
  CHECK(why(big, full(shape, 6, {0, 0, 0, 4})));                                     // sinks without a window
  CHECK(why(big, full(shape, 6, {0, 0, (uint64_t{1} << 48) + 1, 0})) && why(big, full(shape, 6, {0, 0, 5, (uint64_t{1} << 48) + 1})));
  CHECK(!why(big, full(shape, 6, {0, 0, uint64_t{1} << 48, uint64_t{1} << 48})));
  CHECK(why(big, full(but(0, 1 << 23), 6, {0, 0, 0, 0})));                           // rows times heads
  CHECK(why(std::vector<size_t>(9, size_t{1} << 60), full({1, 1024, 16, 4096, 16, 1, 1}, 1024, {0, 0, 0, 0})));
  CHECK(why(big, full(shape, 6, {0, 0, 0})));
  for (size_t j = 0; j < 8; ++j) {
    Launch l(fits, full(shape, 6, {0, 0, 0, 0}));
    l.buf[8] = l.buf[j];
    CHECK(check_attention_pages(l.args(), &call));
  }
""")


def test_draft_verify(tmp_path):
    run_program(tmp_path, r"""
  DraftCall call;
  auto why = [&](std::vector<size_t> b, std::vector<uint64_t> s) { return check_draft_verify(Launch(b, s).args(), &call); };
  const uint64_t one = 0x3F800000, half = 0x3F000000;
  const std::vector<size_t> fits = {4 * 100 * 4, 16, 32, 12, 8, 8};
  CHECK(!why(fits, {4, 100, 2, one, 0}) && call.temperature == 1.0f && !call.draft);
  auto seven = fits;
  seven.push_back(fits[0]);
  CHECK(!why(seven, {4, 100, 2, one, half}) && call.draft && call.draft_temperature == 0.5f);
  CHECK(!why(seven, {4, 100, 2, 0, 0}));                                             // greedy: the draft's is not looked at
  for (size_t i = 0; i < 7; ++i) {
    auto less = seven;
    less[i] -= 4;
    CHECK(why(less, {4, 100, 2, one, one}));
  }
  const std::vector<size_t> big(7, size_t{1} << 46);
  for (size_t i = 0; i < 3; ++i) {
    std::vector<uint64_t> s = {4, 100, 2, one, one};
    s[i] = 0;
    CHECK(why(big, s));
  }
  CHECK(why(big, {(1 << 20) + 1, 100, 2, one, one}) && why(big, {4, (1 << 21) + 1, 2, one, one}) && why(big, {4, 100, 4097, one, one}));
  CHECK(!why(big, {1 << 20, 1 << 21, 4096, one, one}));
  for (uint64_t t : {0xBF800000ull, 0x7F800000ull, 0x7FC00000ull}) CHECK(why(big, {4, 100, 2, t, one}) && why(big, {4, 100, 2, one, t}));
  CHECK(why(big, {4, 100, 2, one, 0}) && why(big, {4, 100, 2, one}) && why({4, 4, 4, 4, 4}, {1, 1, 1, one, one}));
  for (size_t i = 4; i < 6; ++i) for (size_t j = 0; j < 7; ++j) {
    if (i == j) continue;
    Launch l(seven, {4, 100, 2, one, one});
    l.buf[i] = l.buf[j];
    CHECK(check_draft_verify(l.args(), &call));
  }
  Launch l(seven, {4, 100, 2, one, one});
  l.buf[6] = l.buf[0];                                                               // the draft may be the target
  CHECK(!check_draft_verify(l.args(), &call));
""")


def test_what_a_refusal_says(tmp_path):
    run_program(tmp_path, r"""
  PageReadCall call;
  const std::string why = check_pages_read(Launch({}, {}).args(), &call);
  CHECK(why == "pages_read: expects 9 buffers and 8 scalars");
""")

"""What the ids around a tree of drafted tokens refuse (tessera_amd/csrc/tree_args.hpp): host logic without HIP, run here
as a small C++ program; a launch raises the same before any device work (test_gpu_tree_refusals.py)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

HEAD = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "tree_args.hpp"
using namespace qmm;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); std::exit(1); } } while (0)
// A launch over buffers of the given sizes, side by side with gaps.
struct Launch {
  std::vector<size_t> bytes;
  std::vector<uint64_t> sc;
  std::vector<void*> buf;
  Launch(std::vector<size_t> b, std::vector<uint64_t> s) : bytes(b), sc(s) {
    uintptr_t at = 1 << 20;
    for (size_t n : bytes) buf.push_back(reinterpret_cast<void*>(at)), at += (n + 4096) / 256 * 256;
  }
  LaunchArgs args(bool sizes = true) const { return {buf.data(), sizes ? bytes.data() : nullptr, buf.size(), sc.data(), sc.size()}; }
};
"""


def run_program(tmp_path, body):
    if shutil.which("g++") is None:
        pytest.skip("g++ not found")
    src, exe = tmp_path / "args.cpp", tmp_path / "args"
    src.write_text(HEAD + "int main() {\n" + body + "\n}\n")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Wextra", "-I" + os.path.join(ROOT, "tessera_amd", "csrc"), "-o", str(exe), str(src)],
                   check=True, timeout=120)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout


def test_tree_mask(tmp_path):
    run_program(tmp_path, r"""
  auto why = [](std::vector<size_t> b, std::vector<uint64_t> s) { return check_tree_mask(Launch(b, s).args()); };
  CHECK(!why({4, 4, 24}, {1, 0}));
  CHECK(!why({4096, 4096 * 32, 24576}, {1024, uint64_t{1} << 48}));
  CHECK(why({4100, 8192 * 32, 25000}, {1025, 0}));
  CHECK(why({4, 4, 24}, {0, 0}));
  CHECK(why({4, 4, 24}, {1, (uint64_t{1} << 48) + 1}));
  CHECK(why({4, 4, 24}, {1}));
  CHECK(why({4, 4}, {1, 0}));
  CHECK(why({132 - 4, 33 * 8, 33 * 24}, {33, 0}));
  CHECK(why({132, 33 * 8 - 4, 33 * 24}, {33, 0}));
  CHECK(why({132, 33 * 8, 33 * 24 - 8}, {33, 0}));
  CHECK(!why({132, 33 * 8, 33 * 24}, {33, 0}));
  Launch l({132, 33 * 8, 33 * 24}, {33, 0});
  l.buf[1] = l.buf[0];
  CHECK(check_tree_mask(l.args()));
""")


def test_qk_norm(tmp_path):
    run_program(tmp_path, r"""
  const uint64_t theta = 0x461C4000, eps = 0x358637BD;     // 10000, 1e-6
  QkNormCall call;
  // rows 3, heads 4 over 2 of 64
  const std::vector<size_t> fits = {3 * 1024, 3 * 512, 256, 256, 3 * 1024, 3 * 512};
  auto with = [&](std::vector<size_t> b, std::vector<uint64_t> s) { return check_qk_norm(Launch(b, s).args(), false, &call); };
  CHECK(!with(fits, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 0, 0}));
  CHECK(call.q_stride == 256 && call.k_stride == 128 && !call.gated);
  for (size_t i = 0; i < 6; ++i) {
    auto less = fits;
    less[i] -= 4;
    CHECK(with(less, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 0, 0}));
  }
  for (size_t i = 0; i < 5; ++i) {
    std::vector<uint64_t> s = {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 0, 0};
    s[i] = 0;
    CHECK(with(fits, s));
  }
  const std::vector<size_t> big(6, size_t{1} << 40);
  CHECK(with(big, {3, 4, 2, 258, 64, 0, theta, eps, 0, 0, 0, 0}));
  CHECK(with(big, {3, 4, 2, 63, 62, 0, theta, eps, 0, 0, 0, 0}));
  CHECK(with(big, {3, 4, 2, 64, 66, 0, theta, eps, 0, 0, 0, 0}));
  CHECK(with(big, {3, 4, 2, 64, 33, 0, theta, eps, 0, 0, 0, 0}));
  CHECK(with(big, {3, 4, 2, 64, 64, 0, 0, eps, 0, 0, 0, 0}));                 // theta 0
  CHECK(with(big, {3, 4, 2, 64, 64, 0, 0x7FC00000, eps, 0, 0, 0, 0}));        // NaN
  CHECK(with(big, {3, 4, 2, 64, 64, 0, 0x7F800000, eps, 0, 0, 0, 0}));        // infinite
  CHECK(with(big, {3, 4, 2, 64, 64, 0, theta, 0xB58637BD, 0, 0, 0, 0}));      // epsilon below 0
  CHECK(with(big, {3, 4, 2, 64, 64, 0, theta, eps, 255, 0, 0, 0}));           // strides shorter than a row
  CHECK(with(big, {3, 4, 2, 64, 64, 0, theta, eps, 0, 127, 0, 0}));
  CHECK(with(big, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 2, 0}));
  CHECK(with(big, {(1 << 24) + 1, 1, 1, 64, 64, 0, theta, eps, 0, 0, 0, 0}));
  CHECK(with(big, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 0}));
  CHECK(with(fits, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 0, 1}));            // the cache ends before the last row
  CHECK(with(fits, {3, 4, 2, 64, 64, 0, theta, eps, 300, 0, 0, 0}));          // rows further apart
  // fp16 rows of a cache
  CHECK(!with({3 * 1024, 3 * 512, 256, 256, 3 * 1024, 5 * 256}, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 1, 2}));
  CHECK(with({3 * 1024, 3 * 512, 256, 256, 3 * 1024, 5 * 256 - 2}, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 1, 2}));
  // a gate: twice as wide
  CHECK(!with({3 * 2048, 3 * 512, 256, 256, 3 * 1024, 3 * 512, 3 * 1024}, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 0, 0}) && call.gated);
  CHECK(with({3 * 1024, 3 * 512, 256, 256, 3 * 1024, 3 * 512, 3 * 1024}, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 0, 0}));
  CHECK(with({3 * 2048, 3 * 512, 256, 256, 3 * 1024, 3 * 512, 3 * 1024 - 4}, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 0, 0}));
  // in place, and not where the layouts differ
  Launch l(fits, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 0, 0});
  l.buf[4] = l.buf[0], l.buf[5] = l.buf[1];
  CHECK(!check_qk_norm(l.args(), false, &call));
  l.buf[4] = static_cast<char*>(l.buf[0]) + 16;
  CHECK(check_qk_norm(l.args(), false, &call));
  Launch w({3 * 1280, 3 * 512, 256, 256, 3 * 1280, 3 * 512}, {3, 4, 2, 64, 64, 0, theta, eps, 320, 0, 0, 0});
  w.buf[4] = w.buf[0];
  CHECK(check_qk_norm(w.args(), false, &call));
  Launch h(fits, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 1, 0});
  h.buf[5] = h.buf[1];
  CHECK(check_qk_norm(h.args(), false, &call));                               // fp16 over fp32
  Launch o(fits, {3, 4, 2, 64, 64, 0, theta, eps, 0, 0, 0, 0});
  o.buf[5] = o.buf[4];
  CHECK(check_qk_norm(o.args(), false, &call));
  // positions
  auto axes = [&](std::vector<size_t> b, std::vector<uint64_t> s) { return check_qk_norm(Launch(b, s).args(), true, &call); };
  const std::vector<size_t> seven = {3 * 1024, 3 * 512, 256, 256, 72, 3 * 1024, 3 * 512};
  CHECK(!axes(seven, {3, 4, 2, 64, 64, theta, eps, 0, 0, 0, 0, 16, 8, 8}) && call.sec_t == 16 && call.sec_h == 8);
  CHECK(axes(seven, {3, 4, 2, 64, 64, theta, eps, 0, 0, 0, 0, 16, 8, 9}));
  CHECK(axes(seven, {3, 4, 2, 64, 64, theta, eps, 0, 0, 0, 0, ~uint64_t{0}, 8, 9}));
  CHECK(axes({3 * 1024, 3 * 512, 256, 256, 64, 3 * 1024, 3 * 512}, {3, 4, 2, 64, 64, theta, eps, 0, 0, 0, 0, 16, 8, 8}));
  CHECK(axes(seven, {3, 4, 2, 64, 64, theta, eps, 0, 0, 0, 0, 16, 8}));
""")


def test_attention_tree(tmp_path):
    run_program(tmp_path, r"""
  const uint64_t m = 3, n = 50, heads = 4, kv = 2, d = 64, tree = 33;
  const size_t q = m * heads * d * 4, row = kv * d * 2, words = m * 2 * 4;
  const std::vector<size_t> fits = {q, n * row, n * row, words, q};
  auto why = [&](std::vector<size_t> b, std::vector<uint64_t> s) { return check_attention_tree(Launch(b, s).args(), false, 0); };
  CHECK(!why(fits, {m, n, heads, kv, d, tree, 0, 1}));
  for (size_t i = 0; i < 5; ++i) {
    auto less = fits;
    less[i] -= 2;
    CHECK(why(less, {m, n, heads, kv, d, tree, 0, 1}));
  }
  CHECK(why(fits, {m, n, heads, kv, d, tree, 0, 0}));       // fp32 takes twice as much
  for (size_t i = 0; i < 6; ++i) {
    std::vector<uint64_t> s = {m, n, heads, kv, d, tree, 0, 1};
    s[i] = 0;
    CHECK(why(fits, s));
  }
  const std::vector<size_t> big(5, size_t{1} << 50);
  CHECK(!why(big, {m, n, heads, kv, d, n, 0, 1}));
  CHECK(why(big, {m, n, heads, kv, d, n + 1, 0, 1}));
  CHECK(why(big, {m, n, 5, kv, d, tree, 0, 1}));
  CHECK(why(big, {m, n, heads, kv, 257, tree, 0, 1}));
  CHECK(why(big, {m, n, heads, kv, d, tree, 0, 2}));
  CHECK(why(big, {m, (uint64_t{1} << 31) + 1, heads, kv, d, tree, 0, 1}));
  CHECK(why(big, {(1 << 24) + 1, n, heads, kv, d, tree, 0, 1}));
  CHECK(!why(big, {1, 1 << 20, 1, 1, d, 1 << 16, 0, 1}));
  CHECK(why(big, {1, 1 << 20, 1, 1, d, (1 << 16) + 1, 0, 1}));
  CHECK(why(big, {m, n, heads, kv, d, tree, 0}));
  Launch l(fits, {m, n, heads, kv, d, tree, 0, 1});
  l.buf[4] = l.buf[0];
  CHECK(check_attention_tree(l.args(), false, 0));          // rows are read while others are written
  auto quant = [&](std::vector<size_t> b, std::vector<uint64_t> s, uint32_t kind) { return check_attention_tree(Launch(b, s).args(), true, kind); };
  const std::vector<size_t> eight = {q, n * kv * d, n * kv * d, n * 4, n * 4, words, q}, four = {q, n * kv * d / 2, n * kv * d / 2, n * 4, n * 4, words, q};
  CHECK(!quant(eight, {m, n, heads, kv, d, tree, 0}, 2) && !quant(eight, {m, n, heads, kv, d, tree, 0}, 4) && !quant(four, {m, n, heads, kv, d, tree, 0}, 3));
  CHECK(quant(four, {m, n, heads, kv, d, tree, 0}, 2));
  CHECK(quant(four, {m, n, 1, 1, 33, tree, 0}, 3));         // an odd number of codes a key row
  for (size_t i = 0; i < 7; ++i) {
    auto less = eight;
    less[i] -= 1;
    CHECK(quant(less, {m, n, heads, kv, d, tree, 0}, 2));
  }
  CHECK(quant(fits, {m, n, heads, kv, d, tree, 0}, 2));
""")


def test_token_logprobs(tmp_path):
    run_program(tmp_path, r"""
  auto why = [](std::vector<size_t> b, std::vector<uint64_t> s) { return check_token_logprobs(Launch(b, s).args()); };
  const std::vector<size_t> four = {5 * 400, 24, 24, 12}, six = {5 * 400, 24, 24, 12, 3 * 32, 3 * 32};
  CHECK(!why(four, {3, 100, 2, 0, 2}));
  CHECK(!why(six, {3, 100, 2, 8, 2}));
  CHECK(why(four, {3, 100, 2, 8, 2}));
  CHECK(why(six, {3, 100, 2, 0, 2}));
  CHECK(why(six, {3, 100, 2, 8, 3}));
  for (size_t i = 0; i < 6; ++i) {
    auto less = six;
    less[i] -= 4;
    CHECK(why(less, {3, 100, 2, 8, 2}));
  }
  const std::vector<size_t> big(6, size_t{1} << 50);
  CHECK(!why(big, {3, 100, 2, 32, 2}));
  CHECK(why(big, {3, 100, 2, 33, 2}));
  CHECK(why(big, {3, 7, 2, 8, 2}));
  CHECK(why(big, {0, 100, 2, 8, 2}));
  CHECK(why(big, {3, 0, 2, 8, 2}));
  CHECK(why(big, {3, 100, 0, 8, 2}));
  CHECK(why(big, {3, 100, 1025, 8, 2}));
  CHECK(why(big, {3, uint64_t{1} << 31, 2, 8, 2}));
  CHECK(why(big, {3, 100, 2, 8}));
  Launch l(six, {3, 100, 2, 8, 2});
  l.buf[5] = l.buf[4];
  CHECK(check_token_logprobs(l.args()));
""")

// What the ids around a tree of drafted tokens ("tree_mask", "qk_norm_rope", "qk_norm_mrope", "attention_tree*",
// "token_logprobs") refuse.  Host logic only, no HIP calls: each check returns nullptr or why a launch is refused.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cstring>

namespace qmm {

// A launch's arguments as the C ABI hands them over; `bytes` may be null (sizes unknown).
struct LaunchArgs {
  void* const* buf;
  const size_t* bytes;
  size_t nbuf;
  const uint64_t* sc;
  size_t nsc;

  bool fits(size_t i, unsigned __int128 need) const { return bytes == nullptr || static_cast<unsigned __int128>(bytes[i]) >= need; }
  // `need_a` bytes of buffer a and `need_b` of buffer b share some.
  bool overlap(size_t a, unsigned __int128 need_a, size_t b, unsigned __int128 need_b) const {
    const unsigned __int128 x = reinterpret_cast<uintptr_t>(buf[a]), y = reinterpret_cast<uintptr_t>(buf[b]);
    return x < y + need_b && y < x + need_a;
  }
};

inline float scalar_f32(uint64_t bits) {
  const uint32_t low = static_cast<uint32_t>(bits);
  float v;
  std::memcpy(&v, &low, 4);
  return v;
}

constexpr uint32_t kTreeMaskMost = 1024;        // nodes of "tree_mask"
constexpr uint64_t kTreeKeysMost = 1 << 16;     // of "attention_tree", which counts a row's bits word by word under a window
constexpr uint64_t kLogprobTokensMost = 1024, kLogprobTopMost = 32;

// "tree_mask": buffers Parents, Mask, Positions; scalars nodes, base.
inline const char* check_tree_mask(const LaunchArgs& c) {
  if (c.nbuf != 3 || c.nsc != 2) return "tree_mask: expects 3 buffers and 2 scalars";
  const uint64_t nodes = c.sc[0];
  if (nodes == 0 || nodes > kTreeMaskMost || c.sc[1] > (uint64_t{1} << 48)) return "tree_mask: 1 to 1024 nodes, base at most 2^48";
  const uint64_t need[3] = {nodes * 4, nodes * ((nodes + 31) / 32) * 4, nodes * 24};
  for (size_t i = 0; i < 3; ++i) {
    if (!c.fits(i, need[i])) return "tree_mask: a buffer is smaller than the nodes require";
  }
  if (c.overlap(0, need[0], 1, need[1]) || c.overlap(0, need[0], 2, need[2]) || c.overlap(1, need[1], 2, need[2])) {
    return "tree_mask: buffers must not overlap";
  }
  return nullptr;
}

// "qk_norm_rope": buffers Q, K, Wq, Wk, Qout, Kout[, Gate]; scalars rows, heads, kv_heads, head_dim, rope_dim, pos_base,
// theta, eps, q_stride, k_stride, k_f16, k_row.  "qk_norm_mrope": Pos after Wk, no pos_base, then sec_t, sec_h, sec_w.
struct QkNormCall {
  uint64_t rows, heads, kv_heads, head_dim, rope_dim, pos_base, q_stride, k_stride, k_f16, k_row, sec_t, sec_h;
  float theta, eps;
  bool gated;
  size_t q_out;        // buffers q_out, q_out + 1, q_out + 2
};
inline const char* check_qk_norm(const LaunchArgs& c, bool axes, QkNormCall* out) {
  const size_t base = axes ? 7 : 6;
  if ((c.nbuf != base && c.nbuf != base + 1) || c.nsc != (axes ? 14u : 12u)) {
    return "qk_norm_rope/mrope: expects 6 (7 with positions) buffers, one more with a gate, and 12 (14) scalars";
  }
  const uint64_t* s = c.sc + (axes ? 5 : 6);
  QkNormCall a{c.sc[0], c.sc[1], c.sc[2], c.sc[3], c.sc[4], axes ? 0 : c.sc[5], s[2], s[3], s[4], s[5],
               axes ? s[6] : 0, axes ? s[7] : 0, scalar_f32(s[0]), scalar_f32(s[1]), c.nbuf == base + 1, axes ? 5u : 4u};
  if (a.rows == 0 || a.heads == 0 || a.kv_heads == 0 || a.head_dim == 0 || a.rope_dim == 0) {
    return "qk_norm_rope/mrope: rows, heads, kv_heads, head_dim, rope_dim must be non-zero";
  }
  if (a.head_dim > 256 || a.head_dim % 2 != 0 || a.rope_dim % 2 != 0 || a.rope_dim > a.head_dim) {
    return "qk_norm_rope/mrope: head_dim and rope_dim must be even, head_dim at most 256, rope_dim at most head_dim";
  }
  if (a.rows > (1u << 24) || a.heads > (1u << 16) || a.kv_heads > (1u << 16) || a.pos_base > (uint64_t{1} << 48) ||
      a.q_stride > (uint64_t{1} << 32) || a.k_stride > (uint64_t{1} << 32) || a.k_row > (uint64_t{1} << 40) || a.k_f16 > 1 ||
      a.rows * (a.heads + a.kv_heads) > 0x3FFFFFCull) {               // (a wavefront each: fewer than 2^32 threads)
    return "qk_norm_rope/mrope: a scalar is out of range";
  }
  if (!(a.theta > 0.0f) || a.theta > 3.4e38f || !(a.eps >= 0.0f) || a.eps > 3.4e38f) {
    return "qk_norm_rope/mrope: theta must be positive, eps not negative, both finite";
  }
  if (axes) {
    const uint64_t sec_w = s[8];
    if (a.sec_t > a.rope_dim || a.sec_h > a.rope_dim || sec_w > a.rope_dim || a.sec_t + a.sec_h + sec_w > a.rope_dim / 2) {
      return "qk_norm_mrope: the sections hold more pairs than rope_dim / 2";
    }
  }
  const uint64_t q_row = a.heads * a.head_dim * (a.gated ? 2 : 1), k_row = a.kv_heads * a.head_dim;
  if (a.q_stride == 0) a.q_stride = q_row;
  if (a.k_stride == 0) a.k_stride = k_row;
  if (a.q_stride < q_row || a.k_stride < k_row) return "qk_norm_rope/mrope: a stride is shorter than a row";
  using u128 = unsigned __int128;
  const u128 q_in = (static_cast<u128>(a.rows - 1) * a.q_stride + q_row) * 4, k_in = (static_cast<u128>(a.rows - 1) * a.k_stride + k_row) * 4;
  const u128 q_bytes = static_cast<u128>(a.rows) * a.heads * a.head_dim * 4, elem = a.k_f16 != 0 ? 2 : 4;
  const u128 k_all = static_cast<u128>(a.k_row + a.rows) * k_row * elem, w = a.head_dim * 4;
  const size_t o = a.q_out;
  if (!c.fits(0, q_in) || !c.fits(1, k_in) || !c.fits(2, w) || !c.fits(3, w) || (axes && !c.fits(4, static_cast<u128>(a.rows) * 24)) ||
      !c.fits(o, q_bytes) || !c.fits(o + 1, k_all) || (a.gated && !c.fits(o + 2, q_bytes))) {
    return "qk_norm_rope/mrope: a buffer is smaller than the scalars require";
  }
  // An output may be its own input where the two have the same layout; any other overlap is refused.
  const bool q_same = c.buf[o] == c.buf[0] && !a.gated && a.q_stride == q_row;
  const bool k_same = c.buf[o + 1] == c.buf[1] && a.k_f16 == 0 && a.k_row == 0 && a.k_stride == k_row;
  const u128 in[5] = {q_in, k_in, w, w, static_cast<u128>(a.rows) * 24}, res[3] = {q_bytes, k_all, q_bytes};
  for (size_t i = 0; i < (a.gated ? 3u : 2u); ++i) {
    for (size_t j = 0; j < (axes ? 5u : 4u); ++j) {
      if ((i == 0 && j == 0 && q_same) || (i == 1 && j == 1 && k_same)) continue;
      if (c.overlap(o + i, res[i], j, in[j])) return "qk_norm_rope/mrope: an output overlaps an input of another layout";
    }
    for (size_t j = 0; j < i; ++j) {
      if (c.overlap(o + i, res[i], o + j, res[j])) return "qk_norm_rope/mrope: outputs overlap";
    }
  }
  *out = a;
  return nullptr;
}

// "attention_tree": buffers Q, K, V, Mask, Out; scalars m, n, heads, kv_heads, head_dim, tree, window, kv_f16.
// "attention_tree_q8" / "_q4" / "_fp8" (kind 2, 3, 4): Q, K, V, Ks, Vs, Mask, Out; without kv_f16.
inline const char* check_attention_tree(const LaunchArgs& c, bool quantized, uint32_t kind) {
  if (c.nbuf != (quantized ? 7u : 5u) || c.nsc != (quantized ? 7u : 8u)) {
    return "attention_tree: expects 5 buffers and 8 scalars (over a quantized cache 7 and 7)";
  }
  const uint64_t m = c.sc[0], n = c.sc[1], heads = c.sc[2], kv_heads = c.sc[3], head_dim = c.sc[4], tree = c.sc[5];
  if (m == 0 || n == 0 || heads == 0 || kv_heads == 0 || head_dim == 0 || heads % kv_heads != 0) {
    return "attention_tree: m, n, heads, kv_heads, head_dim must be non-zero and heads a multiple of kv_heads";
  }
  if (head_dim > 256) return "attention_tree: head_dim must be at most 256";
  if (tree == 0 || tree > n || tree > kTreeKeysMost) return "attention_tree: the tree holds one key at least, n and 65536 at most";
  if (!quantized && c.sc[7] > 1) return "attention_tree: kv_f16 is 0 or 1";
  if (kind == 3 && (kv_heads * head_dim) % 2 != 0) return "attention_tree_q4: a key row must hold an even number of codes";
  if (m > (1u << 24) || n > (uint64_t{1} << 31) || heads > (1u << 16) || c.sc[6] > (uint64_t{1} << 48) || m * heads > 0xFFFFFFull) {
    return "attention_tree: a scalar is out of range";
  }
  using u128 = unsigned __int128;
  const u128 q = static_cast<u128>(m) * heads * head_dim * 4, codes = static_cast<u128>(n) * kv_heads * head_dim;
  const u128 kv = kind == 3 ? codes / 2 : quantized ? codes : codes * (c.sc[7] != 0 ? 2 : 4);
  const u128 mask = static_cast<u128>(m) * ((tree + 31) / 32) * 4;
  const size_t at = quantized ? 5 : 3;
  bool ok = c.fits(0, q) && c.fits(1, kv) && c.fits(2, kv) && c.fits(at, mask) && c.fits(at + 1, q);
  if (quantized) ok = ok && c.fits(3, static_cast<u128>(n) * 4) && c.fits(4, static_cast<u128>(n) * 4);
  if (!ok) return "attention_tree: a buffer is smaller than the scalars require";
  for (size_t i = 0; i <= at; ++i) {
    const u128 need = i == 0 ? q : i <= 2 ? kv : i == at ? mask : static_cast<u128>(n) * 4;
    if (c.overlap(at + 1, q, i, need)) return "attention_tree: the output overlaps an input";
  }
  return nullptr;
}

// "token_logprobs": buffers Logits, Tokens, Logprobs, Entropy[, TopTokens, TopLogprobs]; scalars rows, vocab, tokens, top_k, row_base.
inline const char* check_token_logprobs(const LaunchArgs& c) {
  if (c.nsc != 5 || (c.nbuf != 4 && c.nbuf != 6)) return "token_logprobs: expects 4 buffers (6 with top_k) and 5 scalars";
  const uint64_t rows = c.sc[0], vocab = c.sc[1], tokens = c.sc[2], top_k = c.sc[3], row_base = c.sc[4];
  if (rows == 0 || vocab == 0 || tokens == 0) return "token_logprobs: rows, vocab and tokens must be non-zero";
  if (rows > (1u << 30) || vocab > 0x7FFFFFFFull || row_base > (uint64_t{1} << 40) || tokens > kLogprobTokensMost) {
    return "token_logprobs: a scalar is out of range (at most 1024 tokens a row)";
  }
  if (top_k > kLogprobTopMost || top_k > vocab || (top_k != 0) != (c.nbuf == 6)) {
    return "token_logprobs: top_k is 0 (4 buffers) or 1..32 and at most vocab (6 buffers)";
  }
  using u128 = unsigned __int128;
  const u128 need[6] = {static_cast<u128>(row_base + rows) * vocab * 4, static_cast<u128>(rows) * tokens * 4, static_cast<u128>(rows) * tokens * 4,
                        static_cast<u128>(rows) * 4, static_cast<u128>(rows) * top_k * 4, static_cast<u128>(rows) * top_k * 4};
  for (size_t i = 0; i < c.nbuf; ++i) {
    if (!c.fits(i, need[i])) return "token_logprobs: a buffer is smaller than the scalars require";
  }
  for (size_t i = 2; i < c.nbuf; ++i) {
    for (size_t j = 0; j < i; ++j) {
      if (c.overlap(i, need[i], j, need[j])) return "token_logprobs: an output overlaps another buffer";
    }
  }
  return nullptr;
}

}  // namespace qmm

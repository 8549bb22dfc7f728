// What the ids around a paged cache ("pages_write_q8", "pages_write_fp8", "pages_read_q8", "pages_read_fp8", "attention_pages_q8",
// "attention_pages_fp8") and "draft_verify" refuse.  Host logic only, no HIP calls: each check returns nullptr or why a launch
// is refused.  What lies in device memory (starts, lengths, page numbers, tokens) cannot be refused: the kernels leave out what
// does not hold.
#pragma once

#include "tree_args.hpp"

namespace qmm {

constexpr uint64_t kPageSequencesMost = 4096;            // a wavefront walks their starts 64 at a time
constexpr uint64_t kPagePositionsMost = uint64_t{1} << 30;   // of a sequence: 32-bit arithmetic on positions stays in range
constexpr uint64_t kDraftVocabMost = uint64_t{1} << 21;

// The batch and the pool, as all three families take them.
struct PageCall {
  uint64_t rows, kv_heads, head_dim, sequences, block, pages, width;
  // Pages that `rows` rows of `sequences` sequences lie in, at most.
  uint64_t touched() const {
    const uint64_t some = rows / block + 2 * sequences;
    return rows < some ? rows : some;
  }
  unsigned __int128 codes() const { return static_cast<unsigned __int128>(pages) * kv_heads * block * head_dim; }
  unsigned __int128 scales() const { return static_cast<unsigned __int128>(pages) * kv_heads * 4; }
  unsigned __int128 table() const { return static_cast<unsigned __int128>(sequences) * width * 4; }
};

inline const char* check_page_call(const PageCall& a) {
  if (a.rows == 0 || a.kv_heads == 0 || a.head_dim == 0 || a.sequences == 0 || a.pages == 0 || a.width == 0) {
    return "rows, heads, head_dim, sequences, pages and width must be non-zero";
  }
  if (a.head_dim % 16 != 0 || a.head_dim > 256) return "head_dim must be a multiple of 16, at most 256";
  if (a.block != 16 && a.block != 32 && a.block != 64 && a.block != 128) return "a page holds 16, 32, 64 or 128 positions";
  if (a.rows > (1u << 24) || a.kv_heads > (1u << 12) || a.sequences > kPageSequencesMost || a.pages > 0x7FFFFFFFull ||
      a.width > kPagePositionsMost || a.width * a.block > kPagePositionsMost) {
    return "a scalar is out of range (at most 2^24 rows, 4096 sequences and key heads, 2^30 positions a sequence)";
  }
  return nullptr;
}

// A text that says which id it is about.
inline const char* about(const char* id, const char* why) {
  static thread_local char text[192];
  if (why == nullptr) return nullptr;
  size_t at = 0;
  for (const char* p = id; *p != 0 && at < sizeof(text) - 3; ++p) text[at++] = *p;
  text[at++] = ':', text[at++] = ' ';
  for (const char* p = why; *p != 0 && at < sizeof(text) - 1; ++p) text[at++] = *p;
  text[at] = 0;
  return text;
}

// No written buffer shares memory with another.
template <size_t N>
inline bool page_buffers_apart(const LaunchArgs& c, const unsigned __int128 (&need)[N], const bool (&written)[N]) {
  for (size_t i = 0; i < N; ++i) {
    for (size_t j = 0; j < i; ++j) {
      if ((written[i] || written[j]) && c.overlap(i, need[i], j, need[j])) return false;
    }
  }
  return true;
}
template <size_t N>
inline bool page_buffers_fit(const LaunchArgs& c, const unsigned __int128 (&need)[N]) {
  for (size_t i = 0; i < N; ++i) {
    if (!c.fits(i, need[i])) return false;
  }
  return true;
}

// "pages_write_*": buffers K, V, Table, Starts, Lens, Kp, Vp, Ks, Vs; scalars rows, kv_heads, head_dim, sequences, block, pages,
// width, k_stride, v_stride.
struct PageWriteCall {
  PageCall page;
  uint64_t k_stride, v_stride;
};
inline const char* check_pages_write(const LaunchArgs& c, PageWriteCall* out) {
  const char* id = "pages_write";
  if (c.nbuf != 9 || c.nsc != 9) return about(id, "expects 9 buffers and 9 scalars");
  PageWriteCall a{{c.sc[0], c.sc[1], c.sc[2], c.sc[3], c.sc[4], c.sc[5], c.sc[6]}, c.sc[7], c.sc[8]};
  if (const char* why = check_page_call(a.page)) return about(id, why);
  const uint64_t row = a.page.kv_heads * a.page.head_dim;
  if (a.k_stride == 0) a.k_stride = row;
  if (a.v_stride == 0) a.v_stride = row;
  if (a.k_stride < row || a.v_stride < row || a.k_stride % 4 != 0 || a.v_stride % 4 != 0 || a.k_stride > (uint64_t{1} << 32) ||
      a.v_stride > (uint64_t{1} << 32)) {
    return about(id, "a stride is a multiple of 4 floats, no shorter than a row and at most 2^32");
  }
  if (a.page.touched() * a.page.kv_heads >= (1u << 22)) return about(id, "more pages and heads than a launch holds (2^22)");
  using u128 = unsigned __int128;
  const u128 k = (static_cast<u128>(a.page.rows - 1) * a.k_stride + row) * 4, v = (static_cast<u128>(a.page.rows - 1) * a.v_stride + row) * 4;
  const u128 need[9] = {k, v, a.page.table(), (a.page.sequences + 1) * 4, a.page.sequences * 4, a.page.codes(), a.page.codes(), a.page.scales(), a.page.scales()};
  if (!page_buffers_fit(c, need)) return about(id, "a buffer is smaller than the scalars require");
  const bool written[9] = {false, false, false, false, false, true, true, true, true};
  if (!page_buffers_apart(c, need, written)) return about(id, "the pool overlaps another buffer");
  *out = a;
  return nullptr;
}

// "pages_read_*": buffers Kp, Vp, Ks, Vs, Table, Starts, Lens, K, V; scalars rows, kv_heads, head_dim, sequences, block, pages,
// width, out_f16.
struct PageReadCall {
  PageCall page;
  bool f16;
};
inline const char* check_pages_read(const LaunchArgs& c, PageReadCall* out) {
  const char* id = "pages_read";
  if (c.nbuf != 9 || c.nsc != 8) return about(id, "expects 9 buffers and 8 scalars");
  const PageReadCall a{{c.sc[0], c.sc[1], c.sc[2], c.sc[3], c.sc[4], c.sc[5], c.sc[6]}, c.sc[7] == 1};
  if (const char* why = check_page_call(a.page)) return about(id, why);
  if (c.sc[7] > 1) return about(id, "out_f16 is 0 or 1");
  if (a.page.touched() * a.page.kv_heads >= (1u << 22)) return about(id, "more pages and heads than a launch holds (2^22)");
  using u128 = unsigned __int128;
  const u128 rows = static_cast<u128>(a.page.rows) * a.page.kv_heads * a.page.head_dim * (a.f16 ? 2 : 4);
  const u128 need[9] = {a.page.codes(), a.page.codes(), a.page.scales(), a.page.scales(), a.page.table(), (a.page.sequences + 1) * 4, a.page.sequences * 4, rows, rows};
  if (!page_buffers_fit(c, need)) return about(id, "a buffer is smaller than the scalars require");
  const bool written[9] = {false, false, false, false, false, false, false, true, true};
  if (!page_buffers_apart(c, need, written)) return about(id, "an output overlaps another buffer");
  *out = a;
  return nullptr;
}

// "attention_pages_*": buffers Q, Kp, Vp, Ks, Vs, Table, Starts, Lens, Out; scalars rows, heads, kv_heads, head_dim, sequences,
// block, pages, width, max_rows, max_len, window, sinks.
struct PageAttentionCall {
  PageCall page;
  uint64_t heads, max_rows, max_len, window, sinks;
};
inline const char* check_attention_pages(const LaunchArgs& c, PageAttentionCall* out) {
  const char* id = "attention_pages";
  if (c.nbuf != 9 || c.nsc != 12) return about(id, "expects 9 buffers and 12 scalars");
  PageAttentionCall a{{c.sc[0], c.sc[2], c.sc[3], c.sc[4], c.sc[5], c.sc[6], c.sc[7]}, c.sc[1], c.sc[8], c.sc[9], c.sc[10], c.sc[11]};
  if (const char* why = check_page_call(a.page)) return about(id, why);
  if (a.heads == 0 || a.heads % a.page.kv_heads != 0 || a.heads > (1u << 16)) return about(id, "heads is a multiple of kv_heads, at most 65536");
  if (a.page.rows * a.heads > 0xFFFFFFull || a.page.sequences * a.page.kv_heads > (1u << 21)) {
    return about(id, "at most 2^24 - 1 rows times heads and 2^21 sequences times kv_heads");      // (a grid of fewer than 2^32 threads)
  }
  const uint64_t most = a.page.width * a.page.block;
  if (a.max_rows > a.page.rows || a.max_len > most) return about(id, "max_rows is at most rows, max_len at most width times block (0: just that)");
  if (a.max_rows == 0) a.max_rows = a.page.rows;
  if (a.max_len == 0) a.max_len = most;
  if (a.window > (uint64_t{1} << 48) || a.sinks > (uint64_t{1} << 48)) return about(id, "window and sinks are at most 2^48");
  if (a.window == 0 && a.sinks != 0) return about(id, "sinks go with a window (without one every position is seen)");
  using u128 = unsigned __int128;
  const u128 q = static_cast<u128>(a.page.rows) * a.heads * a.page.head_dim * 4;
  const u128 need[9] = {q, a.page.codes(), a.page.codes(), a.page.scales(), a.page.scales(), a.page.table(), (a.page.sequences + 1) * 4, a.page.sequences * 4, q};
  if (!page_buffers_fit(c, need)) return about(id, "a buffer is smaller than the scalars require");
  const bool written[9] = {false, false, false, false, false, false, false, false, true};
  if (!page_buffers_apart(c, need, written)) return about(id, "the output overlaps an input");
  *out = a;
  return nullptr;
}

// "draft_verify": buffers Logits, Tokens, Random, Starts, Accepted, Next[, DraftLogits]; scalars rows, vocab, sequences,
// temperature, draft_temperature.
struct DraftCall {
  uint64_t rows, vocab, sequences;
  float temperature, draft_temperature;
  bool draft;
};
inline const char* check_draft_verify(const LaunchArgs& c, DraftCall* out) {
  const char* id = "draft_verify";
  if ((c.nbuf != 6 && c.nbuf != 7) || c.nsc != 5) return about(id, "expects 6 buffers (7 with the draft's logits) and 5 scalars");
  const DraftCall a{c.sc[0], c.sc[1], c.sc[2], scalar_f32(c.sc[3]), scalar_f32(c.sc[4]), c.nbuf == 7};
  if (a.rows == 0 || a.vocab == 0 || a.sequences == 0) return about(id, "rows, vocab and sequences must be non-zero");
  if (a.rows > (1u << 20) || a.vocab > kDraftVocabMost || a.sequences > kPageSequencesMost) {
    return about(id, "at most 2^20 rows, a vocabulary of 2^21 and 4096 sequences");
  }
  if (!(a.temperature >= 0.0f) || a.temperature > 3.4e38f) return about(id, "temperature is 0 (the likeliest token) or positive and finite");
  if (a.draft && a.temperature > 0.0f && (!(a.draft_temperature > 0.0f) || a.draft_temperature > 3.4e38f)) {
    return about(id, "draft_temperature is positive and finite");
  }
  using u128 = unsigned __int128;
  const u128 logits = static_cast<u128>(a.rows) * a.vocab * 4;
  const u128 need[7] = {logits, a.rows * 4, a.rows * 8, (a.sequences + 1) * 4, a.sequences * 4, a.sequences * 4, a.draft ? logits : 0};
  for (size_t i = 0; i < c.nbuf; ++i) {
    if (!c.fits(i, need[i])) return about(id, "a buffer is smaller than the scalars require");
  }
  for (size_t i = 4; i < 6; ++i) {
    for (size_t j = 0; j < c.nbuf; ++j) {
      if (i != j && c.overlap(i, need[i], j, need[j])) return about(id, "an output overlaps another buffer");
    }
  }
  *out = a;
  return nullptr;
}

}  // namespace qmm

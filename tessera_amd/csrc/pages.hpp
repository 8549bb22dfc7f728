// A pool of pages of 8-bit keys and values, and the batch of sequences that lies in it: what the kernels of "pages_write_*",
// "pages_read_*" and "attention_pages_*" share.
//
// A page holds `block` positions of one sequence.  Keys lie [page][kv_head][position][element], values
// [page][kv_head][element][position], each under one fp32 scale for a page and key head ([page][kv_head]): a run of sixteen bytes of
// either is what a lane of the matrix instruction takes, elements of a key for the scores, positions of an element for the sums,
// so that no value is transposed on its way there.  Sequence s has Lens[s] positions, of which the call's rows Starts[s] ..
// Starts[s + 1] - 1 are the last; its page j is Table[s * width + j].
#pragma once

#include <type_traits>

#include "page_args.hpp"
#include "qmm_device.hpp"

namespace qmm {

enum class PageKind { Q8, Fp8 };

struct PageBatch {
  const uint32_t *table, *starts, *lens;
  uint32_t rows, sequences, pages, width, max_rows, max_len;
  uint32_t kv_heads, head_dim, log_block;
};
PageBatch page_batch(const PageCall& call, const uint32_t* table, const uint32_t* starts, const uint32_t* lens);

namespace {

constexpr float page_largest(PageKind kind) { return kind == PageKind::Q8 ? 127.0f : 448.0f; }

// A sequence of the batch: its rows of the call (from `first` on) and its length.  What does not hold (no rows, rows behind the
// call's last or beyond what the launch was made for, more rows than positions, more positions than the table has) counts as no rows.
struct PageSequence {
  uint32_t first, rows, len;
};
__device__ __forceinline__ PageSequence page_sequence(const PageBatch& b, uint32_t s) {
  const uint32_t first = b.starts[s], end = b.starts[s + 1u], len = b.lens[s];
  const bool holds = first < end && end <= b.rows && end - first <= len && end - first <= b.max_rows && len <= b.max_len;
  return PageSequence{first, holds ? end - first : 0u, len};
}

// Sums over the lanes up to this one (of a wavefront whose lanes are all there): in rows of sixteen, then from row to row.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  auto add = [&](auto ctrl, auto rows) { v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), ctrl.value, rows.value, 0xF, false)); };
  add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});
  add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
  add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
  add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});     // a row's last to the next row
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});     // the second row's last to the upper two
  return v;
}

// The unit `unit` of the batch, `of(sequence)` to each: its sequence and its place among that one's.  All lanes of a wavefront
// call it alike; false: there are fewer units.
struct PageUnit {
  uint32_t s, at;
  PageSequence seq;
};
template <class Of>
__device__ __forceinline__ bool find_unit(const PageBatch& b, uint32_t unit, Of of, PageUnit* out) {
  const uint32_t lane = threadIdx.x & 63u;
  for (uint32_t base = 0; base < b.sequences; base += 64u) {
    const uint32_t s = base + lane;
    PageSequence seq{0u, 0u, 0u};
    if (s < b.sequences) seq = page_sequence(b, s);
    const uint32_t own = seq.rows == 0u ? 0u : of(seq);
    const uint32_t sum = wave_scan(own);
    const uint32_t all = __builtin_amdgcn_readlane(sum, 63);
    if (unit < all) {
      const int hit = __ffsll(static_cast<unsigned long long>(__ballot(sum > unit))) - 1;
      auto from = [&](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), hit)); };
      out->s = base + static_cast<uint32_t>(hit);
      out->at = unit - (from(sum) - from(own));
      out->seq = PageSequence{from(seq.first), from(seq.rows), from(seq.len)};
      return true;
    }
    unit -= all;
  }
  return false;
}

// Pages that the rows of a sequence lie in.
__device__ __forceinline__ uint32_t touched_pages(const PageBatch& b, const PageSequence& seq) {
  return ((seq.len - 1u) >> b.log_block) - ((seq.len - seq.rows) >> b.log_block) + 1u;
}

}  // namespace
}  // namespace qmm

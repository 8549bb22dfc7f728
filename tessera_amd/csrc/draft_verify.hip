// "draft_verify": how many of each sequence's drafted tokens stand, and the token that follows them.
//
// Row i of a sequence holds the target's logits for the token after Tokens[i]; Tokens[i + 1] was drafted for it, but for the last row.
// With p = softmax(logits / temperature) and q the draft's likewise (none: the draft is one token, q = 1), the draft's token x
// stands where u q(x) < p(x), u the row's first random number.  At the first that does not the next token is drawn from max(p - q, 0)
// (none: p without x), behind the last one from p: the first whose running sum exceeds the row's second random number times the
// whole.  Temperature 0: a token stands where it is the likeliest, the lowest of equals.
//
// Which token it is hangs on sums next to a border, so everything from the logits on is fp64: exponentials to 2^-39, sums over chunks of
// 512 columns, a wavefront each, and then over chunks, in an order that the vocabulary alone decides.  What is left of a row but for
// a token, or of all of it, is known from the chunks' statistics; max(p - q, 0) takes another pass over the two rows.
//
// Two launches: the statistics of all rows, a wavefront a chunk; then a workgroup a sequence, or where drafts have probabilities as
// many as fill the chip, of which the last to arrive draws.  Without scratch a workgroup takes a sequence, with the same bits.
// The first is bound by the fp64 instructions, some twenty a logit (100 rows of 131072 of target and draft each: 29 us, 3.6 TB/s), the
// second by one way to memory after the other (8 us without the draft's probabilities, 13 with them, 20 for 32 sequences): nothing is to
// keep it waiting besides, above all no array or struct with padding that the compiler would put into LDS by the dispatch packet's sizes,
// which lies in the host's memory (22 us of 32).

#include "page_args.hpp"
#include "qmm_device.hpp"
#include "qmm_kernels.hpp"

namespace qmm {
namespace {

constexpr uint32_t kEach = 8, kChunk = 64 * kEach, kWaves = 8, kThreads = 64 * kWaves, kChunksMost = static_cast<uint32_t>(kDraftVocabMost) / kChunk;
constexpr uint32_t kNoToken = 0xFFFFFFFFu;

// Of a chunk of a row: the largest logit (NaN: there is a NaN or +infinity), where (the lowest of equals), the sum of exp relative to it.
struct ChunkStats {
  double sum;
  float most;
  uint32_t arg;
};

struct DraftArgs {
  const float *logits, *draft, *random;
  const uint32_t *tokens, *starts;
  uint32_t *accepted, *next;
  uint32_t rows, vocab, sequences, chunks, groups;    // groups: workgroups of a sequence in the second launch
  double scale, draft_scale;         // 1 / (temperature ln 2); 0: the likeliest token
  ChunkStats* stats;                 // (plane, row, chunk)
  double* rest;                      // (sequence, chunk)
  uint32_t* arrived;                 // (sequence): workgroups whose chunks are there
};

// 2^y for y <= 0: 2^n 2^f, |f| <= 1/2, 2^f by the polynomial of degree 8 that meets it at the nine Chebyshev points, of which one is 0: off
// by 1.1e-12 at most.  n is what adding 1.5 2^52 leaves in the low bits; below y = -1000 it is 2^-1000 (in a sum beside a 1: nothing).
__device__ __forceinline__ double exp2_near(double y) {
  y = fmax(y, -1000.0);
  const double whole = y + 0x1.8p52, f = y - (whole - 0x1.8p52);
  double s = 0x1.63d1363a681b4p-20;
  s = fma(s, f, 0x1.00dc4a5344ef5p-16);
  s = fma(s, f, 0x1.4308ac85a69f8p-13);
  s = fma(s, f, 0x1.5d8745a728209p-10);
  s = fma(s, f, 0x1.3b2ab7181b77dp-7);
  s = fma(s, f, 0x1.c6b08dd6fd236p-5);
  s = fma(s, f, 0x1.ebfbdff823cedp-3);
  s = fma(s, f, 0x1.62e42fef84cf0p-1);
  s = fma(s, f, 1.0);
  const uint64_t bits = bit_cast<uint64_t>(s);
  const uint32_t high = static_cast<uint32_t>(bits >> 32) + (static_cast<uint32_t>(bit_cast<uint64_t>(whole)) << 20);
  return bit_cast<double>(static_cast<uint64_t>(high) << 32 | static_cast<uint32_t>(bits));
}
__device__ __forceinline__ double power_near(float logit, double most, double scale) {
  return exp2_near((static_cast<double>(logit) - most) * scale);
}
// 0 where the probability is (and below 2^-1000).
__device__ __forceinline__ double power(float logit, float most, double scale) {
  const double y = (static_cast<double>(logit) - static_cast<double>(most)) * scale;
  return y > -1000.0 ? exp2_near(y) : 0.0;
}

// ---- over a wavefront, within its registers ------------------------------------------------------

// v moved across lanes by `CTRL`; `otherwise` where no lane reaches.
template <int CTRL, int ROWS = 0xF, class T>
__device__ __forceinline__ T moved(T v, T otherwise) {
  if constexpr (sizeof(T) == 4) {
    return bit_cast<T>(__builtin_amdgcn_update_dpp(bit_cast<int>(otherwise), bit_cast<int>(v), CTRL, ROWS, 0xF, false));
  } else {
    const uint64_t x = bit_cast<uint64_t>(v), y = bit_cast<uint64_t>(otherwise);
    const uint32_t low = moved<CTRL, ROWS>(static_cast<uint32_t>(x), static_cast<uint32_t>(y));
    const uint32_t high = moved<CTRL, ROWS>(static_cast<uint32_t>(x >> 32), static_cast<uint32_t>(y >> 32));
    return bit_cast<T>(static_cast<uint64_t>(high) << 32 | low);
  }
}
template <class T>
__device__ __forceinline__ T lane_of(T v, uint32_t lane) {
  if constexpr (sizeof(T) == 4) {
    return bit_cast<T>(__builtin_amdgcn_readlane(bit_cast<int>(v), static_cast<int>(lane)));
  } else {
    const uint64_t x = bit_cast<uint64_t>(v);
    return bit_cast<T>(static_cast<uint64_t>(lane_of(static_cast<uint32_t>(x >> 32), lane)) << 32 | lane_of(static_cast<uint32_t>(x), lane));
  }
}
// with(a, b) over all lanes up to a lane's own (`zero`: what changes nothing); lane 63 has the whole.
template <class T, class With>
__device__ __forceinline__ T scan(T v, T zero, With with) {
  v = with(moved<0x111>(v, zero), v);        // row_shr:1, 2, 4, 8
  v = with(moved<0x112>(v, zero), v);
  v = with(moved<0x114>(v, zero), v);
  v = with(moved<0x118>(v, zero), v);
  v = with(moved<0x142, 0xA>(v, zero), v);   // row_bcast:15, 31
  return with(moved<0x143, 0xC>(v, zero), v);
}
__device__ __forceinline__ double scan_sum(double v) {
  return scan(v, 0.0, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ double whole_sum(double v) { return lane_of(scan_sum(v), 63); }
__device__ __forceinline__ float whole_max(float v) {
  return lane_of(scan(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); }), 63);
}
__device__ __forceinline__ uint32_t whole_min(uint32_t v) {
  return lane_of(scan(v, ~0u, [](uint32_t a, uint32_t b) { return a < b ? a : b; }), 63);
}

// ---- a row's statistics --------------------------------------------------------------------------

// A lane's logits of a chunk, 64 apart; past the row's end -infinity.  (Four in a row a lane, where rows begin at 16 bytes, took as long.)
struct Columns {
  float x[kEach];
};
__device__ __forceinline__ Columns columns_of(const float* row, uint32_t vocab, uint32_t chunk) {
  const uint32_t first = chunk * kChunk + (threadIdx.x & 63u);
  Columns c;
  if (chunk * kChunk + kChunk <= vocab) {                           // wavefront-uniform
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) c.x[j] = row[first + 64u * j];
  } else {
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
      const uint32_t e = first + 64u * j;
      const float v = row[e < vocab ? e : vocab - 1u];
      c.x[j] = e < vocab ? v : -INFINITY;
    }
  }
  return c;
}
// By a wavefront, in every lane.  `scale` 0: no sum, else no place.
__device__ __forceinline__ ChunkStats chunk_stats(const Columns& c, uint32_t chunk, double scale) {
  const uint32_t first = chunk * kChunk + (threadIdx.x & 63u);
  float most = c.x[0];
  bool bad = !(c.x[0] < INFINITY);
#pragma unroll
  for (uint32_t j = 1; j < kEach; ++j) bad = bad || !(c.x[j] < INFINITY), most = fmaxf(most, c.x[j]);
  most = whole_max(most);
  bad = __any(bad);
  uint32_t arg = kNoToken;
  double sum = 0.0;
  if (scale == 0.0) {
#pragma unroll
    for (uint32_t j = kEach; j-- > 0;) {
      if (c.x[j] == most) arg = first + 64u * j;
    }
    arg = whole_min(most == -INFINITY ? kNoToken : arg);
  } else if (!bad && most > -INFINITY) {
    const double to = static_cast<double>(most);
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) sum += power_near(c.x[j], to, scale);
    sum = whole_sum(sum);
  }
  return ChunkStats{sum, bad ? bit_cast<float>(0x7FC00000u) : most, arg};
}

// From its chunks', by a wavefront, in every lane.  A row that is no distribution (NaN or +infinity, or -infinity alone) has NaN as its
// largest.
struct RowStats {
  double sum;
  float most;
  uint32_t arg;
};
__device__ __forceinline__ bool is_bad(const RowStats& r) { return r.most != r.most; }
constexpr uint32_t kAhead = 4;                                      // chunks a lane that are asked for at once
struct Held {
  ChunkStats of[kAhead];
};
// What lies past the last chunk changes nothing.
__device__ __forceinline__ Held hold(const ChunkStats* chunks, uint32_t count, uint32_t base) {
  Held h;
#pragma unroll
  for (uint32_t i = 0; i < kAhead; ++i) {
    const uint32_t c = base + (threadIdx.x & 63u) + 64u * i;
    h.of[i] = chunks[c < count ? c : 0u];
    if (c >= count) h.of[i] = ChunkStats{0.0, -INFINITY, kNoToken};
  }
  return h;
}
__device__ __forceinline__ RowStats row_stats(const Held& first, const ChunkStats* chunks, uint32_t count, double scale) {
  double sum = 0.0;
  float most = -INFINITY;
  uint32_t arg = kNoToken;
  bool bad = false;
  Held h = first;
  auto each = [&](auto with) {                                      // (more chunks than are held: a second and third time from memory)
    for (uint32_t base = 0;;) {
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i) with(h.of[i]);
      base += 64u * kAhead;
      if (base >= count) break;
      h = hold(chunks, count, base);
    }
    if (count > 64u * kAhead) h = first;
  };
  each([&](const ChunkStats& c) { bad = bad || c.most != c.most, most = fmaxf(most, c.most); });
  most = whole_max(most);
  if (__any(bad) || most == -INFINITY) return RowStats{0.0, bit_cast<float>(0x7FC00000u), kNoToken};
  if (scale == 0.0) {
    each([&](const ChunkStats& c) { arg = c.most == most && c.arg < arg ? c.arg : arg; });
    return RowStats{0.0, most, whole_min(arg)};
  }
  each([&](const ChunkStats& c) { sum += c.sum * power(c.most, most, scale); });
  return RowStats{whole_sum(sum), most, kNoToken};
}

// ---- where a sequence's draft ends ---------------------------------------------------------------

// (without padding: what is copied between registers and LDS is registers)
struct Verdict {
  RowStats target, draft;
  uint32_t row, at, token, is;       // of the call; of the sequence; the draft's token; kEnds ..
};
constexpr uint32_t kEnds = 1, kRefused = 2, kBad = 4;               // it is the last; the draft's token does not stand; the row says nothing
__device__ __forceinline__ bool sequence_rows(const DraftArgs& a, uint32_t s, uint32_t* first, uint32_t* rows) {
  const uint32_t begin = a.starts[s], end = a.starts[s + 1u];
  *first = begin, *rows = end - begin;
  return begin < end && end <= a.rows;
}
// Row `at` of a sequence, by a wavefront, from its chunks' statistics; `draft` those of the draft's row, unless `of_draft` is `known`.
__device__ __forceinline__ Verdict verdict_of(const DraftArgs& a, const ChunkStats* target, const ChunkStats* draft, uint32_t first, uint32_t rows, uint32_t at,
                                         bool known, RowStats of_draft) {
  Verdict v;
  v.draft = of_draft;
  v.row = first + at, v.at = at;
  const bool last = at + 1u == rows, both = !last && a.draft != nullptr && !known;
  const uint32_t token = a.tokens[v.row + (last ? 0u : 1u)];
  const Held of_target = hold(target, a.chunks, 0u);
  Held of_q = of_target;
  if (both) of_q = hold(draft, a.chunks, 0u);
  v.token = last ? 0u : token;
  const uint64_t place = static_cast<uint64_t>(v.row) * a.vocab + (!last && v.token < a.vocab ? v.token : 0u);
  const float logit = a.logits[place], of_draft_logit = a.draft != nullptr ? a.draft[place] : 0.0f, u = a.random[2u * static_cast<uint64_t>(v.row)];
  v.target = row_stats(of_target, target, a.chunks, a.scale);
  if (both) v.draft = row_stats(of_q, draft, a.chunks, a.draft_scale);
  if (is_bad(v.target) || (!last && a.draft != nullptr && is_bad(v.draft))) {
    v.is = kEnds | kBad;
  } else if (last) {
    v.is = kEnds;
  } else if (a.scale == 0.0) {
    v.is = v.target.arg != v.token ? kEnds | kRefused : 0u;
  } else {
    double p = 0.0, q = 1.0;
    if (v.token < a.vocab) {
      p = power(logit, v.target.most, a.scale) / v.target.sum;
      if (a.draft != nullptr) q = power(of_draft_logit, v.draft.most, a.draft_scale) / v.draft.sum;
    }
    v.is = static_cast<double>(u) * q < p ? 0u : kEnds | kRefused;
  }
  return v;
}

// ---- what is left of the row that is drawn from --------------------------------------------------

// Relative to the row's largest probability, so that equal logits have sums without rounding and two rows alike have nothing left.
__device__ __forceinline__ double rest_of(const DraftArgs& a, const Verdict& v, double share, float logit, float of_draft, uint32_t e) {
  const double p = power(logit, v.target.most, a.scale);
  if ((v.is & kRefused) == 0u) return p;
  if (a.draft == nullptr) return e == v.token ? 0.0 : p;
  const double less = p - power(of_draft, v.draft.most, a.draft_scale) * share;
  return less > 0.0 ? less : 0.0;
}
__device__ __forceinline__ double share_of(const DraftArgs& a, const Verdict& v) { return a.draft != nullptr && (v.is & kRefused) != 0u ? v.target.sum / v.draft.sum : 0.0; }
// A lane's columns of a chunk, apart by `step` from `from` on.
__device__ __forceinline__ void chunk_rest(const DraftArgs& a, const Verdict& v, uint32_t chunk, uint32_t from, uint32_t step, double (&rest)[kEach]) {
  const double share = share_of(a, v);
  const bool both = a.draft != nullptr && (v.is & kRefused) != 0u;
  const uint64_t row = static_cast<uint64_t>(v.row) * a.vocab;
  const uint32_t base = chunk * kChunk + from;
  float x[kEach], y[kEach];
#pragma unroll
  for (uint32_t j = 0; j < kEach; ++j) x[j] = a.logits[row + (base + step * j < a.vocab ? base + step * j : 0u)];
#pragma unroll
  for (uint32_t j = 0; j < kEach; ++j) y[j] = both ? a.draft[row + (base + step * j < a.vocab ? base + step * j : 0u)] : 0.0f;
#pragma unroll
  for (uint32_t j = 0; j < kEach; ++j) {
    const uint32_t e = base + step * j;
    const double r = rest_of(a, v, share, x[j], y[j], e);
    rest[j] = e < a.vocab ? r : 0.0;
  }
}
// The chunk's sum, by a wavefront, in every lane.
__device__ __forceinline__ double chunk_sum(const DraftArgs& a, const Verdict& v, uint32_t chunk) {
  double rest[kEach], sum = 0.0;
  chunk_rest(a, v, chunk, threadIdx.x & 63u, 64u, rest);
#pragma unroll
  for (uint32_t j = 0; j < kEach; ++j) sum += rest[j];
  return whole_sum(sum);
}

// The draw, by a wavefront, in every lane: `stats` are the target row's chunks, `rest` the chunks' sums where the draft has probabilities and
// was refused.  A lane has a run of chunks, then of columns.
__device__ __forceinline__ uint32_t draw_token(const DraftArgs& a, Verdict v, const ChunkStats* stats, const double* rest) {
  const uint32_t lane = threadIdx.x & 63u, per = (a.chunks + 63u) / 64u, first = lane * per, end = first + per < a.chunks ? first + per : a.chunks;
  const float u = a.random[2u * static_cast<uint64_t>(v.row) + 1u];
  // a chunk without the refused token is what its statistics say; the other is summed without it
  const uint32_t without = (v.is & kRefused) != 0u && a.draft == nullptr && v.token < a.vocab ? v.token / kChunk : kNoToken;
  const double special = without != kNoToken ? chunk_sum(a, v, without) : 0.0;
  auto sum_of = [&](uint32_t c) {
    if ((v.is & kRefused) != 0u && a.draft != nullptr) return __hip_atomic_load(rest + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (c == without && (v.is & kRefused) != 0u) return special;
    const ChunkStats& s = stats[c];
    return s.most > -INFINITY ? s.sum * power(s.most, v.target.most, a.scale) : 0.0;
  };
  auto own_sum = [&] {
    double own = 0.0;
    for (uint32_t c = first; c < end; ++c) own += sum_of(c);
    return own;
  };
  double own = own_sum(), run = scan_sum(own), whole = lane_of(run, 63);
  if (!(whole > 0.0)) {                                             // the draft accounts for all of p: p itself
    v.is &= ~kRefused;
    own = own_sum(), run = scan_sum(own), whole = lane_of(run, 63);
  }
  // (a number outside [0, 1) is the nearest in it)
  const double goal = (u >= 0.0f ? static_cast<double>(fminf(u, 0x1.fffffep-1f)) : 0.0) * whole;
  // The first with something whose running sum exceeds the goal; where rounding leaves none, the last with something.  (Running sums of
  // lanes are not of one order of additions: by a rounding that of a lane with nothing may exceed the goal where the one before does not.)
  auto first_over = [](bool over, bool any) {
    const uint64_t some = __ballot(over && any), last = __ballot(any);
    return some != 0u ? static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(some)) - 1)
                      : 63u - static_cast<uint32_t>(__clzll(static_cast<unsigned long long>(last | 1u)));
  };
  uint32_t holds = first_over(run > goal, own > 0.0), chunk = first;
  double before = run - own, to = before;
  for (uint32_t c = first; c < end && lane == holds; ++c) {
    const double s = sum_of(c);
    if (s > 0.0) chunk = c, before = to;
    to += s;
    if (to > goal) break;
  }
  chunk = lane_of(chunk, holds);
  const double left = goal - lane_of(before, holds);
  double column[kEach];
  chunk_rest(a, v, chunk, lane * kEach, 1u, column);
  own = 0.0;
#pragma unroll
  for (uint32_t j = 0; j < kEach; ++j) own += column[j];
  run = scan_sum(own);
  holds = first_over(run > left, own > 0.0);
  to = run - own;
  uint32_t token = 0u;
  bool found = false;
#pragma unroll
  for (uint32_t j = 0; j < kEach; ++j) {
    to += column[j];
    if (column[j] > 0.0 && !found) token = j, found = to > left;
  }
  return chunk * kChunk + lane_of(lane * kEach + token, holds);
}

__device__ __forceinline__ void put(const DraftArgs& a, uint32_t s, const Verdict& v, uint32_t token) {
  if ((threadIdx.x & 63u) == 0u) a.accepted[s] = v.at, a.next[s] = (v.is & kBad) != 0u ? kNoToken : token;
}

// ---- in two launches -----------------------------------------------------------------------------

// A wavefront goes from chunk to chunk, the next one's loads under way.
__global__ __launch_bounds__(kThreads) void draft_stats_kernel(DraftArgs a, uint32_t all) {
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), step = gridDim.x * kWaves;
  for (uint32_t i = blockIdx.x * kThreads + threadIdx.x; i < a.sequences; i += gridDim.x * kThreads) a.arrived[i] = 0u;
  auto columns = [&](uint32_t at) {
    const uint32_t chunk = at % a.chunks, rest = at / a.chunks, row = rest % a.rows;
    return columns_of((rest < a.rows ? a.logits : a.draft) + static_cast<uint64_t>(row) * a.vocab, a.vocab, chunk);
  };
  uint32_t at = blockIdx.x * kWaves + wave;
  if (at >= all) return;
  Columns now = columns(at);
  for (; at < all; at += step) {
    const Columns next = columns(at + step < all ? at + step : at);
    const ChunkStats s = chunk_stats(now, at % a.chunks, at / a.chunks < a.rows ? a.scale : a.draft_scale);
    if ((threadIdx.x & 63u) == 0u) a.stats[at] = s;
    now = next;
  }
}

struct RestShared {
  Verdict of[kWaves];
  uint32_t before;
};
// The row at which a sequence's draft ends, by a workgroup, a wavefront a row, from all rows' statistics.
__device__ __forceinline__ Verdict find_end(const DraftArgs& a, uint32_t first, uint32_t rows, RestShared& sh) {
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
  for (uint32_t base = 0;; base += kWaves) {
    __syncthreads();
    if (base + wave < rows) {
      const uint64_t at = static_cast<uint64_t>(first + base + wave) * a.chunks;
      const Verdict v = verdict_of(a, a.stats + at, a.stats + static_cast<uint64_t>(a.rows) * a.chunks + at, first, rows, base + wave, false, RowStats{0.0, 0.0f, 0u});
      if (lane == 0u) sh.of[wave] = v;
    } else if (lane == 0u) {
      sh.of[wave].is = 0u;
    }
    __syncthreads();
    const uint64_t ends = __ballot(lane < kWaves && (sh.of[lane % kWaves].is & kEnds) != 0u);
    if (ends != 0u) return sh.of[__ffsll(static_cast<unsigned long long>(ends)) - 1];      // (the last row does)
  }
}

__global__ __launch_bounds__(kThreads) void draft_rest_kernel(DraftArgs a) {
  __shared__ RestShared sh;
  const uint32_t each = a.groups, s = blockIdx.x / each, share = blockIdx.x % each;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t first, rows;
  if (!sequence_rows(a, s, &first, &rows)) return;
  const Verdict v = find_end(a, first, rows, sh);
  const bool apart = a.draft != nullptr && (v.is & kRefused) != 0u;      // its sums are formed by all of the sequence's workgroups
  if (!apart && share != 0u) return;
  double* rest = a.rest + static_cast<uint64_t>(s) * a.chunks;
  if (apart) {
    for (uint32_t chunk = share * kWaves + wave; chunk < a.chunks; chunk += each * kWaves) {
      const double sum = chunk_sum(a, v, chunk);
      if ((threadIdx.x & 63u) == 0u) __hip_atomic_store(rest + chunk, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // The sums go from XCD to XCD within the launch, past the L2s: each wavefront's is there before its workgroup is counted.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0u) sh.before = __hip_atomic_fetch_add(a.arrived + s, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (sh.before + 1u != each) return;                             // workgroup-uniform
  }
  if (wave != 0u) return;
  uint32_t token = v.target.arg;
  if (a.scale != 0.0 && (v.is & kBad) == 0u) token = draw_token(a, v, a.stats + static_cast<uint64_t>(v.row) * a.chunks, rest);
  put(a, s, v, token);
}

// ---- a workgroup a sequence ----------------------------------------------------------------------

struct AloneShared {
  ChunkStats stats[kChunksMost];
  double rest[kChunksMost];
};
__global__ __launch_bounds__(kThreads) void draft_alone_kernel(DraftArgs a) {
  __shared__ AloneShared sh;
  const uint32_t s = blockIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t first, rows;
  if (!sequence_rows(a, s, &first, &rows)) return;
  auto gather = [&](const float* plane, uint32_t row, double scale) {
    __syncthreads();
    for (uint32_t c = wave; c < a.chunks; c += kWaves) {
      const ChunkStats x = chunk_stats(columns_of(plane + static_cast<uint64_t>(row) * a.vocab, a.vocab, c), c, scale);
      if ((threadIdx.x & 63u) == 0u) sh.stats[c] = x;
    }
    __syncthreads();
  };
  Verdict v;
  v.is = 0u;
  for (uint32_t at = 0; at < rows && (v.is & kEnds) == 0u; ++at) {
    RowStats draft{0.0, 0.0f, 0u};                                               // the draft's first, of which only the row's statistics are kept
    if (a.draft != nullptr && at + 1u < rows) {
      gather(a.draft, first + at, a.draft_scale);
      draft = row_stats(hold(sh.stats, a.chunks, 0u), sh.stats, a.chunks, a.draft_scale);
    }
    gather(a.logits, first + at, a.scale);
    v = verdict_of(a, sh.stats, nullptr, first, rows, at, true, draft);
  }
  if (a.draft != nullptr && (v.is & kRefused) != 0u) {
    for (uint32_t c = wave; c < a.chunks; c += kWaves) {
      const double sum = chunk_sum(a, v, c);
      if ((threadIdx.x & 63u) == 0u) sh.rest[c] = sum;
    }
    __syncthreads();
  }
  if (wave != 0u) return;
  uint32_t token = v.target.arg;
  if (a.scale != 0.0 && (v.is & kBad) == 0u) token = draw_token(a, v, sh.stats, sh.rest);
  put(a, s, v, token);
}

uint32_t chunks_of(const DraftCall& c) { return static_cast<uint32_t>((c.vocab + kChunk - 1) / kChunk); }
bool reads_draft(const DraftCall& c) { return c.draft && c.temperature > 0.0f; }

}  // namespace

size_t draft_verify_scratch_bytes(const DraftCall& c) {
  return static_cast<size_t>((c.rows * (reads_draft(c) ? 2 : 1) * sizeof(ChunkStats) + c.sequences * sizeof(double)) * chunks_of(c) + c.sequences * sizeof(uint32_t));
}

hipError_t launch_draft_verify(const DraftCall& c, const float* logits, const uint32_t* tokens, const float* random, const uint32_t* starts,
                               uint32_t* accepted, uint32_t* next, const float* draft, void* scratch, hipStream_t stream) {
  DraftArgs a{};
  a.logits = logits, a.draft = reads_draft(c) ? draft : nullptr, a.random = random, a.tokens = tokens, a.starts = starts;
  a.accepted = accepted, a.next = next;
  a.rows = static_cast<uint32_t>(c.rows), a.vocab = static_cast<uint32_t>(c.vocab), a.sequences = static_cast<uint32_t>(c.sequences);
  a.chunks = chunks_of(c);
  constexpr double kLog2E = 1.4426950408889634074;
  a.scale = c.temperature > 0.0f ? kLog2E / static_cast<double>(c.temperature) : 0.0;
  a.draft_scale = a.draft != nullptr ? kLog2E / static_cast<double>(c.draft_temperature) : 0.0;
  if (scratch == nullptr) {
    hipLaunchKernelGGL(draft_alone_kernel, dim3(a.sequences), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  }
  const uint32_t planes = a.draft != nullptr ? 2u : 1u, all = planes * a.rows * a.chunks;
  a.stats = static_cast<ChunkStats*>(scratch);
  a.rest = reinterpret_cast<double*>(a.stats + all);
  a.arrived = reinterpret_cast<uint32_t*>(a.rest + static_cast<size_t>(a.sequences) * a.chunks);
  const uint32_t cus = static_cast<uint32_t>(num_cus()), needed = (all + kWaves - 1u) / kWaves;
  hipLaunchKernelGGL(draft_stats_kernel, dim3(needed < 4u * cus ? needed : 4u * cus), dim3(kThreads), 0, stream, a, all);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  a.groups = 1u;
  if (a.draft != nullptr) {
    const uint32_t fill = (2u * cus + a.sequences - 1u) / a.sequences, most = (a.chunks + kWaves - 1u) / kWaves;
    a.groups = fill < most ? fill : most;
  }
  hipLaunchKernelGGL(draft_rest_kernel, dim3(a.sequences * a.groups), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace qmm

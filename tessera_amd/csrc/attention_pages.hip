// "attention_pages_q8", "attention_pages_fp8": the rows of a batch of sequences against their pages of 8-bit keys and values.
//
// Row i of a sequence, at position p, sees the positions up to p; under a window those of them that are among the last `window` or
// the first `sinks` of the sequence.  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = q . k_j / sqrt(head_dim), in one pass
// over the keys with a running reference m.
//
// What is fp32 enters the matrix instructions in pieces.  Over int8 pages a query is an integer of 23 bits and a sign under its row's
// largest element, in three int8 limbs: an element is carried to 2^-23 of the largest, products and sums are exact.  Else it is two fp16
// terms, x = hi + lo, hi = RN16(x), lo = RN16(x - hi), under a power of two that brings a query's largest element to 2^13 .. 2^14 (an
// element is carried to 2^-22 of itself down to 2^-16 of the largest, below to 2^-38 of that), the largest of a row's weights times their
// values' scales so far to 2^9 .. 2^15 (to 2^-22 of itself down to 2^-12 of the largest, below to 2^-34 of that; 2^10 coarser where weights
// are below 2^-116).  Codes enter exactly; a key's scale multiplies its fp32 score.  Scores, references, sums and results are fp32.

#include <type_traits>

#include "launch_rules.hpp"
#include "pages.hpp"
#include "qmm_kernels.hpp"

namespace qmm {
namespace {

constexpr float kLog2E = 1.44269504088896340736f;

struct PageAttention {
  PageBatch batch;
  const float* q;
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  float* out;
  float *part_sum, *part_most, *part_total;   // (unit, key head, part, one of `stored` columns): the part's result; its reference in powers of two; its weights' sum
  uint32_t heads, group, window, sinks;       // window 0: every position
  uint32_t log_tile, parts, part_tiles, stored, even;   // positions a tile; tiles a part; columns of a unit that a part has room for; workgroups of an even split, or 0
};

// ---- which positions a unit walks ----------------------------------------------------------------
//
// A unit is COLUMNS (row, head) pairs of a key head in one sequence, `group` pairs to a row.  It walks tiles of 64 positions, or of 32 where
// pages_log_tile says so: those with sinks that lie before its windows, then those from the first row's window to the last row's position.
struct UnitTiles {
  uint32_t columns;               // that there are
  uint32_t first_col;             // its first among the sequence's
  uint32_t low, high;             // the first and the last row's positions
  uint32_t sink_tiles, from_tile, tiles;
};
__device__ __forceinline__ UnitTiles tiles_between(const PageAttention& a, uint32_t low, uint32_t high) {
  UnitTiles w{};
  w.low = low, w.high = high;
  const uint32_t begin = a.window != 0u && w.low + 1u > a.window ? w.low + 1u - a.window : 0u;
  const uint32_t sinks = a.sinks < begin ? a.sinks : begin;
  w.sink_tiles = (sinks + (1u << a.log_tile) - 1u) >> a.log_tile;
  w.from_tile = begin >> a.log_tile > w.sink_tiles ? begin >> a.log_tile : w.sink_tiles;
  w.tiles = w.sink_tiles + ((w.high >> a.log_tile) + 1u - w.from_tile);
  return w;
}
// The one unit of a sequence whose pairs all fit.
__device__ __forceinline__ UnitTiles sequence_tiles(const PageAttention& a, const PageSequence& seq) {
  UnitTiles w = tiles_between(a, seq.len - seq.rows, seq.len - 1u);
  w.columns = seq.rows * a.group;
  return w;
}
__device__ __forceinline__ UnitTiles unit_tiles(const PageAttention& a, const PageUnit& u, uint32_t most_columns) {
  const uint32_t all = u.seq.rows * a.group, first = u.at * most_columns, columns = all - first < most_columns ? all - first : most_columns;
  const uint32_t past = u.seq.len - u.seq.rows;
  UnitTiles w = tiles_between(a, past + first / a.group, past + (first + columns - 1u) / a.group);
  w.first_col = first, w.columns = columns;
  return w;
}
__device__ __forceinline__ uint32_t tile_at(const UnitTiles& w, uint32_t i) { return i < w.sink_tiles ? i : w.from_tile + (i - w.sink_tiles); }

// What is loaded of a page that the pool has not: a head's keys or values at most, all 0.  (Its positions are hidden, but a code that is NaN
// would reach the sums through a weight of 0.)
alignas(16) __device__ const uint8_t g_no_page[256 * 128] = {};
// (An address of global memory as such: of a choice between that and a buffer's the compiler knows no more than that it is one.)
typedef const __attribute__((address_space(1))) uint8_t* PageBytes;
template <class T>
__device__ __forceinline__ T load_page(PageBytes from) {
  typedef uint32_t words __attribute__((ext_vector_type(sizeof(T) / 4)));
  return bit_cast<T>(*(const __attribute__((address_space(1))) words*)from);
}
__device__ __forceinline__ PageBytes page_bytes_of(const uint8_t* pool, bool held, uint64_t at) { return held ? (PageBytes)pool + at : (PageBytes)g_no_page; }

// ---- operands ------------------------------------------------------------------------------------

// Eight codes (two dwords) as fp16.  The half 0x6400 | u is 1024 + u.
template <PageKind KIND>
__device__ __forceinline__ half8_t operand(uint32_t w0, uint32_t w1) {
  if constexpr (KIND == PageKind::Q8) {
    auto two = [](uint32_t biased, uint32_t sel) {
      const half2_t x = bit_cast<half2_t>(__builtin_amdgcn_perm(0x64646464u, biased, sel));
      return bit_cast<uint32_t>(x - half2_t{static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)});
    };
    const uint32_t x = w0 ^ 0x80808080u, y = w1 ^ 0x80808080u;
    return bit_cast<half8_t>(uint4{two(x, 0x04010400u), two(x, 0x04030402u), two(y, 0x04010400u), two(y, 0x04030402u)});
  } else {
    auto two = [](uint32_t w, auto high) { return bit_cast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, decltype(high)::value)); };
    return bit_cast<half8_t>(uint4{two(w0, std::false_type{}), two(w0, std::true_type{}), two(w1, std::false_type{}), two(w1, std::true_type{})});
  }
}

// Largest / sum over the four groups of sixteen lanes.
__device__ __forceinline__ float groups_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
  v = fmaxf(bit_cast<float>(a[0]), bit_cast<float>(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
  return fmaxf(bit_cast<float>(b[0]), bit_cast<float>(b[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
  v = bit_cast<float>(a[0]) + bit_cast<float>(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
  return bit_cast<float>(b[0]) + bit_cast<float>(b[1]);
}
// 2^(target - exponent of v) for v > 0, within what fp32 can hold.
__device__ __forceinline__ float power_to(float v, int target) {
  const int s = 254 + target - static_cast<int>(bit_cast<uint32_t>(v) >> 23 & 255u);
  return bit_cast<float>(static_cast<uint32_t>(s > 254 ? 254 : s < 1 ? 1 : s) << 23);
}
__device__ __forceinline__ float from_reference(float ref) { return ref == -INFINITY ? 0.0f : ref; }

// Sums times corr, now and then.  In place, by hand: of a branch around products the compiler makes a second set of registers and moves
// the sums from one to the other in every tile.  (The matrix instructions behind the sums have been
// waited for: at most sixteen passes of four cycles.)
template <int N>
__device__ __forceinline__ void scale_sums(float4_t (&o)[N], float corr) {
  asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15\n\ts_nop 15" ::);
#pragma unroll
  for (int x = 0; x < N; ++x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v = o[x][e];
      asm volatile("v_mul_f32 %0, %1, %0" : "+v"(v) : "v"(corr));
      o[x][e] = v;
    }
  }
  asm volatile("s_nop 1" ::);                                       // (before a matrix instruction takes them)
}

// What a sum of weights times values is multiplied by, of weights that are `total` together.  Before all else: a result is no larger than
// its values are, where their sum could be past fp32's range.
__device__ __forceinline__ float share_of(float total) { return total == 0.0f ? 0.0f : 1.0f / total; }

// Weights are taken relative to a reference that follows a column's largest score only where that would leave it by 2^kSlack.
constexpr float kSlack = 3.0f;

// A column's running state in one wavefront: lanes r, 16 + r, 32 + r, 48 + r hold a quarter of each tile's positions.
struct Column {
  float ref = -INFINITY;          // in powers of two
  float sum = 0.0f;               // of weights, this lane's share
  float most = 0.0f;              // a weight times its value's scale that was met, the largest where it was looked for, this lane's
  float up = 0x1p127f;            // the power of two over those
};

// Products to weights times the values' scale, as two terms; `scale` makes a product a score in powers of two.  COUNT of a lane's positions
// of the tile; bit i of `shown`: the column sees the i-th; ALL: every column sees all.  A weight is below 2^kSlack, so that with
// v_scale * up below 2^12 all is as it should be; else, and where the reference moves, the sums so far are to be scaled by *corr (true).
template <bool ALL, int COUNT>
__device__ __forceinline__ bool weigh(Column& c, float (&s)[COUNT], float scale, uint32_t shown, float v_scale, half8_t (&hi)[COUNT / 8],
                                      half8_t (&lo)[COUNT / 8], float* corr) {
  scale = scale == 0.0f ? 0x1p-126f : scale;      // (keys that are all 0: a hidden product stays -infinity)
  if constexpr (!ALL) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) s[i] = (shown >> i & 1u) != 0u ? s[i] : -INFINITY;
  }
  float most = s[0];
#pragma unroll
  for (int i = 1; i < COUNT; ++i) most = fmaxf(most, s[i]);
  most *= scale;
  const bool moves = __any(most > c.ref + kSlack || (c.ref == -INFINITY && most > -INFINITY) || !(v_scale * c.up < 0x1p12f));
  if (moves) {
    const float before = c.ref;
    c.ref = fmaxf(c.ref, groups_max(most));
    float by = before == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(before - c.ref);
    c.sum *= by;
    // A weight counts as 2^-116 at least, so that v_scale * up is finite (the least is 2^-126: their terms begin 2^10 lower at most);
    // without any the scale may be as large as it likes, and nothing is weighed under it.  (NaN stays.)
    const float weight = __builtin_amdgcn_exp2f(most - from_reference(c.ref));
    c.most = fmaxf(c.most * by, (weight > 0.0f ? fmaxf(weight, 0x1p-116f) : 0.0f) * v_scale);
    v_scale = weight == 0.0f && v_scale < INFINITY ? 0.0f : v_scale;
    const float largest = groups_max(c.most), scaled = largest * c.up;
    if (largest > 0.0f && !(scaled >= 0x1p9f && scaled < 0x1p12f)) {
      const float up = power_to(largest, 10);
      by *= up * (1.0f / c.up);                   // (powers of two)
      c.up = up;
    }
    *corr = by;
  }
  const float to = from_reference(c.ref), factor = v_scale * c.up;
  typedef float float2_v __attribute__((ext_vector_type(2)));
  float minus_one = -1.0f;
  asm("" : "+s"(minus_one));                                      // (a product with the fp16 number as it is, not its conversion and a difference)
#pragma unroll
  for (int i = 0; i < COUNT; i += 2) {
    float2_v w;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float p = __builtin_amdgcn_exp2f(fmaf(s[i + e], scale, -to));
      if constexpr (!ALL) p = (shown >> (i + e) & 1u) != 0u ? p : 0.0f;                             // (a hidden position's scales may be NaN)
      c.sum += p;
      w[e] = p * factor;
      if constexpr (!ALL) w[e] = (shown >> (i + e) & 1u) != 0u ? w[e] : 0.0f;
    }
    const half2_t h = __builtin_convertvector(w, half2_t);
    const float2_v rest = {fmaf(static_cast<float>(h[0]), minus_one, w[0]), fmaf(static_cast<float>(h[1]), minus_one, w[1])};
    const half2_t l = __builtin_convertvector(rest, half2_t);
    hi[i / 8][i % 8] = h[0], hi[i / 8][i % 8 + 1] = h[1], lo[i / 8][i % 8] = l[0], lo[i / 8][i % 8 + 1] = l[1];
  }
  return moves;
}

// ---- an even split -------------------------------------------------------------------------------
//
// Of units that are a sequence each: all their tiles, a sequence's heads one behind the other, in runs of equal cost, one a workgroup.
// To begin a head costs what begin_tiles do: so many lie before its first, with nothing in them.  A run that covers a head whole gives
// its result, else it leaves its own for the merge: in the workgroup's first place that of its first head, in its second that of
// a later one.
__device__ __forceinline__ uint32_t even_of(const PageAttention& a, const PageSequence& seq) {
  return seq.rows == 0u ? 0u : sequence_tiles(a, seq).tiles + begin_tiles(a.log_tile);
}
struct EvenTiles {
  uint32_t before, all;           // of a head of the sequences before the s-th; of all
};
__device__ __forceinline__ EvenTiles even_tiles(const PageAttention& a, uint32_t s) {
  uint32_t before = 0u, all = 0u;
  for (uint32_t at = threadIdx.x & 63u; at < a.batch.sequences; at += 64u) {
    const uint32_t own = even_of(a, page_sequence(a.batch, at));
    all += own, before += at < s ? own : 0u;
  }
  auto last = [](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(wave_scan(v)), 63)); };
  return EvenTiles{last(before), last(all)};
}
__device__ __forceinline__ uint32_t even_share(const PageAttention& a, uint32_t all) {
  const uint32_t share = (all * a.batch.kv_heads + a.even - 1u) / a.even, least = begin_tiles(a.log_tile) + 4u;
  return all != 0u && share < least ? least : share;    // (a tile a wavefront)
}

// ---- few columns ---------------------------------------------------------------------------------
//
// Bound by reading the pages.  16 CG columns a workgroup; each wavefront takes every NW-th tile of positions on its own, with no barrier
// between.  S^T = K Q^T and O^T = V^T P^T by matrix instructions of 16 x 16.  Row 4 g + e of the t-th of a tile's key operands is position
// 16 g + 4 t + e (of 32 positions 8 g + 4 t + e), so that lane group g ends up with the scores of the tile's g-th quarter (which lies in
// one page: one scale a lane), and those are the ones of the value operands that it loads: no score changes its lane.  A register that
// an operand was made from takes the next tile's at once, so that a tile's loads have a whole tile's time.  The queries' operands lie in LDS, one
// copy for all wavefronts.
// 48 sequences of up to 8000 positions, 24 heads over 4 of 256, int8, 395 MB: 82 us, 4.8 TB/s; 5 rows on 65000, 32 over 8 of 128, E4M3, 133 MB:
// 33 us, of which 5 pass until the first tile is there and 4 until the last workgroup has begun; 1 row on 1187, 16 over 4 of 64: 9 us,
// of which 2.2 go by before the sequence is found, 2 before its tiles are there, 1.5 a tile for the longest wavefront.
constexpr int query_operands(PageKind kind, int dp) { return kind == PageKind::Q8 ? 3 * (dp / 64) : 2 * (dp / 32); }

template <PageKind KIND, int DP, int CG, int NW>
struct FewShared {
  union {
    uint4 q[CG][query_operands(KIND, DP)][64];
    alignas(16) float o[NW][16 * CG][DP + 4];
  };
  float ref[NW][16 * CG], sum[NW][16 * CG];
};

// A row's elements 64 x + 16 g + e of lane group g.
template <int DP>
__device__ __forceinline__ void query_load(const float* q, uint32_t D, float (&raw)[DP / 64][16]) {
  const uint32_t g = (threadIdx.x & 63u) >> 4;
#pragma unroll
  for (int x = 0; x < DP / 64; ++x) {
    const uint32_t d = 64u * x + 16u * g;
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const float4 v = *reinterpret_cast<const float4*>(q + (d < D ? d : 0u) + e);
      raw[x][e] = d < D ? v.x : 0.0f, raw[x][e + 1] = d < D ? v.y : 0.0f, raw[x][e + 2] = d < D ? v.z : 0.0f, raw[x][e + 3] = d < D ? v.w : 0.0f;
    }
  }
}

// Those as operands: over int8 pages the limbs of three of them, else two terms of the sixteen in two steps.  Returns what a score is to
// be multiplied by.  Only the operands of steps `x % step == own` are written.
template <PageKind KIND, int DP>
__device__ __forceinline__ float query_terms(const float (&raw)[DP / 64][16], uint32_t D, uint4 (*to)[64], uint32_t own, uint32_t step) {
  const uint32_t lane = threadIdx.x & 63u;
  float most = 0.0f;
  bool odd = false;
#pragma unroll
  for (int x = 0; x < DP / 64; ++x) {
#pragma unroll
    for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(raw[x][e])), odd = odd || !(fabsf(raw[x][e]) < INFINITY);
  }
  most = groups_max(most);
  const float natural = kLog2E / sqrtf(static_cast<float>(D));
  if constexpr (KIND == PageKind::Q8) {
    constexpr float kMost = 8355584.0f;                            // three limbs hold 127 more, which rounding cannot reach
    const float up = most == 0.0f ? 1.0f : power_to(most, 0), whole = most == 0.0f ? 1.0f : most * up, scale = kMost / whole;
    odd = groups_max(odd ? 1.0f : 0.0f) != 0.0f;
#pragma unroll
    for (int x = 0; x < DP / 64; ++x) {
      if (static_cast<uint32_t>(x) % step != own) continue;
      uint32_t limb[3][4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t n[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // two's complement with each byte's carry into the next: n + 0x8080 has bytes limb + 128 but for the highest
          n[e] = (static_cast<uint32_t>(static_cast<int>(__builtin_rintf(raw[x][4 * w + e] * up * scale))) + 0x8080u) ^ 0x8080u;
        }
#pragma unroll
        for (uint32_t i = 0; i < 3; ++i) {
          const uint32_t low = __builtin_amdgcn_perm(n[1], n[0], 0x0C0C0400u + 0x0101u * i), high = __builtin_amdgcn_perm(n[3], n[2], 0x04000C0Cu + 0x01010000u * i);
          limb[i][w] = low | high;
        }
      }
#pragma unroll
      for (int i = 0; i < 3; ++i) to[3 * x + i][lane] = uint4{limb[i][0], limb[i][1], limb[i][2], limb[i][3]};
    }
    // (an infinity or NaN: all scores NaN)
    return odd ? bit_cast<float>(0x7FC00000u) : natural * (whole / kMost) / up;
  } else {
    const float up = most == 0.0f ? 1.0f : power_to(most, 13);
#pragma unroll
    for (int x = 0; x < DP / 32; ++x) {
      if (static_cast<uint32_t>(x) % step != own) continue;
      half8_t hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = raw[x / 2][8 * (x % 2) + e] * up;
        hi[e] = static_cast<_Float16>(v);
        lo[e] = static_cast<_Float16>(v - static_cast<float>(hi[e]));
      }
      to[2 * x][lane] = bit_cast<uint4>(hi), to[2 * x + 1][lane] = bit_cast<uint4>(lo);
    }
    return natural / up;
  }
}

typedef int int4_t __attribute__((ext_vector_type(4)));


template <PageKind KIND, int DP, int CG, int NW>
__global__ __launch_bounds__(NW * 64, 2) void attention_pages_few_kernel(PageAttention a) {
  constexpr int KL = DP / 64, VL = DP / 16, C = 16 * CG;
  constexpr uint32_t TILE = 1u << pages_log_tile(DP, C), OWN = TILE / 4;      // positions of a tile, and of a lane's
  constexpr int NT = TILE / 16;                                     // key operands
  __shared__ FewShared<KIND, DP, CG, NW> sh;
  const PageBatch& b = a.batch;
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = __builtin_amdgcn_readfirstlane(t >> 6), r = lane & 15u, g = lane >> 4;
  const uint32_t D = b.head_dim, block = 1u << b.log_block;
  uint32_t at_tile = 0u, last_tile = 0u;
  if (a.even != 0u) {
    const uint32_t share = even_share(a, even_tiles(a, 0u).all);
    at_tile = blockIdx.x * share, last_tile = at_tile + share;
  }
  for (bool first_run = true;; first_run = false) {
    PageUnit u;
    UnitTiles w;
    uint32_t kv, begin, end;
    uint64_t slot;
    if (a.even != 0u) {
      if (at_tile >= last_tile || !find_unit(b, at_tile, [&](const PageSequence& q) { return even_of(a, q) * b.kv_heads; }, &u)) return;
      const uint32_t in = u.at;
      w = sequence_tiles(a, u.seq);
      constexpr uint32_t EMPTY = begin_tiles(TILE == 32 ? 5 : 6);
      const uint32_t wide = w.tiles + EMPTY, from = in % wide, left = last_tile - at_tile, to = wide - from < left ? wide : from + left;
      kv = in / wide;
      if (to <= EMPTY) return;                                       // (the next workgroup begins it)
      begin = from > EMPTY ? from - EMPTY : 0u, end = to - EMPTY;
      slot = 2u * static_cast<uint64_t>(blockIdx.x) + (first_run ? 0u : 1u);
      at_tile += to - from;
    } else {
      const uint32_t rest = blockIdx.x / b.kv_heads, part = rest % a.parts;
      if (!first_run || !find_unit(b, rest / a.parts, [](const PageSequence&) { return 1u; }, &u)) return;
      w = sequence_tiles(a, u.seq);
      kv = blockIdx.x % b.kv_heads, begin = part * a.part_tiles;
      if (begin >= w.tiles) return;
      end = w.tiles - begin < a.part_tiles ? w.tiles : begin + a.part_tiles;
      slot = (static_cast<uint64_t>(rest / a.parts) * b.kv_heads + kv) * a.parts + part;
    }
    const uint32_t past = u.seq.len - u.seq.rows;

    // Page numbers of a tile's quarters r / 4 (keys) and g (values, scores).  Positions behind the last are the last page's.
    const uint32_t* table = b.table + static_cast<uint64_t>(u.s) * b.width;
    const uint32_t last_slot = (u.seq.len - 1u) >> b.log_block;
    auto slot_of = [&](uint32_t position) {
      const uint32_t s = position >> b.log_block;
      return s < last_slot ? s : last_slot;
    };
    struct Numbers {
      uint32_t k, v;
    };
    auto numbers = [&](uint32_t i) {
      const uint32_t p0 = tile_at(w, i) * TILE;
      return Numbers{table[slot_of(p0 + (r >> 2) * OWN)], table[slot_of(p0 + g * OWN)]};
    };
    uint4 kr[NT][KL];
    std::conditional_t<OWN == 16, uint4, uint2> vr[VL];
    float ks, vs;
    bool known;
    const uint64_t page_bytes = static_cast<uint64_t>(b.kv_heads) * block * D;
    // Where a lane's runs of a tile begin.  (Elements past head_dim meet zeros of the queries, or are not stored.)
    const uint32_t past_end = 16u * g < D % 64u ? 0u : 16u * g - (D % 64u == 0u ? 0u : D % 64u - 16u);       // in a run of 64 that is not whole
    auto keys_at = [&](uint32_t i, const Numbers& n) {
      const uint32_t at = (tile_at(w, i) * TILE + (r >> 2) * OWN) & (block - 1u);
      return page_bytes_of(a.k, n.k < b.pages, n.k * page_bytes + kv * block * D) + ((at + (r & 3u)) * D + 16u * g);
    };
    auto values_at = [&](uint32_t i, const Numbers& n) {
      const uint32_t at = (tile_at(w, i) * TILE + g * OWN) & (block - 1u);
      return page_bytes_of(a.v, n.v < b.pages, n.v * page_bytes + kv * block * D) + (r * block + at);
    };
    auto fetch_keys = [&](PageBytes from, int y, int x) {
      const PageBytes at = 64u * x + 64u <= D ? from : from - past_end;
      kr[y][x] = load_page<uint4>(at + (4u * y * D + (64u * x < D ? 64u * x : 0u)));
    };
    auto fetch_values = [&](PageBytes from, int x) {
      const PageBytes at = from + (16u * x < D ? 16u * x * block : 0u);   // (uniform: no register of its own)
      vr[x] = load_page<std::remove_reference_t<decltype(vr[x])>>(at);
    };
    auto fetch_scales = [&](const Numbers& n) {
      known = n.v < b.pages;
      const uint64_t at = static_cast<uint64_t>(known ? n.v : 0u) * b.kv_heads + kv;
      ks = a.k_scale[at], vs = a.v_scale[at];
    };

    // This lane's columns; past the last one, the last.  Their loads are before the tile's, behind whose numbers they need not wait.
    // (No branches: where they meet again everything would be waited for.  A wavefront without a tile loads the last one.)
    uint32_t i = begin + wave;
    const uint32_t own = i < end ? i : end - 1u;
    const Numbers now = numbers(own);
    Numbers next = numbers(i + NW < end ? i + NW : own);
    uint32_t pos[CG];
    float q_scale[CG], raw[CG][DP / 64][16];
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) {
      const uint32_t at = cg * 16u + r, col = at < w.columns ? at : w.columns - 1u, row = col / a.group;
      pos[cg] = past + row;
      query_load<DP>(a.q + (static_cast<uint64_t>(u.seq.first + row) * a.heads + kv * a.group + col % a.group) * D, D, raw[cg]);
    }
    {
      const PageBytes from_k = keys_at(own, now), from_v = values_at(own, now);
      fetch_scales(now);
#pragma unroll
      for (int y = 0; y < NT; ++y) {
#pragma unroll
        for (int x = 0; x < KL; ++x) fetch_keys(from_k, y, x);
      }
#pragma unroll
      for (int x = 0; x < VL; ++x) fetch_values(from_v, x);
    }
    // Each wavefront makes a share of the operands.
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) q_scale[cg] = query_terms<KIND, DP>(raw[cg], D, sh.q[cg], wave, NW);
    lds_barrier();

    Column col[CG];
    float4_t o[CG][VL];
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
      for (int x = 0; x < VL; ++x) o[cg][x] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    auto tile = [&](auto last) {
      constexpr bool MORE = !decltype(last)::value;
      const uint32_t first = tile_at(w, i) * TILE;
      const float k_scale = ks, v_scale = vs;
      const bool in_pool = known;
      PageBytes from_k = nullptr, from_v = nullptr;
      if constexpr (MORE) from_k = keys_at(i + NW, next), from_v = values_at(i + NW, next);
      float4_t acc[CG][NT];
      if constexpr (KIND == PageKind::Q8) {
        constexpr int YB = CG == 2 ? 1 : 2;                            // key operands that share a query operand's way from LDS
#pragma unroll
        for (int y0 = 0; y0 < NT; y0 += YB) {
          uint32_t from = lane;
          if constexpr (YB == 1) asm volatile("" : "+v"(from));         // (the queries are read once more, not held)
          int4_t sum[CG][YB][3];
#pragma unroll
          for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
            for (int y = 0; y < YB; ++y) sum[cg][y][0] = sum[cg][y][1] = sum[cg][y][2] = int4_t{0, 0, 0, 0};
          }
#pragma unroll
          for (int x = 0; x < KL; ++x) {
#pragma unroll
            for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
              for (int n = 0; n < 3; ++n) {
                const int4_t q = bit_cast<int4_t>(sh.q[cg][3 * x + n][from]);
#pragma unroll
                for (int y = 0; y < YB; ++y) {
                  sum[cg][y][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bit_cast<int4_t>(kr[y0 + y][x]), q, sum[cg][y][n], 0, 0, 0);
                }
              }
            }
            if constexpr (MORE) {
#pragma unroll
              for (int y = 0; y < YB; ++y) fetch_keys(from_k, y0 + y, x);
            }
          }
#pragma unroll
          for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
            for (int y = 0; y < YB; ++y) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                // (the lower two together are below 2^31)
                const float low = static_cast<float>((sum[cg][y][1][e] << 8) + sum[cg][y][0][e]);
                acc[cg][y0 + y][e] = fmaf(static_cast<float>(sum[cg][y][2][e]), 65536.0f, low);
              }
            }
          }
        }
      } else {
#pragma unroll
        for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
          for (int y = 0; y < NT; ++y) acc[cg][y] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int x = 0; x < 2 * KL; ++x) {
          half8_t hi[CG], lo[CG];
#pragma unroll
          for (int cg = 0; cg < CG; ++cg) hi[cg] = bit_cast<half8_t>(sh.q[cg][2 * x][lane]), lo[cg] = bit_cast<half8_t>(sh.q[cg][2 * x + 1][lane]);
#pragma unroll
          for (int y = 0; y < NT; ++y) {
            const uint4 run = kr[y][x / 2];
            const half8_t key = x % 2 == 0 ? operand<KIND>(run.x, run.y) : operand<KIND>(run.z, run.w);
#pragma unroll
            for (int cg = 0; cg < CG; ++cg) {
              acc[cg][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, lo[cg], acc[cg][y], 0, 0, 0);
              acc[cg][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, hi[cg], acc[cg][y], 0, 0, 0);
            }
            if constexpr (MORE) {
              if (x % 2 == 1) fetch_keys(from_k, y, x / 2);
            }
          }
        }
      }
      if constexpr (MORE) {
        fetch_scales(next);
        if (i + 2 * NW < end) next = numbers(i + 2 * NW);
      }
      // Every column sees every position of the tile, or it goes by bits.
      const bool all = first + (TILE - 1u) <= w.low && (a.window == 0u || first + a.window > w.high) && __all(in_pool);
      half8_t p_hi[CG][OWN / 8], p_lo[CG][OWN / 8];
#pragma unroll
      for (int cg = 0; cg < CG; ++cg) {
        float s[OWN], corr;
#pragma unroll
        for (uint32_t e = 0; e < OWN; ++e) s[e] = acc[cg][e / 4][e % 4];
        bool moves;
        if (all) {
          moves = weigh<true>(col[cg], s, q_scale[cg] * k_scale, 0u, v_scale, p_hi[cg], p_lo[cg], &corr);
        } else {
          const uint32_t p0 = first + OWN * g;
          uint32_t shown = 0u;
#pragma unroll
          for (uint32_t e = 0; e < OWN; ++e) {
            const uint32_t p = p0 + e;
            const bool sees = (p <= pos[cg]) & ((a.window == 0u) | (pos[cg] - p < a.window) | (p < a.sinks)) & in_pool;
            shown |= (sees ? 1u : 0u) << e;
          }
          moves = weigh<false>(col[cg], s, q_scale[cg] * k_scale, shown, v_scale, p_hi[cg], p_lo[cg], &corr);
        }
        if (moves) scale_sums(o[cg], corr);
      }
#pragma unroll
      for (int x = 0; x < VL; ++x) {
        half8_t value[OWN / 8];
        value[0] = operand<KIND>(vr[x].x, vr[x].y);
        if constexpr (OWN == 16) value[1] = operand<KIND>(vr[x].z, vr[x].w);
#pragma unroll
        for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
          for (uint32_t n = 0; n < OWN / 8; ++n) o[cg][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value[n], p_lo[cg][n], o[cg][x], 0, 0, 0);
#pragma unroll
          for (uint32_t n = 0; n < OWN / 8; ++n) o[cg][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value[n], p_hi[cg][n], o[cg][x], 0, 0, 0);
        }
        if constexpr (MORE) fetch_values(from_v, x);
      }
    };
    for (; i + NW < end; i += NW) tile(std::false_type{});
    if (i < end) tile(std::true_type{});

    // Merge of the wavefronts' results by the weights that they have under the largest reference.
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) {
      col[cg].sum = groups_sum(col[cg].sum);
      if (g == 0u) sh.ref[wave][cg * 16u + r] = col[cg].ref, sh.sum[wave][cg * 16u + r] = col[cg].sum;
    }
    __syncthreads();                                                  // (no wavefront reads the queries any more)
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) {
      const float share = share_of(col[cg].sum), factor = 1.0f / col[cg].up;
#pragma unroll
      for (int x = 0; x < VL; ++x) *reinterpret_cast<float4_t*>(&sh.o[wave][cg * 16u + r][16 * x + 4 * g]) = o[cg][x] * share * factor;
    }
    __syncthreads();
    const bool whole = begin == 0u && end == w.tiles;                 // no other part has tiles
    slot *= a.stored;
    for (uint32_t e = t; e < w.columns * (D / 4u); e += NW * 64u) {
      const uint32_t c = e / (D / 4u), d = e % (D / 4u) * 4u;
      float top = -INFINITY;
#pragma unroll
      for (int n = 0; n < NW; ++n) top = fmaxf(top, sh.ref[n][c]);
      float weight[NW], total = 0.0f;
#pragma unroll
      for (int n = 0; n < NW; ++n) weight[n] = __builtin_amdgcn_exp2f(sh.ref[n][c] - from_reference(top)) * sh.sum[n][c], total += weight[n];
      const float share = share_of(total);
      float4_t x = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int n = 0; n < NW; ++n) x += *reinterpret_cast<const float4_t*>(&sh.o[n][c][d]) * (weight[n] * share);
      if (total == 0.0f) x = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
      if (whole) {
        const uint32_t pair = c;
        float* to = a.out + (static_cast<uint64_t>(u.seq.first + pair / a.group) * a.heads + kv * a.group + pair % a.group) * D + d;
        *reinterpret_cast<float4_t*>(to) = x;
      } else {
        *reinterpret_cast<float4_t*>(a.part_sum + (slot + c) * D + d) = x;
        if (d == 0u) a.part_most[slot + c] = top, a.part_total[slot + c] = total;
      }
    }
    lds_barrier();                                                    // the next run's queries go where these sums are
  }
}

// ---- many columns --------------------------------------------------------------------------------
//
// Bound by the matrix instructions and the vector instructions beside them.  A workgroup takes 128 columns, a wavefront 16 CG of them and all
// of a tile of 64 positions (HALVES 1); or, where 64 are enough, those, 4 / CG groups of 16 CG times two halves of a tile: of each page's
// sixteen positions of the tile a wavefront takes the first or the last eight, and the halves are merged in the end.  (CG 2 reads half as much
// of the LDS; of heads of 256, and of 128 with all of a tile, its sums are more registers than there are.)  2 x 1500 rows over up to 2000
// more, 24 heads over 4 of 256, 137 GFLOP: 244 us (E4M3 248); 48 over 8 of 128: 281, 282; 32 over 8 of 64: 143, 127 (pages_rule has those of 64
// columns).  As the terms have it, int8 products at twice the rate, that is 1.75 and 2 times the work of fp16 products: 1.0 and 1.1, 0.85 and
// 1.0, 0.55 and 0.7 PFLOP/s.  Of heads of 256 over int8 pages the matrix instructions are busy in two fifths of the cycles, the vector instructions
// (three beside each of the others) in another third, the wavefronts of a SIMD between the same barriers.  (Halves that take turns at
// them, with barriers between, were slower: their registers did not suffice.  So were priorities by half or by phase.)
// The tile's operands lie in LDS, made once for all columns: keys' as few_kernel's (int8 codes as they are), values' as fp16,
// each operand's 64 lanes side by side, so that every write and read is whole lines.  While a tile is multiplied the next one goes to the
// other half of the LDS and the one after that is under way.
template <PageKind KIND, int DP, int HALVES>
struct TileShared {
  static constexpr int KEYS = (KIND == PageKind::Q8 ? 4 : 8) * (DP / 64), VALUES = 2 * (DP / 16);   // operands of a tile
  static constexpr int QUERIES = query_operands(KIND, DP);
  union {
    uint4 stage[2][KEYS + VALUES][64];
    uint4 q[8 / HALVES][QUERIES][64];                               // of groups of 16 columns, before the first tile
    float4_t o[4][DP / 16][HALVES == 2 ? 64 : 1];                   // of the second half, behind the last
  };
  float scale[128 / HALVES], ref[HALVES][128 / HALVES], sum[HALVES][128 / HALVES];
};

template <PageKind KIND, int DP, int CG, int HALVES>
__global__ __launch_bounds__(512 / CG, 2) void attention_pages_tile_kernel(PageAttention a) {
  constexpr int KL = DP / 64, VL = DP / 16, C = 128 / HALVES, WAVES = 8 / CG, GROUPS = WAVES / HALVES;
  constexpr int OWN = 16 / HALVES, NT = 4 / HALVES, SETS = C / 16;  // places of a tile that are a lane's; key operands; groups of 16 columns
  constexpr int KOWN = 4 * KL / WAVES, VOWN = VL / WAVES;           // a thread's runs of a tile
  using Shared = TileShared<KIND, DP, HALVES>;
  __shared__ Shared sh;
  const PageBatch& b = a.batch;
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = __builtin_amdgcn_readfirstlane(t >> 6), r = lane & 15u, g = lane >> 4;
  const uint32_t group = wave % GROUPS, half = wave / GROUPS;
  const uint32_t kv = blockIdx.x % b.kv_heads, rest = blockIdx.x / b.kv_heads, part = rest % a.parts, unit = rest / a.parts;
  PageUnit u;
  if (!find_unit(b, unit, [&](const PageSequence& q) { return (q.rows * a.group + C - 1u) / C; }, &u)) return;
  u.at = (u.seq.rows * a.group + C - 1u) / C - 1u - u.at;           // the last rows, which see most, first
  const UnitTiles w = unit_tiles(a, u, C);
  const uint32_t begin = part * a.part_tiles;
  if (begin >= w.tiles) return;                                     // workgroup-uniform
  const uint32_t end = w.tiles - begin < a.part_tiles ? w.tiles : begin + a.part_tiles;
  const uint32_t D = b.head_dim, block = 1u << b.log_block, past = u.seq.len - u.seq.rows;

  const uint32_t* table = b.table + static_cast<uint64_t>(u.s) * b.width;
  const uint32_t last_slot = (u.seq.len - 1u) >> b.log_block;
  auto slot_of = [&](uint32_t position) {
    const uint32_t s = position >> b.log_block;
    return s < last_slot ? s : last_slot;
  };
  struct Numbers {
    uint32_t k, v;
  };
  auto numbers = [&](uint32_t i) {
    const uint32_t p0 = tile_at(w, i < end ? i : end - 1u) * 64u;
    return Numbers{table[slot_of(p0 + (r >> 2) * 16u)], table[slot_of(p0 + g * 16u)]};
  };
  // A thread's share of a tile: key operand wave % 4, runs wave / 4, ...; value operands wave, wave + WAVES, ...; and its lane's scales.
  uint4 kr[KOWN], vr[VOWN];
  struct Scales {
    float k, v;
    uint32_t known;
  };
  const uint64_t page_bytes = static_cast<uint64_t>(b.kv_heads) * block * D;
  auto key_run = [&](int x) { return (WAVES / 4u) * x + wave / 4u; };
  auto fetch_keys = [&](uint32_t i, const Numbers& n) {
    const uint32_t at = (tile_at(w, i < end ? i : end - 1u) * 64u + (r >> 2) * 16u) & (block - 1u);
    const PageBytes from = page_bytes_of(a.k, n.k < b.pages, n.k * page_bytes + kv * block * D) + (at + (r & 3u) + 4u * (wave & 3u)) * D;
#pragma unroll
    for (int x = 0; x < KOWN; ++x) {
      const uint32_t d = 64u * key_run(x) + 16u * g;
      kr[x] = load_page<uint4>(from + (d < D ? d : 0u));
    }
  };
  auto fetch_values = [&](uint32_t i, const Numbers& n) {
    const uint32_t at = (tile_at(w, i < end ? i : end - 1u) * 64u + g * 16u) & (block - 1u);
    const PageBytes from = page_bytes_of(a.v, n.v < b.pages, n.v * page_bytes + kv * block * D) + at;
#pragma unroll
    for (int x = 0; x < VOWN; ++x) {
      const uint32_t d = 16u * (WAVES * x + wave) + r;
      vr[x] = load_page<uint4>(from + (d < D ? d : r) * block);
    }
  };
  auto fetch_scales = [&](const Numbers& n) {
    const uint32_t known = n.v < b.pages ? 1u : 0u;
    const uint64_t at = static_cast<uint64_t>(known != 0u ? n.v : 0u) * b.kv_heads + kv;
    return Scales{a.k_scale[at], a.v_scale[at], known};
  };
  auto stash_keys = [&](uint32_t to, int x) {
    const uint32_t at = (wave & 3u) * KL + key_run(x);
    if constexpr (KIND == PageKind::Q8) {
      sh.stage[to][at][lane] = kr[x];
    } else {
      sh.stage[to][2u * at][lane] = bit_cast<uint4>(operand<KIND>(kr[x].x, kr[x].y));
      sh.stage[to][2u * at + 1u][lane] = bit_cast<uint4>(operand<KIND>(kr[x].z, kr[x].w));
    }
  };
  auto stash_values = [&](uint32_t to, int x) {
    const uint32_t at = Shared::KEYS + 2u * (WAVES * x + wave);
    sh.stage[to][at][lane] = bit_cast<uint4>(operand<KIND>(vr[x].x, vr[x].y));
    sh.stage[to][at + 1u][lane] = bit_cast<uint4>(operand<KIND>(vr[x].z, vr[x].w));
  };

  const Numbers of_first = numbers(begin), of_second = numbers(begin + 1u);
  Numbers next = numbers(begin + 2u);                               // of the tile after the next
  fetch_keys(begin, of_first);
  fetch_values(begin, of_first);
  Scales scales = fetch_scales(of_first), of_next = fetch_scales(of_second);

  // The queries' operands: a wavefront makes those of 16 columns (of eight wavefronts two share them), and takes those of its own.
  auto column_row = [&](uint32_t at) {
    const uint32_t col = w.first_col + (at < w.columns ? at : w.columns - 1u);
    return col / a.group;
  };
  constexpr uint32_t SHARE = WAVES > SETS ? WAVES / SETS : 1;
#pragma unroll
  for (uint32_t own = wave % SETS; own < SETS; own += WAVES) {
    const uint32_t at = own * 16u + r, col = w.first_col + (at < w.columns ? at : w.columns - 1u), row = col / a.group;
    float raw[DP / 64][16];
    query_load<DP>(a.q + (static_cast<uint64_t>(u.seq.first + row) * a.heads + kv * a.group + col % a.group) * D, D, raw);
    const float scale = query_terms<KIND, DP>(raw, D, sh.q[own], wave / SETS, SHARE);
    if (g == 0u) sh.scale[own * 16u + r] = scale;
  }
  lds_barrier();
  uint4 q[CG][Shared::QUERIES];
  uint32_t pos[CG];
  float q_scale[CG];
#pragma unroll
  for (int cg = 0; cg < CG; ++cg) {
    const uint32_t from = group * CG + cg;
#pragma unroll
    for (int x = 0; x < Shared::QUERIES; ++x) q[cg][x] = sh.q[from][x][lane];
    q_scale[cg] = sh.scale[from * 16u + r];
    pos[cg] = past + column_row(from * 16u + r);
  }
  lds_barrier();                                                    // the first tile goes where they were
#pragma unroll
  for (int x = 0; x < KOWN; ++x) stash_keys(0u, x);
#pragma unroll
  for (int x = 0; x < VOWN; ++x) stash_values(0u, x);
  fetch_keys(begin + 1u, of_second);
  fetch_values(begin + 1u, of_second);
  lds_barrier();

  Column col[CG];
  float4_t o[CG][VL];
#pragma unroll
  for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
    for (int x = 0; x < VL; ++x) o[cg][x] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  for (uint32_t i = begin, buf = 0u; i < end; ++i, buf ^= 1u) {
    const uint32_t first = tile_at(w, i) * 64u;
    const Scales after = fetch_scales(next);
    const Numbers further = numbers(i + 3u);
    // Scores of the key operands 2 half, 2 half + 1.
    float s[CG][OWN];
    if constexpr (KIND == PageKind::Q8) {
#pragma unroll
      for (int y = 0; y < NT; ++y) {
        int4_t sum[CG][3];
#pragma unroll
        for (int cg = 0; cg < CG; ++cg) sum[cg][0] = sum[cg][1] = sum[cg][2] = int4_t{0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < KL; ++x) {
          const int4_t key = bit_cast<int4_t>(sh.stage[buf][(NT * half + y) * KL + x][lane]);
#pragma unroll
          for (int n = 0; n < 3; ++n) {
#pragma unroll
            for (int cg = 0; cg < CG; ++cg) sum[cg][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(key, bit_cast<int4_t>(q[cg][3 * x + n]), sum[cg][n], 0, 0, 0);
          }
          constexpr int EACH = NT * KL / KOWN;
          if ((KL * y + x) % EACH == EACH - 1) stash_keys(buf ^ 1u, (KL * y + x) / EACH);
        }
#pragma unroll
        for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[cg][4 * y + e] = fmaf(static_cast<float>(sum[cg][2][e]), 65536.0f, static_cast<float>((sum[cg][1][e] << 8) + sum[cg][0][e]));
          }
        }
      }
    } else {
      float4_t acc[CG][NT];
#pragma unroll
      for (int y = 0; y < CG * NT; ++y) acc[y / NT][y % NT] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int x = 0; x < 2 * KL; ++x) {
        half8_t key[NT];
#pragma unroll
        for (int y = 0; y < NT; ++y) key[y] = bit_cast<half8_t>(sh.stage[buf][(NT * half + y) * (2 * KL) + x][lane]);
#pragma unroll
        for (int term = 1; term >= 0; --term) {
#pragma unroll
          for (int y = 0; y < NT; ++y) {
#pragma unroll
            for (int cg = 0; cg < CG; ++cg) acc[cg][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key[y], bit_cast<half8_t>(q[cg][2 * x + term]), acc[cg][y], 0, 0, 0);
          }
        }
        if (x % (2 * KL / KOWN) == 1) stash_keys(buf ^ 1u, x / (2 * KL / KOWN));
      }
#pragma unroll
      for (int cg = 0; cg < CG; ++cg) {
#pragma unroll
        for (int e = 0; e < OWN; ++e) s[cg][e] = acc[cg][e / 4][e % 4];
      }
    }
    fetch_keys(i + 2u, next);
    // The first values' operands are on their way while the weights are formed.  (Not of heads of 64, which with 64 columns of E4M3 are three
    // wavefronts a SIMD without.)
    constexpr bool EARLY = DP > 64;
    constexpr int EACH = 4 / CG, STEPS = 2 * VL / HALVES / EACH;    // value operands of a step
    half8_t ahead[EACH];
    auto element = [](int step) { return HALVES == 2 ? step * EACH : step / 2 * EACH; };      // its first set of sixteen elements
    auto read_values = [&](int step) {
      const uint32_t eights = HALVES == 2 ? half : static_cast<uint32_t>(step) % 2u;          // of the places
#pragma unroll
      for (int y = 0; y < EACH; ++y) ahead[y] = bit_cast<half8_t>(sh.stage[buf][Shared::KEYS + 2 * (element(step) + y) + eights][lane]);
    };
    if constexpr (EARLY) read_values(0);
    const bool all = first + 63u <= w.low && (a.window == 0u || first + a.window > w.high) && __all(scales.known != 0u);
    half8_t p_hi[CG][OWN / 8], p_lo[CG][OWN / 8];
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) {
      float corr;
      bool moves;
      if (all) {
        moves = weigh<true>(col[cg], s[cg], q_scale[cg] * scales.k, 0u, scales.v, p_hi[cg], p_lo[cg], &corr);
      } else {
        const uint32_t p0 = first + 16u * g + OWN * half;
        uint32_t shown = 0u;
#pragma unroll
        for (uint32_t e = 0; e < OWN; ++e) {
          const uint32_t p = p0 + e;
          const bool sees = (p <= pos[cg]) & ((a.window == 0u) | (pos[cg] - p < a.window) | (p < a.sinks)) & (scales.known != 0u);
          shown |= (sees ? 1u : 0u) << e;
        }
        moves = weigh<false>(col[cg], s[cg], q_scale[cg] * scales.k, shown, scales.v, p_hi[cg], p_lo[cg], &corr);
      }
      if (moves) scale_sums(o[cg], corr);
    }
#pragma unroll
    for (int step = 0; step < STEPS; ++step) {
      if constexpr (!EARLY) read_values(step);
      half8_t value[EACH];
#pragma unroll
      for (int y = 0; y < EACH; ++y) value[y] = ahead[y];
      if (EARLY && step + 1 < STEPS) read_values(step + 1);
      const int x = element(step), of = HALVES == 2 ? 0 : step % 2, done = element(step + 1);
#pragma unroll
      for (int term = 1; term >= 0; --term) {                       // (the same sum's products four apart)
#pragma unroll
        for (int y = 0; y < EACH; ++y) {
#pragma unroll
          for (int cg = 0; cg < CG; ++cg) {
            o[cg][x + y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value[y], term == 1 ? p_lo[cg][of] : p_hi[cg][of], o[cg][x + y], 0, 0, 0);
          }
        }
      }
      if (done != x && done % WAVES == 0) stash_values(buf ^ 1u, done / WAVES - 1);
    }
    fetch_values(i + 2u, next);
    scales = of_next, of_next = after, next = further;
    lds_barrier();                                                  // (the loads stay under way)
  }

  // Merge of the halves.
  float factor[CG], top[CG], total[CG];
  if constexpr (HALVES == 1) {
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) top[cg] = col[cg].ref, total[cg] = groups_sum(col[cg].sum), factor[cg] = 1.0f / col[cg].up;
  } else {
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) {
      const float total = groups_sum(col[cg].sum);
      if (g == 0u) sh.ref[half][(group * CG + cg) * 16u + r] = col[cg].ref, sh.sum[half][(group * CG + cg) * 16u + r] = total;
    }
    lds_barrier();
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) {
      const uint32_t at = (group * CG + cg) * 16u + r;
      const float ref0 = sh.ref[0][at], ref1 = sh.ref[1][at];
      top[cg] = fmaxf(ref0, ref1);
      const float to = from_reference(top[cg]);
      total[cg] = fmaf(__builtin_amdgcn_exp2f(ref1 - to), sh.sum[1][at], __builtin_amdgcn_exp2f(ref0 - to) * sh.sum[0][at]);
      factor[cg] = __builtin_amdgcn_exp2f(col[cg].ref - to) / col[cg].up;
      if (half == 1u) {
#pragma unroll
        for (int x = 0; x < VL; ++x) sh.o[group * CG + cg][x][lane] = o[cg][x] * share_of(total[cg]) * factor[cg];
      }
    }
    lds_barrier();
    if (half == 1u) return;
  }
  const bool whole = w.tiles <= a.part_tiles;                       // no other part has tiles
  const uint64_t slot = ((static_cast<uint64_t>(unit) * b.kv_heads + kv) * a.parts + part) * a.stored;
#pragma unroll
  for (int cg = 0; cg < CG; ++cg) {
    const uint32_t c = (group * CG + cg) * 16u + r;
    if (c >= w.columns) continue;
    const uint32_t at = w.first_col + c;
    float* to = whole ? a.out + (static_cast<uint64_t>(u.seq.first + at / a.group) * a.heads + kv * a.group + at % a.group) * D : a.part_sum + (slot + c) * D;
    const float share = share_of(total[cg]);
    if (!whole && g == 0u) a.part_most[slot + c] = top[cg], a.part_total[slot + c] = total[cg];
#pragma unroll
    for (int x = 0; x < VL; ++x) {
      const uint32_t d = 16u * x + 4u * g;
      float4_t v = o[cg][x] * share * factor[cg];
      if constexpr (HALVES == 2) v += sh.o[group * CG + cg][x][lane];
      if (total[cg] == 0.0f) v = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
      if (d < D) *reinterpret_cast<float4_t*>(to + d) = v;
    }
  }
}

// ---- the parts' merge ----------------------------------------------------------------------------

// A workgroup a column: its parts' results by the weights that they have under the largest of their references, the first parts' loads under
// way at once.
template <int C>
__global__ __launch_bounds__(256) void attention_pages_merge_kernel(PageAttention a) {
  __shared__ float of_wave[2][4], weight[kPagePartsMost];
  __shared__ alignas(16) float4_t piece[256];
  const PageBatch& b = a.batch;
  const uint32_t c = blockIdx.x % a.stored, rest = blockIdx.x / a.stored, kv = rest % b.kv_heads, unit = rest / b.kv_heads, t = threadIdx.x;
  PageUnit u;
  if (!find_unit(b, unit, [&](const PageSequence& q) { return C < 64 ? 1u : (q.rows * a.group + C - 1u) / C; }, &u)) return;
  if constexpr (C >= 64) u.at = (u.seq.rows * a.group + C - 1u) / C - 1u - u.at;      // as the tiles' kernel has it
  const UnitTiles w = C < 64 ? sequence_tiles(a, u.seq) : unit_tiles(a, u, C);
  if (c >= w.columns) return;                                       // workgroup-uniform, as the next ones
  // Places of the parts: the first one's, then from `then` on, `step` apart.
  uint64_t place, then, step;
  uint32_t parts;
  if (a.even != 0u) {
    const EvenTiles tiles = even_tiles(a, u.s);
    const uint32_t share = even_share(a, tiles.all), empty = begin_tiles(a.log_tile), from = tiles.before * b.kv_heads + kv * (w.tiles + empty);
    const uint32_t first = (from + empty) / share;
    parts = (from + empty + w.tiles - 1u) / share - first + 1u;
    place = 2u * static_cast<uint64_t>(first) + (first * share < from ? 1u : 0u), then = 2u * static_cast<uint64_t>(first + 1u), step = 2u;
  } else {
    parts = (w.tiles + a.part_tiles - 1u) / a.part_tiles;
    place = (static_cast<uint64_t>(unit) * b.kv_heads + kv) * a.parts, then = place + 1u, step = 1u;
  }
  if (parts == 1u) return;
  const uint32_t D = b.head_dim, runs = D / 4u;
  auto column = [&](uint32_t p) { return (p == 0u ? place : then + (p - 1u) * step) * a.stored + c; };
  // 256 / runs threads a run of four elements; the first parts' results are asked for before their weights are there
  constexpr uint32_t AHEAD = 8, OWN = kPagePartsMost / 256u;
  float own[OWN], sum[OWN], most = -INFINITY;
#pragma unroll
  for (uint32_t i = 0; i < OWN; ++i) {
    const uint32_t p = t + 256u * i;
    own[i] = p < parts ? a.part_most[column(p)] : -INFINITY, sum[i] = p < parts ? a.part_total[column(p)] : 0.0f;
    most = fmaxf(most, own[i]);
  }
  const uint32_t lanes = 256u / runs, mine = t / runs, d = t % runs * 4u;
  float4_t x = float4_t{0.0f, 0.0f, 0.0f, 0.0f}, early[AHEAD];
  auto load = [&](uint32_t p) { return p < parts && mine < lanes ? *reinterpret_cast<const float4_t*>(a.part_sum + column(p) * D + d) : x; };
#pragma unroll
  for (uint32_t i = 0; i < AHEAD; ++i) early[i] = load(mine + i * lanes);
  most = wave_max(most);
  if ((t & 63u) == 0u) of_wave[0][t >> 6] = most;
  __syncthreads();
  const float top = fmaxf(fmaxf(of_wave[0][0], of_wave[0][1]), fmaxf(of_wave[0][2], of_wave[0][3]));
  float all = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < OWN; ++i) {
    const float f = t + 256u * i < parts ? __builtin_amdgcn_exp2f(own[i] - from_reference(top)) * sum[i] : 0.0f;
    weight[t + 256u * i] = f;
    all += f;
  }
  all = wave_sum(all);
  if ((t & 63u) == 0u) of_wave[1][t >> 6] = all;
  __syncthreads();
  const float total = (of_wave[1][0] + of_wave[1][1]) + (of_wave[1][2] + of_wave[1][3]), share = share_of(total);
#pragma unroll
  for (uint32_t i = 0; i < AHEAD; ++i) {
    if (mine + i * lanes < parts) x += early[i] * (weight[mine + i * lanes] * share);
  }
#pragma unroll 4
  for (uint32_t p = mine + AHEAD * lanes; p < parts; p += lanes) {
    if (mine < lanes) x += *reinterpret_cast<const float4_t*>(a.part_sum + column(p) * D + d) * (weight[p] * share);
  }
  piece[t] = x;
  __syncthreads();
  if (mine != 0u) return;
  for (uint32_t n = 1; n < lanes; ++n) x += piece[n * runs + t];
  const uint32_t pair = w.first_col + c;
  float* out = a.out + (static_cast<uint64_t>(u.seq.first + pair / a.group) * a.heads + kv * a.group + pair % a.group) * D + d;
  *reinterpret_cast<float4_t*>(out) = total == 0.0f ? float4_t{0.0f, 0.0f, 0.0f, 0.0f} : x;
}

}  // namespace

static PagesCall sizes_of(const PageAttentionCall& c) {
  return PagesCall{c.page.rows, c.page.sequences, c.heads / c.page.kv_heads, c.page.kv_heads, c.page.head_dim, c.max_rows, c.max_len, c.window, c.sinks};
}
size_t attention_pages_parts_bytes(const PageAttentionCall& c, const PagesShape& shape) { return pages_bytes(sizes_of(c), shape); }
PagesShape attention_pages_shape(const PageAttentionCall& c, bool in_parts) {
  return pages_rule(sizes_of(c), static_cast<uint64_t>(num_cus()), in_parts ? kAttentionPartsMost : 0);
}

hipError_t launch_attention_pages(bool fp8, const PageAttentionCall& c, const PagesShape& shape, const float* q, const uint8_t* k, const uint8_t* v,
                                  const float* ks, const float* vs, const uint32_t* table, const uint32_t* starts, const uint32_t* lens, float* out,
                                  void* scratch, hipStream_t stream) {
  PageAttention a{};
  a.batch = page_batch(c.page, table, starts, lens);
  a.batch.max_rows = static_cast<uint32_t>(c.max_rows), a.batch.max_len = static_cast<uint32_t>(c.max_len);
  a.q = q, a.k = k, a.v = v, a.k_scale = ks, a.v_scale = vs, a.out = out;
  a.heads = static_cast<uint32_t>(c.heads), a.group = static_cast<uint32_t>(c.heads / c.page.kv_heads);
  // (a window or sinks past every position are all positions)
  a.window = c.window >= c.max_len ? 0u : static_cast<uint32_t>(c.window);
  a.sinks = static_cast<uint32_t>(c.sinks < c.max_len ? c.sinks : c.max_len);
  a.parts = static_cast<uint32_t>(shape.parts), a.part_tiles = static_cast<uint32_t>(shape.part_tiles);
  a.stored = static_cast<uint32_t>(pages_stored(sizes_of(c), shape.columns)), a.log_tile = pages_log_tile(c.page.head_dim, shape.columns);
  const uint64_t groups = pages_units(sizes_of(c), shape.columns) * c.page.kv_heads;
  a.even = static_cast<uint32_t>(shape.even);
  const bool split = shape.parts > 1 || shape.even != 0;
  if (split) {
    const uint64_t columns = (shape.even != 0 ? 2 * shape.even : groups * shape.parts) * a.stored;
    a.part_sum = static_cast<float*>(scratch);
    a.part_most = a.part_sum + columns * c.page.head_dim;
    a.part_total = a.part_most + columns;
  }
  auto tile = [&](auto kind, auto dim) {
    constexpr int CG = decltype(dim)::value == 256 ? 1 : 2;
    const dim3 grid(static_cast<uint32_t>(groups * shape.parts));
    constexpr int TALL = decltype(dim)::value == 64 ? 2 : 1;
    if (shape.columns == 128) {
      hipLaunchKernelGGL((attention_pages_tile_kernel<decltype(kind)::value, decltype(dim)::value, TALL, 1>), grid, dim3(512 / TALL), 0, stream, a);
      return;
    }
    hipLaunchKernelGGL((attention_pages_tile_kernel<decltype(kind)::value, decltype(dim)::value, CG, 2>), grid, dim3(512 / CG), 0, stream, a);
  };
  auto few = [&](auto kind, auto dim, auto cg) {
    constexpr int DP = decltype(dim)::value, CG = decltype(cg)::value;
    const dim3 grid(static_cast<uint32_t>(shape.even != 0 ? shape.even : groups * shape.parts));
    if (shape.waves == 8) hipLaunchKernelGGL((attention_pages_few_kernel<decltype(kind)::value, DP, CG, 8>), grid, dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((attention_pages_few_kernel<decltype(kind)::value, DP, CG, 4>), grid, dim3(256), 0, stream, a);
  };
  auto with_columns = [&](auto kind, auto dim) {
    if (shape.columns >= 64) return tile(kind, dim);
    if constexpr (decltype(dim)::value <= 128) {
      if (shape.columns == 32) return few(kind, dim, std::integral_constant<int, 2>{});
    }
    few(kind, dim, std::integral_constant<int, 1>{});
  };
  auto with_dim = [&](auto kind) {
    const uint64_t D = c.page.head_dim;
    D <= 64 ? with_columns(kind, std::integral_constant<int, 64>{}) : D <= 128 ? with_columns(kind, std::integral_constant<int, 128>{})
                                                                     : with_columns(kind, std::integral_constant<int, 256>{});
  };
  fp8 ? with_dim(std::integral_constant<PageKind, PageKind::Fp8>{}) : with_dim(std::integral_constant<PageKind, PageKind::Q8>{});
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !split) return e;
  auto merge = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(groups * a.stored)), dim3(256), 0, stream, a); };
  shape.columns == 16 ? merge(attention_pages_merge_kernel<16>) : shape.columns == 32 ? merge(attention_pages_merge_kernel<32>)
  : shape.columns == 64 ? merge(attention_pages_merge_kernel<64>) : merge(attention_pages_merge_kernel<128>);
  return hipGetLastError();
}

}  // namespace qmm

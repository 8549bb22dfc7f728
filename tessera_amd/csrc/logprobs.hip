// "token_logprobs": log probabilities of given tokens, the entropy and the largest entries of every row of logits.
//
//   m = max x,  S = sum e^(x - m),  W = sum (x - m) e^(x - m)
//   log p(t) = (x_t - m) - log S,  entropy = log S - W / S        (both terms of the entropy are positive: nothing cancels)
//
// A logit of -infinity has probability 0 and adds nothing to the entropy; NaN or +infinity in a row make its log
// probabilities and entropy NaN, and so does a row of -infinity alone.  The largest entries go by value, then by column;
// -0 and +0 tie, NaN ranks below everything.  A token id of vocab or more has log probability -infinity.

#include "qmm_device.hpp"
#include "launch_rules.hpp"
#include "qmm_kernels.hpp"
#include "tree_args.hpp"

namespace qmm {
namespace {

constexpr float kLog2E = 1.44269504088896340736f;
constexpr uint32_t kEach = kLogprobEach;
constexpr uint32_t kMost = kLogprobTopMost, kListMost = 1024;

struct LogprobArgs {
  const float* logits;               // of the first row
  const uint32_t* tokens;
  float *logprobs, *entropy;
  uint32_t* top_tokens;
  float* top_logprobs;
  uint64_t vocab;
  uint32_t count, top_k;             // tokens a row
  uint32_t width, tiles, shares;     // columns of a tile, a multiple of four; tiles of a row a workgroup; workgroups a row
  float* stats;                      // rows x shares x {m, S, W}
  uint64_t* keys;                    // rows x shares x top_k
};

// Maximum over the wavefront, the same in every lane.  NaN counts for nothing.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ float dpp_max(float v) {
  const int moved = __builtin_amdgcn_update_dpp(bit_cast<int>(v), bit_cast<int>(v), kCtrl, kRowMask, 0xF, false);
  return fmaxf(v, bit_cast<float>(moved));
}
__device__ __forceinline__ float wave_most(float v) {
  v = dpp_max<0xB1, 0xF>(v);   // quad_perm [1,0,3,2]
  v = dpp_max<0x4E, 0xF>(v);   // quad_perm [2,3,0,1]
  v = dpp_max<0x141, 0xF>(v);  // row_half_mirror
  v = dpp_max<0x140, 0xF>(v);  // row_mirror
  v = dpp_max<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v = dpp_max<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return bit_cast<float>(__builtin_amdgcn_readlane(bit_cast<int>(v), 63));
}
__device__ __forceinline__ float wave_total(float v) { return bit_cast<float>(__builtin_amdgcn_readlane(bit_cast<int>(wave_sum_last(v)), 63)); }

// How many of the list's `count` keys lie above `mine`; four of them under way at a time (the list ends on a multiple of four).
__device__ __forceinline__ uint32_t keys_above(const uint64_t* list, uint32_t count, uint64_t mine) {
  uint32_t above = 0u;
  for (uint32_t o = 0; o < count; o += 4u) {
    uint64_t k[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) k[i] = list[o + i];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) above += o + i < count && k[i] > mine ? 1u : 0u;
  }
  return above;
}

// Larger first: by value, then by column.  0 is no key.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t bits = bit_cast<uint32_t>(v == 0.0f ? 0.0f : v);
  return v != v ? 0u : (bits & 0x80000000u) != 0u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float v, uint32_t column) { return static_cast<uint64_t>(order_of(v)) << 32 | ~column; }
__device__ __forceinline__ uint32_t column_of(uint64_t key) { return ~static_cast<uint32_t>(key); }
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return o == 0u ? NAN : bit_cast<float>((o & 0x80000000u) != 0u ? o & 0x7FFFFFFFu : ~o);
}

// A row's sums under a reference m: of two such, the second brought under the larger.
struct Sums {
  float m, s, w;
};
__device__ __forceinline__ Sums moved(Sums a, float m) {      // (no terms: s = w = 0 whatever the reference)
  if (a.m == m || a.m == -INFINITY) return Sums{m, a.s, a.w};
  const float d = a.m - m, e = expf(d);
  return Sums{m, a.s * e, e * fmaf(fmaxf(d, -200.0f), a.s, a.w)};
}

// What a row comes to, from its sums and the sorted keys of its largest entries.
__device__ __forceinline__ float logit_of(const LogprobArgs& a, uint64_t row, uint32_t i) {
  const uint32_t token = a.tokens[row * a.count + i];
  return token < a.vocab ? a.logits[row * a.vocab + token] : -INFINITY;
}
// `own`: the logit of the row's token t, loaded early.
__device__ __forceinline__ void finish(const LogprobArgs& a, uint64_t row, Sums sums, const uint64_t* top, float own, uint32_t t, uint32_t threads) {
  const float log_s = logf(sums.s);
  const bool none = sums.m == -INFINITY;                      // nothing above -infinity (or only NaN)
  for (uint32_t i = t; i < a.count; i += threads) {
    const float v = i == t ? own : logit_of(a, row, i);
    a.logprobs[row * a.count + i] = none ? NAN : (v - sums.m) - log_s;
  }
  if (t == 0u) a.entropy[row] = none ? NAN : log_s - sums.w / sums.s;
  if (t < a.top_k) {
    a.top_tokens[row * a.top_k + t] = column_of(top[t]);
    a.top_logprobs[row * a.top_k + t] = none ? NAN : (value_of(top[t]) - sums.m) - log_s;
  }
}

// One workgroup of THREADS for `tiles` tiles of a row, up to eight entries of a tile a thread; the next tile is under way while this one is
// summed.  Every thread keeps sums of its own under its own largest entry, so that the tiles meet at one barrier each, that of
// the largest entries: from the largest thread maxima of every wavefront of the first tile comes a bound that top_k entries
// reach, what reaches it goes to a list in LDS, and where the list has grown its top_k-th entry becomes the bound.
template <uint32_t THREADS>
__global__ __launch_bounds__(THREADS, THREADS == 1024 ? 8 : 4) void logprob_tiles_kernel(LogprobArgs a) {
  constexpr uint32_t kThreads = THREADS, kWaves = THREADS / 64, kTops = kMost / kWaves;   // thread maxima of a wavefront
  static_assert(kTops * kWaves == 32 && kWaves <= 16);
  __shared__ uint64_t list[kListMost], best[kMost];
  __shared__ float wave_top[32], wave_sums[32], bound_s;
  __shared__ uint32_t count_s[3], total_s[2];
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
  const uint64_t row = blockIdx.x / a.shares;
  const uint32_t share = blockIdx.x % a.shares;
  const float* x = a.logits + row * a.vocab;
  const uint32_t vocab = static_cast<uint32_t>(a.vocab), shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x) >> 2) & 3u;
  const float* from = x - shift;                              // on 16 bytes: entry i of it is column i - shift
  const uint32_t end = vocab + shift, kTile = a.width, all_tiles = (end + kTile - 1u) / kTile;
  const uint32_t first = share * a.tiles, last = first + a.tiles < all_tiles ? first + a.tiles : all_tiles;   // (the last share may be empty)

  // A value the compiler takes for a new one: what is needed now and then is formed there, not held along the tiles.
  auto again = [](uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
  };
  // The next tile's entries, through a view of it whose end the hardware checks.
  float next[kEach];
  auto load = [&](uint32_t tile) {
    const uint64_t at = reinterpret_cast<uint64_t>(from) + static_cast<uint64_t>(tile) * kTile * 4u;
    const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at)), high = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32));
    const uint32_t left = tile < all_tiles ? end - tile * kTile : 0u;
    const auto view = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(static_cast<uint64_t>(high) << 32 | low), 0,
                                                        static_cast<int>(__builtin_amdgcn_readfirstlane((left < kTile ? left : kTile) * 4u)), 0x00020000);
#pragma unroll
    for (uint32_t j = 0; j < kEach / 4; ++j) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(view, (j * 4u * kThreads + 4u * t) * 4u, 0, 0);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) next[4 * j + e] = bit_cast<float>(v[e]);
    }
  };
  load(first);
  Sums run = {-INFINITY, 0.0f, 0.0f};                         // this thread's
  const float own = a.shares == 1u && t < a.count ? logit_of(a, row, t) : 0.0f;
  // The list's entries before this tile; what an entry has to reach, or (`above`) exceed, since what is kept comes before it;
  // whether the last one kept is NaN, so that -infinity counts; the columns so far.
  uint32_t held = 0, columns = 0;
  float bound = -INFINITY;
  bool exceed = false, below = false;
  if (t < 3u) count_s[t] = 0u;
  // The top_k first of the list's `count` entries in order to `best` and back to its start; -> how many there are.
  auto rank = [&](uint32_t count) {
    for (uint32_t i = t; i < count; i += kThreads) {
      const uint64_t mine = list[i];
      const uint32_t above = keys_above(list, count, mine);
      if (above < a.top_k) best[above] = mine;
    }
    __syncthreads();
    const uint32_t kept = count < a.top_k ? count : a.top_k;
    if (t < kept) list[t] = best[t];
    if (kept == a.top_k) {
      const uint64_t least = best[kept - 1u];
      below = (least >> 32) == 0u, exceed = !below;
      bound = below ? -INFINITY : value_of(least);
    }
    __syncthreads();
    return kept;
  };
  for (uint32_t tile = first; tile < last; ++tile) {
    const uint32_t thread = again(t);
    auto column = [&](uint32_t j) {                           // outside the tile or the row: vocab or more
      const uint32_t in = (j / 4u) * (4u * kThreads) + 4u * thread;
      return in < kTile ? tile * kTile + in + j % 4u - shift : ~0u;
    };
    float v[kEach], most = -INFINITY;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) v[j] = next[j];
    if (tile == 0u || tile + 1u == all_tiles || kTile != kThreads * kEach) {
#pragma unroll
      for (uint32_t j = 0; j < kEach; ++j) v[j] = column(j) < vocab ? v[j] : -INFINITY;
    }
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) most = fmaxf(most, v[j]);
    if (tile + 1u < last) load(tile + 1u);

    const float m = fmaxf(run.m, most), ref = m == -INFINITY ? 0.0f : m;
    const float d0 = run.m - ref, e0 = run.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(d0 * kLog2E);
    run.w = e0 * fmaf(fmaxf(d0, -200.0f), run.s, run.w), run.s *= e0, run.m = m;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
      const float d = v[j] - ref, e = __builtin_amdgcn_exp2f(d * kLog2E);
      run.s += e;
      run.w = fmaf(fmaxf(d, -200.0f), e, run.w);
    }
    if (a.top_k == 0u) continue;

    if (tile == first) {
      float rest = most;
#pragma unroll
      for (uint32_t i = 0; i < kTops; ++i) {
        const float one = wave_most(rest);
        if (lane == 0u) wave_top[i * kWaves + wave] = one;
        rest = rest == one ? -INFINITY : rest;
      }
      lds_barrier();
      if (wave == 0u) {
        const uint32_t own_lane = again(lane);
        const float mine = wave_top[own_lane & 31u];
        uint32_t above = 0u;
#pragma unroll
        for (uint32_t i = 0; i < 32u; ++i) {
          const float o = wave_top[i];
          above += (o > mine || (o == mine && i < own_lane)) ? 1u : 0u;
        }
        if (own_lane < 32u && above == a.top_k - 1u) bound_s = mine;
      }
      lds_barrier();
      bound = bound_s;
    }
    const uint32_t counter = tile % 3u;
    if (most >= bound) {
#pragma unroll
      for (uint32_t j = 0; j < kEach; ++j) {
        if (v[j] >= bound && !(exceed && v[j] == bound) && (v[j] != -INFINITY || below) && column(j) < vocab) {
          const uint32_t at = held + atomicAdd(&count_s[counter], 1u);
          if (at < kListMost) list[at] = key_of(v[j], column(j));
        }
      }
    }
    if (t == 0u) count_s[(tile + 1u) % 3u] = 0u;              // (read last two barriers ago)
    lds_barrier();
    uint32_t count = held + count_s[counter];
    const uint32_t here = tile + 1u < all_tiles ? (tile == 0u ? kTile - shift : kTile) : end - tile * kTile - (tile == 0u ? shift : 0u);
    columns += here;
    const uint32_t need = a.top_k < columns ? a.top_k : columns;
    const bool exactly = count > kListMost || count < need;
    if (exactly) {
      // Too many alike, or too few that are numbers: exactly the `want` first entries of the tile, those above a value `least`
      // and the first columns of it (behind -infinity, of NaN).
      const uint32_t want = a.top_k < here ? a.top_k : here;
      uint32_t round = 0u;
      auto total = [&](auto counts) {                             // of the tile's entries; one barrier
        uint32_t mine = 0u;
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) mine += column(j) < vocab && counts(j) ? 1u : 0u;
        const float sum = wave_total(static_cast<float>(mine));
        if (lane == 0u) atomicAdd(&total_s[round & 1u], static_cast<uint32_t>(sum));
        lds_barrier();
        const uint32_t all = total_s[round & 1u];
        lds_barrier();
        if (t == 0u) total_s[round & 1u] = 0u;
        ++round;
        return all;
      };
      if (t < 2u) total_s[t] = 0u;
      __syncthreads();
      float least = count < need ? -INFINITY : bound;
      uint32_t more = total([&](uint32_t j) { return v[j] > least; });
      if (more >= want) {                                           // bit by bit, the largest that `want` entries reach
        uint32_t order = 0u;
        for (uint32_t bit = 0x80000000u; bit != 0u; bit >>= 1) {
          if (total([&](uint32_t j) { return order_of(v[j]) >= (order | bit); }) >= want) order |= bit;
        }
        least = value_of(static_cast<uint64_t>(order) << 32);
        more = total([&](uint32_t j) { return v[j] > least; });
      }
      if (t == 0u) total_s[0] = total_s[1] = 0u;
      __syncthreads();
#pragma unroll
      for (uint32_t j = 0; j < kEach; ++j) {
        if (v[j] > least && column(j) < vocab) list[held + atomicAdd(&total_s[0], 1u)] = key_of(v[j], column(j));
      }
      if (wave == 0u) {                                             // the rest: along the columns
        const uint32_t begin = tile == 0u ? 0u : tile * kTile - shift, stop = begin + here;
        uint32_t at = more;
        for (int nan = 0; nan < 2 && at < want; ++nan) {
          for (uint32_t c = begin; c < stop && at < want; c += 64u) {
            const float value = c + lane < stop ? x[c + lane] : 0.0f;
            const bool hit = c + lane < stop && (nan == 0 ? value == least : value != value);
            const uint64_t hits = __ballot(hit);
            const uint32_t place = at + __popcll(hits & ((uint64_t{1} << lane) - 1u));
            if (hit && place < want) list[held + place] = key_of(value, c + lane);
            at += __popcll(hits);
          }
        }
      }
      __syncthreads();
      count = held + want;
    }
    held = exactly || count > 2u * a.top_k + 32u || tile + 1u == last ? rank(count) : count;
  }
  const float m = wave_most(run.m);
  run = moved(run, m);
  const float s = wave_sum_last(run.s), w = wave_sum_last(run.w);
  if (lane == 63u) wave_top[wave] = m, wave_sums[2u * wave] = s, wave_sums[2u * wave + 1u] = w;
  __syncthreads();
  const uint32_t i = lane & 15u;                              // a lane a wavefront's
  Sums all = i < kWaves ? Sums{wave_top[i], wave_sums[2u * i], wave_sums[2u * i + 1u]} : Sums{-INFINITY, 0.0f, 0.0f};
  all = moved(all, wave_most(all.m));
  all.s = row16_sum(all.s), all.w = row16_sum(all.w);
  if (a.shares == 1u) {
    finish(a, row, all, best, own, t, kThreads);
    return;
  }
  const size_t at = blockIdx.x;
  if (t == 0u) a.stats[3u * at] = all.m, a.stats[3u * at + 1u] = all.s, a.stats[3u * at + 2u] = all.w;
  if (t < a.top_k) a.keys[at * a.top_k + t] = t < held ? best[t] : 0ull;
}

// The shares of a row (at most kSharesMost): their sums under the largest reference; of their sorted keys those that reach
// a bound that top_k of them do, each counting those above it.
constexpr uint32_t kSharesMost = kLogprobShares, kMergeThreads = 256;
__global__ __launch_bounds__(kMergeThreads) void logprob_merge_kernel(LogprobArgs a) {
  constexpr uint32_t kKeys = kSharesMost * kMost / kMergeThreads;   // a thread's
  __shared__ uint64_t list[kSharesMost * kMost], best[kMost], level[kSharesMost], bound_s;
  __shared__ uint32_t count_s;
  const uint32_t t = threadIdx.x, lane = t & 63u;
  const uint64_t row = blockIdx.x;
  const float* stats = a.stats + row * a.shares * 3u;
  const uint64_t* keys = a.keys + row * a.shares * a.top_k;
  const uint32_t all_keys = a.shares * a.top_k;
  // Of the shares' `deep`-th keys the `nth` largest has deep * nth >= top_k keys at or above it.
  const uint32_t deep = (a.top_k + a.shares - 1u) / a.shares, nth = a.top_k == 0u ? 0u : (a.top_k + deep - 1u) / deep;
  const uint64_t mine_level = a.top_k != 0u && t < a.shares ? keys[t * a.top_k + deep - 1u] : 0ull;
  uint64_t held[kKeys];
#pragma unroll
  for (uint32_t i = 0; i < kKeys; ++i) held[i] = t + i * kMergeThreads < all_keys ? keys[t + i * kMergeThreads] : 0ull;
  const Sums mine = lane < a.shares ? Sums{stats[3u * lane], stats[3u * lane + 1u], stats[3u * lane + 2u]} : Sums{-INFINITY, 0.0f, 0.0f};
  const float own = t < a.count ? logit_of(a, row, t) : 0.0f;
  if (a.top_k != 0u) {
    if (t < kSharesMost) level[t] = mine_level;
    if (t == 0u) count_s = 0u, bound_s = 0ull;
    __syncthreads();
    if (t < a.shares) {                                         // (equal ones are 0, which as a bound keeps every key)
      if (keys_above(level, a.shares, mine_level) == nth - 1u) bound_s = mine_level;
    }
    __syncthreads();
    const uint64_t bound = bound_s;
#pragma unroll
    for (uint32_t i = 0; i < kKeys; ++i) {
      if (held[i] >= bound && held[i] != 0ull) list[atomicAdd(&count_s, 1u)] = held[i];
    }
    __syncthreads();
    const uint32_t count = count_s;
    for (uint32_t i = t; i < count; i += kMergeThreads) {
      const uint64_t key = list[i];
      const uint32_t above = keys_above(list, count, key);
      if (above < a.top_k) best[above] = key;
    }
    __syncthreads();
  }
  Sums all = moved(mine, wave_most(mine.m));
  all.s = wave_total(all.s), all.w = wave_total(all.w);
  finish(a, row, all, best, own, t, kMergeThreads);
}

LogprobPlan plan_of(uint64_t rows, uint64_t vocab, uint32_t top_k, size_t most) {
  return logprob_plan(rows, vocab, top_k, static_cast<uint64_t>(num_cus()), most);
}

}  // namespace

size_t token_logprobs_scratch_bytes(uint64_t rows, uint64_t vocab, uint32_t top_k, size_t most) {
  return logprob_bytes(plan_of(rows, vocab, top_k, most), rows, top_k);
}

hipError_t launch_token_logprobs(const float* logits, const uint32_t* tokens, float* logprobs, float* entropy, uint32_t* top_tokens,
                                 float* top_logprobs, uint64_t rows, uint64_t vocab, uint32_t count, uint32_t top_k, uint64_t row_base,
                                 void* scratch, size_t most, hipStream_t stream) {
  const LogprobPlan plan = plan_of(rows, vocab, top_k, scratch != nullptr ? most : 0);
  for (uint64_t r = 0; r < rows; r += kLogprobRows) {
    const uint32_t here = static_cast<uint32_t>(rows - r < kLogprobRows ? rows - r : kLogprobRows);
    LogprobArgs a{logits + (row_base + r) * vocab, tokens + r * count, logprobs + r * count, entropy + r,
                  top_k == 0 ? nullptr : top_tokens + r * top_k, top_k == 0 ? nullptr : top_logprobs + r * top_k, vocab, count, top_k,
                  plan.width, plan.tiles, plan.shares, nullptr, nullptr};
    if (plan.shares > 1) {
      a.keys = static_cast<uint64_t*>(scratch);
      a.stats = reinterpret_cast<float*>(a.keys + size_t{here} * plan.shares * top_k);
    }
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(here * plan.shares), dim3(plan.threads), 0, stream, a); };
    if (plan.threads == 256) go(logprob_tiles_kernel<256>);
    else if (plan.threads == 512) go(logprob_tiles_kernel<512>);
    else go(logprob_tiles_kernel<1024>);
    if (plan.shares > 1) hipLaunchKernelGGL(logprob_merge_kernel, dim3(here), dim3(kMergeThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace qmm

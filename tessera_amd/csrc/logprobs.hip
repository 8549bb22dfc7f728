// "token_logprobs": log probabilities of given tokens, the entropy and the largest entries of every row of logits.
//
//   m = max x,  S = sum e^(x - m),  W = sum (x - m) e^(x - m)
//   log p(t) = (x_t - m) - log S,  entropy = log S - W / S        (both terms of the entropy are positive: nothing cancels)
//
// A logit of -infinity has probability 0 and adds nothing to the entropy; NaN or +infinity in a row make its log
// probabilities and entropy NaN, and so does a row of -infinity alone.  The largest entries go by value, then by column;
// -0 and +0 tie, NaN ranks below everything.  A token id of vocab or more has log probability -infinity.

#include "qmm_device.hpp"
#include "qmm_kernels.hpp"
#include "tree_args.hpp"

namespace qmm {
namespace {

constexpr float kLog2E = 1.44269504088896340736f;
constexpr uint32_t kThreads = 1024, kWaves = kThreads / 64, kEach = 8, kTile = kThreads * kEach;
constexpr uint32_t kMost = kLogprobTopMost, kListMost = 1024;

struct LogprobArgs {
  const float* logits;               // of the first row
  const uint32_t* tokens;
  float *logprobs, *entropy;
  uint32_t* top_tokens;
  float* top_logprobs;
  uint64_t vocab;
  uint32_t count, top_k, tiles, shares;      // tokens a row; tiles of a row a workgroup; workgroups a row
  float* stats;                      // rows x shares x {m, S, W}
  uint64_t* keys;                    // rows x shares x top_k
};

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
__device__ __forceinline__ void finish(const LogprobArgs& a, uint64_t row, Sums sums, const uint64_t* top, uint32_t t, uint32_t threads) {
  const float* x = a.logits + row * a.vocab;
  const float log_s = logf(sums.s);
  const bool none = sums.m == -INFINITY;                      // nothing above -infinity (or only NaN)
  for (uint32_t i = t; i < a.count; i += threads) {
    const uint32_t token = a.tokens[row * a.count + i];
    const float v = token < a.vocab ? x[token] : -INFINITY;
    a.logprobs[row * a.count + i] = none ? NAN : (v - sums.m) - log_s;
  }
  if (t == 0u) a.entropy[row] = none ? NAN : log_s - sums.w / sums.s;
  if (t < a.top_k) {
    a.top_tokens[row * a.top_k + t] = column_of(top[t]);
    a.top_logprobs[row * a.top_k + t] = none ? NAN : (value_of(top[t]) - sums.m) - log_s;
  }
}

// One workgroup for `tiles` tiles of a row, eight entries of a tile a thread.  The row is read once: the next tile is
// under way while this one is summed.  Its largest entries: from the two largest thread maxima of every wavefront comes a
// bound that top_k entries of the tile reach, so that only some tens of them go to a list, where each counts those above it.
__global__ __launch_bounds__(kThreads) void logprob_tiles_kernel(LogprobArgs a) {
  __shared__ uint64_t list[kListMost + kMost], best[kMost];
  __shared__ float wave_top[2 * kWaves], wave_sums[2 * kWaves], bound_s;
  __shared__ uint32_t count_s, total_s[2];
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
  const uint64_t row = blockIdx.x / a.shares;
  const uint32_t share = blockIdx.x % a.shares;
  const float* x = a.logits + row * a.vocab;
  const uint32_t vocab = static_cast<uint32_t>(a.vocab), shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x) >> 2) & 3u;
  const float* from = x - shift;                              // on 16 bytes: entry i of it is column i - shift
  const uint32_t end = vocab + shift, all_tiles = (end + kTile - 1u) / kTile;
  const uint32_t first = share * a.tiles, last = first + a.tiles < all_tiles ? first + a.tiles : all_tiles;   // (the last share may be empty)

  float next[kEach];
  auto load = [&](uint32_t tile) {
#pragma unroll
    for (uint32_t j = 0; j < kEach / 4; ++j) {
      const uint32_t i = tile * kTile + j * (4u * kThreads) + 4u * t;
      if (i >= shift && i + 4u <= end) {
        const float4 v = *reinterpret_cast<const float4*>(from + i);
        next[4 * j] = v.x, next[4 * j + 1] = v.y, next[4 * j + 2] = v.z, next[4 * j + 3] = v.w;
      } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) next[4 * j + e] = i + e >= shift && i + e < end ? from[i + e] : -INFINITY;
      }
    }
  };
  load(first);
  Sums run = {-INFINITY, 0.0f, 0.0f};                         // this thread's, m the same in all
  uint32_t kept = 0;                                          // keys in `best`
  if (t == 0u) count_s = 0u;
  for (uint32_t tile = first; tile < last; ++tile) {
    float v[kEach], most = -INFINITY;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) v[j] = next[j], most = fmaxf(most, v[j]);
    if (tile + 1u < last) load(tile + 1u);
    auto column = [&](uint32_t j) { return tile * kTile + (j / 4u) * (4u * kThreads) + 4u * t + j % 4u - shift; };   // outside: vocab or more

    const float one = wave_max(most), two = wave_max(most == one ? -INFINITY : most);
    if (lane == 0u) wave_top[2u * wave] = one, wave_top[2u * wave + 1u] = two;
    __syncthreads();
    const float tops = wave_top[lane & 31u], m = fmaxf(run.m, wave_max(tops));
    if (a.top_k != 0u && wave == 0u) {
      uint32_t above = 0u;
      for (uint32_t i = 0; i < 2u * kWaves; ++i) {
        const float o = wave_top[i];
        above += (o > tops || (o == tops && i < lane)) ? 1u : 0u;
      }
      if (lane < 32u && above == a.top_k - 1u) bound_s = tops;
    }
    run = moved(run, m);
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
      const float d = v[j] - ref, e = __builtin_amdgcn_exp2f(d * kLog2E);
      run.s += e;
      run.w = fmaf(fmaxf(d, -200.0f), e, run.w);
    }
    if (a.top_k == 0u) {
      __syncthreads();
      continue;
    }
    __syncthreads();
    // Entries that reach the bound and, where there are top_k before this tile, the least of those.
    float bound = bound_s;
    if (kept == a.top_k) bound = fmaxf(bound, value_of(best[kept - 1u]));
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
      if (v[j] >= bound && (bound != -INFINITY || v[j] != -INFINITY)) {
        const uint32_t at = atomicAdd(&count_s, 1u);
        if (at < kListMost) list[at] = key_of(v[j], column(j));
      }
    }
    __syncthreads();
    uint32_t count = count_s;
    const uint32_t here = tile + 1u < all_tiles ? (tile == 0u ? kTile - shift : kTile) : end - tile * kTile - (tile == 0u ? shift : 0u);
    const uint32_t want = a.top_k < here ? a.top_k : here;
    if (count > kListMost || (kept < a.top_k && count < want)) {
      // Too many alike, or too few that are numbers: exactly the `want` first entries of the tile.  Bit by bit, the largest
      // `least` that `want` entries reach, then among those at `least` the columns up to `until`.
      auto total = [&](auto counts) {
        uint32_t mine = 0u;
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) mine += column(j) < vocab && counts(j) ? 1u : 0u;
        const uint32_t sum = static_cast<uint32_t>(wave_sum(static_cast<float>(mine)));
        __syncthreads();
        if (t == 0u) total_s[0] = 0u;
        __syncthreads();
        if (lane == 0u) atomicAdd(&total_s[0], sum);
        __syncthreads();
        return total_s[0];
      };
      uint32_t least = 0u, until = 0u;
      for (uint32_t bit = 0x80000000u; bit != 0u; bit >>= 1) {
        if (total([&](uint32_t j) { return order_of(v[j]) >= (least | bit); }) >= want) least |= bit;
      }
      const uint32_t rest = want - total([&](uint32_t j) { return order_of(v[j]) > least; });
      for (uint32_t bit = 0x80000000u; bit != 0u; bit >>= 1) {         // `until`: fewer than `rest` such columns lie below it
        if (total([&](uint32_t j) { return order_of(v[j]) == least && column(j) < (until | bit); }) < rest) until |= bit;
      }
      __syncthreads();
      if (t == 0u) count_s = 0u;
      __syncthreads();
#pragma unroll
      for (uint32_t j = 0; j < kEach; ++j) {
        const uint32_t o = order_of(v[j]);
        if (column(j) < vocab && (o > least || (o == least && column(j) <= until))) list[atomicAdd(&count_s, 1u)] = key_of(v[j], column(j));
      }
      __syncthreads();
      count = count_s;
    }
    if (t < kept) list[count + t] = best[t];
    __syncthreads();
    count += kept;
    kept = count < a.top_k ? count : a.top_k;
    for (uint32_t i = t; i < count; i += kThreads) {
      const uint64_t mine = list[i];
      uint32_t above = 0u;
      for (uint32_t o = 0; o < count; ++o) above += list[o] > mine ? 1u : 0u;
      if (above < a.top_k) best[above] = mine;
    }
    if (t == 0u) count_s = 0u;
    __syncthreads();
  }
  const float s = wave_sum_last(run.s), w = wave_sum_last(run.w);
  if (lane == 63u) wave_sums[2u * wave] = s, wave_sums[2u * wave + 1u] = w;
  __syncthreads();
  Sums all = {run.m, 0.0f, 0.0f};
#pragma unroll
  for (uint32_t i = 0; i < kWaves; ++i) all.s += wave_sums[2u * i], all.w += wave_sums[2u * i + 1u];
  if (a.shares == 1u) {
    finish(a, row, all, best, t, kThreads);
    return;
  }
  const size_t at = blockIdx.x;
  if (t == 0u) a.stats[3u * at] = all.m, a.stats[3u * at + 1u] = all.s, a.stats[3u * at + 2u] = all.w;
  if (t < a.top_k) a.keys[at * a.top_k + t] = t < kept ? best[t] : 0ull;
}

// The shares of a row (at most kSharesMost): their sums under the largest reference; of their sorted keys those that reach
// a bound that top_k of them do, each counting those above it.
constexpr uint32_t kSharesMost = 64, kMergeThreads = 256;
__global__ __launch_bounds__(kMergeThreads) void logprob_merge_kernel(LogprobArgs a) {
  __shared__ uint64_t list[kSharesMost * kMost], best[kMost];
  __shared__ uint64_t level[kSharesMost], bound_s;
  __shared__ uint32_t count_s;
  const uint32_t t = threadIdx.x, lane = t & 63u;
  const uint64_t row = blockIdx.x;
  const float* stats = a.stats + row * a.shares * 3u;
  const uint64_t* keys = a.keys + row * a.shares * a.top_k;
  const Sums mine = lane < a.shares ? Sums{stats[3u * lane], stats[3u * lane + 1u], stats[3u * lane + 2u]} : Sums{-INFINITY, 0.0f, 0.0f};
  const float m = wave_max(mine.m);
  Sums all = moved(mine, m);
  all.s = wave_sum(all.s), all.w = wave_sum(all.w);
  if (a.top_k != 0u) {
    // Of the shares' `deep`-th keys the `nth` largest has deep * nth >= top_k keys at or above it.
    const uint32_t deep = (a.top_k + a.shares - 1u) / a.shares, nth = (a.top_k + deep - 1u) / deep;
    if (t < a.shares) level[t] = keys[t * a.top_k + deep - 1u];
    if (t == 0u) count_s = 0u, bound_s = 0ull;
    __syncthreads();
    if (t < a.shares) {
      const uint64_t own = level[t];
      uint32_t above = 0u;
      for (uint32_t i = 0; i < a.shares; ++i) above += (level[i] > own || (level[i] == own && i < t)) ? 1u : 0u;
      if (above == nth - 1u) bound_s = own;
    }
    __syncthreads();
    const uint64_t bound = bound_s;
    for (uint32_t i = t; i < a.shares * a.top_k; i += kMergeThreads) {
      const uint64_t key = keys[i];
      if (key >= bound && key != 0ull) list[atomicAdd(&count_s, 1u)] = key;
    }
    __syncthreads();
    const uint32_t count = count_s;
    for (uint32_t i = t; i < count; i += kMergeThreads) {
      const uint64_t own = list[i];
      uint32_t above = 0u;
      for (uint32_t o = 0; o < count; ++o) above += list[o] > own ? 1u : 0u;
      if (above < a.top_k) best[above] = own;
    }
    __syncthreads();
  }
  finish(a, row, all, best, t, kMergeThreads);
}

uint32_t tiles_of(uint64_t vocab) { return static_cast<uint32_t>((vocab + 3u + kTile - 1u) / kTile); }   // (3: the alignment)

struct Plan {
  uint32_t tiles, shares;
};
Plan plan_of(uint64_t rows, uint64_t vocab, bool shared) {
  const uint32_t all = tiles_of(vocab);
  if (!shared) return Plan{all, 1};
  const uint32_t tiles = (all + kSharesMost - 1) / kSharesMost;
  return Plan{tiles, (all + tiles - 1) / tiles};
}
constexpr uint64_t kRowsMost = uint64_t{1} << 20;                 // rows of a launch: 64 workgroups of 1024 threads each stay a grid
size_t bytes_a_row(const Plan& plan, uint32_t top_k) { return plan.shares < 2 ? 0 : size_t{plan.shares} * (12u + 8u * top_k); }

}  // namespace

// What the shares of all rows take, or of as many rows as fit `most` bytes.
size_t token_logprobs_scratch_bytes(uint64_t rows, uint64_t vocab, uint32_t top_k, size_t most) {
  const size_t each = bytes_a_row(plan_of(rows, vocab, true), top_k);
  if (each == 0) return 0;
  const uint64_t at_once = most / each < rows ? most / each : rows;
  return static_cast<size_t>(at_once) * each + 16;
}

hipError_t launch_token_logprobs(const float* logits, const uint32_t* tokens, float* logprobs, float* entropy, uint32_t* top_tokens,
                                 float* top_logprobs, uint64_t rows, uint64_t vocab, uint32_t count, uint32_t top_k, uint64_t row_base,
                                 void* scratch, size_t scratch_bytes, hipStream_t stream) {
  const Plan plan = plan_of(rows, vocab, scratch != nullptr);
  const size_t each = bytes_a_row(plan, top_k);
  uint64_t at_once = each == 0 ? rows : (scratch_bytes - 16) / each;
  if (at_once > kRowsMost / 64) at_once = kRowsMost / 64;
  for (uint64_t r = 0; r < rows; r += at_once) {
    const uint32_t here = static_cast<uint32_t>(rows - r < at_once ? rows - r : at_once);
    LogprobArgs a{logits + (row_base + r) * vocab, tokens + r * count, logprobs + r * count, entropy + r,
                  top_k == 0 ? nullptr : top_tokens + r * top_k, top_k == 0 ? nullptr : top_logprobs + r * top_k, vocab, count, top_k,
                  plan.tiles, plan.shares, nullptr, nullptr};
    if (plan.shares > 1) {
      a.keys = static_cast<uint64_t*>(scratch);
      a.stats = reinterpret_cast<float*>(a.keys + size_t{here} * plan.shares * top_k);
    }
    hipLaunchKernelGGL(logprob_tiles_kernel, dim3(here * plan.shares), dim3(kThreads), 0, stream, a);
    if (plan.shares > 1) hipLaunchKernelGGL(logprob_merge_kernel, dim3(here), dim3(kMergeThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace qmm

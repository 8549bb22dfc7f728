// "draft_verify": how many of each sequence's drafted tokens stand, and the token that follows them.
//
// Row i of a sequence holds the target's logits for the token after Tokens[i]; Tokens[i + 1] was drafted for it, but for the last row.
// With p = softmax(logits / temperature) and q the draft's likewise (none: the draft is one token, q = 1), the draft's token x
// stands where u q(x) < p(x), u the row's first random number.  At the first that does not the next token is drawn from max(p - q, 0)
// (none: p without x), behind the last one from p: the first whose running sum exceeds the row's second random number times the
// whole.  Temperature 0: a token stands where it is the likeliest, the lowest of equals.
//
// Which token it is hangs on sums next to a border, so everything from the logits on is fp64: exponentials to 2^-42, sums over chunks of
// 4096 columns and then over chunks, in an order that the vocabulary alone decides.  Two forms of launch, with the same bits:
// a workgroup for a chunk, in three launches (statistics of all rows; the remaining sums of the row that is drawn from; the draw),
// or, without scratch, a workgroup for a sequence.  Bound by reading the logits.

#include "page_args.hpp"
#include "qmm_device.hpp"
#include "qmm_kernels.hpp"

namespace qmm {
namespace {

constexpr uint32_t kChunk = 4096, kThreads = 256, kEach = kChunk / kThreads, kChunksMost = static_cast<uint32_t>(kDraftVocabMost) / kChunk;
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
  uint32_t rows, vocab, sequences, chunks;
  double scale, draft_scale;         // 1 / (temperature ln 2); 0: the likeliest token
  ChunkStats* stats;                 // (plane, row, chunk)
  double* rest;                      // (sequence, chunk)
};

// 2^y for y <= 0, below 2^-1022 as 0: 2^n 2^f, |f| <= 1/2, by the power series of exp(f ln 2) to its eleventh term (the next is
// 2^-46 of the sum).
__device__ __forceinline__ double exp2_of(double y) {
  const double n = __builtin_rint(y), x = (y - n) * 0.69314718055994530942;
  double s = 1.0 / 39916800.0;
  s = fma(s, x, 1.0 / 3628800.0);
  s = fma(s, x, 1.0 / 362880.0);
  s = fma(s, x, 1.0 / 40320.0);
  s = fma(s, x, 1.0 / 5040.0);
  s = fma(s, x, 1.0 / 720.0);
  s = fma(s, x, 1.0 / 120.0);
  s = fma(s, x, 1.0 / 24.0);
  s = fma(s, x, 1.0 / 6.0);
  s = fma(s, x, 0.5);
  s = fma(s, x, 1.0);
  s = fma(s, x, 1.0);
  if (!(y >= -1022.0)) return 0.0;
  return s * bit_cast<double>(static_cast<uint64_t>(static_cast<int64_t>(static_cast<int32_t>(n)) + 1023) << 52);
}
__device__ __forceinline__ double power(float logit, float most, double scale) {
  return exp2_of((static_cast<double>(logit) - static_cast<double>(most)) * scale);
}

struct BlockShared {
  double sum[kThreads / 64];
  float most[kThreads / 64];
  uint32_t arg[kThreads / 64];
};
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}
// The sum over the workgroup, in every thread.
__device__ __forceinline__ double block_sum(double v, BlockShared& sh) {
  v = wave_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0u) sh.sum[threadIdx.x >> 6] = v;
  __syncthreads();
  double all = sh.sum[0];
#pragma unroll
  for (uint32_t i = 1; i < kThreads / 64u; ++i) all += sh.sum[i];
  return all;
}
// The larger logit, of equals the one further in front.
__device__ __forceinline__ void take_larger(float& most, uint32_t& arg, float other, uint32_t at) {
  if (other > most || (other == most && at < arg)) most = other, arg = at;
}

// By a workgroup; thread 0 returns it.  `scale` 0: no sum.
__device__ __forceinline__ ChunkStats chunk_stats(const float* row, uint32_t vocab, uint32_t chunk, double scale, BlockShared& sh) {
  const uint32_t t = threadIdx.x, first = chunk * kChunk + t;
  float x[kEach], most = -INFINITY;
  uint32_t arg = kNoToken;
  bool bad = false;
#pragma unroll
  for (uint32_t j = 0; j < kEach; ++j) {
    const uint32_t e = first + j * kThreads;
    x[j] = e < vocab ? row[e] : -INFINITY;
    bad = bad || !(x[j] < INFINITY);
    if (x[j] > most) most = x[j], arg = e;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float other = __shfl_xor(most, off, kWave);
    const uint32_t at = __shfl_xor(arg, off, kWave);
    take_larger(most, arg, other, at);
  }
  bad = __any(bad);
  __syncthreads();
  if ((t & 63u) == 0u) sh.most[t >> 6] = bad ? bit_cast<float>(0x7FC00000u) : most, sh.arg[t >> 6] = arg;
  __syncthreads();
  most = -INFINITY, arg = kNoToken, bad = false;
#pragma unroll
  for (uint32_t i = 0; i < kThreads / 64u; ++i) {
    bad = bad || sh.most[i] != sh.most[i];
    take_larger(most, arg, sh.most[i], sh.arg[i]);
  }
  double sum = 0.0;
  if (scale != 0.0 && !bad && most > -INFINITY) {                   // workgroup-uniform
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) sum += power(x[j], most, scale);
    sum = block_sum(sum, sh);
  }
  return ChunkStats{sum, bad ? bit_cast<float>(0x7FC00000u) : most, arg};
}

// A row's statistics from its chunks', by a wavefront, in every lane.  `bad`: NaN or +infinity, or -infinity alone.
struct RowStats {
  double sum;
  float most;
  uint32_t arg;
  bool bad;
};
__device__ __forceinline__ RowStats row_stats(const ChunkStats* chunks, uint32_t count, double scale) {
  const uint32_t lane = threadIdx.x & 63u;
  RowStats r{0.0, -INFINITY, kNoToken, false};
  for (uint32_t c = lane; c < count; c += 64u) {
    const float m = chunks[c].most;
    r.bad = r.bad || m != m;
    take_larger(r.most, r.arg, m, chunks[c].arg);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float other = __shfl_xor(r.most, off, kWave);
    const uint32_t at = __shfl_xor(r.arg, off, kWave);
    take_larger(r.most, r.arg, other, at);
  }
  r.bad = __any(r.bad) || r.most == -INFINITY;
  if (r.bad || scale == 0.0) return r;
  for (uint32_t c = lane; c < count; c += 64u) {
    if (chunks[c].most > -INFINITY) r.sum += chunks[c].sum * power(chunks[c].most, r.most, scale);
  }
  r.sum = wave_sum64(r.sum);
  return r;
}

// ---- where a sequence's draft ends ---------------------------------------------------------------

struct Verdict {
  RowStats target, draft;
  uint32_t row, at, token;           // of the call; of the sequence; the refused token
  bool ends, refused;                // refused: the draft's token does not stand there
};
__device__ __forceinline__ bool sequence_rows(const DraftArgs& a, uint32_t s, uint32_t* first, uint32_t* rows) {
  const uint32_t begin = a.starts[s], end = a.starts[s + 1u];
  *first = begin, *rows = end - begin;
  return begin < end && end <= a.rows;
}
// Row `at` of a sequence, by a wavefront, from its chunks' statistics; `draft` those of the draft's row,
// unless `of_draft` is `known`.
__device__ __forceinline__ Verdict judge(const DraftArgs& a, const ChunkStats* target, const ChunkStats* draft, uint32_t first, uint32_t rows, uint32_t at,
                                         bool known = false, RowStats of_draft = RowStats{}) {
  Verdict v{};
  v.row = first + at, v.at = at;
  v.target = row_stats(target, a.chunks, a.scale);
  const bool last = at + 1u == rows;
  if (!last) v.token = a.tokens[v.row + 1u];
  if (a.scale == 0.0) {
    v.refused = !last && v.target.arg != v.token;
    v.ends = v.target.bad || last || v.refused;
    return v;
  }
  bool bad = v.target.bad;
  if (!last && a.draft != nullptr) {
    v.draft = known ? of_draft : row_stats(draft, a.chunks, a.draft_scale);
    bad = bad || v.draft.bad;
  }
  v.target.bad = bad;
  if (bad || last) {
    v.ends = true;
    return v;
  }
  double p = 0.0, q = 1.0;
  if (v.token < a.vocab) {
    const uint64_t place = static_cast<uint64_t>(v.row) * a.vocab + v.token;
    p = power(a.logits[place], v.target.most, a.scale) / v.target.sum;
    if (a.draft != nullptr) q = power(a.draft[place], v.draft.most, a.draft_scale) / v.draft.sum;
  }
  v.refused = !(static_cast<double>(a.random[2u * static_cast<uint64_t>(v.row)]) * q < p);
  v.ends = v.refused;
  return v;
}

// What is left of column e of the row that is drawn from, relative to its largest probability (so that equal logits have sums
// without rounding, and two rows alike have nothing left).
__device__ __forceinline__ double rest_of(const DraftArgs& a, const Verdict& v, double share, uint32_t e) {
  const uint64_t place = static_cast<uint64_t>(v.row) * a.vocab + e;
  const double p = power(a.logits[place], v.target.most, a.scale);
  if (!v.refused) return p;
  if (a.draft == nullptr) return e == v.token ? 0.0 : p;
  const double less = p - power(a.draft[place], v.draft.most, a.draft_scale) * share;
  return less > 0.0 ? less : 0.0;
}
__device__ __forceinline__ double share_of(const DraftArgs& a, const Verdict& v) { return a.draft != nullptr && v.refused ? v.target.sum / v.draft.sum : 0.0; }
__device__ __forceinline__ double chunk_rest(const DraftArgs& a, const Verdict& v, uint32_t chunk, BlockShared& sh) {
  const double share = share_of(a, v);
  double sum = 0.0;
#pragma unroll 4
  for (uint32_t j = 0; j < kEach; ++j) {
    const uint32_t e = chunk * kChunk + j * kThreads + threadIdx.x;
    if (e < a.vocab) sum += rest_of(a, v, share, e);
  }
  return block_sum(sum, sh);
}

struct DrawShared {
  double sums[kChunksMost];
  double rest[kChunk];
  double before;
  uint32_t chunk, token;
};
// The draw: `rest` holds the chunks' sums; `stats` the target row's chunks.
__device__ __forceinline__ uint32_t draw_token(const DraftArgs& a, Verdict v, const double* rest, const ChunkStats* stats, DrawShared& d, BlockShared& sh) {
  const uint32_t t = threadIdx.x;
  for (uint32_t c = t; c < a.chunks; c += kThreads) d.sums[c] = rest[c];
  __syncthreads();
  auto total = [&] {
    double all = 0.0;
    for (uint32_t c = 0; c < a.chunks; ++c) all += d.sums[c];
    return all;
  };
  double whole = total();
  if (!(whole > 0.0)) {                                             // the draft accounts for all of p: p itself
    __syncthreads();
    v.refused = false;
    for (uint32_t c = t; c < a.chunks; c += kThreads) {
      d.sums[c] = stats[c].most > -INFINITY ? stats[c].sum * power(stats[c].most, v.target.most, a.scale) : 0.0;
    }
    __syncthreads();
    whole = total();
  }
  const float u = a.random[2u * static_cast<uint64_t>(v.row) + 1u];
  const double goal = (u >= 0.0f ? static_cast<double>(u) : 0.0) * whole;
  if (t == 0u) {
    double sum = 0.0, last_before = 0.0;
    uint32_t chunk = kNoToken, last = 0u;
    for (uint32_t c = 0; c < a.chunks && chunk == kNoToken; ++c) {
      const double now = sum + d.sums[c];
      if (d.sums[c] > 0.0) last = c, last_before = sum;
      if (now > goal) chunk = c, last_before = sum;
      sum = now;
    }
    d.chunk = chunk == kNoToken ? last : chunk, d.before = last_before, d.token = kNoToken;
  }
  __syncthreads();
  // The chunk's running sums: sixteen columns a thread in a row.
  const uint32_t base = d.chunk * kChunk;
  const double left = goal - d.before, share = share_of(a, v);
  for (uint32_t j = 0; j < kEach; ++j) {
    const uint32_t e = base + j * kThreads + t;
    d.rest[j * kThreads + t] = e < a.vocab ? rest_of(a, v, share, e) : 0.0;
  }
  __syncthreads();
  double own = 0.0;
  uint32_t last = kNoToken;
  for (uint32_t j = 0; j < kEach; ++j) {
    const double r = d.rest[t * kEach + j];
    own += r;
    if (r > 0.0) last = t * kEach + j;
  }
  double sum = own;                                                 // inclusive, over threads
  const uint32_t lane = t & 63u;
#pragma unroll
  for (uint32_t off = 1u; off < 64u; off <<= 1) {
    const double before = __shfl_up(sum, off, kWave);
    if (lane >= off) sum += before;
  }
  __syncthreads();
  if (lane == 63u) sh.sum[t >> 6] = sum;
  __syncthreads();
  for (uint32_t i = 0; i < (t >> 6); ++i) sum += sh.sum[i];
  double run = sum - own;
  uint32_t found = kNoToken;
  for (uint32_t j = 0; j < kEach && found == kNoToken; ++j) {
    const double r = d.rest[t * kEach + j];
    run += r;
    if (r > 0.0 && run > left) found = t * kEach + j;
  }
  // The first that exceeds it; where rounding leaves none, the last that is left at all.
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint32_t other = __shfl_xor(found, off, kWave), behind = __shfl_xor(last, off, kWave);
    found = other < found ? other : found;
    if (last == kNoToken || (behind != kNoToken && behind > last)) last = behind;
  }
  __syncthreads();
  if (lane == 0u) sh.arg[t >> 6] = found, sh.most[t >> 6] = bit_cast<float>(last);
  __syncthreads();
  found = kNoToken, last = kNoToken;
#pragma unroll
  for (uint32_t i = 0; i < kThreads / 64u; ++i) {
    const uint32_t behind = bit_cast<uint32_t>(sh.most[i]);
    found = sh.arg[i] < found ? sh.arg[i] : found;
    if (behind != kNoToken) last = behind;
  }
  return base + (found != kNoToken ? found : last);
}

// ---- a workgroup a chunk -------------------------------------------------------------------------

__global__ __launch_bounds__(kThreads) void draft_stats_kernel(DraftArgs a) {
  __shared__ BlockShared sh;
  const uint32_t chunk = blockIdx.x % a.chunks, rest = blockIdx.x / a.chunks, row = rest % a.rows, plane = rest / a.rows;
  const float* from = (plane == 0u ? a.logits : a.draft) + static_cast<uint64_t>(row) * a.vocab;
  const ChunkStats s = chunk_stats(from, a.vocab, chunk, plane == 0u ? a.scale : a.draft_scale, sh);
  if (threadIdx.x == 0u) a.stats[blockIdx.x] = s;
}

struct VerdictShared {
  Verdict of[kThreads / 64];
};
// The row at which a sequence's draft ends, by a workgroup, a wavefront a row, from all rows' statistics.
__device__ __forceinline__ Verdict find_end(const DraftArgs& a, uint32_t first, uint32_t rows, VerdictShared& sh) {
  const uint32_t wave = threadIdx.x >> 6;
  for (uint32_t base = 0;; base += kThreads / 64u) {
    Verdict v{};
    if (base + wave < rows) {
      const uint64_t at = static_cast<uint64_t>(first + base + wave) * a.chunks;
      v = judge(a, a.stats + at, a.stats + static_cast<uint64_t>(a.rows) * a.chunks + at, first, rows, base + wave);
    }
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) sh.of[wave] = v;
    __syncthreads();
    for (uint32_t i = 0; i < kThreads / 64u; ++i) {
      if (sh.of[i].ends) return sh.of[i];                           // (the last row does)
    }
  }
}
__device__ __forceinline__ void put(const DraftArgs& a, uint32_t s, const Verdict& v, uint32_t token) {
  a.accepted[s] = v.at, a.next[s] = v.target.bad ? kNoToken : token;
}

__global__ __launch_bounds__(kThreads) void draft_rest_kernel(DraftArgs a) {
  __shared__ BlockShared sh;
  __shared__ VerdictShared verdicts;
  const uint32_t each = a.scale == 0.0 ? 1u : a.chunks, s = blockIdx.x / each, chunk = blockIdx.x % each;
  uint32_t first, rows;
  if (!sequence_rows(a, s, &first, &rows)) return;
  const Verdict v = find_end(a, first, rows, verdicts);
  if (a.scale == 0.0 || v.target.bad) {
    if (chunk == 0u && threadIdx.x == 0u) put(a, s, v, v.target.arg);
    return;
  }
  const double sum = chunk_rest(a, v, chunk, sh);
  if (threadIdx.x == 0u) a.rest[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kThreads) void draft_draw_kernel(DraftArgs a) {
  __shared__ BlockShared sh;
  __shared__ VerdictShared verdicts;
  __shared__ DrawShared draw;
  const uint32_t s = blockIdx.x;
  uint32_t first, rows;
  if (!sequence_rows(a, s, &first, &rows)) return;
  const Verdict v = find_end(a, first, rows, verdicts);
  if (v.target.bad) return;
  const uint32_t token = draw_token(a, v, a.rest + static_cast<uint64_t>(s) * a.chunks, a.stats + static_cast<uint64_t>(v.row) * a.chunks, draw, sh);
  if (threadIdx.x == 0u) put(a, s, v, token);
}

// ---- a workgroup a sequence ----------------------------------------------------------------------

struct AloneShared {
  ChunkStats stats[kChunksMost];
  Verdict verdict;
};
__global__ __launch_bounds__(kThreads) void draft_alone_kernel(DraftArgs a) {
  __shared__ BlockShared sh;
  __shared__ AloneShared alone;
  __shared__ DrawShared draw;
  const uint32_t s = blockIdx.x, t = threadIdx.x;
  uint32_t first, rows;
  if (!sequence_rows(a, s, &first, &rows)) return;
  auto gather = [&](const float* plane, uint32_t row, double scale) {
    __syncthreads();
    for (uint32_t c = 0; c < a.chunks; ++c) {
      const ChunkStats x = chunk_stats(plane + static_cast<uint64_t>(row) * a.vocab, a.vocab, c, scale, sh);
      if (t == 0u) alone.stats[c] = x;
    }
    __syncthreads();
  };
  Verdict v{};
  for (uint32_t at = 0; at < rows && !v.ends; ++at) {
    // the draft's first, of which only the row's statistics are kept
    RowStats draft{};
    if (a.draft != nullptr && a.scale != 0.0 && at + 1u < rows) {
      gather(a.draft, first + at, a.draft_scale);
      draft = row_stats(alone.stats, a.chunks, a.draft_scale);
    }
    gather(a.logits, first + at, a.scale);
    v = judge(a, alone.stats, nullptr, first, rows, at, true, draft);
  }
  if (a.scale == 0.0 || v.target.bad) {
    if (t == 0u) put(a, s, v, v.target.arg);
    return;
  }
  double* rest = draw.rest;                                         // (the draw copies the sums out of it before it uses it)
  for (uint32_t c = 0; c < a.chunks; ++c) {
    const double sum = chunk_rest(a, v, c, sh);
    if (t == 0u) rest[c] = sum;
  }
  __syncthreads();
  const uint32_t token = draw_token(a, v, rest, alone.stats, draw, sh);
  if (t == 0u) put(a, s, v, token);
}

uint32_t chunks_of(const DraftCall& c) { return static_cast<uint32_t>((c.vocab + kChunk - 1) / kChunk); }
bool reads_draft(const DraftCall& c) { return c.draft && c.temperature > 0.0f; }

}  // namespace

size_t draft_verify_scratch_bytes(const DraftCall& c) {
  return static_cast<size_t>((c.rows * (reads_draft(c) ? 2 : 1) * sizeof(ChunkStats) + c.sequences * sizeof(double)) * chunks_of(c));
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
  const uint32_t planes = a.draft != nullptr ? 2u : 1u;
  a.stats = static_cast<ChunkStats*>(scratch);
  a.rest = reinterpret_cast<double*>(a.stats + static_cast<size_t>(planes) * a.rows * a.chunks);
  hipLaunchKernelGGL(draft_stats_kernel, dim3(planes * a.rows * a.chunks), dim3(kThreads), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(draft_rest_kernel, dim3(a.scale == 0.0 ? a.sequences : a.sequences * a.chunks), dim3(kThreads), 0, stream, a);
  if ((e = hipGetLastError()) != hipSuccess || a.scale == 0.0) return e;
  hipLaunchKernelGGL(draft_draw_kernel, dim3(a.sequences), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace qmm

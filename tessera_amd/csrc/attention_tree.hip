// "attention_tree" and its forms over quantized caches: the rows of a drafted tree against the keys before it and the
// tree's own, as each row's bits say (attention_kernels.hpp: TREE).

#include "attention_kernels.hpp"

namespace qmm {
namespace {

// ---- a workgroup shares its keys among 64 (row, head) pairs ---------------------------------------
//
// The pairs of a key head, `group` to a row, are the columns of the contractions S^T = K Q^T and O^T = V^T P^T on
// v_mfma_f32_16x16x32_f16.  Eight wavefronts, two a SIMD: four groups of 16 columns times two halves of a tile of 64 keys.  A tile is
// made fp16 (exactly: fp16 numbers or codes) once, on its way into LDS, keys row by row, values transposed; all columns read the
// same operands.
//
// What is fp32 enters as two fp16 terms under a power of two that brings the largest of its head, key or row near 2^14: hi =
// RN16(x) and lo = RN16(2^11 (x - hi)), 2^-23 of x down to 2^-28 of the largest and 2^-50 of that below.  Of a query, and of an fp32
// key under a power of two of its own, the products with a second term have sums of their own, scaled once a tile.  Values and
// weights have one sum of all, as registers for two are not to be had and the vector unit takes 0.8 us a tile to add them up: an
// fp32 value's second term is multiplied by 2^-11 of the weight, and a weight's is RN16(x - hi), which leaves 2^-23 of a weight (times its
// value's power of two or scale) down to 2^-11 of its row's largest and 2^-34 of that below.  Of fp32 keys and values the product of
// two second terms, 2^-22 of the whole at most, is left out.
//
// Bound by the matrix instructions and what does not go on beside them, as all wavefronts are at the same place.  So nothing
// is done to the running sums but by the matrix instructions: weights are taken relative to a reference that follows the
// largest score only where it would leave 2^kSlack of it, and just then the sums are scaled; and the next tile goes to LDS a
// piece at a time between them.  64 rows of 24 heads of 256 over 4 on 32832 fp16 keys in ten parts: 111 us (702 with a
// workgroup a row and key head); a tile of 64 keys 1.47 us, 1.79 with the next one's way to LDS in one go, 2.57 with every
// tile's sums added to the running ones by the vector unit.  Two terms of 64 fp32 keys of 256 fill the LDS: their tiles go
// there between two barriers, 5 us each (of 128 3, of 64 2.1), the next one's loads under way meanwhile.  64 rows of 24
// heads of 256 over 4 on 8192 fp32 keys: 87 us (220 by the kernel below).
constexpr float kSlack = 4.0f;                    // in powers of two

template <int DP>
struct TreeTile {
  static constexpr uint32_t kKeyBytes = 64 * DP * 2, kStage = 2 * kKeyBytes;
  alignas(16) uint8_t stage[2][kStage];           // 64 keys, then two times 32 keys' values transposed
  float scales[2][2][64];                         // keys', values'
  float ref[2][64], sum[2][64], up[2][64];        // the halves'
  uint32_t start[64];                             // of the keys that a column sees, where that is not the first
  uint32_t low[4], high[4], special;
};

// BYTES (1 to 32) at `offset` of a buffer whose end the hardware checks: what lies past it reads as 0.
template <int BYTES>
__device__ __forceinline__ void load_run(__amdgpu_buffer_rsrc_t from, uint32_t offset, uint32_t (&r)[(BYTES + 3) / 4]) {
  if constexpr (BYTES == 1) {
    r[0] = __builtin_amdgcn_raw_buffer_load_b8(from, offset, 0, 0);
  } else if constexpr (BYTES == 2) {
    r[0] = __builtin_amdgcn_raw_buffer_load_b16(from, offset, 0, 0);
  } else if constexpr (BYTES == 4) {
    r[0] = __builtin_amdgcn_raw_buffer_load_b32(from, offset, 0, 0);
  } else if constexpr (BYTES == 8) {
    const auto v = __builtin_amdgcn_raw_buffer_load_b64(from, offset, 0, 0);
    r[0] = v[0], r[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(from, offset + 16u * i, 0, 0);
      r[4 * i] = v[0], r[4 * i + 1] = v[1], r[4 * i + 2] = v[2], r[4 * i + 3] = v[3];
    }
  }
}

// A key of an fp32 cache is taken under a power of two of its own, as its codes' scale is of a quantized one: `up` brings its largest
// element to 2^14 .. 2^15.  The largest of a key's elements in the LANES lanes that hold them (with 32: lanes apart by 16 hold
// two keys where `apart`).
template <int LANES>
__device__ __forceinline__ float key_most(float v, bool apart) {
  auto step = [&](auto ctrl) {
    constexpr int kCtrl = decltype(ctrl)::value;
    v = fmaxf(v, bit_cast<float>(__builtin_amdgcn_update_dpp(0, bit_cast<int>(v), kCtrl, 0xF, 0xF, true)));
  };
  step(std::integral_constant<int, 0xB1>{});     // quad_perm [1,0,3,2]
  step(std::integral_constant<int, 0x4E>{});     // quad_perm [2,3,0,1]
  step(std::integral_constant<int, 0x141>{});    // row_half_mirror
  if constexpr (LANES >= 16) step(std::integral_constant<int, 0x140>{});   // row_mirror
  if constexpr (LANES == 32) {
    const uint32_t x = bit_cast<uint32_t>(v);
    if (apart) {
      const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
      v = fmaxf(bit_cast<float>(b[0]), bit_cast<float>(b[1]));
    } else {
      const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
      v = fmaxf(bit_cast<float>(b[0]), bit_cast<float>(b[1]));
    }
  }
  return v;
}
// The two terms of x under `up`, the second one times 2^11.
struct Terms {
  _Float16 hi, lo;
};
__device__ __forceinline__ Terms terms_of(uint32_t x, float up) {
  const float v = bit_cast<float>(x) * up;
  const _Float16 hi = static_cast<_Float16>(v);
  return Terms{hi, static_cast<_Float16>((v - static_cast<float>(hi)) * 0x1p11f)};
}

// A value the compiler takes for a new one: what is needed only now and then or after the walk over the keys is formed from
// the thread's number or the head size again, not held, where the registers are just enough.
__device__ __forceinline__ uint32_t again(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

// (row, head) pair `pair` over the keys of start .. last that its row sees, in fp32 by THREADS threads (256 at least): where
// infinities or NaN keep the matrix instructions from it.  Keys 64 at a time, a wavefront's lanes along head_dim for a score, a
// thread or two an element of the sum.
struct PairShared {
  float score[64], weight[64], sum[512];
};
template <KvKind KV, uint32_t THREADS>
__device__ __forceinline__ void attend_pair(const AttentionArgs& a, TreePair which, uint32_t kv, uint64_t start, uint64_t last, uint32_t s_part,
                                            PairShared& sh) {
  constexpr uint32_t kHalves = THREADS / 256u, kWaves = THREADS / 64u;
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6, D = a.head_dim, e = t & 255u, half = t >> 8;
  const uint64_t pair = which.at;
  const uint32_t* bits = a.mask + static_cast<uint64_t>(which.row) * a.words;
  {
    uint64_t row_start, row_last;
    key_range<true>(a, which.row, row_start, row_last);
    start = row_start > start ? row_start : start;
  }
  const float scale = 1.0f / sqrtf(static_cast<float>(again(D)));
  float run_max = -INFINITY, run_sum = 0.0f, acc = 0.0f;
  for (uint64_t j0 = start; j0 <= last; j0 += 64u) {
    const uint32_t count = last - j0 < 63u ? static_cast<uint32_t>(last - j0) + 1u : 64u;
    const uint32_t low = tree_keys(a, bits, j0), high = count > 32u ? tree_keys(a, bits, j0 + 32u) : 0u;
    auto sees = [&](uint32_t k) { return k < count && ((k < 32u ? low >> k : high >> (k - 32u)) & 1u) != 0u; };
    for (uint32_t k = wave; k < 64u; k += kWaves) {
      float dot = 0.0f;
      if (sees(k)) {
        for (uint32_t d = lane; d < D; d += 64u) {
          dot = fmaf(a.q[pair * D + d], cache_element<KV>(a.k, a.k_scale, j0 + k, ((j0 + k) * a.kv_heads + kv) * D + d), dot);
        }
      }
      dot = wave_sum(dot);
      if (lane == 0u) sh.score[k] = sees(k) ? dot * scale : -INFINITY;
    }
    __syncthreads();
    const float s = sh.score[lane], most = fmaxf(run_max, wave_max(s)), to = reference_score(most);
    const float w = sees(lane) ? expf(s - to) : 0.0f, corr = expf(run_max - to);      // (the same in every wavefront)
    if (wave == 0u) sh.weight[lane] = w;
    run_sum = fmaf(corr, run_sum, wave_sum(w));
    run_max = most;
    __syncthreads();
    float x = 0.0f;
    for (uint32_t k = half; k < count && e < D && half < kHalves; k += kHalves) {
      if (sees(k)) x = fmaf(sh.weight[k], cache_element<KV>(a.v, a.v_scale, j0 + k, ((j0 + k) * a.kv_heads + kv) * D + e), x);
    }
    acc = fmaf(corr, acc, x);
  }
  if constexpr (kHalves == 2) {
    if (half < 2u) sh.sum[t] = acc;
  }
  __syncthreads();
  if (t < D) {
    const float x = kHalves == 2 ? acc + sh.sum[t + 256u] : acc;
    if (a.part.split != 0) a.part.pacc[(pair * a.part.split + s_part) * D + t] = x;
    else a.out[pair * D + t] = run_sum == 0.0f ? 0.0f : x / run_sum;
  }
  if (t == 0u && a.part.split != 0) a.part.pmax[pair * a.part.split + s_part] = run_max, a.part.psum[pair * a.part.split + s_part] = run_sum;
  __syncthreads();
}

template <KvKind KV, int DP>
__global__ __launch_bounds__(512, 2) void attention_tree_kernel(AttentionArgs a) {
  constexpr bool F32 = KV == KvKind::F32, QUANT = kv_quantized(KV), SCALED = QUANT || F32;
  constexpr bool LATE = F32 && DP == 256;                          // the next values' way begins behind the products: no registers before
  constexpr int BITS = kv_bits(KV);
  constexpr int STEPS = DP / 32;                                   // matrix instructions of a score, in two sums
  constexpr int VE = DP / 16, RE = DP / 32;                        // elements of a row of the result, of a value run
  constexpr int CHUNKS = DP / 8;                                   // runs of eight elements of a key
  constexpr int KLOADS = 64 * CHUNKS / 512;
  constexpr int EARLY = LATE ? KLOADS / 2 : KLOADS;
  constexpr int KDW = 8 * BITS / 32, VDW = (RE * BITS + 31) / 32;
  using Shared = TreeTile<DP>;
  __shared__ Shared sh;

  const uint32_t t = threadIdx.x, lane = t & 63u, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t r = lane & 15u, g = lane >> 4, col_group = wave & 3u, half = wave >> 2;
  const uint32_t D = a.head_dim, group = a.heads / a.kv_heads;
  const uint32_t split = a.part.split == 0 ? 1u : static_cast<uint32_t>(a.part.split);
  const uint32_t kv = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads, s_part = unit % split;
  const uint32_t columns = static_cast<uint32_t>(a.rows * group);
  const uint32_t c0 = unit / split * 64u;
  const uint32_t c_end = c0 + 64u < columns ? c0 + 64u : columns;
  // A lane's column of the workgroup's, past the last one the last.
  struct Column {
    uint32_t row, head;
  };
  auto column = [&](uint32_t thread) {
    const uint32_t at = c0 + col_group * 16u + (thread & 15u), col = at < c_end ? at : c_end - 1u;
    const uint32_t per = again(group);
    return Column{col / per, kv * group + col % per};
  };

  // The keys that the columns' rows see begin in no order: the earliest start and the latest.  Past the prefix a tile goes by
  // the rows' bits.
  const uint32_t prefix = static_cast<uint32_t>(a.n - a.tree);
  uint32_t wg_start, latest_start, wg_last = static_cast<uint32_t>(a.n - 1);
  {
    uint64_t first_key, last_key;
    key_range<true>(a, column(t).row, first_key, last_key);
    uint32_t low = static_cast<uint32_t>(first_key), high = low;
    if (a.window != 0 || prefix == 0u) {
      if (g == 0u && half == 0u) sh.start[col_group * 16u + r] = low;
#pragma unroll
      for (uint32_t off = 8u; off > 0u; off >>= 1) {
        const uint32_t l = __shfl_xor(low, off, kWave), h = __shfl_xor(high, off, kWave);
        low = l < low ? l : low, high = h > high ? h : high;
      }
      if (lane == 0u && half == 0u) sh.low[col_group] = low, sh.high[col_group] = high;
      __syncthreads();
      low = ~0u, high = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) low = sh.low[i] < low ? sh.low[i] : low, high = sh.high[i] > high ? sh.high[i] : high;
    }
    wg_start = __builtin_amdgcn_readfirstlane(low < wg_last ? low : wg_last);
    latest_start = __builtin_amdgcn_readfirstlane(high);
  }
  if (split > 1u) {                                                // whole tiles of the workgroup's keys a part
    const uint32_t chunk = ((wg_last - wg_start + split) / split + 63u) / 64u * 64u;
    if (static_cast<uint64_t>(s_part) * chunk > wg_last - wg_start) {
      for (uint32_t c = c0; c < c_end; ++c) empty_part<512, true>(a, c / group, kv * group + c % group, 1, s_part);
      return;
    }
    wg_start += s_part * chunk;
    if (wg_last - wg_start >= chunk) wg_last = wg_start + chunk - 1u;
  }

  const uint32_t stride = a.kv_heads * D * BITS / 8;               // (times 64 below 2^31: the caller)
  // This thread's share of a tile's loads: chunk k_chunk of keys k_key + (512 / CHUNKS) i, elements RE v_run.. of keys
  // 4 v_four.. (lanes l and l + 16 write the halves of a chunk).  Elements past head_dim are read as the row's first: the
  // queries are 0 there, of the result they are not stored.  Keys past the last read as 0; no column sees them.
  const uint32_t k_key = t / CHUNKS, k_chunk = t % CHUNKS;
  const uint32_t v_run = (t & 15u) * 2u + (t >> 5 & 1u), v_four = half * 8u + (t >> 4 & 1u) * 4u + col_group;
  const uint32_t head_at = kv * D * BITS / 8;
  const uint32_t k_off = k_key * stride + head_at + (k_chunk * 8u < D ? k_chunk * BITS : 0u);
  const uint32_t v_off = v_four * 4u * stride + head_at + (v_run * RE < D ? v_run * RE * BITS / 8 : 0u);
  auto tile_of = [&](const void* base, uint32_t j0, uint32_t row_bytes) {
    const uint32_t rows = j0 > wg_last ? 0u : wg_last - j0 < 64u ? wg_last - j0 + 1u : 64u;
    const uint64_t at = reinterpret_cast<uint64_t>(base) + static_cast<uint64_t>(j0) * row_bytes;
    const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at)), high = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(static_cast<uint64_t>(high) << 32 | low), 0,
                                             static_cast<int>(__builtin_amdgcn_readfirstlane(rows * row_bytes)), 0x00020000);
  };
  uint32_t kr[KLOADS][KDW], vr[4][VDW], sr = 0u;
  auto fetch_keys = [&](uint32_t j0, int i) { load_run<BITS>(tile_of(a.k, j0, stride), k_off + i * (512u / CHUNKS) * stride, kr[i]); };
  auto fetch_values = [&](uint32_t j0) {
    const auto tile = tile_of(a.v, j0, stride);
#pragma unroll
    for (int e = 0; e < 4; ++e) load_run<RE * BITS / 8>(tile, v_off + e * stride, vr[e]);
  };
  auto fetch_scales = [&](uint32_t j0) {
    if constexpr (QUANT) {
      if (wave < 2u) sr = __builtin_amdgcn_raw_buffer_load_b32(tile_of(wave == 0u ? a.k_scale : a.v_scale, j0, 4u), lane * 4u, 0, 0);
    }
  };
  // A key's row in LDS: its chunks of sixteen bytes at c ^ swizzle, so that neighbouring keys' chunks fall on
  // different banks; 256 bytes hold 16 chunks.
  auto key_swizzle = [](uint32_t key) { return CHUNKS >= 16 ? key & 15u : (key >> 1) & 7u; };
  // Block j of 32 keys' values holds elements 16 j .. 16 j + 15, a row each of four chunks of sixteen bytes, chunk c of keys 4c..
  // and 16 + 4c..; chunk c of row r is at place (4 r + c) ^ (r & 12) ^ j of the block, which puts the sixteen blocks or
  // rows that sixteen lanes write at once on sixteen bank groups.
  auto stash_keys = [&](uint32_t b, int i) {
    const uint32_t key = k_key + i * (512u / CHUNKS);
    *reinterpret_cast<half8_t*>(sh.stage[b] + key * (DP * 2u) + ((k_chunk ^ key_swizzle(key)) * 16u)) = key_operand<KV>(kr[i]);
  };
  const uint32_t v_row = v_run * RE & 15u, v_block = v_run * RE / 16u;
  const uint32_t v_to = Shared::kKeyBytes + half * (DP * 64u) + v_block * 1024u +
                        (((v_row * 4u + (v_four & 3u)) ^ (v_row & 12u) ^ v_block) * 16u) + (v_four >> 2 & 1u) * 8u;
  auto stash_values = [&](uint32_t b, int j) {
    const uint32_t to = v_to ^ static_cast<uint32_t>(((4 * j) ^ (j & 12)) * 16);   // (the bits of v_row + j and of v_row are apart)
    *reinterpret_cast<uint2*>(sh.stage[b] + to) = uint2{value_pair<KV>(vr[0], vr[1], j), value_pair<KV>(vr[2], vr[3], j)};
  };
  auto stash_scales = [&](uint32_t b) {
    if constexpr (QUANT) {
      if (wave < 2u) {
        const float x = bit_cast<float>(sr);
        sh.scales[b][wave][lane] = x;
        if (wave == 0u && !(fabsf(x) < INFINITY)) sh.special = 1u;   // such a key's score says nothing of its weight here
      }
    }
  };

  // An fp32 tile's terms: the first in stage 0, the second in stage 1.
  auto stash_f32 = [&] {
    if constexpr (F32) {
      const uint32_t now = again(t), to_key = now / CHUNKS, to_chunk = now % CHUNKS;
#pragma unroll
      for (int i = 0; i < KLOADS; ++i) {
        const uint32_t key = to_key + i * (512u / CHUNKS);
        float most = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(bit_cast<float>(kr[i][e])));
        most = key_most<CHUNKS>(most, false);
        const float up = most == 0.0f ? 1.0f : power_of_two_to(most, 14);
        if (!(most < INFINITY)) sh.special = 1u;
        if (to_chunk == 0u) sh.scales[0][0][key] = 1.0f / up;
        half8_t hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const Terms x = terms_of(kr[i][e], up);
          hi[e] = x.hi, lo[e] = x.lo;
        }
        const uint32_t to = key * (DP * 2u) + ((to_chunk ^ key_swizzle(key)) * 16u);
        *reinterpret_cast<half8_t*>(sh.stage[0] + to) = hi;
        *reinterpret_cast<half8_t*>(sh.stage[1] + to) = lo;
      }
      const uint32_t to_run = (now & 15u) * 2u + (now >> 5 & 1u), to_four = half * 8u + (now >> 4 & 1u) * 4u + col_group;
      const uint32_t to_row = to_run * RE & 15u, to_block = to_run * RE / 16u;
      const uint32_t v_base = Shared::kKeyBytes + half * (DP * 64u) + to_block * 1024u +
                              (((to_row * 4u + (to_four & 3u)) ^ (to_row & 12u) ^ to_block) * 16u) + (to_four >> 2 & 1u) * 8u;
      float ups[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float most = 0.0f;
#pragma unroll
        for (int e = 0; e < RE; ++e) most = fmaxf(most, fabsf(bit_cast<float>(vr[k][e])));
        most = key_most<32>(most, true);
        ups[k] = most == 0.0f ? 1.0f : power_of_two_to(most, 14);
        if (to_run == 0u) sh.scales[0][1][to_four * 4u + k] = 1.0f / ups[k];
      }
#pragma unroll
      for (int j = 0; j < RE; ++j) {
        __attribute__((ext_vector_type(4))) _Float16 hi, lo;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const Terms x = terms_of(vr[k][j], ups[k]);
          hi[k] = x.hi, lo[k] = x.lo;
        }
        const uint32_t to = v_base ^ static_cast<uint32_t>(((4 * j) ^ (j & 12)) * 16);
        *reinterpret_cast<uint2*>(sh.stage[0] + to) = bit_cast<uint2>(hi);
        *reinterpret_cast<uint2*>(sh.stage[1] + to) = bit_cast<uint2>(lo);
      }
    }
  };

  if (t == 0) sh.special = 0u;
  fetch_scales(wg_start);
#pragma unroll
  for (int i = 0; i < KLOADS; ++i) fetch_keys(wg_start, i);
  fetch_values(wg_start);

  // The queries' terms: each half makes those of half the steps and takes the others from LDS.
  half8_t q_hi[STEPS], q_lo[STEPS];
  float score_scale = kLog2E / sqrtf(static_cast<float>(D));
  {
    constexpr int OWN = STEPS / 2;
    const Column mine = column(t);
    const float* qp = a.q + (static_cast<uint64_t>(mine.row) * a.heads + mine.head) * D;
    float raw[OWN][8], most = 0.0f;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const uint32_t d = (half * OWN + i) * 32u + g * 8u;
      const float4 x = d < D ? *reinterpret_cast<const float4*>(qp + d) : float4{0.0f, 0.0f, 0.0f, 0.0f};
      const float4 y = d < D ? *reinterpret_cast<const float4*>(qp + d + 4) : float4{0.0f, 0.0f, 0.0f, 0.0f};
      raw[i][0] = x.x, raw[i][1] = x.y, raw[i][2] = x.z, raw[i][3] = x.w;
      raw[i][4] = y.x, raw[i][5] = y.y, raw[i][6] = y.z, raw[i][7] = y.w;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(raw[i][e]));
    }
    most = groups_max(most);
    if (g == 0u) sh.ref[half][col_group * 16u + r] = most;
    __syncthreads();                                               // (and `special` is set up)
    most = fmaxf(sh.ref[0][col_group * 16u + r], sh.ref[1][col_group * 16u + r]);
    const float up = most == 0.0f ? 1.0f : power_of_two_to(most, 14);
    score_scale /= up;
    half8_t* swap = reinterpret_cast<half8_t*>(sh.stage[1]) + col_group * (STEPS * 128) + lane;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      half8_t hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = raw[i][kq_dim<KV>(e)] * up;
        hi[e] = static_cast<_Float16>(v);
        lo[e] = static_cast<_Float16>((v - static_cast<float>(hi[e])) * 0x1p11f);
      }
      swap[(half * OWN + i) * 128u] = hi, swap[(half * OWN + i) * 128u + 64u] = lo;
    }
    if constexpr (!F32) {
      stash_scales(0);
      fetch_scales(wg_start + 64u);
#pragma unroll
      for (int i = 0; i < KLOADS; ++i) stash_keys(0, i), fetch_keys(wg_start + 64u, i);
#pragma unroll
      for (int j = 0; j < RE; ++j) stash_values(0, j);
      fetch_values(wg_start + 64u);
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < STEPS; ++i) q_hi[i] = swap[i * 128], q_lo[i] = swap[i * 128 + 64];
    lds_barrier();                                                 // the next tile goes where they were
  }
  float4_t o[VE];
#pragma unroll
  for (int j = 0; j < VE; ++j) o[j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float ref = -INFINITY, origin = 0.0f, run_sum = 0.0f;            // origin: ref, 0 while there is none
  float lane_most = 0.0f, value_up = SCALED ? power_of_two_to(0.0f, 14) : 0x1p10f;
  const uint32_t key_row = (half * 32u + r) * (DP * 2u), key_swz = key_swizzle(r);
  const uint32_t value_row = Shared::kKeyBytes + half * (DP * 64u) + (((r * 4u + g) ^ (r & 12u)) * 16u);
  // While a tile is multiplied the next one goes to LDS, a piece at a time between the matrix instructions, and the registers
  // of every piece take the tile after that one's.
  for (uint32_t j0 = wg_start, b = 0; j0 <= wg_last; j0 += 64u, b ^= 1u) {
    const uint8_t* stage = sh.stage[F32 ? 0 : b];
    if constexpr (F32) {
      stash_f32();
#pragma unroll
      for (int i = 0; i < EARLY; ++i) fetch_keys(j0 + 64u, i);
      if constexpr (!LATE) fetch_values(j0 + 64u);
      lds_barrier();
    }

    // Element 4 h + e of a lane: key 16 h + 4 g + e of the wavefront's 32.  Operands are read DEEP steps ahead of
    // their matrix instructions; the barriers keep the compiler from moving each read to its use.
    float4_t acc[2][2];                                            // of the first terms, and of those that stand for 2^-11
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      acc[h][0] = SCALED ? float4_t{0.0f, 0.0f, 0.0f, 0.0f} : float4_t{-origin, -origin, -origin, -origin};
      acc[h][1] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    constexpr int DEEP = 2;
    half8_t kf[DEEP + 1][2], kl[F32 ? DEEP + 1 : 1][2];
    auto read_keys = [&](int step) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* from = stage + key_row + h * (16u * DP * 2u) + (((4u * step + g) ^ key_swz) * 16u);
        kf[step % (DEEP + 1)][h] = *reinterpret_cast<const half8_t*>(from);
        if constexpr (F32) kl[step % (DEEP + 1)][h] = *reinterpret_cast<const half8_t*>(from + Shared::kStage);
      }
    };
#pragma unroll
    for (int i = 0; i < DEEP; ++i) read_keys(i);
    if constexpr (!F32) {
      stash_scales(b ^ 1u);
      fetch_scales(j0 + 128u);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int step = 0; step < STEPS; ++step) {
      if (step + DEEP < STEPS) read_keys(step + DEEP);
      if constexpr (F32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) acc[h][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl[step % (DEEP + 1)][h], q_hi[step], acc[h][1], 0, 0, 0);
      }
#pragma unroll
      for (int term = 0; term < 2; ++term) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float4_t& x = acc[h][term];
          x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[step % (DEEP + 1)][h], term == 0 ? q_hi[step] : q_lo[step], x, 0, 0, 0);
        }
      }
      if constexpr (!F32) {
        if (step % 2 == 1) stash_keys(b ^ 1u, step / 2), fetch_keys(j0 + 128u, step / 2);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // The values' operands, read AHEAD blocks ahead of their matrix instructions, two blocks at a time.
    constexpr int AHEAD = 2;
    half8_t vf[AHEAD + 2], vl[F32 ? AHEAD + 2 : 1];
    auto read_values = [&](int j) {
      const uint8_t* from = stage + (value_row ^ static_cast<uint32_t>(j * 16)) + j * 1024u;
      vf[j % (AHEAD + 2)] = *reinterpret_cast<const half8_t*>(from);
      if constexpr (F32) vl[j % (AHEAD + 2)] = *reinterpret_cast<const half8_t*>(from + Shared::kStage);
    };
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) read_values(j);

    float s[8];
    float4 vsv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = fmaf(acc[h][1][e], 0x1p-11f, acc[h][0][e]);
      if constexpr (SCALED) {
        const uint32_t at = half * 32u + h * 16u + g * 4u, of = F32 ? 0u : b;
        const float4 ks = *reinterpret_cast<const float4*>(&sh.scales[of][0][at]);
        vsv[h] = *reinterpret_cast<const float4*>(&sh.scales[of][1][at]);
        s[4 * h] = fmaf(x[0], ks.x, -origin), s[4 * h + 1] = fmaf(x[1], ks.y, -origin);
        s[4 * h + 2] = fmaf(x[2], ks.z, -origin), s[4 * h + 3] = fmaf(x[3], ks.w, -origin);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * h + e] = x[e];
      }
    }
    if (j0 + 64u > prefix || j0 < latest_start || wg_last - j0 < 64u) {   // some column does not see some key of the tile
      const uint32_t now = again(t), key0 = j0 + half * 32u, from = 4u * (now >> 4 & 3u);
      const uint32_t row = column(now).row;
      uint32_t shown = key0 <= wg_last ? tree_keys(a, a.mask + static_cast<uint64_t>(row) * a.words, key0) : 0u;
      const uint32_t start = a.window == 0 ? 0u : sh.start[col_group * 16u + (now & 15u)];   // (with no window, rows that see nothing have no bits)
      if (start > key0) shown = start - key0 < 32u ? shown & ~0u << (start - key0) : 0u;
      if (wg_last - key0 < 31u) shown &= (2u << (wg_last - key0)) - 1u;
      shown >>= from;
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = (shown >> (16 * (e / 4) + e % 4) & 1u) != 0u ? s[e] : -INFINITY;
    }
    float most = s[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) most = fmaxf(most, s[e]);
    float corr = 1.0f;
    // Scores are formed as differences from the reference, and only those are brought to units of log2: what rounding takes from a
    // large score would else be a power of two to scale by.
    if (__any(most * score_scale > kSlack || (ref == -INFINITY && most > ref))) {
      const float before = ref;                                    // the same in all lanes of the column
      ref = fmaxf(ref, groups_max(most + origin));
      corr = before == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((before - ref) * score_scale);
      const float to = reference_score(ref);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = (s[e] + origin) - to;
      origin = to;
    }
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s[e] = __builtin_amdgcn_exp2f(s[e] * score_scale);
      sum += s[e];
    }
    run_sum = fmaf(corr, run_sum, sum);
    if constexpr (SCALED) {
      // The values' scales enter the weights, under a power of two that keeps the largest contribution so far
      // between 2^9 and 2^15.
      lane_most *= corr;
      float here = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[e] *= (&vsv[e / 4].x)[e % 4];
        here = fmaxf(here, fabsf(s[e]));
      }
      lane_most = fmaxf(lane_most, here);
      if (__any(corr != 1.0f || !(here * value_up < 0x1p15f))) {
        const float largest = groups_max(lane_most), scaled = largest * value_up;
        if (largest > 0.0f && !(scaled >= 0x1p9f && scaled < 0x1p15f)) {
          const float up = power_of_two_to(largest, 13);
          corr *= up / value_up;
          value_up = up;
        }
      }
    }
    if (__any(corr != 1.0f)) {
#pragma unroll
      for (int j = 0; j < VE; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] *= corr;
      }
    }
    half8_t p_hi, p_lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = s[e] * value_up;
      const _Float16 hi = static_cast<_Float16>(x);
      p_hi[e] = hi;
      p_lo[e] = static_cast<_Float16>(x - static_cast<float>(hi));
    }
    half8_t p_down;                                                // for the values' second terms
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) p_down[e] = p_hi[e] * static_cast<_Float16>(0x1p-11f);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < VE; j += 2) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (j + AHEAD + i < VE) read_values(j + AHEAD + i);
      }
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 2; ++i) o[j + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl[(j + i) % (AHEAD + 2)], p_down, o[j + i], 0, 0, 0);
      }
#pragma unroll
      for (int term = 0; term < 2; ++term) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          o[j + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[(j + i) % (AHEAD + 2)], term == 0 ? p_lo : p_hi, o[j + i], 0, 0, 0);
        }
      }
      if constexpr (!F32) stash_values(b ^ 1u, j / 2);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (!F32) fetch_values(j0 + 128u);
    if constexpr (LATE) {
#pragma unroll
      for (int i = EARLY; i < KLOADS; ++i) fetch_keys(j0 + 64u, i);
      fetch_values(j0 + 64u);
    }
    lds_barrier();                                                 // (the loads stay under way)
  }
  __syncthreads();

  // Merge of the halves under the larger reference, each for half the elements; the lanes' shares of the sums of weights first.
  run_sum = groups_sum(run_sum);
  const uint32_t late = again(t), late_g = late >> 4 & 3u, own_at = col_group * 16u + (late & 15u);
  constexpr int VH = VE / 2;
  float4_t* pieces = reinterpret_cast<float4_t*>(sh.stage[0]) + col_group * (VE * 64u) + (late & 63u);
  if (late_g == 0u) sh.ref[half][own_at] = ref, sh.sum[half][own_at] = run_sum, sh.up[half][own_at] = value_up;
#pragma unroll
  for (int j = 0; j < VH; ++j) pieces[(half * VH + j) * 64u] = half == 0u ? o[VH + j] : o[j];
  __syncthreads();
  const float ref0 = sh.ref[0][own_at], ref1 = sh.ref[1][own_at], top = fmaxf(ref0, ref1), to = reference_score(top);
  const float w0 = __builtin_amdgcn_exp2f((ref0 - to) * score_scale), w1 = __builtin_amdgcn_exp2f((ref1 - to) * score_scale);
  const float total = fmaf(w1, sh.sum[1][own_at], w0 * sh.sum[0][own_at]);
  const float f0 = w0 / sh.up[0][own_at], f1 = w1 / sh.up[1][own_at];
  float4_t merged[VH];                                             // elements 16 (half * VH + j) + 4 g ..
  bool finite = fabsf(total) < INFINITY;
#pragma unroll
  for (int j = 0; j < VH; ++j) {
    const float4_t own = half == 0u ? o[j] : o[VH + j], other = pieces[((1u - half) * VH + j) * 64u];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      merged[j][e] = half == 0u ? fmaf(other[e], f1, own[e] * f0) : fmaf(own[e], f1, other[e] * f0);
      finite = finite && fabsf(merged[j][e]) < INFINITY;
    }
  }
  if (!finite) sh.special = 1u;
  __syncthreads();
  // Infinities and NaN were not kept apart: whatever met one has left a sum that is not finite, or set `special`, and the
  // workgroup's columns are done again one by one.  That is meant for the exception: NaN among the values that no row sees, 64 rows of 24
  // heads over 4 of 256 on 32832 fp16 keys, make 33 ms of 0.13.
  if (__builtin_amdgcn_readfirstlane(sh.special) != 0u) {          // workgroup-uniform
    __syncthreads();
    for (uint32_t c = c0; c < c_end; ++c) {
      const TreePair pair{c / group, c / group * a.heads + kv * group + c % group};
      attend_pair<KV, 512>(a, pair, kv, wg_start, wg_last, s_part, *reinterpret_cast<PairShared*>(sh.stage[0]));
    }
    return;
  }
  if (c0 + own_at >= c_end) return;
  const Column mine = column(late);
  const uint64_t pair = static_cast<uint64_t>(mine.row) * a.heads + mine.head;
  float* out = a.out + pair * D;
  float factor = total == 0.0f ? 0.0f : 1.0f / total;
  if (split > 1u) {
    const uint64_t part = pair * split + s_part;
    out = a.part.pacc + part * D;
    const float natural = score_scale * kLn2, largest = top * natural;
    factor = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(part_move<true>(fmaf(top, natural, -largest)));
    if (late_g == 0u && half == 0u) a.part.pmax[part] = largest, a.part.psum[part] = total * factor;
  }
#pragma unroll
  for (int j = 0; j < VH; ++j) {
    const uint32_t d = (half * VH + j) * 16u + late_g * 4u;
    if (d < D) *reinterpret_cast<float4_t*>(out + d) = merged[j] * factor;
  }
}

// ---- few pairs a workgroup: eight at most, sixteen over an fp32 cache -------------------------------------------------------
//
// attend_row with `each` (row, head) pairs in place of a row's heads, so that a key is read once for all of them: sixteen fp32
// pairs or a row's heads, as tree_rule says.  10 rows of 8 heads over 8 of 128 on 4565 fp32 keys 49 us by rows, 15.7 by sixteen
// pairs; few keys are the other way round, 46 rows of 8 heads over 1 of 128 on 52 7.6 and 9.4, as the sums of sixteen are merged.
// The shortest calls are a launch and its latencies: 10 rows of 12 heads over 2 of 64 on 62 fp16 keys 5.5 us (an empty launch
// among others 3.5).
template <KvKind KV, int DP, int NW>
__global__ __launch_bounds__(NW * 64, 1) void attention_pairs_kernel(AttentionArgs a, uint32_t each) {
  union Lds {
    RowsShared<KV, DP, NW> merge;
    PairShared pair;
    __device__ Lds() {}
  };
  __shared__ Lds lds;
  __shared__ TreeRows rows;
  const uint32_t t = threadIdx.x, split = a.part.split == 0 ? 1u : static_cast<uint32_t>(a.part.split);
  const uint32_t kv = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads, s_part = unit % split;
  const uint32_t pairs = static_cast<uint32_t>(a.rows) * (a.heads / a.kv_heads), first = unit / split * each;
  const uint32_t here = pairs - first < each ? pairs - first : each;
  if (t < here) rows.at[t] = tree_pair(a, kv, first + t).at;
  if (t == 0u) rows.special = 0u;
  // From the earliest key that a row sees.
  uint64_t start = 0, last = a.n - 1;
  if (a.window != 0 || a.n == a.tree) {
    const uint32_t own = t % 16u;
    uint64_t row_last;
    key_range<true>(a, tree_pair(a, kv, first + (own < here ? own : here - 1u)).row, start, row_last);
#pragma unroll
    for (uint32_t off = 8u; off > 0u; off >>= 1) {
      const uint64_t other = __shfl_xor(static_cast<unsigned long long>(start), off, kWave);
      start = other < start ? other : start;
    }
    const uint32_t high = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(start >> 32));
    start = static_cast<uint64_t>(high) << 32 | __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(start));
  }
  if (a.part.split != 0 && !key_chunk(a, s_part, start, last)) {   // workgroup-uniform
    for (uint32_t i = 0; i < here; ++i) {
      const TreePair pair = tree_pair(a, kv, first + i);
      empty_part<NW * 64, true>(a, pair.row, pair.at - pair.row * a.heads, 1, s_part);
    }
    return;
  }
  attend_row<KV, DP, NW, KV == KvKind::F32 ? 16 : 32, true>(a, first, kv, 0, here, start, last, s_part, lds.merge, &rows);
  __syncthreads();
  if (__builtin_amdgcn_readfirstlane(rows.special) == 0u) return;       // workgroup-uniform
  for (uint32_t i = 0; i < here; ++i) attend_pair<KV, NW * 64>(a, tree_pair(a, kv, first + i), kv, start, last, s_part, lds.pair);
}

// (The wavefronts of a workgroup under a window go by the whole cache's keys: by those that are walked, 11 windows of 8 to 512
// keys took 0.98 to 1.06 of the time, as more wavefronts are sooner through the loads of few keys.)
template <KvKind KV>
hipError_t launch_pairs(const AttentionArgs& a, uint64_t each, hipStream_t stream) {
  const uint64_t workgroups = (a.rows * (a.heads / a.kv_heads) + each - 1) / each * a.kv_heads * (a.part.split == 0 ? 1 : a.part.split);
  return with_waves<KV>(a, workgroups, [&](auto dim, auto waves) {
    hipLaunchKernelGGL((attention_pairs_kernel<KV, decltype(dim)::value, decltype(waves)::value>), dim3(static_cast<uint32_t>(workgroups)),
                       dim3(decltype(waves)::value * 64u), 0, stream, a, static_cast<uint32_t>(each));
  });
}

template <KvKind KV>
hipError_t launch_tree_tiles(const AttentionArgs& a, hipStream_t stream) {
  const uint64_t split = a.part.split == 0 ? 1 : a.part.split;
  const AttentionCall call{a.rows, a.n, a.heads, a.kv_heads, a.head_dim, 0, false};
  const dim3 grid(static_cast<uint32_t>(attention_pairs64(call) * split));
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(512), 0, stream, a); };
  a.head_dim <= 64 ? go(attention_tree_kernel<KV, 64>) : a.head_dim <= 128 ? go(attention_tree_kernel<KV, 128>) : go(attention_tree_kernel<KV, 256>);
  return hipGetLastError();
}

}  // namespace

TreeShape attention_tree_shape(uint32_t kind, uint64_t m, uint64_t n, uint64_t heads, uint64_t kv_heads, uint64_t head_dim,
                               uint64_t window, const void* out, uint64_t most_parts) {
  const uint32_t dim = static_cast<uint32_t>(head_dim);
  const bool by_rows = with_kind(kind, [&](auto tag) { return runs_fit<decltype(tag)::value>(dim); });
  // (a tile's rows lie within 2^31 bytes, its loads are runs of eight elements)
  const bool shared = reinterpret_cast<uintptr_t>(out) % 16 == 0 && kv_heads * head_dim * (kind == 0 ? 4 : 2) < (1u << 25) &&
                      n < (1u << 31) && dim % 8 == 0;
  const TreeCall call{m, window != 0 && window < n ? window : n, heads, kv_heads, head_dim, padded_head(dim), kind == 0, kind > 1, by_rows, shared};
  if (by_rows || shared) return tree_rule(call, static_cast<uint64_t>(num_cus()), most_parts, kAttentionPartsMost);
  uint64_t parts = 2 * static_cast<uint64_t>(num_cus()) / (m * heads);      // a workgroup a row and head
  if (parts > call.keys / 128) parts = call.keys / 128;
  if (parts > most_parts) parts = most_parts;
  while (parts > 1 && attention_parts_size(m, heads, head_dim, parts) > kAttentionPartsMost) --parts;
  return TreeShape{false, 1, parts < 2 ? 1 : parts};
}

hipError_t launch_attention_tree(uint32_t kind, const float* q, const void* k, const void* v, const float* k_scale, const float* v_scale,
                                 const uint32_t* mask, float* out, uint64_t m, uint64_t n, uint64_t heads, uint64_t kv_heads,
                                 uint64_t head_dim, uint64_t tree, uint64_t window, const TreeShape& shape, void* scratch, hipStream_t stream) {
  const uint64_t parts = shape.parts;
  AttentionArgs a = args_of(q, k, v, k_scale, v_scale, out, n, heads, kv_heads, head_dim, 0, 0, window, false, m);
  a.mask = mask, a.tree = static_cast<uint32_t>(tree), a.words = static_cast<uint32_t>((tree + 31) / 32);
  if (parts > 1) {
    float* acc = static_cast<float*>(scratch);
    float* most = acc + m * heads * parts * head_dim;
    a.part = SplitOut{acc, most, most + m * heads * parts, parts};
  }
  const hipError_t e = with_kind(kind, [&](auto tag) {
    constexpr KvKind KV = decltype(tag)::value;
    if (shape.tile) return launch_tree_tiles<KV>(a, stream);
    if (runs_fit<KV>(a.head_dim)) return launch_pairs<KV>(a, shape.pairs, stream);
    hipLaunchKernelGGL((attention_any_kernel<KV, true>), dim3(static_cast<uint32_t>(m * heads * (parts < 2 ? 1 : parts))), dim3(256), 0, stream, a);
    return hipGetLastError();
  });
  if (e != hipSuccess || parts <= 1) return e;
  return launch_combine<true>(a.part.pacc, a.part.pmax, a.part.psum, out, m, heads, head_dim, parts, stream);
}

}  // namespace qmm

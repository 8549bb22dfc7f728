// "qk_norm_rope", "qk_norm_mrope": RMS norm of every query and key head and its rotary embedding in one pass over the
// projection's rows, which "qgate_split", "rmsnorm", "rope" and "cast_f32_f16" do in up to six.

#include <cmath>

#include "qmm_device.hpp"
#include "qmm_kernels.hpp"
#include "tree_args.hpp"

namespace qmm {
namespace {

struct QkNormArgs {
  const float *q, *k, *wq, *wk;
  const uint64_t* pos3;              // null: positions pos_base + row
  float *q_out, *gate;               // gate null: the query heads lie side by side
  void* k_out;                       // from its first row on
  uint64_t rows, pos_base, q_stride, k_stride;
  uint32_t heads, kv_heads, head_dim, rope_dim, sec_t, sec_h, each, chunks;
  float eps;
  double turn[7];                    // theta^(-2 2^b / rope_dim)
};

// cos and sin of position * theta^(-2 j / rope_dim), formed in 64 bits and rounded once, as "rope" does.  theta^(-2 j /
// rope_dim) is the product of the powers turn[b] of j's bits (at most six roundings of 2^-53); the angle is taken modulo
// pi/2, which three parts hold to more than 2^-150 of it, and the Taylor sums up to x^13 and x^12 miss by less than 2^-40 there.
__device__ __forceinline__ float2 cos_sin(const QkNormArgs& a, uint64_t row, uint32_t j) {
  uint64_t p = a.pos_base + row;
  if (a.pos3 != nullptr) p = a.pos3[row * 3 + (j < a.sec_t ? 0u : j < a.sec_t + a.sec_h ? 1u : 2u)];
  if (p > (uint64_t{1} << 50)) p = uint64_t{1} << 50;              // above, n below is off by more than one
  double f = 1.0;
#pragma unroll
  for (uint32_t b = 0; b < 7; ++b) f *= (j >> b & 1u) != 0u ? a.turn[b] : 1.0;
  const double angle = static_cast<double>(p) * f;
  const double n = rint(angle * 0.63661977236758134308);
  double x = fma(n, -0x1.921fb54442d18p+0, angle);
  x = fma(n, -0x1.1a62633145c07p-54, x);
  x = fma(n, 0x1.f1976b7ed8fbcp-110, x);
  const uint32_t quarter = static_cast<uint32_t>(static_cast<int>(n - 4.0 * floor(0.25 * n)));
  const double z = x * x;
  double sn = fma(z, 1.0 / 6227020800.0, -1.0 / 39916800.0), cs = fma(z, 1.0 / 479001600.0, -1.0 / 3628800.0);
  sn = fma(z, sn, 1.0 / 362880.0), cs = fma(z, cs, 1.0 / 40320.0);
  sn = fma(z, sn, -1.0 / 5040.0), cs = fma(z, cs, -1.0 / 720.0);
  sn = fma(z, sn, 1.0 / 120.0), cs = fma(z, cs, 1.0 / 24.0);
  sn = fma(z, sn, -1.0 / 6.0), cs = fma(z, cs, -0.5);
  sn = fma(x * z, sn, x), cs = fma(z, cs, 1.0);
  const float sin_x = static_cast<float>(sn), cos_x = static_cast<float>(cs);
  const float c = (quarter & 1u) != 0u ? sin_x : cos_x, s = (quarter & 1u) != 0u ? cos_x : sin_x;
  return float2{quarter == 1u || quarter == 2u ? -c : c, quarter >= 2u ? -s : s};
}

// Sum over each run of LANES lanes, in every lane of it.
template <int LANES>
__device__ __forceinline__ float run_sum(float v) {
  v = row16_sum(v);
  if constexpr (LANES >= 32) {
    const auto b = __builtin_amdgcn_permlane16_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
    v = bit_cast<float>(b[0]) + bit_cast<float>(b[1]);
  }
  if constexpr (LANES == 64) {
    const auto b = __builtin_amdgcn_permlane32_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
    v = bit_cast<float>(b[0]) + bit_cast<float>(b[1]);
  }
  return v;
}

// A wavefront takes `each` times 64 / LANES heads of one row, LANES lanes with four elements each to a head, and forms the
// angles of its lanes' elements once; the other element of a pair is four lanes' worth away and comes across the wavefront.
// A head's elements are read once, all before any is written.
template <int LANES, bool F16>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkNormArgs a) {
  constexpr uint32_t kHeads = 64 / LANES;
  const uint32_t lane = threadIdx.x & 63u, at = lane % LANES, slot = lane / LANES;
  const uint64_t unit = static_cast<uint64_t>(blockIdx.x) * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint64_t row = unit / a.chunks;
  if (row >= a.rows) return;                                        // wave-uniform
  const uint32_t all = a.heads + a.kv_heads, D = a.head_dim, pairs = a.rope_dim / 2u;
  const uint32_t head0 = static_cast<uint32_t>(unit % a.chunks) * a.each * kHeads + slot;
  const uint32_t e = at * 4u;                                       // this lane's elements e .. e + 3
  const bool inside = e < D;
  const uint32_t wide = a.gate != nullptr ? 2u * D : D;
  const float *qr = a.q + row * a.q_stride, *kr = a.k + row * a.k_stride;
  auto source = [&](uint32_t h) { return h < a.heads ? qr + static_cast<size_t>(h) * wide : kr + static_cast<size_t>(h - a.heads) * D; };
  auto four = [](bool there, const float* from) {
    if (!there) return float4{0.0f, 0.0f, 0.0f, 0.0f};
    return *reinterpret_cast<const float4*>(from);
  };
  auto load = [&](uint32_t h) { return four(inside && h < all, source(h) + e); };
  auto load_gate = [&](uint32_t h) { return four(a.gate != nullptr && inside && h < a.heads, source(h) + D + e); };
  float4 next = load(head0), next_gate = load_gate(head0);
  const float4 wq = four(inside, a.wq + e), wk = four(inside, a.wk + e);

  // y' = y cos +- partner sin: the first half of the pairs minus, the second plus, elements past rope_dim as they are.
  float c[4] = {1.0f, 1.0f, 1.0f, 1.0f}, s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  int partner = static_cast<int>(lane);
  if (e < a.rope_dim) {
    const bool second = e >= pairs;
    partner += second ? -static_cast<int>(pairs / 4u) : static_cast<int>(pairs / 4u);
    const uint32_t j = second ? e - pairs : e;
    const float2 t0 = cos_sin(a, row, j), t1 = cos_sin(a, row, j + 1u), t2 = cos_sin(a, row, j + 2u), t3 = cos_sin(a, row, j + 3u);
    c[0] = t0.x, c[1] = t1.x, c[2] = t2.x, c[3] = t3.x;
    s[0] = t0.y, s[1] = t1.y, s[2] = t2.y, s[3] = t3.y;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) s[i] = second ? s[i] : -s[i];
  }
  const float part = 1.0f / static_cast<float>(D);
  for (uint32_t n = 0; n < a.each; ++n) {
    const uint32_t h = head0 + n * kHeads;
    const float4 x = next, g = next_gate;
    if (n + 1u < a.each) next = load(h + kHeads), next_gate = load_gate(h + kHeads);
    float sum = x.x * x.x;
    sum = fmaf(x.y, x.y, sum);
    sum = fmaf(x.z, x.z, sum);
    sum = fmaf(x.w, x.w, sum);
    sum = run_sum<LANES>(sum);
    const float gain = 1.0f / sqrtf(sum * part + a.eps);
    const bool query = h < a.heads;
    const float4 w = {query ? wq.x : wk.x, query ? wq.y : wk.y, query ? wq.z : wk.z, query ? wq.w : wk.w};
    const float y[4] = {x.x * gain * w.x, x.y * gain * w.y, x.z * gain * w.z, x.w * gain * w.w};
    float z[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) z[i] = fmaf(y[i], c[i], __shfl(y[i], partner, kWave) * s[i]);
    if (!inside || h >= all) continue;
    if (query) {
      const size_t to = (row * a.heads + h) * D + e;
      *reinterpret_cast<float4*>(a.q_out + to) = float4{z[0], z[1], z[2], z[3]};
      if (a.gate != nullptr) *reinterpret_cast<float4*>(a.gate + to) = g;
    } else {
      const size_t to = (row * a.kv_heads + (h - a.heads)) * D + e;
      if constexpr (F16) {
        const half2_t low = {static_cast<_Float16>(z[0]), static_cast<_Float16>(z[1])}, high = {static_cast<_Float16>(z[2]), static_cast<_Float16>(z[3])};
        *reinterpret_cast<uint2*>(static_cast<_Float16*>(a.k_out) + to) = uint2{bit_cast<uint32_t>(low), bit_cast<uint32_t>(high)};
      } else {
        *reinterpret_cast<float4*>(static_cast<float*>(a.k_out) + to) = float4{z[0], z[1], z[2], z[3]};
      }
    }
  }
}

// Head sizes, rotated parts and strides that runs of four elements do not divide: a wavefront a head, an element a lane at a
// time, pairs through LDS.
template <bool F16>
__global__ __launch_bounds__(256) void qk_norm_rope_any_kernel(QkNormArgs a) {
  __shared__ float held[4][256];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t all = a.heads + a.kv_heads, D = a.head_dim, pairs = a.rope_dim / 2u;
  const uint64_t unit = static_cast<uint64_t>(blockIdx.x) * 4u + wave, row = unit / all;
  const uint32_t h = static_cast<uint32_t>(unit % all);
  const bool here = row < a.rows, query = h < a.heads;
  const float* from = !here ? nullptr : query ? a.q + row * a.q_stride + static_cast<size_t>(h) * (a.gate != nullptr ? 2u * D : D)
                                              : a.k + row * a.k_stride + static_cast<size_t>(h - a.heads) * D;
  float x[4], sum = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const uint32_t e = lane + 64u * i;
    x[i] = here && e < D ? from[e] : 0.0f;
    sum = fmaf(x[i], x[i], sum);
  }
  sum = run_sum<64>(sum);
  const float gain = 1.0f / sqrtf(sum * (1.0f / static_cast<float>(D)) + a.eps);
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const uint32_t e = lane + 64u * i;
    if (here && e < D) held[wave][e] = x[i] * gain * (query ? a.wq : a.wk)[e];
  }
  __syncthreads();
  if (!here) return;
  const size_t to = query ? (row * a.heads + h) * D : (row * a.kv_heads + (h - a.heads)) * D;
  for (uint32_t e = lane; e < D; e += 64u) {
    float z = held[wave][e];
    if (e < a.rope_dim) {
      const bool second = e >= pairs;
      const float2 turned = cos_sin(a, row, second ? e - pairs : e);
      z = fmaf(z, turned.x, held[wave][second ? e - pairs : e + pairs] * (second ? turned.y : -turned.y));
    }
    if (query) {
      a.q_out[to + e] = z;
      if (a.gate != nullptr) a.gate[to + e] = from[D + e];
    } else if constexpr (F16) {
      static_cast<_Float16*>(a.k_out)[to + e] = static_cast<_Float16>(z);
    } else {
      static_cast<float*>(a.k_out)[to + e] = z;
    }
  }
}

}  // namespace

hipError_t launch_qk_norm_rope(const QkNormCall& call, const float* q, const float* k, const float* wq, const float* wk, const uint64_t* pos3,
                               float* q_out, void* k_out, float* gate, hipStream_t stream) {
  QkNormArgs a{};
  a.q = q, a.k = k, a.wq = wq, a.wk = wk, a.pos3 = pos3, a.q_out = q_out, a.gate = gate;
  const uint64_t k_row = call.kv_heads * call.head_dim, first = call.k_row * k_row * (call.k_f16 != 0 ? 2 : 4);
  a.k_out = static_cast<uint8_t*>(k_out) + first;
  a.rows = call.rows, a.pos_base = call.pos_base, a.q_stride = call.q_stride, a.k_stride = call.k_stride;
  a.heads = static_cast<uint32_t>(call.heads), a.kv_heads = static_cast<uint32_t>(call.kv_heads);
  a.head_dim = static_cast<uint32_t>(call.head_dim), a.rope_dim = static_cast<uint32_t>(call.rope_dim);
  a.sec_t = static_cast<uint32_t>(call.sec_t), a.sec_h = static_cast<uint32_t>(call.sec_h), a.eps = call.eps;
  for (uint32_t b = 0; b < 7; ++b) {
    a.turn[b] = std::pow(static_cast<double>(call.theta), -2.0 * static_cast<double>(1u << b) / static_cast<double>(call.rope_dim));
  }
  const uint64_t all = call.heads + call.kv_heads;
  const bool f16 = call.k_f16 != 0;
  auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  auto grid = [](uint64_t waves) { return dim3(static_cast<uint32_t>((waves + 3) / 4)); };
  if (call.head_dim % 4 != 0 || call.rope_dim % 8 != 0 || call.q_stride % 4 != 0 || call.k_stride % 4 != 0 || !aligned(a.k_out)) {
    a.each = a.chunks = 0;
    const dim3 g = grid(call.rows * all);
    if (f16) hipLaunchKernelGGL(qk_norm_rope_any_kernel<true>, g, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(qk_norm_rope_any_kernel<false>, g, dim3(256), 0, stream, a);
    return hipGetLastError();
  }
  auto go = [&](auto lanes) {
    constexpr int LANES = decltype(lanes)::value;
    const uint64_t groups = (all + 64 / LANES - 1) / (64 / LANES);
    // With many heads a wavefront takes several of a row, which share its angles and hide each other's way to memory (us, 1 / 2
    // / 4 / 7 / 14 at a time: 2048 rows of 28 heads of 256 with fp16 keys 44 / 30 / 24.3 / 25.4 / 26, 4.7 TB/s of them; 512 rows 12.7 / 9.2 /
    // 8.5 / 8.2 / 10.7, 128 rows 5.3 / 4.5 / 5.0 / 6.3 / 9.7, one row 3.4 / 3.4 / 4.4 / 5.6 / 8.7).
    const uint64_t units = call.rows * groups;
    a.each = units >= 8192 ? 4 : units >= 2048 ? 2 : 1;
    a.chunks = static_cast<uint32_t>((groups + a.each - 1) / a.each);
    const dim3 g = grid(call.rows * a.chunks);
    if (f16) hipLaunchKernelGGL((qk_norm_rope_kernel<LANES, true>), g, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((qk_norm_rope_kernel<LANES, false>), g, dim3(256), 0, stream, a);
  };
  if (call.head_dim <= 64) go(std::integral_constant<int, 16>{});
  else if (call.head_dim <= 128) go(std::integral_constant<int, 32>{});
  else go(std::integral_constant<int, 64>{});
  return hipGetLastError();
}

}  // namespace qmm

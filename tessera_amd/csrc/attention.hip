// Dispatch of the "attention" ids, their flash-decoding forms and the merge of those (kernels: attention_kernels.hpp).

#include "attention_kernels.hpp"

namespace qmm {
namespace {

hipError_t launch_attention_as(uint32_t kind, const AttentionArgs& a, uint64_t m, hipStream_t stream) {
  return with_kind(kind, [&](auto tag) {
    constexpr KvKind KV = decltype(tag)::value;
    if (runs_fit<KV>(a.head_dim)) return launch_rows<KV>(a, m, stream);
    const uint64_t parts = a.part.split == 0 ? 1 : a.part.split;
    hipLaunchKernelGGL(attention_any_kernel<KV>, dim3(static_cast<uint32_t>(m * a.heads * parts)), dim3(256), 0, stream, a);
    return hipGetLastError();
  });
}

}  // namespace

uint64_t attention_parts(uint32_t kind, uint64_t m, uint64_t n, uint64_t heads, uint64_t kv_heads, uint64_t head_dim,
                         uint64_t q_base, uint64_t window, bool causal, const void* out, uint64_t most_parts) {
  if (kind == 0 || m < 17 || n >= (1u << 31) || reinterpret_cast<uintptr_t>(out) % 16 != 0) return 0;
  const uint32_t dim = static_cast<uint32_t>(head_dim);
  if (!with_kind(kind, [&](auto tag) { return runs_fit<decltype(tag)::value>(dim); })) return 0;
  if (kv_heads * head_dim * 2 >= (1u << 25)) return 0;             // a tile's rows lie within 2^31 bytes
  uint64_t keys = causal && q_base + m < n ? q_base + m : n;
  if (causal && window != 0 && window < keys) keys = window;
  const AttentionCall call{m, keys, heads, kv_heads, head_dim, padded_head(dim), kind != 1};
  if (attention_pairs64(call) >= kMaxGridThreads / 512u) return 0;
  return attention_rule(call, static_cast<uint64_t>(num_cus()), most_parts, kAttentionPartsMost);
}

size_t attention_parts_bytes(uint64_t m, uint64_t heads, uint64_t head_dim, uint64_t parts) {
  return attention_parts_size(m, heads, head_dim, parts);
}

// kind: 0 fp32, 1 fp16 keys and values; 2 int8, 3 4-bit, 4 E4M3 codes with one scale per key row (always causal).
hipError_t launch_attention(uint32_t kind, const float* q, const void* k, const void* v, const float* k_scale, const float* v_scale,
                            float* out, uint64_t m, uint64_t n, uint64_t heads, uint64_t kv_heads, uint64_t head_dim,
                            uint64_t q_base, uint64_t row_base, uint64_t window, bool causal, uint64_t parts, void* scratch,
                            hipStream_t stream) {
  AttentionArgs a = args_of(q, k, v, k_scale, v_scale, out, n, heads, kv_heads, head_dim, q_base, row_base, window, causal, m);
  if (parts == 0) return launch_attention_as(kind, a, m, stream);
  if (parts > 1) {
    float* acc = static_cast<float*>(scratch);
    float* most = acc + m * heads * parts * head_dim;
    a.part = SplitOut{acc, most, most + m * heads * parts, parts};
  }
  const hipError_t e = with_kind(kind, [&](auto tag) {
    if constexpr (decltype(tag)::value == KvKind::F32) return hipErrorInvalidValue;
    else return launch_tiles<decltype(tag)::value>(a, stream);
  });
  if (e != hipSuccess || parts == 1) return e;
  return launch_attention_combine(a.part.pacc, a.part.pmax, a.part.psum, out + row_base * heads * head_dim, m, heads, head_dim, parts, stream);
}

// The split-N form: kv_kind as launch_attention_as (0 fp32, 1 fp16, 2.. quantized with scales).
hipError_t launch_attention_split(const float* q, const void* k, const void* v, const float* k_scale, const float* v_scale,
                                  float* pacc, float* pmax, float* psum, uint64_t m, uint64_t n, uint64_t heads,
                                  uint64_t kv_heads, uint64_t head_dim, uint64_t q_base, uint64_t window, uint32_t kv_kind,
                                  bool causal, uint64_t split, hipStream_t stream) {
  AttentionArgs a = args_of(q, k, v, k_scale, v_scale, nullptr, n, heads, kv_heads, head_dim, q_base, 0, window, causal, m);
  a.part = SplitOut{pacc, pmax, psum, split};
  return launch_attention_as(kv_kind, a, m, stream);
}

hipError_t launch_attention_combine(const float* pacc, const float* pmax, const float* psum, float* out, uint64_t m,
                                    uint64_t heads, uint64_t head_dim, uint64_t split, hipStream_t stream) {
  return launch_combine<false>(pacc, pmax, psum, out, m, heads, head_dim, split, stream);
}

}  // namespace qmm

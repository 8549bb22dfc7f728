// "attention_tree" and its forms over quantized caches: the rows of a drafted tree against the keys before it and the
// tree's own, as each row's bits say (attention_kernels.hpp: TREE).

#include "attention_kernels.hpp"

namespace qmm {

uint64_t attention_tree_parts(uint32_t kind, uint64_t m, uint64_t n, uint64_t heads, uint64_t kv_heads, uint64_t head_dim,
                              uint64_t window, uint64_t most_parts) {
  const uint64_t keys = window != 0 && window < n ? window : n, per = kind == 0 ? 16 : 8;
  const uint64_t units = m * kv_heads * ((heads / kv_heads + per - 1) / per);
  uint64_t parts = 2 * static_cast<uint64_t>(num_cus()) / units;
  if (parts > keys / 128) parts = keys / 128;
  if (parts > most_parts) parts = most_parts;
  while (parts > 1 && attention_parts_size(m, heads, head_dim, parts) > kAttentionPartsMost) --parts;
  return parts == 0 ? 1 : parts;
}

hipError_t launch_attention_tree(uint32_t kind, const float* q, const void* k, const void* v, const float* k_scale, const float* v_scale,
                                 const uint32_t* mask, float* out, uint64_t m, uint64_t n, uint64_t heads, uint64_t kv_heads,
                                 uint64_t head_dim, uint64_t tree, uint64_t window, uint64_t parts, void* scratch, hipStream_t stream) {
  AttentionArgs a = args_of(q, k, v, k_scale, v_scale, out, n, heads, kv_heads, head_dim, 0, 0, window, false, m);
  a.mask = mask, a.tree = static_cast<uint32_t>(tree), a.words = static_cast<uint32_t>((tree + 31) / 32);
  if (parts > 1) {
    float* acc = static_cast<float*>(scratch);
    float* most = acc + m * heads * parts * head_dim;
    a.part = SplitOut{acc, most, most + m * heads * parts, parts};
  }
  const hipError_t e = launch_attention_as<true>(kind, a, m, stream);
  if (e != hipSuccess || parts <= 1) return e;
  return launch_combine<true>(a.part.pacc, a.part.pmax, a.part.psum, out, m, heads, head_dim, parts, stream);
}

}  // namespace qmm

// "tree_mask": what the nodes of a drafted tree see, from their parents.

#include "qmm_device.hpp"
#include "qmm_kernels.hpp"
#include "tree_args.hpp"

namespace qmm {
namespace {

// Node i follows node parents[i] < i, or the cache's last token (kRoot).  It sees itself and what its parent sees; its
// position is `base` plus its depth.  Any other parent marks a place that holds no node (padding): that place and all that
// follow it see nothing, at position `base`.
//
// Bound by latency.  An ancestor chain has up to `nodes` links, so it is not walked link by link: all nodes first walk
// the links inside their own 32 (one word of the bits, at most 31 links) and keep those bits and the ancestor outside
// (`leave`); then a node needs one step a word.  A workgroup does the first for every node before its last one and the
// second for 64 of its own, whose rows it gathers in LDS to write them whole.  16 nodes 3.5 us among others
// (an empty launch), 1000 nodes 5.8.
constexpr uint32_t kRoot = 0xFFFFFFFFu, kPadding = 0xFFFFFFFEu;
constexpr uint32_t kTreeNodes = 64, kTreeThreads = 256;

__global__ __launch_bounds__(kTreeThreads) void tree_mask_kernel(const uint32_t* __restrict__ parents, uint32_t* __restrict__ mask,
                                                                 uint64_t* __restrict__ positions, uint32_t nodes, uint64_t base) {
  constexpr uint32_t kWords = kTreeMaskMost / 32u;
  __shared__ uint32_t up[kTreeMaskMost], near_bits[kTreeMaskMost], leave[kTreeMaskMost], rows[kTreeNodes][kWords + 1];
  const uint32_t t = threadIdx.x, first = blockIdx.x * kTreeNodes, words = (nodes + 31u) / 32u;
  const uint32_t end = first + kTreeNodes < nodes ? first + kTreeNodes : nodes;
  for (uint32_t i = t; i < end; i += kTreeThreads) {
    const uint32_t p = parents[i];
    up[i] = p == kRoot ? kRoot : p < i ? p : kPadding;
  }
  for (uint32_t i = t; i < kTreeNodes * (kWords + 1u); i += kTreeThreads) (&rows[0][0])[i] = 0u;
  __syncthreads();
  for (uint32_t i = t; i < end; i += kTreeThreads) {
    uint32_t bits = 1u << (i & 31u), a = up[i];
    while (a < kTreeMaskMost && (a >> 5) == (i >> 5)) bits |= 1u << (a & 31u), a = up[a];
    near_bits[i] = bits, leave[i] = a;
  }
  __syncthreads();
  const uint32_t i = first + t;
  if (t < kTreeNodes && i < end) {
    uint32_t depth = 0, a = i;
    while (a < kTreeMaskMost) {
      rows[t][a >> 5] = near_bits[a];
      depth += __popc(near_bits[a]);
      a = leave[a];
    }
    if (a == kPadding) {
      depth = 1u;
      for (uint32_t w = 0; w <= i >> 5; ++w) rows[t][w] = 0u;
    }
    const uint64_t position = base + depth - 1u;
#pragma unroll
    for (uint32_t axis = 0; axis < 3; ++axis) positions[i * 3ull + axis] = position;
  }
  __syncthreads();
  for (uint32_t at = t; at < (end - first) * words; at += kTreeThreads) mask[static_cast<size_t>(first) * words + at] = rows[at / words][at % words];
}

}  // namespace

hipError_t launch_tree_mask(const uint32_t* parents, uint32_t* mask, uint64_t* positions, uint32_t nodes, uint64_t base, hipStream_t stream) {
  hipLaunchKernelGGL(tree_mask_kernel, dim3((nodes + kTreeNodes - 1) / kTreeNodes), dim3(kTreeThreads), 0, stream, parents, mask, positions, nodes, base);
  return hipGetLastError();
}

}  // namespace qmm

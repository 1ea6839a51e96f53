// What the kernels of a drafted tree share: its parents, counts and cache slots.
#pragma once

#include "common.hpp"

namespace grpo {

constexpr int TREE_MAX = GRPO_TREE_MAX_NODES;  // nodes of a tree: one per lane
static_assert(TREE_MAX == 64, "one lane per node");

// A node's parent is an earlier node; anything else (-1) is none.
__device__ __forceinline__ int node_parent(int p, int i) { return p >= 0 && p < i ? p : -1; }

// Of every node (lane i < T, p its parent as above) the nodes that it sees: its ancestors and
// itself, as bits. The bits of the node 2^k levels up are joined in step k, six at most.
__device__ __forceinline__ uint64_t ancestors(int p) {
  const int lane = threadIdx.x & 63;
  uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
  while (__ballot(p >= 0)) {
    const int from = p >= 0 ? p : lane;
    const uint32_t l = __shfl((int)lo, from), h = __shfl((int)hi, from);
    const int up = __shfl(p, from);
    lo |= l;
    hi |= h;
    p = p >= 0 ? up : -1;
  }
  return (uint64_t)hi << 32 | lo;
}

// Nodes of sequence b that are in use: none where it has no context length (< 0).
__device__ __forceinline__ int nodes_of(const int32_t* counts, int b, int T, int context) {
  const int n = counts ? min(max(counts[b], 0), T) : T;
  return context < 0 ? 0 : n;
}

// A paged cache [num_blocks][Hkv][block_size][D] and the block tables of its sequences.
struct Pages {
  const int32_t* bt;
  int64_t bts;
  int64_t num_blocks;
  int block_size, max_blocks, Hkv;
  // Row (D values) of head 0 at a sequence's slot, -1 where the table has no block for it;
  // head h is block_size rows further on for each h.
  __device__ __forceinline__ int64_t row(int b, int64_t slot) const {
    if (slot < 0 || slot >= (int64_t)max_blocks * block_size) return -1;
    const int i = (int)slot / block_size;
    const int blk = bt[(int64_t)b * bts + i];
    if (blk < 0 || blk >= num_blocks) return -1;
    return (int64_t)blk * Hkv * block_size + ((int)slot - i * block_size);
  }
};

}  // namespace grpo

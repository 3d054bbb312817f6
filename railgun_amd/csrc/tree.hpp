// What the kernels of a step over drafted tokens share.
#pragma once

#include "rg_common.hpp"

namespace rg {

// Nodes of a tree: their bits in 32 words.
constexpr int kMaxTreeNodes = 1024;

// Refuses max_nodes that no tree has.
int check_tree_nodes(const char* op, int32_t max_nodes);

struct Tree {
  int first, len, nodes;
};
// The nodes of sequence s: what cu_nodes says, held to the packed arrays (len) and to max_nodes (nodes).
__device__ __forceinline__ Tree tree_of(const int32_t* cu, int s, int num_nodes, int max_nodes) {
  const int first = max(0, min(cu[s], num_nodes)), last = max(first, min(cu[s + 1], num_nodes));
  return Tree{first, last - first, min(last - first, max_nodes)};
}

}  // namespace rg

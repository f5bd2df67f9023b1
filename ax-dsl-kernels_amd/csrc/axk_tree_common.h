// Trees of drafted tokens, as the paged attention and the Gated DeltaNet read them: parents[b, t], t < T <= 64, a node's
// parent before it, -1 for the last token of the history, -2 for no node.
#pragma once
#include "axk_common.h"

namespace axk_tree {

constexpr int kMaxNodes = 64;  // one 64-bit word of ancestors a node, one lane a node

// The nodes of a tree as its cache holds them: those up to the last that is one.
AXK_DEV int node_count(int parent) {
  const uint64_t there = __ballot(parent != -2);
  return there ? 64 - __builtin_clzll(there) : 0;
}

// A log decay g whose e^g is zero in 32 bits (-inf too): nothing of what came before it is left. Such a g stays out of sums over
// a branch, where -inf less -inf would be NaN and a huge one would swallow the others; what lies before the branch's last one has
// weight 0 instead. (Parents come before their children, so the last one of a branch has the highest index.)
AXK_DEV bool forgets(float g) { return g < -104.0f; }
AXK_DEV int last_of(uint64_t nodes) { return 63 - __builtin_clzll(nodes | 1); }

// Lane t: node t and its ancestors, by doubling the distance to the farthest known one; zero where t is no node. A parent
// that is no node before it makes t none, and sets *status. With SUM, x becomes its sum over the same nodes.
template <bool SUM>
AXK_DEV uint64_t ancestors_sum(int parent, int nodes, int* status, double& x) {
  const int lane = threadIdx.x & 63;
  const bool bad = parent < -2 || parent >= lane;
  int up = parent == -2 || bad ? -3 : parent;  // -1: beyond the root, -3: not in the tree
  uint64_t seen = 1ull << lane;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const int from = max(up, 0);
    const uint32_t lo = __shfl((uint32_t)seen, from), hi = __shfl((uint32_t)(seen >> 32), from);
    const int next = __shfl(up, from);
    double more = 0.0;
    if constexpr (SUM) more = __shfl(x, from);
    if (up >= 0) {
      seen |= ((uint64_t)hi << 32) | lo;
      up = next;
      x += more;
    }
  }
  if (parent != -2 && up != -1 && lane < nodes && status) *status = 1;
  return up == -1 ? seen : 0;
}
AXK_DEV uint64_t ancestors(int parent, int nodes, int* status) {
  double none = 0.0;
  return ancestors_sum<false>(parent, nodes, status, none);
}

}  // namespace axk_tree

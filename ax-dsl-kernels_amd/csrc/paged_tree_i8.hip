// paged_tree.h for a cache of this stored type (a file of its own, so that the three compile side by side).
#include "paged_tree.h"

namespace axk_tree {
int launch_i8(const TreeArgs& a, int d, int rb, hipStream_t st) { return launch_type<kI8>(a, d, rb, st); }
}  // namespace axk_tree

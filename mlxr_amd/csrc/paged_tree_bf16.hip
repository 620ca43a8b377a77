// Attention of drafted tokens instantiated for one pair of query and cache types (paged_tree.h).
#include "paged_tree.h"

namespace mlxr {
namespace tree {
TreeKern kern_bf16(int dim, int columns, int longest, int out_dtype) {
  return out_dtype == MLXR_F32 ? kern_of<false, false, 3>(dim, columns, longest) : kern_of<false, false, 2>(dim, columns, longest);
}
}  // namespace tree
}  // namespace mlxr

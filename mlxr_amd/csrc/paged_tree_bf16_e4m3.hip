// Attention of drafted tokens instantiated for one pair of query and cache types (paged_tree.h).
#include "paged_tree.h"

namespace mlxr {
namespace tree {
TreeKern kern_bf16_e4m3(int dim, int columns, int longest) { return kern_of<false, true>(dim, columns, longest); }
}  // namespace tree
}  // namespace mlxr

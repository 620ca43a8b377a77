// Decode attention instantiated for one pair of query and cache types (paged_attn.h).
#include "paged_attn.h"

namespace mlxr {
namespace paged {
AttnKern& kern_f16_e4m3(int dim, bool p8) { return kern_of<true, true>(dim, p8); }
}  // namespace paged
}  // namespace mlxr

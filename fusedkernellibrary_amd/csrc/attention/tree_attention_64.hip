// Attention kernels for heads of 64 elements.
#include "tree_attention.hpp"

namespace fkattn {
template int launch_attention<64>(const AttentionArgs&, const AttentionPlan&, void*, Launched&);
}

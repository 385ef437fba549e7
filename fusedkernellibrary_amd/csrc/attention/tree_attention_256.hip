// Attention kernels for heads of 256 elements.
#include "tree_attention.hpp"

namespace fkattn {
template int launch_attention<256>(const AttentionArgs&, const AttentionPlan&, void*, Launched&);
}

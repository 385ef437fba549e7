// Attention kernels for heads of 96 elements.
#include "tree_attention.hpp"

namespace fkattn {
template int launch_attention<96>(const AttentionArgs&, const AttentionPlan&, void*, Launched&);
}

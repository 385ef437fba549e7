// Attention kernels for heads of 192 elements.
#include "tree_attention.hpp"

namespace fkattn {
template int launch_attention<192>(const AttentionArgs&, const AttentionPlan&, void*, Launched&);
}

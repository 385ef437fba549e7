// Attention kernels for heads of 128 elements.
#include "tree_attention.hpp"

namespace fkattn {
template int launch_attention<128>(const AttentionArgs&, const AttentionPlan&, void*, Launched&);
}

// Attention kernels for heads of 96 elements.
#include "tree_attention.hpp"

namespace fkattn {
template <> int launch_attention<96>(const AttentionArgs& a, const AttentionPlan& plan, void* stream, Launched& info) { return start_attention<96, false>(a, plan, stream, info); }
}

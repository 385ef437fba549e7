// Attention kernels for heads of 192 elements.
#include "tree_attention.hpp"

namespace fkattn {
template <> int launch_attention<192>(const AttentionArgs& a, const AttentionPlan& plan, void* stream, Launched& info) { return start_attention<192, false>(a, plan, stream, info); }
}

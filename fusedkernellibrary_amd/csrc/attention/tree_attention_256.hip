// Attention kernels for heads of 256 elements.
#include "tree_attention.hpp"

namespace fkattn {
template <> int launch_attention<256>(const AttentionArgs& a, const AttentionPlan& plan, void* stream, Launched& info) { return start_attention<256, false>(a, plan, stream, info); }
}

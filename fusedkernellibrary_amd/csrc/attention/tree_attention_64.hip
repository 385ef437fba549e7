// Attention kernels for heads of 64 elements.
#include "tree_attention.hpp"

namespace fkattn {
template <> int launch_attention<64>(const AttentionArgs& a, const AttentionPlan& plan, void* stream, Launched& info) { return start_attention<64, false>(a, plan, stream, info); }
}

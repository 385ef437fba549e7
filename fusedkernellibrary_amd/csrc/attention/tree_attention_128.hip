// Attention kernels for heads of 128 elements.
#include "tree_attention.hpp"

namespace fkattn {
template <> int launch_attention<128>(const AttentionArgs& a, const AttentionPlan& plan, void* stream, Launched& info) { return start_attention<128, false>(a, plan, stream, info); }
}

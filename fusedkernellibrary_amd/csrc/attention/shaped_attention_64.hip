// Kernels of attention with scores of another shape, for heads of 64 elements.
#include "tree_attention.hpp"

namespace fkattn {
template <> int launch_attention<64>(const ShapedArgs& a, const AttentionPlan& plan, void* stream, Launched& info) { return start_attention<64, true>(a, plan, stream, info); }
}

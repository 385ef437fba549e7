// Kernels of attention with scores of another shape, for heads of 256 elements.
#include "tree_attention.hpp"

namespace fkattn {
template <> int launch_attention<256>(const ShapedArgs& a, const AttentionPlan& plan, void* stream, Launched& info) { return start_attention<256, true>(a, plan, stream, info); }
}

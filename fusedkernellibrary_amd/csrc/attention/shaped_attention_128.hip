// Kernels of attention with scores of another shape, for heads of 128 elements.
#include "tree_attention.hpp"

namespace fkattn {
template <> int launch_attention<128>(const ShapedArgs& a, const AttentionPlan& plan, void* stream, Launched& info) { return start_attention<128, true>(a, plan, stream, info); }
}

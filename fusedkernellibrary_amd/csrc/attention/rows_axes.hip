// rows_axes.hip -- norm and rotation of heads, and the quantising write, by positions of several axes (heads.hpp).
#include "heads.hpp"

namespace fkattn {
int launch_heads(const AxesHeadArgs& a, int type, bool to_cache, void* stream, Launched& info) { return start_heads_of_any_size<true>(a, type, to_cache, stream, info); }
}

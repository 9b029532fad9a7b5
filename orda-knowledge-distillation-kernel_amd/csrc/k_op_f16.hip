// k_op_f16.hip -- the projection's and the feed-forward block's kernels,
// instantiated for f16.
#include "op_kernels.hpp"

namespace orda {
ORDA_INSTANTIATE_OPS16(f16)
}  // namespace orda

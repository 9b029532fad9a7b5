// k_op_bf16.hip -- the projection's and the feed-forward block's kernels,
// instantiated for bf16.
#include "op_kernels.hpp"

namespace orda {
ORDA_INSTANTIATE_OPS16(bf16)
}  // namespace orda

// The attention kernels of f16 tensors with heads of 65 to 96 elements.
#include "attn.hpp"

namespace orda {
template hipError_t launch_attn<f16, 96>(const AttnParams&, AttnPass, hipStream_t);
}  // namespace orda

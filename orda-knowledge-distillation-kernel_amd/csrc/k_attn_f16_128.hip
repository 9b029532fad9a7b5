// The attention kernels of f16 tensors with heads of 97 to 128 elements.
#include "attn.hpp"

namespace orda {
template hipError_t launch_attn<f16, 128>(const AttnParams&, AttnPass, hipStream_t);
}  // namespace orda

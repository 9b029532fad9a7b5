// The attention kernels of bf16 tensors with heads of 97 to 128 elements.
#include "attn.hpp"

namespace orda {
template hipError_t launch_attn<bf16, 128>(const AttnParams&, AttnPass, hipStream_t);
}  // namespace orda

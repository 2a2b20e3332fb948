// Attention over f16 keys.
#include "attention_kernels.hpp"

namespace kvmem_hip {

template void launch_attention<KVMEM_TYPE_F16>(hipStream_t, int, uint32_t, const AttnPlan &, const AttnParams &);
template bool load_attention<KVMEM_TYPE_F16>();

}  // namespace kvmem_hip

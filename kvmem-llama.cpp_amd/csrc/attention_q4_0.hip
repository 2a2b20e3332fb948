// Attention over q4_0 keys.
#include "attention_kernels.hpp"

namespace kvmem_hip {

template void launch_attention<KVMEM_TYPE_Q4_0>(hipStream_t, int, uint32_t, const AttnPlan &, const AttnParams &);
template bool load_attention<KVMEM_TYPE_Q4_0>();

}  // namespace kvmem_hip

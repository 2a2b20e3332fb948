// Linear attention by chunks, rows of F16 (linear_chunk_kernels.hpp).
#include "linear_chunk_kernels.hpp"

namespace kvmem_hip {

void launch_linear_chunks_f16(hipStream_t stream, const ChunkParams &p) { launch_dims<_Float16>(stream, p); }

bool load_linear_chunks_f16() { return load_kernel_object(&linear_prepare_kernel<_Float16, 64, true>); }

}  // namespace kvmem_hip

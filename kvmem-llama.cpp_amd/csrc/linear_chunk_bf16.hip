// Linear attention by chunks, rows of BF16 (linear_chunk_kernels.hpp).
#include "linear_chunk_kernels.hpp"

namespace kvmem_hip {

void launch_linear_chunks_bf16(hipStream_t stream, const ChunkParams &p) { launch_dims<__bf16>(stream, p); }

bool load_linear_chunks_bf16() { return load_kernel_object(&linear_prepare_kernel<__bf16, 64, true>); }

}  // namespace kvmem_hip

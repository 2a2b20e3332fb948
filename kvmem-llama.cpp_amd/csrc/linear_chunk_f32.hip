// Linear attention by chunks, rows of F32 (linear_chunk_kernels.hpp).
#include "linear_chunk_kernels.hpp"

namespace kvmem_hip {

void launch_linear_chunks_f32(hipStream_t stream, const ChunkParams &p) { launch_dims<float>(stream, p); }

bool load_linear_chunks_f32() { return load_kernel_object(&linear_prepare_kernel<float, 64, true>); }

}  // namespace kvmem_hip

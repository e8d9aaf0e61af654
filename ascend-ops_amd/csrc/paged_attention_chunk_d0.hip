// Instantiations of the chunk attention kernels, two head sizes to a file so that the build is spread over the CPUs.
#include "paged_attention_chunk.h"

namespace aops {
template hipError_t chunk_launch<16>(const ChunkArgs&, hipStream_t);
template hipError_t chunk_launch<256>(const ChunkArgs&, hipStream_t);
}  // namespace aops

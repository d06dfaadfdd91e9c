#include "linear_chunk.cuh"

namespace jvpfa {
namespace linear {
template int launch_chunks<__half>(const Scan& s, bool outputs, cudaStream_t stream);
}  // namespace linear
}  // namespace jvpfa

#include "linear_chunk.cuh"

namespace jvpfa {
namespace linear {
template int launch_chunks<__half>(const Scan& s, bool outputs, cudaStream_t stream);
template int chunk_ctas<__half>(const Scan& s);
}  // namespace linear
}  // namespace jvpfa

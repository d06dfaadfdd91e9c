#include "linear_scan.cuh"

namespace jvpfa {
namespace linear {
template int launch_scan<float, true>(const Scan& s, cudaStream_t stream);
template int launch_scan<float, false>(const Scan& s, cudaStream_t stream);
}  // namespace linear
}  // namespace jvpfa

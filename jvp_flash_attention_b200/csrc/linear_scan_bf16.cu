#include "linear_scan.cuh"

namespace jvpfa {
namespace linear {
template int launch_scan<__nv_bfloat16, true>(const Scan& s, cudaStream_t stream);
template int launch_scan<__nv_bfloat16, false>(const Scan& s, cudaStream_t stream);
}  // namespace linear
}  // namespace jvpfa

#include "norm_bwd.cuh"

namespace jvpfa {
namespace norms {
template int launch_bwd<float>(const jvpfa_norm_args& a, const Cut& c, cudaStream_t s);
}  // namespace norms
}  // namespace jvpfa

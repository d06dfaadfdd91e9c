#include "norm_fwd.cuh"

namespace jvpfa {
namespace norms {
template int launch_fwd<__half>(const jvpfa_norm_args& a, cudaStream_t s);
}  // namespace norms
}  // namespace jvpfa

// Linear attention with a decay l for each head: what its kernels share.
//
// Everything is one causal map, linear in each of three sequences a, b (rows of D entries) and c (of E):
//   out_t = scale sum_{s <= t} l^(t-s) (a_t . b_s) c_s = scale a_t . M_t,   M_t = l M_{t-1} + b_t c_t^T.
// o is that of (q, k, v).  Its gradients are the same map again, dq that of (go, v, k), and with the rows in reverse order dk that of (v, go, q)
// and dv that of (k, q, go); a given state's cotangent is where the reverse M begins.  With tangents all of it holds for dual numbers: of
// (q + tq, k + tk, v + tv) the map's tangent is to, and the gradients of both outputs are value (dtq, dtk, dtv) and tangent (dq, dk, dv) of the maps
// whose cotangent is gto + go, gto the value and go the tangent.
//
// Rows are taken in chunks: within one, the products (a_t . b_s) are a small matrix, weighted by l^(t-s); what came before is M.
#pragma once
#include "common.cuh"

namespace jvpfa {
namespace linear {

constexpr int kSMs = 148;
constexpr float kLowest = -1e4f;  // a lower log_decay counts as this: nothing is left of earlier rows, and 0 * log_decay stays 0

struct Scan {
  int dtype, B, H, L, D, E;
  float scale;
  bool dual, reversed;
  const float* log_decay;
  const int32_t* lengths;
  jvpfa_linear_tensor a, b, c, ta, tb, tc, out, tout;
  // states before the first row and behind the last: entry (d, e) of head i at i * D * E + d * stride[0] + e * stride[1]
  const float *first, *tfirst;
  float *last, *tlast;
  long long first_stride[2], last_stride[2];
  float first_scale, last_scale;
  int ahead;       // the first row sees `first` l^ahead times
  int last_ahead;  // ... and `last` is M's behind the last row l^last_ahead times
  // a head's rows are cut into `segments` of `segment` rows; their states in the workspace, [head][segment][D * E], value and tangent apart,
  // entry (d, e) at d * state_stride[0] + e * state_stride[1]
  int segments, segment;
  float *states, *tstates;
  long long state_stride[2];
};

template <typename T>
int launch_chunks(const Scan& s, bool outputs, cudaStream_t stream);  // 16-bit types (linear_chunk.cuh)
int launch_scan(const Scan& s, bool outputs, cudaStream_t stream);    // float32 (linear_scan.cu)
// CTAs that an SM holds at once of those that form the outputs.
template <typename T>
int chunk_ctas(const Scan& s);
int scan_ctas(const Scan& s);

// Whether a tensor's rows are whole 16-byte pieces.
template <typename T>
bool wide_tensor(const jvpfa_linear_tensor& x, const Scan& s, int width) {
  uint64_t all = (uint64_t)width * sizeof(T) | reinterpret_cast<uint64_t>(x.p);
  const int counts[3] = {s.B, s.H, s.L};
  for (int d = 0; d < 3; ++d)
    if (counts[d] > 1) all |= (uint64_t)x.stride[d] * sizeof(T);
  return all % 16 == 0;
}

inline long long state_bytes(const Scan& s) { return s.segments > 1 ? 4ll * s.B * s.H * s.segments * s.D * s.E : 0; }

__device__ __forceinline__ float decay_of(const float* log_decay, int h) {
  const float w = log_decay ? log_decay[h] : 0.f;
  return w < kLowest ? kLowest : w;  // (a NaN stays one)
}
// l^n as by + keep, keep 1 or 0: next to 1 by its distance from it, which keeps the digits of slow decays, else as it is, which keeps those of
// what little is left.  M l^n + x is fma(M, by, fma(M, keep, x)).
struct Down {
  float by, keep;
};
__device__ __forceinline__ Down down_of(float power, float less1) { return less1 > -0.5f ? Down{less1, 1.f} : Down{power, 0.f}; }
__device__ __forceinline__ int length_of(const int32_t* lengths, int b, int L) { return lengths ? min(max(lengths[b], 0), L) : L; }

}  // namespace linear
}  // namespace jvpfa

// Norms with the residual sum, gate and modulation around them: what the kernels of value and tangent (norm_fwd) and of the gradients
// (norm_bwd) share.  With s = (mean((x - m)^2) + eps)^(-1/2) and n = s (x - m), m the row's mean or 0, the derivative of n is
//   J v = s (v - mean(v) - n mean(n v))                                  (mean(v) only where m is one)
// which is symmetric, so tangents and gradients are the same map:
//   tn = J tr;   of <g, n> + <h, tn>:   dtr = J h,   dr = J (g - s b h) - s (a tn + e n),   a = mean(n h), b = mean(n tr), e = mean(h tn).
// Around it stand sums and products by vectors: the gain G = weight (1 + scale) and the offset O = bias (1 + scale) + shift of a row's
// group, and the gain E = alpha gate post_weight of what is added.
#pragma once
#include "common.cuh"

namespace jvpfa {
namespace norms {

constexpr int kAtMost = 512;  // threads of a row: they may have 128 registers each

// Loads and stores of V entries at once.
template <typename T, int V>
struct Pack {
  static_assert(V == 1 || V * sizeof(T) == 16, "an entry, or 16 bytes");
  T e[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> r;
  if constexpr (V == 1)
    r.e[0] = *p;
  else
    *reinterpret_cast<uint4*>(r.e) = *reinterpret_cast<const uint4*>(p);
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_floats(T* p, const float* x) {
  Pack<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.e[i] = Elem<T>::from_float(x[i]);
  if constexpr (V == 1)
    *p = r.e[0];
  else
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(r.e);
}

// V entries of a vector in its own type, which is T or float; `wide` says that it can be read 16 bytes at a time.
template <typename T, int V>
__device__ __forceinline__ void load_vec(float* to, const void* v, long long at, bool f32, bool wide) {
  if (f32 || sizeof(T) == 4) {
    const float* p = static_cast<const float*>(v) + at;
    if (V > 1 && wide) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(p + i));
        to[i] = x.x, to[i + (V > 1)] = x.y, to[i + 2 * (V > 1)] = x.z, to[i + 3 * (V > 1)] = x.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) to[i] = __ldg(p + i);
    }
    return;
  }
  const T* p = static_cast<const T*>(v) + at;
  if (V > 1 && wide) {
    const Pack<T, V> x = load_pack<T, V>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) to[i] = Elem<T>::to_float(x.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) to[i] = Elem<T>::to_float(p[i]);
  }
}

struct Wide {  // which vectors can be read 16 bytes at a time, a bit for each (tangents from bit 8 on)
  uint32_t bits;
};

template <typename T, int V>
__device__ __forceinline__ bool vec_at(float* to, const jvpfa_norm_args& a, Wide wide, int which, bool tangent, long long group, int col) {
  const jvpfa_norm_vec& x = a.vec[which];
  const void* p = tangent ? x.tv : x.v;
  if (!p) return false;
  const long long at = (x.grouped ? group * (tangent ? x.tv_stride : x.stride) : 0) + col;
  load_vec<T, V>(to, p, at, a.vec_dtype == JVPFA_FP32, (wide.bits >> (which + (tangent ? 8 : 0))) & 1);
  return true;
}

// The gain and offset of n for V columns, and their tangents.
template <typename T, int V, bool TAN>
__device__ __forceinline__ void gain_of(const jvpfa_norm_args& a, Wide wide, long long group, int col, float* G, float* O, float* tG, float* tO) {
  float w[V], b[V], sc[V], x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sc[i] = 0.f, w[i] = 1.f, b[i] = 0.f;
  vec_at<T, V>(w, a, wide, JVPFA_VEC_WEIGHT, false, group, col);
  const bool has_b = vec_at<T, V>(b, a, wide, JVPFA_VEC_BIAS, false, group, col);
  vec_at<T, V>(sc, a, wide, JVPFA_VEC_SCALE, false, group, col);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    sc[i] += 1.f;
    G[i] = w[i] * sc[i], O[i] = has_b ? b[i] * sc[i] : 0.f;
  }
  if (vec_at<T, V>(x, a, wide, JVPFA_VEC_SHIFT, false, group, col)) {
#pragma unroll
    for (int i = 0; i < V; ++i) O[i] += x[i];
  }
  if constexpr (TAN) {
#pragma unroll
    for (int i = 0; i < V; ++i) tG[i] = tO[i] = 0.f;
    if (vec_at<T, V>(x, a, wide, JVPFA_VEC_WEIGHT, true, group, col)) {
#pragma unroll
      for (int i = 0; i < V; ++i) tG[i] = x[i] * sc[i];
    }
    if (vec_at<T, V>(x, a, wide, JVPFA_VEC_BIAS, true, group, col)) {
#pragma unroll
      for (int i = 0; i < V; ++i) tO[i] = x[i] * sc[i];
    }
    if (vec_at<T, V>(x, a, wide, JVPFA_VEC_SCALE, true, group, col)) {
#pragma unroll
      for (int i = 0; i < V; ++i) tG[i] += w[i] * x[i], tO[i] += b[i] * x[i];
    }
    if (vec_at<T, V>(x, a, wide, JVPFA_VEC_SHIFT, true, group, col)) {
#pragma unroll
      for (int i = 0; i < V; ++i) tO[i] += x[i];
    }
  }
}

// The gain of what is added, and its tangent.
template <typename T, int V, bool TAN>
__device__ __forceinline__ void gate_of(const jvpfa_norm_args& a, Wide wide, long long group, int col, float* E, float* tE) {
  float g[V], p[V], x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) g[i] = p[i] = 1.f;
  vec_at<T, V>(g, a, wide, JVPFA_VEC_GATE, false, group, col);
  vec_at<T, V>(p, a, wide, JVPFA_VEC_POST_WEIGHT, false, group, col);
#pragma unroll
  for (int i = 0; i < V; ++i) E[i] = a.alpha * g[i] * p[i];
  if constexpr (TAN) {
#pragma unroll
    for (int i = 0; i < V; ++i) tE[i] = 0.f;
    if (vec_at<T, V>(x, a, wide, JVPFA_VEC_GATE, true, group, col)) {
#pragma unroll
      for (int i = 0; i < V; ++i) tE[i] = a.alpha * x[i] * p[i];
    }
    if (vec_at<T, V>(x, a, wide, JVPFA_VEC_POST_WEIGHT, true, group, col)) {
#pragma unroll
      for (int i = 0; i < V; ++i) tE[i] += a.alpha * x[i] * g[i];
    }
  }
}

// Sums of K values over the threads of a row, which all of them receive, always added in the same order.  A row of one warp needs no shared
// memory; the others take turns with two buffers, so that one barrier a sum is enough: who writes a buffer again has passed the barrier of
// the sum between, which every reader of the first reached after its reading.
struct RowSum {
  float* buf;   // 2 * 8 * 32 floats
  int warps;    // of the row
  int turn = 0;
  template <int K>
  __device__ __forceinline__ void operator()(float (&x)[K]) {
    static_assert(K <= 8, "the buffers' rows");
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int k = 0; k < K; ++k) x[k] += __shfl_xor_sync(0xffffffffu, x[k], o);
    if (warps == 1) return;
    float* b = buf + turn * 256;
    turn ^= 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) b[k * 32 + warp] = x[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float v = lane < warps ? b[k * 32 + lane] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      x[k] = v;
    }
  }
};

// Entries that 16 bytes hold where everything can be read so, else 1.
inline int vector_entries(const jvpfa_norm_args& a) {
  const int size = a.dtype == JVPFA_FP32 ? 4 : 2;
  uint64_t all = (uint64_t)a.C * size;
  for (const void* p : {a.x, a.tx, a.y, a.ty, (const void*)a.r, (const void*)a.tr, (const void*)a.n, (const void*)a.tn, a.gr, a.gtr, a.gn,
                        a.gtn, (const void*)a.dx, (const void*)a.dtx, (const void*)a.dy, (const void*)a.dty})
    all |= reinterpret_cast<uint64_t>(p);
  if (a.M > 1) all |= (uint64_t)(a.x_stride | (a.tx ? a.tx_stride : 0) | (a.y ? a.y_stride : 0) | (a.ty ? a.ty_stride : 0)) * size;
  return all % 16 == 0 ? 16 / size : 1;
}

inline Wide wide_vectors(const jvpfa_norm_args& a) {
  Wide w{0};
  const int size = a.vec_dtype == JVPFA_FP32 ? 4 : 2;
  for (int i = 0; i < 6; ++i)
    for (int t = 0; t < 2; ++t) {
      const jvpfa_norm_vec& x = a.vec[i];
      const void* p = t ? x.tv : x.v;
      const uint64_t all = reinterpret_cast<uint64_t>(p) | (x.grouped ? (uint64_t)(t ? x.tv_stride : x.stride) * size : 0);
      if (p && all % 16 == 0) w.bits |= 1u << (i + 8 * t);
    }
  return w;
}

// CTAs of this size that an SM holds; asked once for each kernel and size.
template <typename K>
int resident(K kernel, int threads, int (&known)[33]) {
  int n = __atomic_load_n(&known[threads / 32], __ATOMIC_RELAXED);
  if (n) return n;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return 1;
  }
  __atomic_store_n(&known[threads / 32], n, __ATOMIC_RELAXED);
  return n;
}

constexpr int kSMs = 148;

}  // namespace norms
}  // namespace jvpfa

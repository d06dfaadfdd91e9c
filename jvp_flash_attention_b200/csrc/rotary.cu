// Rotary positions: every pair (a, b) of a row's entries is turned by the angle position * frequency,
//   (a', b') = amplitude * (a cos - b sin, a sin + b cos),
// up to four tensors (queries, keys, their tangents) in one launch.  The map is linear, so a tangent goes through it as it is, and the
// gradient is the transposed turn (`transposed`: the sine's sign).
//
// Angles.  position * frequency passes 10^6 radians in long contexts, where 32 bits leave no digit of the fraction of a turn that
// counts.  The product is formed in 64 bits as turns, its fraction is exact there, and only that is rounded to 32 bits
// (by at most 2^-26 turns, 9.4e-8 radians, as the fraction is within half a turn) for sincospif.
//
// What bounds it: memory, each tensor read and written once.  A thread takes the pairs of one row's 2 * 16 bytes and goes through
// several heads with the same cosines, so that their cost (a few 64-bit products, some 25 instructions for each pair) is shared.
// Measured on a B200: bf16 B4 H16 L8192 D128, four tensors of 134 MB, 170 us = 6.3 TB/s, 96 % of the measured copy; B4 H16 L2048 D64 26.5 us
// = 5.1 TB/s; fp32 B2 H8 L1023 D128 13.2 us = 5.1 TB/s; eight single tokens 2.7 us.  (Threads 64 / 128 / 256 of a CTA 169 / 170 / 199 us, heads
// whose loads are under way 2 / 4 / 8 179 / 170 / 178 us.)
#include "common.cuh"

namespace jvpfa {

namespace {

constexpr int kThreads = 128;
constexpr int kAtOnce = 4;  // heads whose loads a thread has in flight

template <int BYTES>
struct Piece;
template <>
struct Piece<16> { using type = uint4; };
template <>
struct Piece<4> { using type = uint32_t; };
template <>
struct Piece<2> { using type = uint16_t; };

template <typename T, int V>
union Vec {
  typename Piece<V * (int)sizeof(T)>::type raw;
  T e[V];
  __device__ Vec() {}
};

struct Groups {
  int first[5];  // blockIdx.y at which each tensor's groups of heads begin
  int heads;     // of a group
  int chunks, rot_chunks;
};

template <typename T, int V, bool NEIGHBOURS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ jvpfa_rotary_args a, const __grid_constant__ Groups gr) {
  const long long idx = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row = idx / gr.chunks;
  const int c = (int)(idx - row * gr.chunks);
  if (row >= (long long)a.B * a.L) return;
  const int b = (int)(row / a.L), l = (int)(row - (long long)b * a.L);
  int t = 0;
  while (t + 1 < a.n_tensors && (int)blockIdx.y >= gr.first[t + 1]) ++t;
  const jvpfa_rotary_tensor& x = a.t[t];
  const int h0 = ((int)blockIdx.y - gr.first[t]) * gr.heads, h1 = min(x.H, h0 + gr.heads);

  const bool turned = c < gr.rot_chunks;
  const int i = c * V;  // the chunk's first pair
  const int e0 = turned ? (NEIGHBOURS ? 2 * i : i) : 2 * a.n_freq + (c - gr.rot_chunks) * 2 * V;
  const int e1 = turned && !NEIGHBOURS ? a.n_freq + i : e0 + V;
  const bool both = e1 < a.D;  // (what is not turned may end after an odd number of pieces)
  float cs[V], sn[V];
  if (turned) {
    long long p = a.offset + l;
    if (a.positions) {
      const long long at = b * a.position_stride[0] + l * a.position_stride[1];
      p = a.position_bits == 64 ? static_cast<const long long*>(a.positions)[at] : static_cast<const int*>(a.positions)[at];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double turns = (double)p * (a.freq[i + j] * 0.15915494309189533577);
      sincospif((float)(2.0 * (turns - rint(turns))), &sn[j], &cs[j]);
      cs[j] *= a.amplitude;
      sn[j] *= a.transposed ? -a.amplitude : a.amplitude;
    }
  }
  const T* src = static_cast<const T*>(x.x) + b * x.x_stride[0] + l * x.x_stride[2];
  T* dst = static_cast<T*>(x.y) + b * x.y_stride[0] + l * x.y_stride[2];
  using Raw = typename Piece<V * (int)sizeof(T)>::type;
  for (int h = h0; h < h1; h += kAtOnce) {
    Vec<T, V> v[kAtOnce][2];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (h + k >= h1) break;
      const T* s = src + (h + k) * x.x_stride[1];
      v[k][0].raw = *reinterpret_cast<const Raw*>(s + e0);
      if (both) v[k][1].raw = *reinterpret_cast<const Raw*>(s + e1);
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (h + k >= h1) break;
      if (turned) {
        T* e[2] = {v[k][0].e, v[k][1].e};
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int ia = NEIGHBOURS ? 2 * j : j, ib = NEIGHBOURS ? 2 * j + 1 : V + j;
          const float fa = Elem<T>::to_float(e[ia / V][ia % V]), fb = Elem<T>::to_float(e[ib / V][ib % V]);
          e[ia / V][ia % V] = Elem<T>::from_float(fa * cs[j] - fb * sn[j]);
          e[ib / V][ib % V] = Elem<T>::from_float(fa * sn[j] + fb * cs[j]);
        }
      }
      T* d = dst + (h + k) * x.y_stride[1];
      *reinterpret_cast<Raw*>(d + e0) = v[k][0].raw;
      if (both) *reinterpret_cast<Raw*>(d + e1) = v[k][1].raw;
    }
  }
}

template <typename T, int V>
int launch(const jvpfa_rotary_args& a, cudaStream_t s) {
  Groups g;
  g.rot_chunks = a.n_freq / V;
  g.chunks = g.rot_chunks + (a.D - 2 * a.n_freq + 2 * V - 1) / (2 * V);
  const long long threads = (long long)a.B * a.L * g.chunks;
  const long long blocks = (threads + kThreads - 1) / kThreads;
  int most = 0;
  for (int t = 0; t < a.n_tensors; ++t) most = a.t[t].H > most ? a.t[t].H : most;
  // Heads of a thread: up to 8 while 6 CTAs remain for every SM, more while 12 do.  The first heads share what cosines cost, later ones
  // gain nothing and leave SMs idle at the end (us at heads: fp16 B3 L1330 D64, 12 and 4 heads, 15.6 at 1, 10.8 at 2; bf16 B1 H32 Hk8 L2048
  // D128 9.3 at 4, 8.4 at 8; B4 H16 L2048 D64 with tangents 26.5 at 8, 29.9 at 16).
  g.heads = 1;
  while (g.heads < most && blocks * a.n_tensors * ((most + 2 * g.heads - 1) / (2 * g.heads)) >= 148 * (g.heads < 8 ? 6 : 12)) g.heads *= 2;
  g.first[0] = 0;
  long long groups = 0;
  for (int t = 0; t < a.n_tensors; ++t) {
    groups += (a.t[t].H + g.heads - 1) / g.heads;
    if (groups > 65535) return JVPFA_ERR_TOO_LARGE;  // grid.y limit
    g.first[t + 1] = (int)groups;
  }
  if (blocks > 2147483647LL) return JVPFA_ERR_TOO_LARGE;
  const dim3 grid((unsigned)blocks, (unsigned)groups);
  if (a.interleaved)
    rotary_kernel<T, V, true><<<grid, kThreads, 0, s>>>(a, g);
  else
    rotary_kernel<T, V, false><<<grid, kThreads, 0, s>>>(a, g);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "rotary_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
}

}  // namespace

int launch_rotary(const jvpfa_rotary_args& a, cudaStream_t s) {
  // Entries of a piece: what divides the pairs, the head, every stride and every address.
  const int size = a.dtype == JVPFA_FP32 ? 4 : 2;
  uint64_t all = (uint64_t)a.n_freq | (uint64_t)a.D;
  for (int t = 0; t < a.n_tensors; ++t) {
    const jvpfa_rotary_tensor& x = a.t[t];
    all |= (reinterpret_cast<uint64_t>(x.x) | reinterpret_cast<uint64_t>(x.y)) / size;
    const bool counts[3] = {a.B > 1, x.H > 1, a.L > 1};  // (the stride of a single entry is nothing's)
    for (int d = 0; d < 3; ++d)
      if (counts[d]) all |= (uint64_t)x.x_stride[d] | (uint64_t)x.y_stride[d];
  }
  if (a.dtype == JVPFA_FP32) return all % 4 == 0 ? launch<float, 4>(a, s) : launch<float, 1>(a, s);
  const bool bf16 = a.dtype == JVPFA_BF16;
  if (all % 8 == 0) return bf16 ? launch<__nv_bfloat16, 8>(a, s) : launch<__half, 8>(a, s);
  if (all % 2 == 0) return bf16 ? launch<__nv_bfloat16, 2>(a, s) : launch<__half, 2>(a, s);
  return bf16 ? launch<__nv_bfloat16, 1>(a, s) : launch<__half, 1>(a, s);
}

}  // namespace jvpfa

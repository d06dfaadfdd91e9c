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

constexpr int kSMs = 148;

// V entries in 16 bytes.
template <typename T, int V>
struct alignas(16) Pack {
  static_assert(V * sizeof(T) == 16, "16 bytes");
  T e[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> r;
  *reinterpret_cast<uint4*>(r.e) = *reinterpret_cast<const uint4*>(p);
  return r;
}

// The first `count` of V entries of a vector in its own type, which is T or float, and zeros; `wide` says that all can be read, 16 bytes at a time.
template <typename T, int V>
__device__ __forceinline__ void load_vec(float* to, const void* v, long long at, int count, bool f32, bool wide) {
  if (f32 || sizeof(T) == 4) {
    const float* p = static_cast<const float*>(v) + at;
    if (wide) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(p + i));
        to[i] = x.x, to[i + 1] = x.y, to[i + 2] = x.z, to[i + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) to[i] = i < count ? __ldg(p + i) : 0.f;
    }
    return;
  }
  const T* p = static_cast<const T*>(v) + at;
  if (wide) {
    const Pack<T, V> x = load_pack<T, V>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) to[i] = Elem<T>::to_float(x.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) to[i] = i < count ? Elem<T>::to_float(p[i]) : 0.f;
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
  const int count = a.C - col;
  load_vec<T, V>(to, p, at, count, a.vec_dtype == JVPFA_FP32, count >= V && (wide.bits >> (which + (tangent ? 8 : 0)) & 1));
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

// The threads of a row: warps of a CTA that may hold several rows at once, each with a barrier of its own.
struct Team {
  int index, threads, tid;  // which row of the CTA's, its threads, this one's place among them
  __device__ __forceinline__ void sync() const {
    if (threads == 32)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "r"(threads) : "memory");
  }
};

// Sums of K values over the threads of a row, which all of them receive, always added in the same order.  In a warp, lanes first halve the values that
// they carry on (8 values in 9 shuffles instead of 40).  Warps take turns with two buffers, so that one barrier a sum is enough: who writes
// a buffer again has passed the barrier of the sum between, which every reader of the first reached after its reading.
struct RowSum {
  float* buf;  // of the row: 2 * 16 * 8 floats
  Team team;
  int turn = 0;
  template <int K>
  __device__ __forceinline__ void operator()(float (&x)[K]) {
    constexpr int P = K <= 2 ? 2 : 8;
    static_assert(K <= 8, "the buffers' rows");
    const int lane = threadIdx.x & 31, warps = team.threads >> 5;
    float v[P];
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = k < K ? x[k] : 0.f;
    int which = 0;
#pragma unroll
    for (int o = 16, n = P / 2; o > 0; o >>= 1) {
      if (n > 0) {
        const bool upper = lane & o;
        which = 2 * which + upper;
#pragma unroll
        for (int k = 0; k < n; ++k) {
          const float other = __shfl_xor_sync(0xffffffffu, upper ? v[k] : v[k + n], o);
          v[k] = (upper ? v[k + n] : v[k]) + other;
        }
        n /= 2;
      } else {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
      }
    }
    constexpr int kStride = 32 / P;  // lanes that hold the same value
    if (warps == 1) {
#pragma unroll
      for (int k = 0; k < K; ++k) x[k] = __shfl_sync(0xffffffffu, v[0], k * kStride);
      return;
    }
    float* b = buf + turn * 128;
    turn ^= 1;
    if (lane % kStride == 0) b[(team.tid >> 5) * P + which] = v[0];
    team.sync();
    // lane: value lane % P of warps lane / P, lane / P + 32 / P, ...
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16 * P; i += 32)
      if (i + lane < warps * P) sum += b[i + lane];
#pragma unroll
    for (int o = P; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int k = 0; k < K; ++k) x[k] = __shfl_sync(0xffffffffu, sum, k);
  }
};
constexpr int kSumFloats = 256;  // of a row's RowSum

// Rows of several tensors on their way into shared memory, `depth` rows ahead, 16 bytes at a time.  Thread t's entries are pieces t, t + threads,
// ... of each row.  ALIGNED: rows begin on 16 bytes, a thread fetches what it reads itself, and nobody waits for anybody.  RAGGED: rows begin
// anywhere; the aligned pieces that a row touches are fetched, and a thread takes its entries out of two neighbours.  DIRECT: rows that shared
// memory has no room for, or of more columns than a thread's 16 entries (with no tangents 32 in the forward) reach; read and written as they are.
enum Way { ALIGNED, RAGGED, DIRECT };
constexpr int kMostDepth = 4;
struct Source {
  const void* p;  // NULL: zeros
  long long stride;
};

template <typename T, int NC>
struct Pieces {
  static constexpr int V = 16 / (int)sizeof(T);
  uint32_t words[NC][4];
  __device__ __forceinline__ float at(int j, int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(words[j][i]);
    } else {
      const uint16_t h = (uint16_t)(words[j][i / 2] >> (i % 2 * 16));
      return Elem<T>::to_float(*reinterpret_cast<const T*>(&h));
    }
  }
};

// Eight words, shifted down by `bytes` (the same for all threads): the first four.
__device__ __forceinline__ void shifted(uint32_t (&to)[4], const uint4& a, const uint4& b, int bytes) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  const int bits = bytes % 4 * 8;
  switch (bytes / 4) {
    case 0:
#pragma unroll
      for (int i = 0; i < 4; ++i) to[i] = __funnelshift_r(w[i], w[i + 1], bits);
      break;
    case 1:
#pragma unroll
      for (int i = 0; i < 4; ++i) to[i] = __funnelshift_r(w[i + 1], w[i + 2], bits);
      break;
    case 2:
#pragma unroll
      for (int i = 0; i < 4; ++i) to[i] = __funnelshift_r(w[i + 2], w[i + 3], bits);
      break;
    default:
#pragma unroll
      for (int i = 0; i < 4; ++i) to[i] = __funnelshift_r(w[i + 3], i + 4 < 8 ? w[i + 4] : 0u, bits);
  }
}

template <typename T, int NC, Way WAY>
struct Rows {
  static constexpr int V = 16 / (int)sizeof(T), kSize = (int)sizeof(T);
  int C, M;
  Team team;
  bool wide;  // DIRECT: rows begin on 16 bytes

  __device__ __forceinline__ int piece(int j) const { return j * team.threads + team.tid; }
  // Whether entry i of piece j is one of the row's.
  __device__ __forceinline__ bool on(int j, int i) const { return piece(j) * V + (WAY == ALIGNED ? 0 : i) < C; }
  __device__ __forceinline__ static int offset(const T* row) { return WAY == RAGGED ? (int)(reinterpret_cast<uintptr_t>(row) & 15) : 0; }

  __device__ __forceinline__ void fetch(unsigned char* slot, const Source& s, int row) const {
    if (WAY == DIRECT || !s.p) return;
    const T* from = static_cast<const T*>(s.p) + row * s.stride;
    const int off = offset(from), pieces = (off + C * kSize + 15) / 16;
    const unsigned char* first = reinterpret_cast<const unsigned char*>(from) - off;
    if constexpr (WAY == ALIGNED) {
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int i = piece(j);
        if (i < pieces) cp_async16(slot + i * 16, first + i * 16, 16);
      }
    } else {
      // what a piece has beyond the tensor's first and last entry is not read
      const unsigned char* begin = static_cast<const unsigned char*>(s.p);
      const unsigned char* end = begin + ((long long)(M - 1) * s.stride + C) * kSize;
      for (int i = team.tid; i < pieces; i += team.threads) {
        const unsigned char* from16 = first + i * 16;
        if (from16 >= begin && from16 + 16 <= end) {
          cp_async16(slot + i * 16, from16, 16);
        } else {
          for (int k = 0; k < 16; k += kSize)
            if (from16 + k >= begin && from16 + k + kSize <= end) *reinterpret_cast<T*>(slot + i * 16 + k) = *reinterpret_cast<const T*>(from16 + k);
        }
      }
    }
  }
  __device__ __forceinline__ void read(Pieces<T, NC>& to, const unsigned char* slot, const Source& s, int row) const {
    const T* from = static_cast<const T*>(s.p) + row * s.stride;
    const int off = offset(from);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) to.words[j][i] = 0u;
      const int at = piece(j), left = C - at * V;
      if (!s.p || left <= 0) continue;
      if constexpr (WAY == DIRECT) {
        if (wide) {
          const uint4 a = *reinterpret_cast<const uint4*>(from + at * V);
          to.words[j][0] = a.x, to.words[j][1] = a.y, to.words[j][2] = a.z, to.words[j][3] = a.w;
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            if (i >= left) continue;
            if constexpr (kSize == 4)
              to.words[j][i] = reinterpret_cast<const uint32_t*>(from)[at * V + i];
            else
              to.words[j][i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(from)[at * V + i] << (i % 2 * 16);
          }
        }
      } else {
        const uint4 a = *reinterpret_cast<const uint4*>(slot + at * 16);
        if constexpr (WAY == ALIGNED) {
          to.words[j][0] = a.x, to.words[j][1] = a.y, to.words[j][2] = a.z, to.words[j][3] = a.w;
        } else {
          const uint4 b = *reinterpret_cast<const uint4*>(slot + at * 16 + 16);
          shifted(to.words[j], a, b, off);
          // what is behind the row's end is zero
          if (left < V) {
            constexpr int per = 4 / kSize;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (i * per >= left)
                to.words[j][i] = 0u;
              else if (per == 2 && 2 * i + 1 >= left)
                to.words[j][i] &= 0xffffu;
            }
          }
        }
      }
    }
  }
  // A vector of 32 bits in shared memory: four entries of each piece, then the next four of each, so that neighbours read neighbouring 16 bytes.
  __device__ __forceinline__ float* place(float* vector, int piece_, int i) const { return vector + (i / 4 * ((C + V - 1) / V) + piece_) * 4; }
  __device__ __forceinline__ void vector(float* to, float* from, int j) const {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(place(from, piece(j), i));
      to[i] = x.x, to[i + 1] = x.y, to[i + 2] = x.z, to[i + 3] = x.w;
    }
  }
  // x: V entries of each piece.  RAGGED ones go through `slot`, which nobody may still be reading.
  __device__ __forceinline__ void write(void* p, int row, const float* x, unsigned char* slot) const {
    if (!p) return;
    T* to = static_cast<T*>(p) + (long long)row * C;
    uint4 raw[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      Pack<T, V> r;
#pragma unroll
      for (int i = 0; i < V; ++i) r.e[i] = Elem<T>::from_float(x[j * V + i]);
      raw[j] = *reinterpret_cast<const uint4*>(r.e);
    }
    if constexpr (WAY != RAGGED) {
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        if (WAY == ALIGNED || wide) {
          if (on(j, 0)) *reinterpret_cast<uint4*>(to + piece(j) * V) = raw[j];
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (on(j, i)) to[piece(j) * V + i] = Elem<T>::from_float(x[j * V + i]);
        }
      }
    } else {
      const int off = offset(to), bytes = C * kSize;
#pragma unroll
      for (int j = 0; j < NC; ++j)
        if (on(j, 0)) *reinterpret_cast<uint4*>(slot + 16 + piece(j) * 16) = raw[j];
      team.sync();
      unsigned char* first = reinterpret_cast<unsigned char*>(to) - off;
      for (int i = team.tid; i * 16 < off + bytes; i += team.threads) {
        // bytes i * 16 - off .. + 15 of the row, which stands 16 bytes into the slot
        if (i * 16 >= off && i * 16 + 16 <= off + bytes) {
          const uint4 a = *reinterpret_cast<const uint4*>(slot + i * 16), b = *reinterpret_cast<const uint4*>(slot + i * 16 + 16);
          uint32_t w[4];
          if (off)
            shifted(w, a, b, 16 - off);
          else
            w[0] = b.x, w[1] = b.y, w[2] = b.z, w[3] = b.w;
          *reinterpret_cast<uint4*>(first + i * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
          for (int k = 0; k < 16; k += kSize) {
            const int at = i * 16 + k - off;
            if (at >= 0 && at < bytes) *reinterpret_cast<T*>(first + i * 16 + k) = *reinterpret_cast<const T*>(slot + 16 + at);
          }
        }
      }
    }
  }
};

__device__ __forceinline__ void wait_rows(int depth) {  // for the oldest of `depth` groups
  if (depth == 1)
    cp_async_wait<0>();
  else if (depth == 2)
    cp_async_wait<1>();
  else if (depth == 3)
    cp_async_wait<2>();
  else
    cp_async_wait<3>();
}

// How a launch is laid out: threads of a row, rows of a CTA at once, rows ahead, the shared memory of a row and of a CTA, CTAs of an SM.
struct Layout {
  int threads, teams, depth, slot, team_bytes, bytes, ctas;
};
// `tensors` read and `written`; `parts` of a CTA's sums where several rows share it; `vectors` of 32 bits that it keeps.  Where no row fits, depth is 0.
// As many rows at once as the registers allow: a row alone waits for its sums most of the time.
inline Layout layout_of(const jvpfa_norm_args& a, Way way, int entries, int most_threads, int registers, int tensors, int written, int parts, int vectors) {
  const int size = a.dtype == JVPFA_FP32 ? 4 : 2;
  Layout l;
  l.threads = (a.C + entries * 32 - 1) / (entries * 32) * 32;
  l.slot = way == DIRECT ? 0 : (a.C * size + 15) / 16 * 16 + (way == RAGGED ? 32 : 0);
  const int of_sm = (a.M + kSMs - 1) / kSMs, rows = of_sm < a.group_rows ? of_sm : a.group_rows;
  l.teams = most_threads / l.threads;
  if (l.teams > 15) l.teams = 15;  // (16 barriers, one of them the CTA's)
  if (l.teams > rows) l.teams = rows;
  if (l.teams < 1) l.teams = 1;
  for (;; --l.teams) {
    l.ctas = 65536 / ((registers + 7) / 8 * 8 * l.threads * l.teams);
    if (l.ctas > (of_sm + l.teams - 1) / l.teams) l.ctas = (of_sm + l.teams - 1) / l.teams;
    if (l.ctas > 16) l.ctas = 16;
    if (l.ctas < 1) l.ctas = 1;
    for (; l.ctas >= 1; --l.ctas)
      for (l.depth = way == DIRECT ? 1 : kMostDepth; l.depth >= 1; --l.depth) {
        l.team_bytes = kSumFloats * 4 + (l.depth * tensors + (way == RAGGED ? written : 0)) * l.slot;
        l.bytes = l.teams * l.team_bytes + ((l.teams > 1 ? parts : 0) + vectors) * ((a.C + 7) / 8 * 8) * 4;
        if (l.bytes + 1024 <= 226 * 1024 / l.ctas) return l;
      }
    if (l.teams == 1) return l;
  }
}

// A kernel's registers, asked for once.
template <typename K>
int registers_of(K kernel, int& known) {
  int n = __atomic_load_n(&known, __ATOMIC_RELAXED);
  if (n) return n;
  cudaFuncAttributes at;
  if (cudaFuncGetAttributes(&at, reinterpret_cast<const void*>(kernel)) != cudaSuccess) {
    cudaGetLastError();
    return 128;
  }
  __atomic_store_n(&known, at.numRegs, __ATOMIC_RELAXED);
  return at.numRegs;
}

// Whether all rows begin on 16 bytes and are whole pieces of 16.
inline bool aligned_rows(const jvpfa_norm_args& a) {
  const int size = a.dtype == JVPFA_FP32 ? 4 : 2;
  uint64_t all = (uint64_t)a.C * size;
  for (const void* p : {a.x, a.tx, a.y, a.ty, (const void*)a.r, (const void*)a.tr, (const void*)a.n, (const void*)a.tn, a.gr, a.gtr, a.gn,
                        a.gtn, (const void*)a.dx, (const void*)a.dtx, (const void*)a.dy, (const void*)a.dty})
    all |= reinterpret_cast<uint64_t>(p);
  if (a.M > 1) all |= (uint64_t)(a.x_stride | (a.tx ? a.tx_stride : 0) | (a.y ? a.y_stride : 0) | (a.ty ? a.ty_stride : 0)) * size;
  return all % 16 == 0;
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

// The sums over a group's rows that the vectors' gradients are made of, by their place in the workspace.
enum Part { PG, PO, PE, PtG, PtO, PtE, kParts };  // of gn n + gtn tn, gn, dr N + dtr tN, gtn n, gtn, dtr N

struct Cut {
  int groups, slices;  // of each group's rows
  uint32_t parts;      // which sums are wanted, a bit for each
  int n_parts;
};

}  // namespace norms
}  // namespace jvpfa

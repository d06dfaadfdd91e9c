// What the gated projection's sources share: the activations with their first two derivatives, and the launch of its matrix products.
#pragma once

#include "f32_tc5_common.cuh"

namespace jvpfa {

__device__ __forceinline__ float fast_exp(float x) { return tc5::fast_exp2(x * kLog2e); }

// An activation's value and first two derivatives at g.  EXACT: to fp32's last places, for fp32 tensors; else by the fast exponential and
// reciprocal (off by less than 2^-17 (1 + |g|); 16-bit results are rounded by 2^-9 or 2^-12).  What a caller does not use of the three
// is not computed.
struct Activated {
  float a, d1, d2;
};
// sigmoid(x) and sigmoid(-x), each with its own relative precision: neither is one minus the other.
// (exp(-|x|) cannot overflow, and NaN stays NaN.)
template <bool EXACT>
__device__ __forceinline__ void sigmoids(float x, float& s, float& r) {
  const float e = EXACT ? expf(-fabsf(x)) : fast_exp(-fabsf(x));
  const float big = EXACT ? 1.f / (1.f + e) : __fdividef(1.f, 1.f + e), small = e * big;
  s = x >= 0.f ? big : small;
  r = x >= 0.f ? small : big;
}
// What a decaying factor multiplies: the gate itself up to 32, where that factor has long been zero (gelu: exp(-512); its tanh form: below
// exp(-2000)).  Powers of the gate stay finite, so that zero times one is zero: all finite gates have the limits of a, a' and a''.
__device__ __forceinline__ float within(float g) { return fminf(fmaxf(g, -32.f), 32.f); }
template <int KIND, bool EXACT>
__device__ __forceinline__ Activated activate(float g) {
  Activated y;
  if constexpr (KIND == JVPFA_ACT_SILU || KIND == JVPFA_ACT_SIGMOID) {
    float s, r;
    sigmoids<EXACT>(g, s, r);
    const float d = s * r;
    if constexpr (KIND == JVPFA_ACT_SIGMOID) {
      y.a = s, y.d1 = d, y.d2 = d * (r - s);
    } else {
      y.a = g * s, y.d1 = s + g * d, y.d2 = d * (2.f + g * (r - s));
    }
  } else if constexpr (KIND == JVPFA_ACT_GELU) {
    const float p = normcdff(g), d = 0.3989422804014327f * (EXACT ? expf(-0.5f * g * g) : fast_exp(-0.5f * g * g));
    const float w = within(g);
    y.a = g * p, y.d1 = p + w * d, y.d2 = d * (2.f - w * w);
  } else {
    // 0.5 (1 + tanh z) = sigmoid(2 z), z = c (g + c3 g^3)
    constexpr float c = 0.7978845608028654f, c3 = 0.044715f;
    float s, r;
    sigmoids<EXACT>(2.f * c * (g + c3 * g * g * g), s, r);
    const float w = within(g), z1 = 2.f * c * (1.f + 3.f * c3 * w * w), z2 = 12.f * c * c3 * w, d = s * r;
    y.a = g * s, y.d1 = s + w * d * z1, y.d2 = d * (2.f * z1 + w * (z2 + (r - s) * z1 * z1));
  }
  return y;
}
// f with the activation as a constant: the choice is made once for a block of entries, not for each (32 copies of all four in a row
// are more instructions than the cache next to the SM holds, and a short call spends its time fetching them).
template <int K>
struct Kind {
  static constexpr int value = K;
};
template <typename F>
__device__ __forceinline__ void with_activation(int kind, F f) {
  switch (kind) {
    case JVPFA_ACT_SILU: f(Kind<JVPFA_ACT_SILU>{}); break;
    case JVPFA_ACT_SIGMOID: f(Kind<JVPFA_ACT_SIGMOID>{}); break;
    case JVPFA_ACT_GELU: f(Kind<JVPFA_ACT_GELU>{}); break;
    default: f(Kind<JVPFA_ACT_GELU_TANH>{}); break;
  }
}

// ---- the projections that a backward reads --------------------------------------------------------------------------------
// g and u (with a tangent tg and tu) in the form in which the forward's threads hold them, a row each: blocks of 32 rows x 32 features,
// of each block the tensors one after another, of each tensor pieces of 16 bytes of a row, row by row, so that a warp writes 512
// contiguous bytes.  16-bit tensors keep 24 bits of an entry, its upper 16 (fp32's sign, exponent and 7 bits) and then the next 8: kept in
// 16 bits g and u would be the largest part of the gradients' error (bf16, of their norm: 3.1e-3 instead of 2.3e-3; rounding
// the result alone is 1.7e-3), in 32 a third more memory.  Cut, not rounded: 2^-16 at most, and nothing can carry into an infinity's
// or NaN's exponent.
template <typename T>
struct Kept {
  static constexpr int kEntry = sizeof(T) == 4 ? 4 : 3;
  static constexpr int kBlock = 32 * 32 * kEntry;  // bytes of a block of one tensor
  static constexpr int kPiece = 16 / (sizeof(T) == 4 ? 4 : 2);
};
__host__ __device__ inline int64_t kept_bytes(int dtype, int64_t rows, int64_t cols, bool tangent) {
  return (rows + 31) / 32 * ((cols + 31) / 32) * (tangent ? 4 : 2) * 32 * 32 * (dtype == JVPFA_FP32 ? 4 : 3);
}
// N entries of row `lane` of a tensor's block, from feature `first` of the block on.
template <typename T, int N>
__device__ __forceinline__ void keep(uint8_t* block, int lane, int first, const float (&v)[N]) {
  constexpr int P = Kept<T>::kPiece;
#pragma unroll
  for (int c = 0; c < N / P; ++c) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < P; ++j) w[j] = __float_as_uint(v[c * P + j]);
    uint8_t* at = block + (first / P + c) * 512 + lane * 16;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      *reinterpret_cast<uint4*>(at) = make_uint4(__byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632),
                                                 __byte_perm(w[4], w[5], 0x7632), __byte_perm(w[6], w[7], 0x7632));
      auto four = [&](int k) { return __byte_perm(__byte_perm(w[k], w[k + 1], 0x51), __byte_perm(w[k + 2], w[k + 3], 0x51), 0x5410); };
      *reinterpret_cast<uint2*>(block + 2048 + (first / P + c) * 256 + lane * 8) = make_uint2(four(0), four(4));
    }
  }
}
// One entry.
template <typename T>
__device__ __forceinline__ void keep_entry(uint8_t* block, int row, int f, float v) {
  constexpr int P = Kept<T>::kPiece;
  const uint32_t w = __float_as_uint(v);
  uint8_t* at = block + f / P * 512 + row * 16;
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<uint32_t*>(at)[f % P] = w;
  } else {
    reinterpret_cast<uint16_t*>(at)[f % P] = (uint16_t)(w >> 16);
    block[2048 + f / P * 256 + row * 8 + f % P] = (uint8_t)(w >> 8);
  }
}
// Piece `c` of row `row` of a tensor's block.
template <typename T>
__device__ __forceinline__ void kept_piece(const uint8_t* block, int row, int c, float (&v)[Kept<T>::kPiece]) {
  const uint4 x = *reinterpret_cast<const uint4*>(block + c * 512 + row * 16);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(w[j]);
  } else {
    const uint2 y = *reinterpret_cast<const uint2*>(block + 2048 + c * 256 + row * 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t low = j < 4 ? y.x : y.y;
      // byte j of the lower bytes under the upper half
      v[j] = __uint_as_float(__byte_perm(__byte_perm(low, 0, 0x4404 | (j & 3) << 4), w[j >> 1], j & 1 ? 0x7610 : 0x5410));
    }
  }
}

namespace tc5 {

// A matrix product of the pair kernel (gated_gemm.cu): result tiles of 256 rows x 256 columns, and the operands it is summed from.
enum PairKind {
  kPairGated = 0,      // x (wg | wu)^T, the gate, and h
  kPairGatedDual = 1,  // ... with x's tangent, and th
  kPairDx = 2,         // A contiguous along the contraction, B across it
  kPairDw = 3          // both across it
};
struct PairMaps {
  CUtensorMap a[4], b[2];  // product: a[2 * group + source], b[source]; gated: a = x, tx, b = wg, wu
};
struct PairArgs {
  int groups, rows, cols;            // of the result: `groups` matrices (gated: 1) of rows x cols
  int depth, sources;                // each is a sum over `sources` products of this depth
  int kblocks, pairs, steps;         // ceil(depth / 64); 1, or 6 products of bf16 parts (fp32); k-blocks of a tile
  int chunk;                         // k-blocks summed on the tensor cores before the sum goes on in registers
  int tiles_m, tiles_n, band;        // tiles of a group, and how many rows of tiles are gone through together
  int whole, items;                  // tiles that are computed whole, and what clusters take up: these, then pieces of the others
  int cut, piece;                    // pieces of a tile, and their k-blocks
  float* partial;                    // 256 x 256 sums of each piece
  void* out[2];
  void *h, *th;                      // gated
  uint8_t* kept;
  int activation;
  bool aligned;                      // rows of the result are whole 16-byte pieces
  int* status;
};
// Fills in what follows from the first two lines; workspace() bytes of scratch for `partial`.
int plan_pair(int dtype, int kind, PairArgs& p);
int64_t pair_workspace(const PairArgs& p);
int launch_pair(int dtype, int kind, const PairArgs& p, const PairMaps& maps, cudaStream_t s);

// A product of few rows with the weights (gated_few.cu).
enum FewKind {
  kFewGated = 0,  // x (wg | wu)^T, the gate, h and with a second group th
  kFewDx = 1      // dx, and as a second group dtx
};
struct FewMaps {
  CUtensorMap w[2];     // wg, wu (16-bit types)
  CUtensorMap rows[4];  // gated: x, tx; dx: [2 * group + source], source 0 the gate's cotangents, 1 the other's
};
struct FewArgs {
  int groups, rows;          // 1 or 2 groups (value, tangent) of so many rows
  int features, width;       // of the weights: rows F, columns K
  const void *wg, *wu;       // fp32: read as they are
  int64_t wg_stride, wu_stride;
  bool pieces;               // ... and in whole 16-byte pieces
  int padded, kblocks, steps, tiles, stages, tmem_columns;
  int first, whole, cluster;  // tiles from `first` on; those of whole rounds, one CTA each; CTAs of each of the others
  void *out[2], *h, *th;
  uint8_t* kept;
  int activation;
  int* status;
};
// Fills in what follows from groups, rows, features and width; false: too many rows for these kernels.
bool plan_few(int dtype, int kind, FewArgs& p);
int launch_few(int dtype, int kind, const FewArgs& p, const FewMaps& maps, cudaStream_t s);
int device_sms();  // of the current device
constexpr int kMaxSteps = 1 << 20;  // k-blocks of one sum on the tensor cores
// The map of a (planes of) row-major matrix: boxes of 64 columns x box_rows rows.
bool encode_matrix(CUtensorMap* m, int dtype, const void* ptr, int rows, int cols, int64_t stride, int planes, int box_rows);

}  // namespace tc5
}  // namespace jvpfa

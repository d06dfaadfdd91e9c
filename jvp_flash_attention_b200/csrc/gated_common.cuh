// What the gated projection's sources share: the activations with their first two derivatives, and the launch of its matrix products.
#pragma once

#include "f32_tc5_common.cuh"

namespace jvpfa {

// a, a' and a'' at g.  EXACT: to fp32's last places, for fp32 tensors; else by the fast exponential and division (relative error
// below 2^-18 of the sigmoid for |g| < 64, 2^-9 being what a bf16 result is rounded by, 2^-12 an fp16 one).
struct Activated {
  float a, d1, d2;
};
// sigmoid(x) and sigmoid(-x), each with its own relative precision: neither is one minus the other.
template <bool EXACT>
__device__ __forceinline__ void sigmoids(float x, float& s, float& r) {
  const float e = EXACT ? expf(-fabsf(x)) : __expf(-fabsf(x));
  const float big = EXACT ? 1.f / (1.f + e) : __fdividef(1.f, 1.f + e), small = e * big;
  s = x >= 0.f ? big : small;
  r = x >= 0.f ? small : big;
}
template <bool EXACT>
__device__ __forceinline__ Activated activate(int kind, float g) {
  Activated y;
  if (kind == JVPFA_ACT_SILU || kind == JVPFA_ACT_SIGMOID) {
    float s, r;
    sigmoids<EXACT>(g, s, r);
    const float d = s * r;
    if (kind == JVPFA_ACT_SIGMOID) {
      y.a = s, y.d1 = d, y.d2 = d * (r - s);
    } else {
      y.a = g * s, y.d1 = s + g * d, y.d2 = d * (2.f + g * (r - s));
    }
  } else if (kind == JVPFA_ACT_GELU) {
    const float p = normcdff(g), d = 0.3989422804014327f * (EXACT ? expf(-0.5f * g * g) : __expf(-0.5f * g * g));
    y.a = g * p, y.d1 = p + g * d, y.d2 = d * (2.f - g * g);
  } else {
    // 0.5 (1 + tanh z) = sigmoid(2 z), z = c (g + c3 g^3)
    constexpr float c = 0.7978845608028654f, c3 = 0.044715f;
    float s, r;
    sigmoids<EXACT>(2.f * c * (g + c3 * g * g * g), s, r);
    const float z1 = 2.f * c * (1.f + 3.f * c3 * g * g), z2 = 12.f * c * c3 * g, d = s * r;
    y.a = g * s, y.d1 = s + g * d * z1, y.d2 = d * (2.f * z1 + g * (z2 + (r - s) * z1 * z1));
  }
  return y;
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
  int kblocks, pairs;                // ceil(depth / 64); 1, or 6 products of bf16 parts (fp32)
  int chunk, steps;                  // k-blocks summed on the tensor cores before the sum goes on in registers, of `steps` a tile
  int tiles_m, tiles_n, tiles;       // tiles of a group, and of all
  void* out[2];
  void *h, *th, *g, *u, *tg, *tu;    // gated
  int activation;
  int* status;
};
int launch_pair(int dtype, int kind, PairArgs& p, const PairMaps& maps, cudaStream_t s);
// The map of a (planes of) row-major matrix: boxes of 64 columns x box_rows rows.
bool encode_matrix(CUtensorMap* m, int dtype, const void* ptr, int rows, int cols, int64_t stride, int planes, int box_rows);

}  // namespace tc5
}  // namespace jvpfa

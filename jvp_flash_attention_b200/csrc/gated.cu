// The gated projection: its launches, and what they need besides the matrix products of gated_gemm.cu.
//
// Forward: one launch (value, or value and tangent).  Backward: a pass that turns the cotangents into those of the projections,
//   dg = gh a' u + gth (a'' tg u + a' tu),  du = gh a + gth a' tg,  dtg = gth a' u,  dtu = gth a,
// bound by memory (12 bytes an entry for the value of a 16-bit tensor: gh, 3 each for g and u, dg, du), then a product over the features for dx and dtx, and one over
// the rows for dwg and dwu.  Tangents are further rows of the first (dx beside dtx, the weights shared) and further depth of the second.
// The pass, measured on a B200: bf16 M8192 F11008 171 us = 6.3 TB/s, with tangents (24 bytes an entry) M8192 F2736 86 us = 6.2; rows that are no whole
// pieces, fp16 M3990 F2731, 24.5 us instead of 20.5.
//
// dg, du, dtg and dtu are rounded to the tensors' type, which is that of the tensor cores' operands: as two 16-bit parts each they would double both
// products.  The error of a whole bf16 backward is 2.3e-3 of the norm with it and 1.7e-3 without (rounding the results alone), fp16's 2.9e-4 and 2.1e-4; a
// cotangent beyond fp16's 65504 is infinite, below 2^-25 it is zero.
//
// Up to 128 rows (value and tangent together) the forward and dx are the kernels of gated_few.cu.
//
// Operands go to the tensor cores by TMA, which takes rows of whole 16-byte pieces; others are copied once into the workspace with padded
// rows.  fp32 operands become three planes of bf16 parts there (f32_tc5_common.cuh): both weights of K4096 F11008 152 us = 5.9 TB/s.
#include <algorithm>
#include <initializer_list>

#include "gated_common.cuh"

namespace jvpfa {

using namespace tc5;

namespace {

constexpr int kThreads = 256;

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T e[V];
};

// ---- operands as TMA takes them ------------------------------------------------------------------------------------------
// rows x cols, row stride `stride`, into rows of up8(cols); fp32: into three planes of bf16 parts.  All of a call's in one launch.
struct StageItem {
  const void* src;
  void* dst;
  int rows, cols;
  long long stride;
};
struct StageArgs {
  StageItem item[4];
};

template <typename T, int V>
__device__ __forceinline__ void stage_matrix(const StageItem& m) {
  const int width = (m.cols + 7) / 8 * 8;
  const int per_row = (m.cols + V - 1) / V;
  const long long step = (long long)gridDim.x * kThreads, plane = (long long)m.rows * width;
  long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  long long r = i / per_row;
  int c = (int)(i - r * per_row);
  const long long step_r = step / per_row;
  const int step_c = (int)(step - step_r * per_row);
  for (; r < m.rows; r += step_r, c += step_c) {
    if (c >= per_row) {
      c -= per_row;
      if (++r >= m.rows) break;
    }
    const Pack<T, V> x = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(m.src) + r * m.stride + c * V);
    if constexpr (sizeof(T) == 4) {
      Pack<__nv_bfloat16, V> part[3];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float h, mid, l;
        split3(x.e[j], h, mid, l);
        part[0].e[j] = __float2bfloat16_rn(h), part[1].e[j] = __float2bfloat16_rn(mid), part[2].e[j] = __float2bfloat16_rn(l);
      }
      __nv_bfloat16* d = static_cast<__nv_bfloat16*>(m.dst) + r * width + c * V;
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<Pack<__nv_bfloat16, V>*>(d + k * plane) = part[k];
    } else {
      *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(m.dst) + r * width + c * V) = x;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) stage_kernel(const __grid_constant__ StageArgs a) {
  constexpr int V = 16 / sizeof(T);
  const StageItem& m = a.item[blockIdx.y];
  if (reinterpret_cast<uint64_t>(m.src) % 16 == 0 && m.cols % V == 0 && m.stride % V == 0)
    stage_matrix<T, V>(m);
  else
    stage_matrix<T, 1>(m);
}

// A matrix as the products read it: in place, or in the workspace.
struct Matrix {
  const void* src;
  int rows, cols;
  int64_t stride;  // of src
  int64_t at = -1; // bytes into the workspace
  const void* ptr = nullptr;
  int64_t width;
  int planes;

  Matrix(int dtype, const void* p, int rows_, int cols_, int64_t stride_)
      : src(p), rows(rows_), cols(cols_), stride(rows_ == 1 ? up8(cols_) : stride_), ptr(p), width(stride), planes(dtype == JVPFA_FP32 ? 3 : 1) {}
  // Takes a place in the workspace where it cannot be read in place.
  void use(int64_t& workspace) {
    if (!src) return;
    const bool in_place = planes == 1 && reinterpret_cast<uint64_t>(src) % 16 == 0 && width % 8 == 0 && width >= cols && width < 1ll << 38;
    if (in_place) return;
    at = workspace;
    width = up8(cols);
    workspace += up256(2 * planes * width * rows);
  }
  // Its place in the workspace, and what has to be copied there.
  void put(void* workspace, StageArgs& stage, int& n) {
    if (at < 0) return;
    void* dst = static_cast<char*>(workspace) + at;
    ptr = dst;
    stage.item[n++] = {src, dst, rows, cols, stride};
  }
  bool map(CUtensorMap* m, int dtype, int box_rows) const { return encode_matrix(m, dtype, ptr, rows, cols, width, planes, box_rows); }
};

int map_error() {
  set_last_cuda_error(cudaErrorUnknown, "cuTensorMapEncodeTiled");
  return JVPFA_ERR_CUDA;
}

int stage(int dtype, std::initializer_list<Matrix*> matrices, void* workspace, cudaStream_t s) {
  StageArgs a{};
  int n = 0;
  long long most = 0;
  for (Matrix* m : matrices) {
    m->put(workspace, a, n);
    if (m->at >= 0) most = std::max<long long>(most, (long long)m->rows * m->cols);
  }
  if (n == 0) return JVPFA_OK;
  const dim3 grid((unsigned)std::min<long long>((most + 8 * kThreads - 1) / (8 * kThreads), 148 * 8), n);
  if (dtype == JVPFA_FP32)
    stage_kernel<float><<<grid, kThreads, 0, s>>>(a);
  else
    stage_kernel<__half><<<grid, kThreads, 0, s>>>(a);  // (bits alone are moved)
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return JVPFA_OK;
  set_last_cuda_error(e, "gated stage_kernel");
  return JVPFA_ERR_CUDA;
}

// ---- cotangents of the projections ---------------------------------------------------------------------------------------
struct CotangentArgs {
  const uint8_t* kept;
  const void *gh, *gth;
  void *d, *td;  // [dg | du] and [dtg | dtu], rows of 2 * width; fp32: three planes each
  int rows, cols, width, tensors;  // tensors: that were kept
  long long units;
};

template <typename T, int V>
__device__ __forceinline__ void store_parts(void* base, long long plane, long long at, const float (&v)[V]) {
  if constexpr (sizeof(T) == 4) {
    Pack<__nv_bfloat16, V> part[3];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float h, m, l;
      split3(v[j], h, m, l);
      part[0].e[j] = __float2bfloat16_rn(h), part[1].e[j] = __float2bfloat16_rn(m), part[2].e[j] = __float2bfloat16_rn(l);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<Pack<__nv_bfloat16, V>*>(static_cast<__nv_bfloat16*>(base) + k * plane + at) = part[k];
  } else {
    uint4 x;
    x = make_uint4(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]), Elem<T>::pack(v[4], v[5]), Elem<T>::pack(v[6], v[7]));
    *reinterpret_cast<uint4*>(static_cast<T*>(base) + at) = x;
  }
}

// V entries of a row from column c on; rows that are no whole pieces entry by entry (0 beyond the end).
template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ void load_floats(const void* base, long long at, int left, float (&v)[V]) {
  const T* p = static_cast<const T*>(base) + at;
  Pack<T, V> x;
  if constexpr (ALIGNED) {
    x = *reinterpret_cast<const Pack<T, V>*>(p);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) x.e[j] = j < left ? p[j] : Elem<T>::from_float(0.f);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = Elem<T>::to_float(x.e[j]);
}

// A warp takes an eighth or a quarter of a kept block at a time: 8 rows x 4 pieces.
template <typename T, int KIND, bool DUAL, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) cotangent_kernel(const __grid_constant__ CotangentArgs p) {
  constexpr int V = Kept<T>::kPiece, kParts = 32 / V;  // of a block: 4 x 8 rows, 1 x or 2 x 4 pieces
  constexpr bool EXACT = sizeof(T) == 4;
  const int lane = threadIdx.x & 31, blocks = (p.cols + 31) / 32;
  const long long plane = (long long)p.rows * 2 * p.width;
  for (long long unit = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); unit < p.units; unit += (long long)gridDim.x * (kThreads / 32)) {
    const unsigned block = (unsigned)(unit / kParts), part = (unsigned)(unit % kParts);
    const unsigned rb = block / (unsigned)blocks, fb = block - rb * (unsigned)blocks;
    const int r = (int)(part & 3) * 8 + (lane >> 2), piece = (int)(part >> 2) * 4 + (lane & 3);
    const int c = (int)fb * 32 + piece * V;
    const long long i = (long long)rb * 32 + r;
    if (i >= p.rows || c >= p.cols) continue;
    const uint8_t* kept = p.kept + (size_t)block * p.tensors * Kept<T>::kBlock;
    const long long from = i * p.cols + c, to = i * 2 * p.width + c;
    float g[V], u[V], gh[V], dg[V], du[V];
    kept_piece<T>(kept, r, piece, g);
    kept_piece<T>(kept + Kept<T>::kBlock, r, piece, u);
    if (!DUAL || p.gh) load_floats<T, V, ALIGNED>(p.gh, from, p.cols - c, gh);
    if constexpr (DUAL) {
      float gth[V], tg[V], tu[V];
      load_floats<T, V, ALIGNED>(p.gth, from, p.cols - c, gth);
      kept_piece<T>(kept + 2 * Kept<T>::kBlock, r, piece, tg);
      kept_piece<T>(kept + 3 * Kept<T>::kBlock, r, piece, tu);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const Activated y = activate<KIND, EXACT>(g[j]);
        const float slope = y.d1 * u[j];
        dg[j] = gth[j] * (y.d2 * tg[j] * u[j] + y.d1 * tu[j]);
        du[j] = gth[j] * y.d1 * tg[j];
        if (p.gh) dg[j] += gh[j] * slope, du[j] += gh[j] * y.a;
        tg[j] = gth[j] * slope;
        tu[j] = gth[j] * y.a;
      }
      store_parts<T, V>(p.td, plane, to, tg);
      store_parts<T, V>(p.td, plane, to + p.width, tu);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const Activated y = activate<KIND, EXACT>(g[j]);
        dg[j] = gh[j] * y.d1 * u[j];
        du[j] = gh[j] * y.a;
      }
    }
    store_parts<T, V>(p.d, plane, to, dg);
    store_parts<T, V>(p.d, plane, to + p.width, du);
  }
}

template <typename T, int KIND, bool DUAL>
void run_cotangents(const CotangentArgs& p, cudaStream_t s) {
  const unsigned blocks = (unsigned)std::min<long long>((p.units + kThreads / 32 - 1) / (kThreads / 32), 148 * 16);
  if (p.cols % Kept<T>::kPiece == 0)
    cotangent_kernel<T, KIND, DUAL, true><<<blocks, kThreads, 0, s>>>(p);
  else
    cotangent_kernel<T, KIND, DUAL, false><<<blocks, kThreads, 0, s>>>(p);
}
template <typename T>
void run_cotangents(int kind, CotangentArgs& p, cudaStream_t s) {
  p.units = (long long)((p.rows + 31) / 32) * ((p.cols + 31) / 32) * (32 / Kept<T>::kPiece);
  auto run = [&](auto k) {
    if (p.gth)
      run_cotangents<T, decltype(k)::value, true>(p, s);
    else
      run_cotangents<T, decltype(k)::value, false>(p, s);
  };
  switch (kind) {
    case JVPFA_ACT_SILU: return run(Kind<JVPFA_ACT_SILU>{});
    case JVPFA_ACT_SIGMOID: return run(Kind<JVPFA_ACT_SIGMOID>{});
    case JVPFA_ACT_GELU: return run(Kind<JVPFA_ACT_GELU>{});
    default: return run(Kind<JVPFA_ACT_GELU_TANH>{});
  }
}
int cotangents(int dtype, int kind, CotangentArgs& p, cudaStream_t s) {
  if (dtype == JVPFA_FP32)
    run_cotangents<float>(kind, p, s);
  else if (dtype == JVPFA_BF16)
    run_cotangents<__nv_bfloat16>(kind, p, s);
  else
    run_cotangents<__half>(kind, p, s);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return JVPFA_OK;
  set_last_cuda_error(e, "gated cotangent_kernel");
  return JVPFA_ERR_CUDA;
}

// ---- plans ---------------------------------------------------------------------------------------------------------------
struct FwdPlan {
  int rc = JVPFA_OK;
  int64_t bytes = 0;
  Matrix x, tx, wg, wu;
  int kind;
  int64_t partial_at = 0;
  PairArgs pair{};
  bool is_few;
  FewArgs few{};
  explicit FwdPlan(const jvpfa_gated_fwd_args& a)
      : x(a.dtype, a.x, a.M, a.K, a.x_stride),
        tx(a.dtype, a.tx, a.M, a.K, a.tx_stride),
        wg(a.dtype, a.wg, a.F, a.K, a.wg_stride),
        wu(a.dtype, a.wu, a.F, a.K, a.wu_stride),
        kind(a.tx ? kPairGatedDual : kPairGated) {
    few.groups = a.tx ? 2 : 1, few.rows = a.M, few.features = a.F, few.width = a.K;
    is_few = plan_few(a.dtype, kFewGated, few);
    x.use(bytes), tx.use(bytes);
    if (is_few && a.dtype == JVPFA_FP32) return;  // (reads the weights as they are)
    wg.use(bytes), wu.use(bytes);
    if (is_few) return;
    partial_at = bytes;
    pair.groups = 1, pair.rows = a.M, pair.cols = a.F, pair.depth = a.K, pair.sources = 1;
    rc = plan_pair(a.dtype, kind, pair);
    if (rc == JVPFA_OK) bytes += pair_workspace(pair);
  }
};

struct BwdPlan {
  int rc = JVPFA_OK;
  int64_t bytes = 0;
  int64_t width, d_bytes, d_at, td_at = -1;
  bool data, weights;  // which products are asked for
  Matrix x, tx, wg, wu;
  int64_t partial_at;  // (one product's at a time)
  PairArgs dx{}, dw{};
  bool is_few;
  FewArgs few{};
  explicit BwdPlan(const jvpfa_gated_bwd_args& a)
      : width(up8(a.F)),
        d_bytes(up256(2 * (a.dtype == JVPFA_FP32 ? 3 : 1) * 2 * width * a.M)),
        d_at(take(d_bytes)),
        td_at(a.gth ? take(d_bytes) : -1),
        data(a.dx || a.dtx),
        weights(a.dwg != nullptr),
        x(a.dtype, weights ? a.x : nullptr, a.M, a.K, a.x_stride),
        tx(a.dtype, weights && a.gth ? a.tx : nullptr, a.M, a.K, a.tx_stride),
        wg(a.dtype, data ? a.wg : nullptr, a.F, a.K, a.wg_stride),
        wu(a.dtype, data ? a.wu : nullptr, a.F, a.K, a.wu_stride) {
    few.groups = (a.dx != nullptr) + (a.dtx != nullptr), few.rows = a.M, few.features = a.F, few.width = a.K;
    is_few = data && plan_few(a.dtype, kFewDx, few);
    x.use(bytes), tx.use(bytes);
    if (!is_few || a.dtype != JVPFA_FP32) wg.use(bytes), wu.use(bytes);
    partial_at = bytes;
    int64_t partial = 0;
    if (data && !is_few) {
      dx.groups = (a.dx != nullptr) + (a.dtx != nullptr), dx.rows = a.M, dx.cols = a.K, dx.depth = a.F, dx.sources = 2;
      rc = plan_pair(a.dtype, kPairDx, dx);
      if (rc == JVPFA_OK) partial = pair_workspace(dx);
    }
    if (weights && rc == JVPFA_OK) {
      dw.groups = 2, dw.rows = a.F, dw.cols = a.K, dw.depth = a.M, dw.sources = a.gth ? 2 : 1;
      rc = plan_pair(a.dtype, kPairDw, dw);
      if (rc == JVPFA_OK) partial = std::max(partial, pair_workspace(dw));
    }
    bytes += partial;
  }
  int64_t take(int64_t n) {
    const int64_t at = bytes;
    bytes += n;
    return at;
  }
};

// The weights of a product of few rows: 64 x 64 boxes of 16-bit ones, fp32 ones as they are.
template <typename Args, typename Plan>
void few_weights(const Args& a, Plan& plan, FewMaps& maps, bool& ok) {
  FewArgs& p = plan.few;
  if (a.dtype != JVPFA_FP32) {
    ok = ok && plan.wg.map(&maps.w[0], a.dtype, 64) && plan.wu.map(&maps.w[1], a.dtype, 64);
    return;
  }
  p.wg = a.wg, p.wu = a.wu, p.wg_stride = a.wg_stride, p.wu_stride = a.wu_stride;
  p.pieces = (reinterpret_cast<uint64_t>(a.wg) | reinterpret_cast<uint64_t>(a.wu)) % 16 == 0 && (a.wg_stride | a.wu_stride) % 4 == 0;
}

}  // namespace

int64_t gated_kept_bytes(int dtype, int64_t M, int64_t F, bool tangent) { return kept_bytes(dtype, M, F, tangent); }
int plan_gated_fwd(const jvpfa_gated_fwd_args& a, int64_t* workspace) {
  const FwdPlan plan(a);
  *workspace = plan.bytes;
  return plan.rc;
}
int plan_gated_bwd(const jvpfa_gated_bwd_args& a, int64_t* workspace) {
  const BwdPlan plan(a);
  *workspace = plan.bytes;
  return plan.rc;
}

int launch_gated_fwd(const jvpfa_gated_fwd_args& a, cudaStream_t s) {
  FwdPlan plan(a);
  if (plan.rc) return plan.rc;
  const int rc = stage(a.dtype, {&plan.x, &plan.tx, &plan.wg, &plan.wu}, a.workspace, s);
  if (rc) return rc;
  const bool dual = a.tx != nullptr;
  if (plan.is_few) {
    FewMaps maps;
    FewArgs& p = plan.few;
    bool ok = plan.x.map(&maps.rows[0], a.dtype, p.padded);
    maps.rows[1] = maps.rows[2] = maps.rows[3] = maps.w[0] = maps.w[1] = maps.rows[0];
    if (dual) ok = ok && plan.tx.map(&maps.rows[1], a.dtype, p.padded);
    few_weights(a, plan, maps, ok);
    if (!ok) return map_error();
    p.h = a.h, p.th = a.th, p.kept = static_cast<uint8_t*>(a.kept);
    p.activation = a.activation;
    return launch_few(a.dtype, kFewGated, p, maps, s);
  }
  PairMaps maps;
  bool ok = plan.x.map(&maps.a[0], a.dtype, dual ? 64 : 128) && plan.wg.map(&maps.b[0], a.dtype, 128) && plan.wu.map(&maps.b[1], a.dtype, 128);
  maps.a[1] = maps.a[0];
  if (dual) ok = ok && plan.tx.map(&maps.a[1], a.dtype, 64);
  maps.a[2] = maps.a[3] = maps.a[0];
  if (!ok) return map_error();
  PairArgs& p = plan.pair;
  p.partial = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + plan.partial_at);
  p.h = a.h, p.th = a.th, p.kept = static_cast<uint8_t*>(a.kept);
  p.activation = a.activation;
  return launch_pair(a.dtype, plan.kind, p, maps, s);
}

int launch_gated_bwd(const jvpfa_gated_bwd_args& a, cudaStream_t s) {
  BwdPlan plan(a);
  if (plan.rc) return plan.rc;
  char* const ws = static_cast<char*>(a.workspace);
  CotangentArgs c{};
  c.kept = static_cast<const uint8_t*>(a.kept), c.tensors = a.kept_tangent ? 4 : 2;
  c.gh = a.gh, c.gth = a.gth;
  c.d = ws + plan.d_at;
  c.td = a.gth ? ws + plan.td_at : nullptr;
  c.rows = a.M, c.cols = a.F, c.width = (int)plan.width;
  int rc = cotangents(a.dtype, a.activation, c, s);
  if (!rc) rc = stage(a.dtype, {&plan.x, &plan.tx, &plan.wg, &plan.wu}, a.workspace, s);
  if (rc) return rc;
  const int planes = a.dtype == JVPFA_FP32 ? 3 : 1;
  float* const partial = reinterpret_cast<float*>(ws + plan.partial_at);
  // half of [dg | du] or of [dtg | dtu]
  auto half = [&](CUtensorMap* m, bool tangent, bool up, int box_rows) {
    return encode_matrix(m, a.dtype, static_cast<const char*>(tangent ? c.td : c.d) + (up ? 2 * plan.width : 0), a.M, a.F, 2 * plan.width, planes,
                         box_rows);
  };
  if (plan.is_few) {
    FewMaps maps;
    FewArgs& p = plan.few;
    bool ok = true;
    int group = 0;
    for (int tangent = 0; tangent < 2; ++tangent) {
      if (!(tangent ? a.dtx : a.dx)) continue;
      p.out[group] = tangent ? a.dtx : a.dx;
      for (int up = 0; up < 2; ++up) ok = ok && half(&maps.rows[2 * group + up], tangent, up, p.padded);
      ++group;
    }
    if (group == 1) maps.rows[2] = maps.rows[0], maps.rows[3] = maps.rows[1];
    maps.w[0] = maps.w[1] = maps.rows[0];
    few_weights(a, plan, maps, ok);
    if (!ok) return map_error();
    rc = launch_few(a.dtype, kFewDx, p, maps, s);
    if (rc) return rc;
  } else if (plan.data) {
    PairMaps maps;
    PairArgs& p = plan.dx;
    p.partial = partial;
    bool ok = plan.wg.map(&maps.b[0], a.dtype, 64) && plan.wu.map(&maps.b[1], a.dtype, 64);
    int group = 0;
    for (int tangent = 0; tangent < 2; ++tangent) {
      if (!(tangent ? a.dtx : a.dx)) continue;
      p.out[group] = tangent ? a.dtx : a.dx;
      for (int up = 0; up < 2; ++up) ok = ok && half(&maps.a[2 * group + up], tangent, up, 128);
      ++group;
    }
    if (group == 1) maps.a[2] = maps.a[0], maps.a[3] = maps.a[1];
    if (!ok) return map_error();
    rc = launch_pair(a.dtype, kPairDx, p, maps, s);
    if (rc) return rc;
  }
  if (plan.weights) {
    PairMaps maps;
    PairArgs& p = plan.dw;
    p.partial = partial;
    p.out[0] = a.dwg, p.out[1] = a.dwu;
    bool ok = plan.x.map(&maps.b[0], a.dtype, 64);
    maps.b[1] = maps.b[0];
    if (a.gth) ok = ok && plan.tx.map(&maps.b[1], a.dtype, 64);
    for (int up = 0; up < 2; ++up)
      for (int tangent = 0; tangent < 2; ++tangent) ok = ok && half(&maps.a[2 * up + tangent], tangent && a.gth, up, 64);
    if (!ok) return map_error();
    rc = launch_pair(a.dtype, kPairDw, p, maps, s);
  }
  return rc;
}

}  // namespace jvpfa

// The gated projection: its launches, and what they need besides the matrix products of gated_gemm.cu.
//
// Forward: one launch (value, or value and tangent).  Backward: a pass that turns the cotangents into those of the projections,
//   dg = gh a' u + gth (a'' tg u + a' tu),  du = gh a + gth a' tg,  dtg = gth a' u,  dtu = gth a,
// bound by memory (four tensors read and two written for the value alone), then a product over the features for dx and dtx, and one over
// the rows for dwg and dwu.  Tangents are further rows of the first (dx beside dtx, the weights shared) and further depth of the second.
//
// Operands go to the tensor cores by TMA, which takes rows of whole 16-byte pieces; others are copied once into the workspace with padded
// rows.  fp32 operands become three planes of bf16 parts there (f32_tc5_common.cuh).
#include <algorithm>

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
// rows x cols, row stride `stride`, into rows of `width`; fp32: into three planes of bf16 parts.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) stage_kernel(const T* src, long long rows, int cols, long long stride, void* dst, int width) {
  const long long per_row = (cols + V - 1) / V, total = rows * per_row;
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kThreads) {
    const long long r = i / per_row;
    const int c = (int)(i - r * per_row) * V;
    const Pack<T, V> x = *reinterpret_cast<const Pack<T, V>*>(src + r * stride + c);
    if constexpr (sizeof(T) == 4) {
      const long long plane = rows * width;
      Pack<__nv_bfloat16, V> part[3];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float h, m, l;
        split3(x.e[j], h, m, l);
        part[0].e[j] = __float2bfloat16_rn(h), part[1].e[j] = __float2bfloat16_rn(m), part[2].e[j] = __float2bfloat16_rn(l);
      }
      __nv_bfloat16* d = static_cast<__nv_bfloat16*>(dst) + r * width + c;
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<Pack<__nv_bfloat16, V>*>(d + k * plane) = part[k];
    } else {
      *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(dst) + r * width + c) = x;
    }
  }
}

template <typename T, int V>
int run_stage(const void* src, int rows, int cols, int64_t stride, void* dst, cudaStream_t s) {
  const long long blocks = ((long long)rows * ((cols + V - 1) / V) + kThreads - 1) / kThreads;
  stage_kernel<T, V><<<(unsigned)std::min<long long>(blocks, 148 * 16), kThreads, 0, s>>>(static_cast<const T*>(src), rows, cols, stride, dst,
                                                                                         (int)up8(cols));
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return JVPFA_OK;
  set_last_cuda_error(e, "gated stage_kernel");
  return JVPFA_ERR_CUDA;
}
// `stride` in elements; pieces of 16 bytes where the source has them.
int stage(int dtype, const void* src, int rows, int cols, int64_t stride, void* dst, cudaStream_t s) {
  const uint64_t address = reinterpret_cast<uint64_t>(src);
  if (dtype == JVPFA_FP32)
    return address % 16 == 0 && cols % 4 == 0 && stride % 4 == 0 ? run_stage<float, 4>(src, rows, cols, stride, dst, s)
                                                                 : run_stage<float, 1>(src, rows, cols, stride, dst, s);
  return address % 16 == 0 && cols % 8 == 0 && stride % 8 == 0 ? run_stage<__half, 8>(src, rows, cols, stride, dst, s)
                                                               : run_stage<__half, 1>(src, rows, cols, stride, dst, s);
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

  Matrix(int dtype, const void* p, int rows_, int cols_, int64_t stride_, int64_t& workspace)
      : src(p), rows(rows_), cols(cols_), stride(stride_), ptr(p), width(stride_), planes(dtype == JVPFA_FP32 ? 3 : 1) {
    if (!p) return;
    if (rows == 1) stride = width = up8(cols);
    const bool in_place = dtype != JVPFA_FP32 && reinterpret_cast<uint64_t>(p) % 16 == 0 && width % 8 == 0 && width >= cols && width < 1ll << 38;
    if (in_place) return;
    at = workspace;
    width = up8(cols);
    workspace += up256(2 * planes * width * rows);
  }
  int make(int dtype, void* workspace, cudaStream_t s) {
    if (at < 0) return JVPFA_OK;
    void* dst = static_cast<char*>(workspace) + at;
    ptr = dst;
    return stage(dtype, src, rows, cols, stride, dst, s);
  }
  bool map(CUtensorMap* m, int dtype, int box_rows) const { return encode_matrix(m, dtype, ptr, rows, cols, width, planes, box_rows); }
};

int map_error() {
  set_last_cuda_error(cudaErrorUnknown, "cuTensorMapEncodeTiled");
  return JVPFA_ERR_CUDA;
}

// ---- cotangents of the projections ---------------------------------------------------------------------------------------
struct CotangentArgs {
  const void *g, *u, *tg, *tu, *gh, *gth;
  void *d, *td;  // [dg | du] and [dtg | dtu], rows of 2 * width; fp32: three planes each
  long long rows;
  int cols, width, activation;
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
    Pack<T, V> x;
#pragma unroll
    for (int j = 0; j < V; ++j) x.e[j] = Elem<T>::from_float(v[j]);
    *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(base) + at) = x;
  }
}

template <typename T, int V>
__device__ __forceinline__ void load_floats(const void* base, long long at, float (&v)[V]) {
  const Pack<T, V> x = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(base) + at);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = Elem<T>::to_float(x.e[j]);
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) cotangent_kernel(const __grid_constant__ CotangentArgs p) {
  constexpr bool EXACT = sizeof(T) == 4;
  const long long per_row = p.cols / V, total = p.rows * per_row, plane = p.rows * 2 * p.width;
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kThreads) {
    const long long r = i / per_row;
    const int c = (int)(i - r * per_row) * V;
    const long long from = r * p.cols + c, to = r * 2 * p.width + c;
    float g[V], u[V], gh[V], dg[V], du[V];
    load_floats<T, V>(p.g, from, g);
    load_floats<T, V>(p.u, from, u);
    if (p.gh) load_floats<T, V>(p.gh, from, gh);
    Activated y[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      y[j] = activate<EXACT>(p.activation, g[j]);
      dg[j] = p.gh ? gh[j] * y[j].d1 * u[j] : 0.f;
      du[j] = p.gh ? gh[j] * y[j].a : 0.f;
    }
    if (p.gth) {
      float gth[V], tg[V], tu[V];
      load_floats<T, V>(p.gth, from, gth);
      load_floats<T, V>(p.tg, from, tg);
      load_floats<T, V>(p.tu, from, tu);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        dg[j] += gth[j] * (y[j].d2 * tg[j] * u[j] + y[j].d1 * tu[j]);
        du[j] += gth[j] * y[j].d1 * tg[j];
        tg[j] = gth[j] * y[j].d1 * u[j];
        tu[j] = gth[j] * y[j].a;
      }
      store_parts<T, V>(p.td, plane, to, tg);
      store_parts<T, V>(p.td, plane, to + p.width, tu);
    }
    store_parts<T, V>(p.d, plane, to, dg);
    store_parts<T, V>(p.d, plane, to + p.width, du);
  }
}

template <typename T, int V>
int run_cotangents(const CotangentArgs& p, cudaStream_t s) {
  const long long blocks = (p.rows * (p.cols / V) + kThreads - 1) / kThreads;
  cotangent_kernel<T, V><<<(unsigned)std::min<long long>(blocks, 148 * 8), kThreads, 0, s>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return JVPFA_OK;
  set_last_cuda_error(e, "gated cotangent_kernel");
  return JVPFA_ERR_CUDA;
}
int cotangents(int dtype, const CotangentArgs& p, cudaStream_t s) {
  if (dtype == JVPFA_FP32) return p.cols % 4 == 0 ? run_cotangents<float, 4>(p, s) : run_cotangents<float, 1>(p, s);
  const bool bf16 = dtype == JVPFA_BF16;
  if (p.cols % 8 == 0) return bf16 ? run_cotangents<__nv_bfloat16, 8>(p, s) : run_cotangents<__half, 8>(p, s);
  return bf16 ? run_cotangents<__nv_bfloat16, 1>(p, s) : run_cotangents<__half, 1>(p, s);
}

// ---- plans ---------------------------------------------------------------------------------------------------------------
struct FwdPlan {
  int64_t bytes = 0;
  Matrix x, tx, wg, wu;
  explicit FwdPlan(const jvpfa_gated_fwd_args& a)
      : x(a.dtype, a.x, a.M, a.K, a.x_stride, bytes),
        tx(a.dtype, a.tx, a.M, a.K, a.tx_stride, bytes),
        wg(a.dtype, a.wg, a.F, a.K, a.wg_stride, bytes),
        wu(a.dtype, a.wu, a.F, a.K, a.wu_stride, bytes) {}
};

struct BwdPlan {
  int64_t bytes = 0;
  int64_t width, d_bytes, d_at, td_at = -1;
  bool data, weights;  // which products are asked for
  Matrix x, tx, wg, wu;
  explicit BwdPlan(const jvpfa_gated_bwd_args& a)
      : width(up8(a.F)),
        d_bytes(up256(2 * (a.dtype == JVPFA_FP32 ? 3 : 1) * 2 * width * a.M)),
        d_at(take(d_bytes)),
        td_at(a.gth ? take(d_bytes) : -1),
        data(a.dx || a.dtx),
        weights(a.dwg != nullptr),
        x(a.dtype, weights ? a.x : nullptr, a.M, a.K, a.x_stride, bytes),
        tx(a.dtype, weights && a.gth ? a.tx : nullptr, a.M, a.K, a.tx_stride, bytes),
        wg(a.dtype, data ? a.wg : nullptr, a.F, a.K, a.wg_stride, bytes),
        wu(a.dtype, data ? a.wu : nullptr, a.F, a.K, a.wu_stride, bytes) {}
  int64_t take(int64_t n) {
    const int64_t at = bytes;
    bytes += n;
    return at;
  }
};

}  // namespace

int64_t gated_fwd_workspace(const jvpfa_gated_fwd_args& a) { return FwdPlan(a).bytes; }
int64_t gated_bwd_workspace(const jvpfa_gated_bwd_args& a) { return BwdPlan(a).bytes; }

int launch_gated_fwd(const jvpfa_gated_fwd_args& a, cudaStream_t s) {
  FwdPlan plan(a);
  for (Matrix* m : {&plan.x, &plan.tx, &plan.wg, &plan.wu}) {
    const int rc = m->make(a.dtype, a.workspace, s);
    if (rc) return rc;
  }
  const bool dual = a.tx != nullptr;
  PairMaps maps;
  bool ok = plan.x.map(&maps.a[0], a.dtype, dual ? 64 : 128) && plan.wg.map(&maps.b[0], a.dtype, 128) && plan.wu.map(&maps.b[1], a.dtype, 128);
  maps.a[1] = maps.a[0];
  if (dual) ok = ok && plan.tx.map(&maps.a[1], a.dtype, 64);
  maps.a[2] = maps.a[3] = maps.a[0];
  if (!ok) return map_error();
  PairArgs p{};
  p.groups = 1, p.rows = a.M, p.cols = a.F, p.depth = a.K, p.sources = 1;
  p.h = a.h, p.th = a.th, p.g = a.g, p.u = a.u, p.tg = a.tg, p.tu = a.tu;
  p.activation = a.activation;
  return launch_pair(a.dtype, dual ? kPairGatedDual : kPairGated, p, maps, s);
}

int launch_gated_bwd(const jvpfa_gated_bwd_args& a, cudaStream_t s) {
  BwdPlan plan(a);
  char* const ws = static_cast<char*>(a.workspace);
  CotangentArgs c{};
  c.g = a.g, c.u = a.u, c.tg = a.tg, c.tu = a.tu, c.gh = a.gh, c.gth = a.gth;
  c.d = ws + plan.d_at;
  c.td = a.gth ? ws + plan.td_at : nullptr;
  c.rows = a.M, c.cols = a.F, c.width = (int)plan.width, c.activation = a.activation;
  int rc = cotangents(a.dtype, c, s);
  for (Matrix* m : {&plan.x, &plan.tx, &plan.wg, &plan.wu})
    if (!rc) rc = m->make(a.dtype, a.workspace, s);
  if (rc) return rc;
  const int planes = a.dtype == JVPFA_FP32 ? 3 : 1;
  // half of [dg | du] or of [dtg | dtu]
  auto half = [&](CUtensorMap* m, bool tangent, bool up, int box_rows) {
    return encode_matrix(m, a.dtype, static_cast<const char*>(tangent ? c.td : c.d) + (up ? 2 * plan.width : 0), a.M, a.F, 2 * plan.width, planes,
                         box_rows);
  };
  if (plan.data) {
    PairMaps maps;
    PairArgs p{};
    p.rows = a.M, p.cols = a.K, p.depth = a.F, p.sources = 2;
    bool ok = plan.wg.map(&maps.b[0], a.dtype, 64) && plan.wu.map(&maps.b[1], a.dtype, 64);
    for (int tangent = 0; tangent < 2; ++tangent) {
      if (!(tangent ? a.dtx : a.dx)) continue;
      p.out[p.groups] = tangent ? a.dtx : a.dx;
      for (int up = 0; up < 2; ++up) ok = ok && half(&maps.a[2 * p.groups + up], tangent, up, 128);
      ++p.groups;
    }
    if (p.groups == 1) maps.a[2] = maps.a[0], maps.a[3] = maps.a[1];
    if (!ok) return map_error();
    rc = launch_pair(a.dtype, kPairDx, p, maps, s);
    if (rc) return rc;
  }
  if (plan.weights) {
    PairMaps maps;
    PairArgs p{};
    p.groups = 2, p.rows = a.F, p.cols = a.K, p.depth = a.M, p.sources = a.gth ? 2 : 1;
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

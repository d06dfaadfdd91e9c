// Entries of the norms and residual sums: argument checks, how a backward is cut, and the launch that adds up the parts of the vectors'
// gradients.  With the parts P of a group (norm_common.cuh), sums over all groups for a vector that is not grouped:
//   dweight = (1 + scale) PG + tscale PtG     dscale = weight PG + tweight PtG + bias PO + tbias PtO    dshift = PO
//   dbias = (1 + scale) PO + tscale PtO       dgate = alpha (post PE + tpost PtE)                       dpost = alpha (gate PE + tgate PtE)
// and the tangents' the same with (PtG, PtO, PtE) for (PG, PO, PE) and nothing for their second terms.
#include "norm_common.cuh"

namespace jvpfa {
namespace norms {

// Instances in norm_fwd_*.cu and norm_bwd_*.cu.
template <typename T>
int launch_fwd(const jvpfa_norm_args& a, cudaStream_t s);
template <typename T>
int launch_bwd(const jvpfa_norm_args& a, const Cut& c, cudaStream_t s);

namespace {

constexpr int kCols = 32, kLanes = 32;  // of a CTA that adds up parts: its columns, and how many take turns with the slices
constexpr int kMostChunks = 64;         // of groups, each by CTAs of its own

struct Totals {
  float d[6], dt[6];
};

__device__ __forceinline__ float vec_scalar(const jvpfa_norm_args& a, int which, bool tangent, long long group, int col, float otherwise) {
  const jvpfa_norm_vec& x = a.vec[which];
  const void* p = tangent ? x.tv : x.v;
  if (!p) return otherwise;
  const long long at = (x.grouped ? group * (tangent ? x.tv_stride : x.stride) : 0) + col;
  if (a.vec_dtype == JVPFA_FP32) return static_cast<const float*>(p)[at];
  return a.vec_dtype == JVPFA_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]) : __half2float(static_cast<const __half*>(p)[at]);
}

__device__ __forceinline__ void write_vec(const jvpfa_norm_args& a, void* p, long long at, float x) {
  if (a.vec_dtype == JVPFA_FP32)
    static_cast<float*>(p)[at] = x;
  else if (a.vec_dtype == JVPFA_BF16)
    static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(x);
  else
    static_cast<__half*>(p)[at] = __float2half_rn(x);
}

// Column blockIdx.x * kCols + x of the groups of chunk blockIdx.y, `per` lanes for the slices of one group, so kLanes / per groups at once.  `totals`: 12 rows of
// C values for each chunk, where there are several.  ALL: a group takes all lanes.  (8192 groups of one row of 1024, scale and shift of each: 180 us; with all
// lanes for a group's one slice 4.2 ms.)
template <bool ALL>
__global__ void __launch_bounds__(kCols * kLanes) norm_parts_kernel(const __grid_constant__ jvpfa_norm_args a, const Cut cut, float* totals, const int lanes) {
  __shared__ float part[kParts][kLanes][kCols + 1];
  const int x = threadIdx.x % kCols, lane = threadIdx.x / kCols, col = blockIdx.x * kCols + x;
  const int per = ALL ? kLanes : lanes, sub = lane % per, at = lane / per, at_once = kLanes / per;
  Totals t;
#pragma unroll
  for (int i = 0; i < 6; ++i) t.d[i] = t.dt[i] = 0.f;
  const long long g0 = (long long)cut.groups * blockIdx.y / gridDim.y, g1 = (long long)cut.groups * (blockIdx.y + 1) / gridDim.y;
  for (long long first = g0; first < g1; first += at_once) {
    const long long group = first + at;
    const bool live = col < a.C && group < g1;
    float p[kParts] = {};
    if (live)
#pragma unroll 4
      for (int slice = sub; slice < cut.slices; slice += per) {
        const float* from = static_cast<const float*>(a.workspace) + (group * cut.slices + slice) * cut.n_parts * (long long)a.C + col;
#pragma unroll
        for (int k = 0; k < kParts; ++k)
          if (cut.parts >> k & 1) p[k] += *from, from += a.C;
      }
    if (per > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kParts; ++k) part[k][lane][x] = p[k];
      __syncthreads();
    }
    if (sub != 0 || !live) continue;
    if (per > 1) {
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        p[k] = 0.f;
        for (int l = 0; l < per; ++l) p[k] += part[k][lane + l][x];
      }
    }
    auto v = [&](int which, bool tangent, float otherwise) { return vec_scalar(a, which, tangent, group, col, otherwise); };
    const float w = v(JVPFA_VEC_WEIGHT, false, 1.f), tw = v(JVPFA_VEC_WEIGHT, true, 0.f), b = v(JVPFA_VEC_BIAS, false, 0.f), tb = v(JVPFA_VEC_BIAS, true, 0.f);
    const float sc = 1.f + v(JVPFA_VEC_SCALE, false, 0.f), tsc = v(JVPFA_VEC_SCALE, true, 0.f);
    const float gate = v(JVPFA_VEC_GATE, false, 1.f), tgate = v(JVPFA_VEC_GATE, true, 0.f);
    const float post = v(JVPFA_VEC_POST_WEIGHT, false, 1.f), tpost = v(JVPFA_VEC_POST_WEIGHT, true, 0.f);
    const float d[6] = {sc * p[PG] + tsc * p[PtG], sc * p[PO] + tsc * p[PtO], w * p[PG] + tw * p[PtG] + b * p[PO] + tb * p[PtO], p[PO],
                        a.alpha * (post * p[PE] + tpost * p[PtE]), a.alpha * (gate * p[PE] + tgate * p[PtE])};
    const float dt[6] = {sc * p[PtG], sc * p[PtO], w * p[PtG] + b * p[PtO], p[PtO], a.alpha * post * p[PtE], a.alpha * gate * p[PtE]};
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      if (a.vec[i].grouped) {
        if (a.d[i]) write_vec(a, a.d[i], group * a.C + col, d[i]);
        if (a.dt[i]) write_vec(a, a.dt[i], group * a.C + col, dt[i]);
      } else {
        t.d[i] += d[i], t.dt[i] += dt[i];
      }
    }
  }
  static_assert(kParts >= 6, "a vector's sums go where the parts were");
  if (at_once > 1) {  // what each of them has added up
    auto over_groups = [&](float(&mine)[6]) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 6; ++i)
        if (sub == 0) part[i][at][x] = mine[i];
      __syncthreads();
      if (lane != 0) return;
#pragma unroll
      for (int i = 0; i < 6; ++i) {
        mine[i] = 0.f;
        for (int l = 0; l < at_once; ++l) mine[i] += part[i][l][x];
      }
    };
    over_groups(t.d), over_groups(t.dt);
  }
  if (lane != 0 || col >= a.C) return;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    if (a.vec[i].grouped) continue;
    if (totals) {
      float* to = totals + (long long)blockIdx.y * 12 * a.C + col;
      to[(long long)i * a.C] = t.d[i], to[(long long)(6 + i) * a.C] = t.dt[i];
    } else {
      if (a.d[i]) write_vec(a, a.d[i], col, t.d[i]);
      if (a.dt[i]) write_vec(a, a.dt[i], col, t.dt[i]);
    }
  }
}

// Vectors that are not grouped, over the chunks of groups.
__global__ void __launch_bounds__(128) norm_totals_kernel(const __grid_constant__ jvpfa_norm_args a, const float* totals, int chunks) {
  const int col = blockIdx.x * 128 + threadIdx.x, i = blockIdx.y % 6;
  void* to = blockIdx.y < 6 ? a.d[i] : a.dt[i];
  if (col >= a.C || !to || a.vec[i].grouped) return;
  float s = 0.f;
  for (int c = 0; c < chunks; ++c) s += totals[((long long)c * 12 + blockIdx.y) * a.C + col];
  write_vec(a, to, col, s);
}

int check(const jvpfa_norm_args* a, bool backward) {
  if (!a) return JVPFA_ERR_NULL;
  if (a->struct_size != (int32_t)sizeof(jvpfa_norm_args)) return JVPFA_ERR_STRUCT;
  if (a->dtype != JVPFA_BF16 && a->dtype != JVPFA_FP16 && a->dtype != JVPFA_FP32) return JVPFA_ERR_DTYPE;
  if (a->vec_dtype != a->dtype && a->vec_dtype != JVPFA_FP32) return JVPFA_ERR_DTYPE;
  if (a->M > (1 << 30)) return JVPFA_ERR_TOO_LARGE;
  if (a->M < 1 || a->C < 1 || a->C > JVPFA_NORM_MAX_WIDTH || a->group_rows < 1 || a->M % a->group_rows) return JVPFA_ERR_SHAPE;
  if (a->kind < JVPFA_NORM_NONE || a->kind > JVPFA_NORM_LAYER || a->post < JVPFA_NORM_NONE || a->post > JVPFA_NORM_LAYER) return JVPFA_ERR_UNSUPPORTED;
  const bool y = a->y != nullptr, n = a->kind != JVPFA_NORM_NONE;
  if ((!y && !n) || (!y && (a->post || a->ty))) return JVPFA_ERR_UNSUPPORTED;
  if (!a->x || ((a->tx || a->ty) && !a->dual)) return JVPFA_ERR_NULL;
  if (a->x_stride < 0 || a->tx_stride < 0 || a->y_stride < 0 || a->ty_stride < 0) return JVPFA_ERR_SHAPE;
  const uintptr_t size = a->dtype == JVPFA_FP32 ? 4 : 2, vec_size = a->vec_dtype == JVPFA_FP32 ? 4 : 2;
  uintptr_t all = 0, vecs = 0;
  for (const void* p : {a->x, a->tx, a->y, a->ty}) all |= reinterpret_cast<uintptr_t>(p);
  for (int i = 0; i < 6; ++i) {
    const jvpfa_norm_vec& v = a->vec[i];
    if (v.tv && (!v.v || !a->dual)) return JVPFA_ERR_NULL;
    if (v.v && (i == JVPFA_VEC_GATE || i == JVPFA_VEC_POST_WEIGHT ? !y : !n)) return JVPFA_ERR_UNSUPPORTED;
    if (v.grouped && (v.stride < 0 || v.tv_stride < 0)) return JVPFA_ERR_SHAPE;
    vecs |= reinterpret_cast<uintptr_t>(v.v) | reinterpret_cast<uintptr_t>(v.tv);
    if (!backward) continue;
    if ((a->d[i] && !v.v) || (a->dt[i] && (!v.v || !a->dual))) return JVPFA_ERR_NULL;
    vecs |= reinterpret_cast<uintptr_t>(a->d[i]) | reinterpret_cast<uintptr_t>(a->dt[i]);
  }
  if (!backward) {
    if (y ? !a->r || (a->dual && !a->tr) : a->r || a->tr) return JVPFA_ERR_NULL;
    if (n ? !a->n || (a->dual && !a->tn) : a->n || a->tn) return JVPFA_ERR_NULL;
    for (const void* p : {a->r, a->tr, a->n, a->tn}) all |= reinterpret_cast<uintptr_t>(p);
  } else {
    if (!a->stats || (!y && (a->gr || a->gtr || a->dy || a->dty)) || (!n && (a->gn || a->gtn))) return JVPFA_ERR_NULL;
    if (!a->dual && (a->gtr || a->gtn || a->dtx || a->dty)) return JVPFA_ERR_NULL;
    for (const void* p : {a->gr, a->gtr, a->gn, a->gtn, (const void*)a->dx, (const void*)a->dtx, (const void*)a->dy, (const void*)a->dty})
      all |= reinterpret_cast<uintptr_t>(p);
  }
  if (all % size || vecs % vec_size || reinterpret_cast<uintptr_t>(a->stats) % 16 || reinterpret_cast<uintptr_t>(a->workspace) % 16) return JVPFA_ERR_ALIGN;
  return JVPFA_OK;
}

struct Plan {
  Cut cut;
  int per, chunks;  // lanes for a group where parts are added up; CTAs that share the groups of a column
  int64_t parts_bytes, bytes;
};

// Parts of a group's rows: one for each SM, with at least 4 rows each.
Plan plan_bwd(const jvpfa_norm_args& a) {
  Plan p{};
  p.cut.groups = a.M / a.group_rows;
  int slices = kSMs / p.cut.groups;
  if (slices > a.group_rows / 4) slices = a.group_rows / 4;
  p.cut.slices = slices < 1 ? 1 : slices;
  auto wants = [&](int i) { return a.d[i] || a.dt[i]; };
  if (wants(JVPFA_VEC_WEIGHT) || wants(JVPFA_VEC_SCALE)) p.cut.parts |= 1u << PG;
  if (wants(JVPFA_VEC_BIAS) || wants(JVPFA_VEC_SHIFT) || (wants(JVPFA_VEC_SCALE) && a.vec[JVPFA_VEC_BIAS].v)) p.cut.parts |= 1u << PO;
  if (wants(JVPFA_VEC_GATE) || wants(JVPFA_VEC_POST_WEIGHT)) p.cut.parts |= 1u << PE;
  if (a.dual) p.cut.parts |= p.cut.parts << PtG;
  for (int k = 0; k < kParts; ++k) p.cut.n_parts += p.cut.parts >> k & 1;
  for (p.per = 1; p.per < p.cut.slices && p.per < kLanes;) p.per *= 2;
  p.chunks = (p.cut.groups + kLanes / p.per - 1) / (kLanes / p.per);
  if (p.chunks > kMostChunks) p.chunks = kMostChunks;
  p.parts_bytes = (int64_t)p.cut.groups * p.cut.slices * p.cut.n_parts * a.C * 4;
  p.bytes = p.cut.parts ? p.parts_bytes + (p.chunks > 1 ? (int64_t)p.chunks * 12 * a.C * 4 : 0) : 0;
  return p;
}

}  // namespace
}  // namespace norms
}  // namespace jvpfa

using namespace jvpfa;

extern "C" {

int jvpfa_norm_fwd(const jvpfa_norm_args* a, void* stream) {
  int rc = norms::check(a, false);
  if (rc) return rc;
  rc = check_arch();
  if (rc) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == JVPFA_FP32) return norms::launch_fwd<float>(*a, s);
  return a->dtype == JVPFA_BF16 ? norms::launch_fwd<__nv_bfloat16>(*a, s) : norms::launch_fwd<__half>(*a, s);
}

int64_t jvpfa_norm_bwd_workspace(const jvpfa_norm_args* a) { return norms::check(a, true) == JVPFA_OK ? norms::plan_bwd(*a).bytes : 0; }

int jvpfa_norm_bwd(const jvpfa_norm_args* a, void* stream) {
  int rc = norms::check(a, true);
  if (rc) return rc;
  const norms::Plan p = norms::plan_bwd(*a);
  if (p.bytes && (!a->workspace || a->workspace_bytes < p.bytes)) return JVPFA_ERR_NULL;
  rc = check_arch();
  if (rc) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == JVPFA_FP32)
    rc = norms::launch_bwd<float>(*a, p.cut, s);
  else
    rc = a->dtype == JVPFA_BF16 ? norms::launch_bwd<__nv_bfloat16>(*a, p.cut, s) : norms::launch_bwd<__half>(*a, p.cut, s);
  if (rc || !p.cut.parts) return rc;
  float* totals = p.chunks > 1 ? reinterpret_cast<float*>(static_cast<char*>(a->workspace) + p.parts_bytes) : nullptr;
  const auto parts = p.per == norms::kLanes ? norms::norm_parts_kernel<true> : norms::norm_parts_kernel<false>;
  parts<<<dim3((a->C + norms::kCols - 1) / norms::kCols, p.chunks), norms::kCols * norms::kLanes, 0, s>>>(*a, p.cut, totals, p.per);
  bool ungrouped = false;
  for (int i = 0; i < 6; ++i) ungrouped = ungrouped || (!a->vec[i].grouped && (a->d[i] || a->dt[i]));
  if (totals && ungrouped) norms::norm_totals_kernel<<<dim3((a->C + 127) / 128, 12), 128, 0, s>>>(*a, totals, p.chunks);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "norm_parts_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
}

}  // extern "C"

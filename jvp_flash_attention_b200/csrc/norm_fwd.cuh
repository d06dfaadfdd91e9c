// Value and tangent of the residual sum and the norm behind it (norm_common.cuh has the formulas), one pass over the rows.
//
// A row is held in the registers of 32 to 512 threads, 8 to 32 entries each, from its load to its store; its means are sums over these
// threads, the variance about the mean in a second one (a first pass's sum of squares loses what a large mean has).  A CTA stays on each SM, for
// several rows at once, and takes successive rows, so that the vectors of a group are read once for many of its rows, and up to four rows
// of each are under way while one is worked on.
// What bounds it: memory, each tensor read and written once.
#pragma once
#include "norm_common.cuh"

namespace jvpfa {
namespace norms {

template <typename T, int NC, Way WAY, bool TAN, bool HASY, bool HASN>
__global__ void __launch_bounds__(512) norm_fwd_kernel(const __grid_constant__ jvpfa_norm_args a, const Wide wide, const Layout lay, const bool aligned) {
  constexpr int V = 16 / (int)sizeof(T), E = V * NC, TENSORS = (HASY ? 2 : 1) * (TAN ? 2 : 1);
  extern __shared__ __align__(16) unsigned char smem[];
  const Team team{(int)threadIdx.x / lay.threads, lay.threads, (int)threadIdx.x % lay.threads};
  unsigned char* mine = smem + team.index * lay.team_bytes;
  RowSum row_sum{reinterpret_cast<float*>(mine), team};
  unsigned char* ring = mine + kSumFloats * 4;
  unsigned char* outs = ring + lay.depth * TENSORS * lay.slot;
  const Rows<T, NC, WAY> rows{a.C, a.M, team, aligned};
  const Source sources[4] = {{a.x, a.x_stride}, {HASY ? a.y : a.tx, HASY ? a.y_stride : a.tx_stride}, {a.tx, a.tx_stride}, {a.ty, a.ty_stride}};
  constexpr int kTx = HASY ? 2 : 1;
  const long long workers = (long long)gridDim.x * lay.teams, me = (long long)blockIdx.x * lay.teams + team.index;
  const int first = (int)(a.M * me / workers), end = (int)(a.M * (me + 1) / workers);
  const float by = 1.f / a.C;
  const bool layer = a.kind == JVPFA_NORM_LAYER, post_layer = a.post == JVPFA_NORM_LAYER, post = a.post != JVPFA_NORM_NONE;

  auto fetch = [&](int row) {  // its slot is its place among the worker's rows
    if (row < end) {
      unsigned char* to = ring + (row - first) % lay.depth * TENSORS * lay.slot;
#pragma unroll
      for (int k = 0; k < TENSORS; ++k) rows.fetch(to + k * lay.slot, sources[k], row);
    }
    cp_async_commit();
  };
  if (WAY != DIRECT)
    for (int k = 0; k < lay.depth; ++k) fetch(first + k);

  float G[E], O[E], Eg[E], tG[TAN ? E : 1], tO[TAN ? E : 1], tE[TAN ? E : 1];
  long long group = -1;
  for (int row = first; row < end; ++row) {
    float r[E], tr[TAN ? E : 1], m[HASY ? E : 1], tm[TAN && HASY ? E : 1];
    if (WAY != DIRECT) wait_rows(lay.depth);
    if (WAY == RAGGED) team.sync();
    {
      const unsigned char* from = ring + (row - first) % lay.depth * TENSORS * lay.slot;
      Pieces<T, NC> raw[TENSORS];
#pragma unroll
      for (int k = 0; k < TENSORS; ++k) rows.read(raw[k], from + k * lay.slot, sources[k], row);
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = j * V + i;
          r[e] = raw[0].at(j, i);
          if constexpr (HASY) m[e] = raw[1].at(j, i);
          if constexpr (TAN) tr[e] = raw[kTx].at(j, i);
          if constexpr (TAN && HASY) tm[e] = raw[3].at(j, i);
        }
    }
    if (WAY == RAGGED) team.sync();
    if (WAY != DIRECT) fetch(row + lay.depth);
    if (row / a.group_rows != group) {
      group = row / a.group_rows;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        if (!rows.on(j, 0)) continue;
        if (HASN) gain_of<T, V, TAN>(a, wide, group, rows.piece(j) * V, G + j * V, O + j * V, tG + (TAN ? j * V : 0), tO + (TAN ? j * V : 0));
        if (HASY) gate_of<T, V, TAN>(a, wide, group, rows.piece(j) * V, Eg + j * V, tE + (TAN ? j * V : 0));
      }
    }
    // x (entries), tx -> n, tn; stat: what a backward reads
    auto normed = [&](float* x, float* tx, bool with_mean, float4& stat) {
      float mean = 0.f, tmean = 0.f;
      if (with_mean) {
        float s[TAN ? 2 : 1] = {};
#pragma unroll
        for (int e = 0; e < E; ++e) {
          s[0] += x[e];
          if constexpr (TAN) s[1] += tx[e];
        }
        row_sum(s);
        mean = s[0] * by;
        if constexpr (TAN) tmean = s[1] * by;
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (rows.on(j, i)) {  // (the entries behind a row's end stay zero)
              x[j * V + i] -= mean;
              if (TAN) tx[j * V + i] -= tmean;
            }
      }
      float s[TAN ? 2 : 1] = {};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        s[0] += x[e] * x[e];
        if constexpr (TAN) s[1] += x[e] * tx[e];
      }
      row_sum(s);
      const float inv = rsqrtf(s[0] * by + a.eps);
      float b = 0.f;
      if constexpr (TAN) b = s[1] * by * inv;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[e] *= inv;
        if (TAN) tx[e] = inv * (tx[e] - x[e] * b);
      }
      stat = make_float4(mean, inv, tmean, b);
    };
    float4 stat_y{0.f, 1.f, 0.f, 0.f}, stat_r{0.f, 1.f, 0.f, 0.f};
    if (HASY) {
      if (post) normed(m, tm, post_layer, stat_y);
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        if (!rows.on(j, 0)) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = j * V + i;
          r[e] += Eg[e] * m[e];
          if (TAN) tr[e] += tE[e] * m[e] + Eg[e] * tm[e];
        }
      }
      rows.write(a.r, row, r, outs);
      if (TAN) rows.write(a.tr, row, tr, outs + lay.slot);
    }
    if (HASN) {
      normed(r, tr, layer, stat_r);
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        if (!rows.on(j, 0)) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = j * V + i;
          if (TAN) tr[e] = tr[e] * G[e] + (r[e] * tG[e] + tO[e]);
          r[e] = r[e] * G[e] + O[e];
        }
      }
      rows.write(a.n, row, r, outs + (HASY ? (TAN ? 2 : 1) * lay.slot : 0));
      if (TAN) rows.write(a.tn, row, tr, outs + (HASY ? 3 : 1) * lay.slot);
    }
    if (a.stats && team.tid == 0) {
      float4* st = reinterpret_cast<float4*>(a.stats) + 2ll * row;
      st[0] = stat_y, st[1] = stat_r;
    }
  }
}

template <typename T, int NC, Way WAY, bool TAN, bool HASY, bool HASN>
int launch_fwd(const jvpfa_norm_args& a, bool aligned, cudaStream_t s) {
  const auto kernel = norm_fwd_kernel<T, NC, WAY, TAN, HASY, HASN>;
  static SmemOptIn opt;
  const int sides = TAN ? 2 : 1;
  const Layout lay = layout_of(a, WAY, 16 / (int)sizeof(T) * NC, 512, (HASY ? 2 : 1) * sides, (HASY && HASN ? 2 : 1) * sides, 0);
  if (lay.depth < 1) return JVPFA_ERR_UNSUPPORTED;
  if (!opt.ensure(reinterpret_cast<const void*>(kernel), 225 * 1024)) return JVPFA_ERR_CUDA;
  const int ctas = (a.M + lay.teams - 1) / lay.teams;
  // CTAs of few bytes share an SM
  int each = 227 * 1024 / (lay.bytes + 1024), by_threads = 512 / (lay.threads * lay.teams);
  each = each < by_threads ? each : by_threads;
  const int most = kSMs * (each < 1 ? 1 : each);
  kernel<<<ctas < most ? ctas : most, lay.threads * lay.teams, lay.bytes, s>>>(a, wide_vectors(a), lay, aligned);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "norm_fwd_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
}

template <typename T, int NC, Way WAY>
int launch_fwd(const jvpfa_norm_args& a, bool al, cudaStream_t s) {
  const bool y = a.y != nullptr, n = a.kind != JVPFA_NORM_NONE;
  if (a.dual)
    return !y ? launch_fwd<T, NC, WAY, true, false, true>(a, al, s) : n ? launch_fwd<T, NC, WAY, true, true, true>(a, al, s) : launch_fwd<T, NC, WAY, true, true, false>(a, al, s);
  return !y ? launch_fwd<T, NC, WAY, false, false, true>(a, al, s) : n ? launch_fwd<T, NC, WAY, false, true, true>(a, al, s) : launch_fwd<T, NC, WAY, false, true, false>(a, al, s);
}

// Eight entries a thread up to 4096 of a row, 16 up to 8192 of 16-bit types, 32 and no shared memory beyond.
template <typename T>
int launch_fwd(const jvpfa_norm_args& a, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool aligned = aligned_rows(a);
  if (a.C <= 4096) return aligned ? launch_fwd<T, 8 / V, ALIGNED>(a, true, s) : launch_fwd<T, 8 / V, RAGGED>(a, false, s);
  if constexpr (sizeof(T) == 2)
    if (a.C <= 8192 && aligned) return launch_fwd<T, 16 / V, ALIGNED>(a, true, s);
  return launch_fwd<T, 32 / V, DIRECT>(a, aligned, s);
}

}  // namespace norms
}  // namespace jvpfa

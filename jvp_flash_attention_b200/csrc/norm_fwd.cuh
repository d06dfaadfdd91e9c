// Value and tangent of the residual sum and the norm behind it (norm_common.cuh has the formulas), one pass over the rows.
//
// A row is held in the registers of 32 to 512 threads, 8 to 32 entries each, from its load to its store; its means are sums over these
// threads, the variance about the mean in a second one (a first pass's sum of squares loses what a large mean has).  CTAs stay and take
// successive rows, so that the vectors of a group are read once for many of its rows, and the next row is under way while one is worked on.
// What bounds it: memory, each tensor read and written once.
#pragma once
#include "norm_common.cuh"

namespace jvpfa {
namespace norms {

template <typename T, int V, int NC, bool TAN, bool HASY, bool HASN>
__global__ void __launch_bounds__(kAtMost) norm_fwd_kernel(const __grid_constant__ jvpfa_norm_args a, const Wide wide, const int threads) {
  constexpr int E = V * NC;
  __shared__ float sums[512];
  // rows of one warp: a warp for each; others: the CTA
  const int team = threads == 32 ? (int)threadIdx.x >> 5 : 0, teams = (int)blockDim.x / threads;
  const int tid = threads == 32 ? (int)threadIdx.x & 31 : (int)threadIdx.x;
  RowSum row_sum{sums, threads / 32};
  const long long workers = (long long)gridDim.x * teams, me = (long long)blockIdx.x * teams + team;
  const int first = (int)(a.M * me / workers), end = (int)(a.M * (me + 1) / workers);
  const float by = 1.f / a.C;
  const bool layer = a.kind == JVPFA_NORM_LAYER, post_layer = a.post == JVPFA_NORM_LAYER, post = a.post != JVPFA_NORM_NONE;
  bool live[NC];
  int col[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) col[j] = (j * threads + tid) * V, live[j] = col[j] < a.C;

  Pack<T, V> px[NC], ptx[NC], py[NC], pty[NC];
  auto fetch = [&](int row) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* tx = static_cast<const T*>(a.tx) + row * a.tx_stride;
    const T* y = static_cast<const T*>(a.y) + row * a.y_stride;
    const T* ty = static_cast<const T*>(a.ty) + row * a.ty_stride;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      if (!live[j]) continue;
      px[j] = load_pack<T, V>(x + col[j]);
      if (HASY) py[j] = load_pack<T, V>(y + col[j]);
      if (TAN && a.tx) ptx[j] = load_pack<T, V>(tx + col[j]);
      if (TAN && HASY && a.ty) pty[j] = load_pack<T, V>(ty + col[j]);
    }
  };
  if (first < end) fetch(first);

  float G[E], O[E], Eg[E], tG[TAN ? E : 1], tO[TAN ? E : 1], tE[TAN ? E : 1];
  long long group = -1;
  for (int row = first; row < end; ++row) {
    float r[E], tr[TAN ? E : 1], m[HASY ? E : 1], tm[TAN && HASY ? E : 1];
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = j * V + i;
        r[e] = live[j] ? Elem<T>::to_float(px[j].e[i]) : 0.f;
        if (TAN) tr[e] = live[j] && a.tx ? Elem<T>::to_float(ptx[j].e[i]) : 0.f;
        if (HASY) m[e] = live[j] ? Elem<T>::to_float(py[j].e[i]) : 0.f;
        if (TAN && HASY) tm[e] = live[j] && a.ty ? Elem<T>::to_float(pty[j].e[i]) : 0.f;
      }
    if (row + 1 < end) fetch(row + 1);
    if (row / a.group_rows != group) {
      group = row / a.group_rows;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        if (!live[j]) continue;
        if (HASN) gain_of<T, V, TAN>(a, wide, group, col[j], G + j * V, O + j * V, tG + (TAN ? j * V : 0), tO + (TAN ? j * V : 0));
        if (HASY) gate_of<T, V, TAN>(a, wide, group, col[j], Eg + j * V, tE + (TAN ? j * V : 0));
      }
    }
    // x (entries), tx -> n, tn; stat: what a backward reads
    auto normed = [&](float* x, float* tx, bool with_mean, float4& stat) {
      float mean = 0.f, tmean = 0.f;
      if (with_mean) {
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < E; ++e) {
          s[0] += x[e];
          if (TAN) s[1] += tx[e];
        }
        row_sum(s);
        mean = s[0] * by, tmean = s[1] * by;
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (live[j])  // (the entries behind a row's end stay zero)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              x[j * V + i] -= mean;
              if (TAN) tx[j * V + i] -= tmean;
            }
      }
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        s[0] += x[e] * x[e];
        if (TAN) s[1] += x[e] * tx[e];
      }
      row_sum(s);
      const float inv = rsqrtf(s[0] * by + a.eps), b = s[1] * by * inv;
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
        if (!live[j]) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = j * V + i;
          r[e] += Eg[e] * m[e];
          if (TAN) tr[e] += tE[e] * m[e] + Eg[e] * tm[e];
        }
        store_floats<T, V>(static_cast<T*>(a.r) + (long long)row * a.C + col[j], r + j * V);
        if (TAN) store_floats<T, V>(static_cast<T*>(a.tr) + (long long)row * a.C + col[j], tr + j * V);
      }
    }
    if (HASN) {
      normed(r, tr, layer, stat_r);
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        if (!live[j]) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = j * V + i;
          if (TAN) tr[e] = tr[e] * G[e] + (r[e] * tG[e] + tO[e]);
          r[e] = r[e] * G[e] + O[e];
        }
        store_floats<T, V>(static_cast<T*>(a.n) + (long long)row * a.C + col[j], r + j * V);
        if (TAN) store_floats<T, V>(static_cast<T*>(a.tn) + (long long)row * a.C + col[j], tr + j * V);
      }
    }
    if (a.stats && tid == 0) {
      float4* st = reinterpret_cast<float4*>(a.stats) + 2ll * row;
      st[0] = stat_y, st[1] = stat_r;
    }
  }
}

template <typename T, int V, int NC, bool TAN, bool HASY, bool HASN>
int launch_fwd(const jvpfa_norm_args& a, cudaStream_t s) {
  const auto kernel = norm_fwd_kernel<T, V, NC, TAN, HASY, HASN>;
  static int known[33] = {};
  const int threads = (a.C + V * NC * 32 - 1) / (V * NC * 32) * 32;
  const int cta = threads == 32 ? 128 : threads, teams = cta / threads;
  const long long rows = (a.M + teams - 1) / teams, most = (long long)kSMs * resident(kernel, cta, known);
  kernel<<<(unsigned)(rows < most ? rows : most), cta, 0, s>>>(a, wide_vectors(a), threads);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "norm_fwd_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
}

template <typename T, int V, int NC>
int launch_fwd(const jvpfa_norm_args& a, cudaStream_t s) {
  const bool y = a.y != nullptr, n = a.kind != JVPFA_NORM_NONE;
  if (a.dual) return y ? (n ? launch_fwd<T, V, NC, true, true, true>(a, s) : launch_fwd<T, V, NC, true, true, false>(a, s)) : launch_fwd<T, V, NC, true, false, true>(a, s);
  return y ? (n ? launch_fwd<T, V, NC, false, true, true>(a, s) : launch_fwd<T, V, NC, false, true, false>(a, s)) : launch_fwd<T, V, NC, false, false, true>(a, s);
}

template <typename T>
int launch_fwd(const jvpfa_norm_args& a, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  if (vector_entries(a) == 1) return a.C <= 16 * kAtMost ? launch_fwd<T, 1, 16>(a, s) : launch_fwd<T, 1, 32>(a, s);
  if (a.C <= 8 * kAtMost) return launch_fwd<T, V, 8 / V>(a, s);
  return a.C <= 16 * kAtMost ? launch_fwd<T, V, 16 / V>(a, s) : launch_fwd<T, V, 32 / V>(a, s);
}

}  // namespace norms
}  // namespace jvpfa

// Gradients of the residual sum and the norm behind it (norm_common.cuh has the formulas), one pass over the rows, and the vectors' sums.
//
// A row is formed again from the operands and the four statistics of each norm that the forward kept, in 32 bits as there, so no result that
// was rounded is read.  Two sums over the row's threads (five values each with tangents, two without) are all that its entries exchange.  The
// vectors' gradients are sums over rows: each thread adds up its columns' in registers while its CTA goes through successive rows of one
// group, and leaves them in the workspace; a second launch adds these parts in a fixed order.
// What bounds it: memory, each tensor read and written once, and the parts.
#pragma once
#include "norm_common.cuh"

namespace jvpfa {
namespace norms {

// The sums over a group's rows that the vectors' gradients are made of, by their place in the workspace.
enum Part { PG, PO, PE, PtG, PtO, PtE, kParts };  // of gn n + gtn tn, gn, dr N + dtr tN, gtn n, gtn, dtr N

struct Cut {
  int groups, slices;  // of each group's rows
  uint32_t parts;      // which sums are wanted, a bit for each
  int n_parts;
};

template <typename T, int V, int NC, bool TAN, bool HASY, bool HASN>
__global__ void __launch_bounds__(kAtMost) norm_bwd_kernel(const __grid_constant__ jvpfa_norm_args a, const Wide wide, const int threads, const Cut cut) {
  constexpr int E = V * NC, ET = TAN ? E : 1;
  __shared__ float sums[512];
  const int team = threads == 32 ? (int)threadIdx.x >> 5 : 0, teams = (int)blockDim.x / threads;
  const int tid = threads == 32 ? (int)threadIdx.x & 31 : (int)threadIdx.x;
  RowSum row_sum{sums, threads / 32};
  const long long workers = (long long)gridDim.x * teams, me = (long long)blockIdx.x * teams + team;
  const float by = 1.f / a.C;
  const bool layer = a.kind == JVPFA_NORM_LAYER, post_layer = a.post == JVPFA_NORM_LAYER, post = a.post != JVPFA_NORM_NONE;
  bool live[NC];
  int col[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) col[j] = (j * threads + tid) * V, live[j] = col[j] < a.C;
  auto get = [&](float* to, const void* p, long long at) {  // a row's entries; zeros for an absent tensor and behind the end
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      if (p && live[j]) {
        const Pack<T, V> x = load_pack<T, V>(static_cast<const T*>(p) + at + col[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) to[j * V + i] = Elem<T>::to_float(x.e[i]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) to[j * V + i] = 0.f;
      }
    }
  };
  auto put = [&](void* p, long long at, const float* x) {
    if (!p) return;
#pragma unroll
    for (int j = 0; j < NC; ++j)
      if (live[j]) store_floats<T, V>(static_cast<T*>(p) + at + col[j], x + j * V);
  };

  for (long long unit = me; unit < (long long)cut.groups * cut.slices; unit += workers) {
    const long long group = unit / cut.slices;
    const int slice = (int)(unit - group * cut.slices);
    const int first = (int)(group * a.group_rows + (long long)a.group_rows * slice / cut.slices);
    const int end = (int)(group * a.group_rows + (long long)a.group_rows * (slice + 1) / cut.slices);
    float pG[HASN ? E : 1], pO[HASN ? E : 1], pE[HASY ? E : 1], ptG[HASN ? ET : 1], ptO[HASN ? ET : 1], ptE[HASY ? ET : 1];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (HASN) pG[e] = pO[e] = 0.f;
      if (HASY) pE[e] = 0.f;
      if (HASN && TAN) ptG[e] = ptO[e] = 0.f;
      if (HASY && TAN) ptE[e] = 0.f;
    }
    for (int row = first; row < end; ++row) {
      const long long at = (long long)row * a.C;
      float r[E], tr[ET], m[HASY ? E : 1], tm[HASY ? ET : 1], Eg[HASY ? E : 1], tE[HASY ? ET : 1];
      float dr[E], dtr[ET];
      get(r, a.x, row * a.x_stride);
      if (TAN) get(tr, a.tx, row * a.tx_stride);
      if (HASY) get(m, a.y, row * a.y_stride);
      if (HASY && TAN) get(tm, a.ty, row * a.ty_stride);
      float g[HASN ? E : 1], h[HASN ? ET : 1];
      if (HASN) get(g, a.gn, at);
      if (HASN && TAN) get(h, a.gtn, at);
      get(dr, HASY ? a.gr : nullptr, at);
      if (TAN) get(dtr, HASY ? a.gtr : nullptr, at);
      const float4* st = reinterpret_cast<const float4*>(a.stats) + 2ll * row;
      const float4 sy = st[0], sr = st[1];  // mean, 1 / deviation, the tangent's mean, mean(n tangent)
      if (HASY) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (live[j]) gate_of<T, V, TAN>(a, wide, group, col[j], Eg + j * V, tE + (TAN ? j * V : 0));
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int e = j * V + i;
            if (!live[j]) {
              Eg[e] = 0.f;
              if (TAN) tE[e] = 0.f;
              continue;
            }
            if (post) {
              m[e] = (m[e] - sy.x) * sy.y;
              if (TAN) tm[e] = sy.y * (tm[e] - sy.z - m[e] * sy.w);
            }
            r[e] += Eg[e] * m[e];
            if (TAN) tr[e] += tE[e] * m[e] + Eg[e] * tm[e];
          }
      }
      if (HASN) {
        // s[]: of n g', g', n h, h, h tn
        float s[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          float G[V], O[V], tG[V], tO[V];
          if (!live[j]) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const int e = j * V + i;
              r[e] = g[e] = 0.f;
              if (TAN) tr[e] = h[e] = 0.f;
            }
            continue;
          }
          gain_of<T, V, TAN>(a, wide, group, col[j], G, O, tG, tO);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int e = j * V + i;
            const float n = (r[e] - sr.x) * sr.y;
            r[e] = n;
            pO[e] += g[e];
            pG[e] += g[e] * n;
            if (TAN) {
              const float tn = sr.y * (tr[e] - sr.z - n * sr.w);
              tr[e] = tn;
              ptO[e] += h[e], ptG[e] += h[e] * n, pG[e] += h[e] * tn;
              const float gh = h[e] * G[i];
              g[e] = g[e] * G[i] + h[e] * tG[i] - sr.y * sr.w * gh;
              h[e] = gh;
              s[2] += n * gh, s[3] += gh, s[4] += gh * tn;
            } else {
              g[e] *= G[i];
            }
            s[0] += n * g[e], s[1] += g[e];
          }
        }
        if constexpr (TAN) {
          row_sum(s);
        } else {
          float u[2] = {s[0], s[1]};
          row_sum(u);
          s[0] = u[0], s[1] = u[1];
        }
        const float ng = s[0] * by, mg = layer ? s[1] * by : 0.f, nh = s[2] * by, mh = layer ? s[3] * by : 0.f, htn = s[4] * by;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          dr[e] += sr.y * (g[e] - mg - r[e] * ng);
          if (TAN) {
            dr[e] -= sr.y * (nh * tr[e] + htn * r[e]);
            dtr[e] += sr.y * (h[e] - mh - r[e] * nh);
          }
        }
      }
      put(a.dx, at, dr);
      if (TAN) put(a.dtx, at, dtr);
      if (HASY) {
        float s[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < E; ++e) {
          pE[e] += dr[e] * m[e];
          if (TAN) {
            pE[e] += dtr[e] * tm[e], ptE[e] += dtr[e] * m[e];
            dr[e] = dr[e] * Eg[e] + dtr[e] * tE[e];
            dtr[e] *= Eg[e];
            if (post) {
              dr[e] -= sy.y * sy.w * dtr[e];
              s[2] += m[e] * dtr[e], s[3] += dtr[e], s[4] += dtr[e] * tm[e];
            }
          } else {
            dr[e] *= Eg[e];
          }
          s[0] += m[e] * dr[e], s[1] += dr[e];
        }
        if (post) {
          if constexpr (TAN) {
            row_sum(s);
          } else {
            float u[2] = {s[0], s[1]};
            row_sum(u);
            s[0] = u[0], s[1] = u[1];
          }
          const float ng = s[0] * by, mg = post_layer ? s[1] * by : 0.f, nh = s[2] * by, mh = post_layer ? s[3] * by : 0.f, htn = s[4] * by;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            dr[e] = sy.y * (dr[e] - mg - m[e] * ng);
            if (TAN) {
              dr[e] -= sy.y * (nh * tm[e] + htn * m[e]);
              dtr[e] = sy.y * (dtr[e] - mh - m[e] * nh);
            }
          }
        }
        put(a.dy, at, dr);
        if (TAN) put(a.dty, at, dtr);
      }
    }
    if (cut.parts) {
      float* to = static_cast<float*>(a.workspace) + unit * cut.n_parts * (long long)a.C;
      auto leave = [&](int part, const float* x) {
        if (!(cut.parts >> part & 1)) return;
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (live[j])
#pragma unroll
            for (int i = 0; i < V; ++i) to[col[j] + i] = x[j * V + i];
        to += a.C;
      };
      if (HASN) leave(PG, pG), leave(PO, pO);
      if (HASY) leave(PE, pE);
      if (HASN && TAN) leave(PtG, ptG), leave(PtO, ptO);
      if (HASY && TAN) leave(PtE, ptE);
    }
  }
}

template <typename T, int V, int NC, bool TAN, bool HASY, bool HASN>
int launch_bwd(const jvpfa_norm_args& a, const Cut& cut, cudaStream_t s) {
  const auto kernel = norm_bwd_kernel<T, V, NC, TAN, HASY, HASN>;
  static int known[33] = {};
  const int threads = (a.C + V * NC * 32 - 1) / (V * NC * 32) * 32;
  const int cta = threads == 32 ? 128 : threads, teams = cta / threads;
  const long long units = ((long long)cut.groups * cut.slices + teams - 1) / teams, most = (long long)kSMs * resident(kernel, cta, known);
  kernel<<<(unsigned)(units < most ? units : most), cta, 0, s>>>(a, wide_vectors(a), threads, cut);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "norm_bwd_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
}

template <typename T, int V, int NC>
int launch_bwd(const jvpfa_norm_args& a, const Cut& c, cudaStream_t s) {
  const bool y = a.y != nullptr, n = a.kind != JVPFA_NORM_NONE;
  if (a.dual) return y ? (n ? launch_bwd<T, V, NC, true, true, true>(a, c, s) : launch_bwd<T, V, NC, true, true, false>(a, c, s)) : launch_bwd<T, V, NC, true, false, true>(a, c, s);
  return y ? (n ? launch_bwd<T, V, NC, false, true, true>(a, c, s) : launch_bwd<T, V, NC, false, true, false>(a, c, s)) : launch_bwd<T, V, NC, false, false, true>(a, c, s);
}

template <typename T>
int launch_bwd(const jvpfa_norm_args& a, const Cut& c, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  if (vector_entries(a) == 1) return a.C <= 16 * kAtMost ? launch_bwd<T, 1, 16>(a, c, s) : launch_bwd<T, 1, 32>(a, c, s);
  if (a.C <= 8 * kAtMost) return launch_bwd<T, V, 8 / V>(a, c, s);
  return a.C <= 16 * kAtMost ? launch_bwd<T, V, 16 / V>(a, c, s) : launch_bwd<T, V, 32 / V>(a, c, s);
}

}  // namespace norms
}  // namespace jvpfa

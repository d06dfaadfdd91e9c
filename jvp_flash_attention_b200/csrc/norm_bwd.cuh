// Gradients of the residual sum and the norm behind it (norm_common.cuh has the formulas), one pass over the rows, and the vectors' sums.
//
// A row is formed again from the operands and the four statistics of each norm that the forward kept, in 32 bits as there, so no result that
// was rounded is read.  Two sums over the row's threads (five values each with tangents, two without) are all that its entries exchange.  The
// vectors' gradients are sums over rows: each thread adds up its columns' in registers while its CTA, one on each SM and several rows at once, goes
// through a part of one group's rows, and leaves them in the workspace; a second launch adds these parts in a fixed order.
// What bounds it: memory, each tensor read and written once; with tangents and a residual sum the registers (170 of a thread, 12 warps).  bf16 8192 x 4096 with both norms 120 us (403 MB at 3.4 TB/s; issue slots
// 57 % busy, a row at once on an SM); 8192 x 1024 with tangents the norm 36 and with the residual sum 73; fp16 3990 x 2731 43.
#pragma once
#include "norm_common.cuh"

namespace jvpfa {
namespace norms {

// (One CTA, said so: else the compiler leaves 32 or 64 registers to the instances that hold least of a row in them.)
template <typename T, int NC, Way WAY, bool TAN, bool HASY, bool HASN, int BOUND>
__global__ void __launch_bounds__(BOUND, 1) norm_bwd_kernel(const __grid_constant__ jvpfa_norm_args a, const Wide wide, const Layout lay, const bool aligned, const Cut cut) {
  constexpr int V = 16 / (int)sizeof(T), E = V * NC, ET = TAN ? E : 1, SIDES = TAN ? 2 : 1;
  constexpr int TENSORS = SIDES * ((HASY ? 3 : 1) + (HASN ? 1 : 0));
  extern __shared__ __align__(16) unsigned char smem[];
  const Team team{(int)threadIdx.x / lay.threads, lay.threads, (int)threadIdx.x % lay.threads};
  unsigned char* mine = smem + team.index * lay.team_bytes;
  RowSum row_sum{reinterpret_cast<float*>(mine), team};
  unsigned char* ring = mine + kSumFloats * 4;
  unsigned char* outs = ring + lay.depth * TENSORS * lay.slot;
  // the vectors of the group in work, put together: E, tE, G, tG
  constexpr int VECTORS = SIDES * ((HASY ? 1 : 0) + (HASN ? 1 : 0));
  float* vectors = reinterpret_cast<float*>(smem + lay.teams * lay.team_bytes);
  const int padded = (a.C + V - 1) / V * V;
  float* shared_parts = vectors + (WAY == DIRECT ? 0 : VECTORS * padded);  // (DIRECT ones read the vectors as they are)
  const Rows<T, NC, WAY> rows{a.C, a.M, team, aligned};
  // x, tx, gn, gtn, y, ty, gr, gtr, as far as there are any of them
  Source sources[TENSORS];
  int n_sources = 0;
  auto source = [&](const void* p, long long stride) { sources[n_sources++] = Source{p, stride}; };
  source(a.x, a.x_stride);
  if (TAN) source(a.tx, a.tx_stride);
  if (HASN) source(a.gn, a.C);
  if (HASN && TAN) source(a.gtn, a.C);
  if (HASY) source(a.y, a.y_stride);
  if (HASY && TAN) source(a.ty, a.ty_stride);
  if (HASY) source(a.gr, a.C);
  if (HASY && TAN) source(a.gtr, a.C);
  const float by = 1.f / a.C;
  const bool layer = a.kind == JVPFA_NORM_LAYER, post_layer = a.post == JVPFA_NORM_LAYER, post = a.post != JVPFA_NORM_NONE;

  for (long long unit = blockIdx.x; unit < (long long)cut.groups * cut.slices; unit += gridDim.x) {
    const long long group = unit / cut.slices;
    const int slice = (int)(unit - group * cut.slices);
    const int first = (int)(group * a.group_rows + (long long)a.group_rows * slice / cut.slices) + team.index;
    const int end = (int)(group * a.group_rows + (long long)a.group_rows * (slice + 1) / cut.slices);
    float pG[HASN ? E : 1], pO[HASN ? E : 1], pE[HASY ? E : 1], ptG[HASN ? ET : 1], ptO[HASN ? ET : 1], ptE[HASY ? ET : 1];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (HASN) pG[e] = pO[e] = 0.f;
      if (HASY) pE[e] = 0.f;
      if (HASN && TAN) ptG[e] = ptO[e] = 0.f;
      if (HASY && TAN) ptE[e] = 0.f;
    }
    // (everybody has read the vectors of the unit before: its sums are behind a barrier where several rows share the CTA)
    if (WAY != DIRECT) {
      if (lay.teams == 1 || !cut.parts) __syncthreads();
      for (int col = threadIdx.x * V; col < a.C; col += blockDim.x * V) {
        float x[4][V];
        float O[V], tO[V];
        if (HASY) gate_of<T, V, TAN>(a, wide, group, col, x[0], x[1]);
        if (HASN) gain_of<T, V, TAN>(a, wide, group, col, x[HASY ? SIDES : 0], O, x[HASY ? 3 : 1], tO);
#pragma unroll
        for (int k = 0; k < VECTORS; ++k)
#pragma unroll
          for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(rows.place(vectors + k * padded, col / V, i)) = make_float4(x[k][i], x[k][i + 1], x[k][i + 2], x[k][i + 3]);
      }
      __syncthreads();
    }
    // piece j of one of them
    auto vector = [&](float* to, int which, int j) { rows.vector(to, vectors + which * padded, j); };
    auto fetch = [&](unsigned char* to, int row) {
      if (row < end) {
#pragma unroll
        for (int i = 0; i < TENSORS; ++i) rows.fetch(to + i * lay.slot, sources[i], row);
      }
      cp_async_commit();
    };
    if (WAY != DIRECT)
      for (int k = 0; k < lay.depth; ++k) fetch(ring + k * TENSORS * lay.slot, first + k * lay.teams);
    unsigned char* slot = ring;
    const float4* stats = reinterpret_cast<const float4*>(a.stats);
    float4 next_y = first < end ? stats[2ll * first] : float4{}, next_r = first < end ? stats[2ll * first + 1] : float4{};
    for (int row = first; row < end; row += lay.teams) {
      float r[E], tr[ET], m[HASY ? E : 1], tm[HASY ? ET : 1], Eg[HASY ? E : 1], tE[HASY ? ET : 1];
      float dr[E], dtr[ET], g[HASN ? E : 1], h[HASN ? ET : 1];
      if (WAY != DIRECT) wait_rows(lay.depth);
      if (WAY == RAGGED) team.sync();
      {
        int at = 0;
        auto get = [&](float* to) {
          Pieces<T, NC> raw;
          rows.read(raw, slot + at * lay.slot, sources[at], row);
          ++at;
#pragma unroll
          for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) to[j * V + i] = raw.at(j, i);
        };
        get(r);
        if (TAN) get(tr);
        if (HASN) get(g);
        if (HASN && TAN) get(h);
        if (HASY) get(m);
        if (HASY && TAN) get(tm);
        if (HASY) get(dr);
        if (HASY && TAN) get(dtr);
      }
      if constexpr (!HASY) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          dr[e] = 0.f;
          if (TAN) dtr[e] = 0.f;
        }
      }
      if (WAY == RAGGED) team.sync();
      if (WAY != DIRECT) {
        fetch(slot, row + lay.depth * lay.teams);
        slot += TENSORS * lay.slot;
        if (slot == outs) slot = ring;
      }
      const float4 sy = next_y, sr = next_r;  // mean, 1 / deviation, the tangent's mean, mean(n tangent)
      if (row + lay.teams < end) next_y = stats[2ll * (row + lay.teams)], next_r = stats[2ll * (row + lay.teams) + 1];
      if (HASY) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (rows.on(j, 0)) {
            if (WAY == DIRECT) {
              gate_of<T, V, TAN>(a, wide, group, rows.piece(j) * V, Eg + j * V, tE + (TAN ? j * V : 0));
            } else {
              vector(Eg + j * V, 0, j);
              if (TAN) vector(tE + (TAN ? j * V : 0), 1, j);
            }
          }
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int e = j * V + i;
            if (!rows.on(j, i)) {
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
          if (!rows.on(j, 0)) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const int e = j * V + i;
              r[e] = 0.f;
              if (TAN) tr[e] = 0.f;
            }
            continue;  // (g and h are zero there)
          }
          if (WAY == DIRECT) {
            gain_of<T, V, TAN>(a, wide, group, rows.piece(j) * V, G, O, tG, tO);
          } else {
            vector(G, HASY ? SIDES : 0, j);
            if (TAN) vector(tG, HASY ? 3 : 1, j);
          }
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int e = j * V + i;
            const float n = rows.on(j, i) ? (r[e] - sr.x) * sr.y : 0.f;
            r[e] = n;
            pO[e] += g[e];
            pG[e] += g[e] * n;
            if (TAN) {
              const float tn = rows.on(j, i) ? sr.y * (tr[e] - sr.z - n * sr.w) : 0.f;
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
      rows.write(a.dx, row, dr, outs);
      if (TAN) rows.write(a.dtx, row, dtr, outs + lay.slot);
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
        rows.write(a.dy, row, dr, outs + SIDES * lay.slot);
        if (TAN) rows.write(a.dty, row, dtr, outs + 3 * lay.slot);
      }
    }
    if (cut.parts) {
      float* to = static_cast<float*>(a.workspace) + unit * cut.n_parts * (long long)a.C;
      // the rows of a CTA one after the other, through shared memory
      for (int turn = 0; turn < lay.teams; ++turn) {
        if (turn == team.index) {
          int part = 0;
          auto leave = [&](Part which, const float* x) {
            if (!(cut.parts >> which & 1)) return;
            const bool last = turn == lay.teams - 1;
#pragma unroll
            for (int j = 0; j < NC; ++j)
#pragma unroll
              for (int i = 0; i < V; ++i) {
                if (!rows.on(j, i)) continue;
                const int col = rows.piece(j) * V + i;
                const float sum = turn ? shared_parts[part * a.C + col] + x[j * V + i] : x[j * V + i];
                (last ? to : shared_parts)[part * a.C + col] = sum;
              }
            ++part;
          };
          if (HASN) leave(PG, pG), leave(PO, pO);
          if (HASY) leave(PE, pE);
          if (HASN && TAN) leave(PtG, ptG), leave(PtO, ptO);
          if (HASY && TAN) leave(PtE, ptE);
        }
        if (lay.teams > 1) __syncthreads();
      }
    }
    cp_async_wait<0>();  // (groups without rows)
  }
}

constexpr int kDoesNotFit = 1;

template <typename T, int E, Way WAY, bool TAN, bool HASY, bool HASN, int BOUND>
int launch_bwd(const jvpfa_norm_args& a, const Cut& cut, bool aligned, cudaStream_t s) {
  constexpr int NC = E * (int)sizeof(T) / 16, SIDES = TAN ? 2 : 1;
  const auto kernel = norm_bwd_kernel<T, NC, WAY, TAN, HASY, HASN, BOUND>;
  static SmemOptIn opt;
  static int registers = 0;
  const Layout lay = layout_of(a, WAY, E, BOUND, registers_of(kernel, registers), SIDES * ((HASY ? 3 : 1) + (HASN ? 1 : 0)), SIDES * (HASY ? 2 : 1), cut.n_parts,
                               WAY == DIRECT ? 0 : SIDES * ((HASY ? 1 : 0) + (HASN ? 1 : 0)));
  if (lay.depth < 1) return kDoesNotFit;
  if (!opt.ensure(reinterpret_cast<const void*>(kernel), 225 * 1024)) return JVPFA_ERR_CUDA;
  const long long units = (long long)cut.groups * cut.slices, most = kSMs * lay.ctas;
  kernel<<<(unsigned)(units < most ? units : most), lay.threads * lay.teams, lay.bytes, s>>>(a, wide_vectors(a), lay, aligned, cut);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "norm_bwd_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
}

// Entries of a thread: 8 with tangents or with the sum and its norm, else 16 of rows that give them to a whole warp; threads have 170 registers
// with 16 entries or tangents, where a row takes at most 384 of them, else 128.  (us at 8 / 16 entries, 512 threads / 16 and 384: the norm of
// fp16 3990 x 2731 rows 58 / 46 / 43, bf16 8192 x 4096 with sum and both norms 121 / 165 / 149, where 16 entries and their sums leave the
// registers or, with 384 threads, one row in work on an SM.)  With tangents 16 from 4097 columns on, and 32 of any row from 8193 on, which
// registers hold in part alone: 0.3 to 3.5 KB of a thread are in local memory with 16, 0.5 to 7.5 with 32 (bf16 2048 rows with tangents, the norm / sum and
// both norms: 4096 columns 34 / 121 us; 4104 77 / 303, with 32 entries in 64 registers 336 / 1065; 8192 110 / 527, so 495 / 1499; 8200 287 / 1343).
template <typename T, Way WAY, bool TAN, bool HASY, bool HASN>
int launch_bwd(const jvpfa_norm_args& a, const Cut& c, bool al, cudaStream_t s) {
  if constexpr (WAY == DIRECT) {
    if (a.C <= 8192) return launch_bwd<T, 16, WAY, TAN, HASY, HASN, 512>(a, c, al, s);
    return launch_bwd<T, 32, WAY, TAN, HASY, HASN, 512>(a, c, al, s);
  } else if constexpr (TAN) {
    if (a.C <= 8 * 384) return launch_bwd<T, 8, WAY, TAN, HASY, HASN, 384>(a, c, al, s);
    if (a.C <= 4096) return launch_bwd<T, 8, WAY, TAN, HASY, HASN, 512>(a, c, al, s);
    return a.C <= 8192 ? launch_bwd<T, 16, WAY, TAN, HASY, HASN, 512>(a, c, al, s) : kDoesNotFit;
  } else {
    if (a.C <= 256 || (HASY && HASN && a.C <= 4096)) return launch_bwd<T, 8, WAY, TAN, HASY, HASN, 512>(a, c, al, s);
    if (a.C <= 16 * 384) return launch_bwd<T, 16, WAY, TAN, HASY, HASN, 384>(a, c, al, s);
    return a.C <= 8192 ? launch_bwd<T, 16, WAY, TAN, HASY, HASN, 512>(a, c, al, s) : kDoesNotFit;
  }
}

template <typename T, Way WAY>
int launch_bwd(const jvpfa_norm_args& a, const Cut& c, bool al, cudaStream_t s) {
  const bool y = a.y != nullptr, n = a.kind != JVPFA_NORM_NONE;
  if (a.dual)
    return !y ? launch_bwd<T, WAY, true, false, true>(a, c, al, s) : n ? launch_bwd<T, WAY, true, true, true>(a, c, al, s) : launch_bwd<T, WAY, true, true, false>(a, c, al, s);
  return !y ? launch_bwd<T, WAY, false, false, true>(a, c, al, s) : n ? launch_bwd<T, WAY, false, true, true>(a, c, al, s) : launch_bwd<T, WAY, false, true, false>(a, c, al, s);
}

template <typename T>
int launch_bwd(const jvpfa_norm_args& a, const Cut& c, cudaStream_t s) {
  const bool aligned = aligned_rows(a);
  const int rc = aligned ? launch_bwd<T, ALIGNED>(a, c, true, s) : launch_bwd<T, RAGGED>(a, c, false, s);
  return rc == kDoesNotFit ? launch_bwd<T, DIRECT>(a, c, aligned, s) : rc;
}

}  // namespace norms
}  // namespace jvpfa

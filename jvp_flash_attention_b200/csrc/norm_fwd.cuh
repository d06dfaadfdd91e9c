// Value and tangent of the residual sum and the norm behind it (norm_common.cuh has the formulas), one pass over the rows.
//
// A row is held in the registers of 32 to 512 threads, 8 to 32 entries each, from its load to its store; its means are sums over these
// threads, the variance about the mean in a second one (a first pass's sum of squares loses what a large mean has).  CTAs take a part of one
// group's rows, several rows at once, with the group's vectors put together in shared memory, and up to four rows of each are under way while one
// is worked on.  What bounds it: memory, each tensor read and written once, as long as a thread has entries enough: sums, addresses and
// waits of a row cost it about 250 instructions, its own work 10 an entry.  bf16 8192 x 4096 with both norms 47 us (268 MB at 5.7 TB/s, 87 % of a copy); 8192 x 1024 with
// tangents the norm 23 and with the residual sum 31 (134 MB); fp16 3990 x 2731, rows that begin anywhere, 24.
#pragma once
#include "norm_common.cuh"

namespace jvpfa {
namespace norms {

template <typename T, int NC, Way WAY, bool TAN, bool HASY, bool HASN>
__global__ void __launch_bounds__(512) norm_fwd_kernel(const __grid_constant__ jvpfa_norm_args a, const Wide wide, const Layout lay, const bool aligned, const int slices) {
  constexpr int V = 16 / (int)sizeof(T), E = V * NC, TENSORS = (HASY ? 2 : 1) * (TAN ? 2 : 1);
  extern __shared__ __align__(16) unsigned char smem[];
  const Team team{(int)threadIdx.x / lay.threads, lay.threads, (int)threadIdx.x % lay.threads};
  unsigned char* mine = smem + team.index * lay.team_bytes;
  RowSum row_sum{reinterpret_cast<float*>(mine), team};
  unsigned char* ring = mine + kSumFloats * 4;
  unsigned char* outs = ring + lay.depth * TENSORS * lay.slot;
  // the vectors of the group in work, put together: E, tE, G, tG, O, tO
  constexpr int SIDES = TAN ? 2 : 1, VECTORS = SIDES * ((HASY ? 1 : 0) + (HASN ? 2 : 0)), AT_G = HASY ? SIDES : 0, AT_O = AT_G + SIDES;
  float* vectors = reinterpret_cast<float*>(smem + lay.teams * lay.team_bytes);
  const int padded = (a.C + V - 1) / V * V;
  const Rows<T, NC, WAY> rows{a.C, a.M, team, aligned};
  const Source sources[4] = {{a.x, a.x_stride}, {HASY ? a.y : a.tx, HASY ? a.y_stride : a.tx_stride}, {a.tx, a.tx_stride}, {a.ty, a.ty_stride}};
  constexpr int kTx = HASY ? 2 : 1;
  const float by = 1.f / a.C;
  const bool layer = a.kind == JVPFA_NORM_LAYER, post_layer = a.post == JVPFA_NORM_LAYER, post = a.post != JVPFA_NORM_NONE;

  const long long units = (long long)(a.M / a.group_rows) * slices;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
  const int group = (int)(unit / slices), slice = (int)(unit - (long long)group * slices);
  const int first = (int)(group * a.group_rows + (long long)a.group_rows * slice / slices) + team.index;
  const int end = (int)(group * a.group_rows + (long long)a.group_rows * (slice + 1) / slices);
  auto fetch = [&](unsigned char* to, int row) {
    if (row < end) {
#pragma unroll
      for (int k = 0; k < TENSORS; ++k) rows.fetch(to + k * lay.slot, sources[k], row);
    }
    cp_async_commit();
  };
  if (WAY != DIRECT) {
    for (int k = 0; k < lay.depth; ++k) fetch(ring + k * TENSORS * lay.slot, first + k * lay.teams);
    __syncthreads();  // everybody has read the vectors of the unit before
    for (int col = threadIdx.x * V; col < a.C; col += blockDim.x * V) {
      float x[6][V];
      if (HASY) gate_of<T, V, TAN>(a, wide, group, col, x[0], x[1]);
      if (HASN) gain_of<T, V, TAN>(a, wide, group, col, x[AT_G], x[AT_O], x[AT_G + 1], x[AT_O + 1]);
#pragma unroll
      for (int k = 0; k < VECTORS; ++k)
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(rows.place(vectors + k * padded, col / V, i)) = make_float4(x[k][i], x[k][i + 1], x[k][i + 2], x[k][i + 3]);
    }
    __syncthreads();
  }
  // piece j of one of them
  auto vector = [&](float* to, int which, int j) { rows.vector(to, vectors + which * padded, j); };
  unsigned char* slot = ring;  // of the row in work; the one that follows as many rows behind as the ring has takes it next
  for (int row = first; row < end; row += lay.teams) {
    float r[E], tr[TAN ? E : 1], m[HASY ? E : 1], tm[TAN && HASY ? E : 1];
    if (WAY != DIRECT) wait_rows(lay.depth);
    if (WAY == RAGGED) team.sync();
    {
      Pieces<T, NC> raw[TENSORS];
#pragma unroll
      for (int k = 0; k < TENSORS; ++k) rows.read(raw[k], slot + k * lay.slot, sources[k], row);
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
    if (WAY != DIRECT) {
      fetch(slot, row + lay.depth * lay.teams);
      slot += TENSORS * lay.slot;
      if (slot == outs) slot = ring;
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
        float gate[V], tgate[V];
        if (WAY == DIRECT) {
          gate_of<T, V, TAN>(a, wide, group, rows.piece(j) * V, gate, tgate);
        } else {
          vector(gate, 0, j);
          if (TAN) vector(tgate, 1, j);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = j * V + i;
          r[e] += gate[i] * m[e];
          if (TAN) tr[e] += tgate[i] * m[e] + gate[i] * tm[e];
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
        float gain[V], offset[V], tgain[V], toffset[V];
        if (WAY == DIRECT) {
          gain_of<T, V, TAN>(a, wide, group, rows.piece(j) * V, gain, offset, tgain, toffset);
        } else {
          vector(gain, AT_G, j), vector(offset, AT_O, j);
          if (TAN) vector(tgain, AT_G + 1, j), vector(toffset, AT_O + 1, j);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = j * V + i;
          if (TAN) tr[e] = tr[e] * gain[i] + (r[e] * tgain[i] + toffset[i]);
          r[e] = r[e] * gain[i] + offset[i];
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
  cp_async_wait<0>();  // (groups without rows)
  }
}

constexpr int kDoesNotFit = 1;

template <typename T, int E, Way WAY, bool TAN, bool HASY, bool HASN>
int launch_fwd(const jvpfa_norm_args& a, bool aligned, cudaStream_t s) {
  constexpr int NC = E * (int)sizeof(T) / 16, SIDES = TAN ? 2 : 1;
  const auto kernel = norm_fwd_kernel<T, NC, WAY, TAN, HASY, HASN>;
  static SmemOptIn opt;
  static int registers = 0;
  const Layout lay = layout_of(a, WAY, E, 512, registers_of(kernel, registers), SIDES * (HASY ? 2 : 1), SIDES * (HASY && HASN ? 2 : 1), 0,
                               WAY == DIRECT ? 0 : SIDES * ((HASY ? 1 : 0) + (HASN ? 2 : 0)));
  if (lay.depth < 1) return kDoesNotFit;
  if (!opt.ensure(reinterpret_cast<const void*>(kernel), 225 * 1024)) return JVPFA_ERR_CUDA;
  // parts of each group's rows: together as many as CTAs, and a row for each of a CTA's at least
  const long long groups = a.M / a.group_rows, most = (long long)kSMs * lay.ctas, least = (a.group_rows + lay.teams - 1) / lay.teams;
  long long slices = most / groups;
  slices = slices < 1 ? 1 : slices > least ? least : slices;
  const long long units = groups * slices;
  kernel<<<(unsigned)(units < most ? units : most), lay.threads * lay.teams, lay.bytes, s>>>(a, wide_vectors(a), lay, aligned, (int)slices);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "norm_fwd_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
}

// Entries of a thread: as many as leave a row a whole warp, up to 32, with tangents up to 16; 8 where every row has an SM and the time is one row's.
// (us at 8 / 16 / 32 entries: bf16 8192 x 4096 with sum and both norms 76 / 57 / 49, fp16 3990 x 2731 47 / 31 / 24, bf16 8192 x 1024 with tangents
// 24.5 / 22.4, eight rows of 1024 3.4 / 3.8 / 4.7.)
template <typename T, Way WAY, bool TAN, bool HASY, bool HASN>
int launch_fwd(const jvpfa_norm_args& a, bool al, cudaStream_t s) {
  if constexpr (WAY == DIRECT) {
    return launch_fwd<T, 32, WAY, TAN, HASY, HASN>(a, al, s);
  } else {
    if (a.C <= 256 || (a.M <= kSMs && a.C <= 4096)) return launch_fwd<T, 8, WAY, TAN, HASY, HASN>(a, al, s);
    if (TAN || a.C <= 512) return a.C <= 8192 ? launch_fwd<T, 16, WAY, TAN, HASY, HASN>(a, al, s) : kDoesNotFit;
    if constexpr (!TAN) return launch_fwd<T, 32, WAY, TAN, HASY, HASN>(a, al, s);
  }
  return kDoesNotFit;
}

template <typename T, Way WAY>
int launch_fwd(const jvpfa_norm_args& a, bool al, cudaStream_t s) {
  const bool y = a.y != nullptr, n = a.kind != JVPFA_NORM_NONE;
  if (a.dual)
    return !y ? launch_fwd<T, WAY, true, false, true>(a, al, s) : n ? launch_fwd<T, WAY, true, true, true>(a, al, s) : launch_fwd<T, WAY, true, true, false>(a, al, s);
  return !y ? launch_fwd<T, WAY, false, false, true>(a, al, s) : n ? launch_fwd<T, WAY, false, true, true>(a, al, s) : launch_fwd<T, WAY, false, true, false>(a, al, s);
}

template <typename T>
int launch_fwd(const jvpfa_norm_args& a, cudaStream_t s) {
  const bool aligned = aligned_rows(a);
  const int rc = aligned ? launch_fwd<T, ALIGNED>(a, true, s) : launch_fwd<T, RAGGED>(a, false, s);
  return rc == kDoesNotFit ? launch_fwd<T, DIRECT>(a, aligned, s) : rc;
}

}  // namespace norms
}  // namespace jvpfa

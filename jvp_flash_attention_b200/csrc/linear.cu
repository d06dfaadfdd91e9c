// Entries of linear attention: argument checks, the cut of long sequences into segments, the launches that the outputs and gradients are made
// of, and the form for one more token.
#include "linear_common.cuh"

namespace jvpfa {
namespace linear {

namespace {

constexpr int kMostSegments = 128;

template <int V>
struct alignas(4 * V) Entries { float x[V]; };

int launch_of_type(const Scan& s, bool outputs, cudaStream_t stream) {
  if (s.dtype == JVPFA_FP32) return launch_scan(s, outputs, stream);
  return s.dtype == JVPFA_BF16 ? launch_chunks<__nv_bfloat16>(s, outputs, stream) : launch_chunks<__half>(s, outputs, stream);
}

// The states that the segments begin with, from those that each one's own rows leave, in place and segment after segment; V successive entries of M
// a thread, value or tangent.  Memory-bound, though what it reads was just written and is in L2: B4 H16 L8192 D128 in 9
// segments, 38 MB read and written, 14 us (an entry a thread: 33).
template <int V>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Scan p) {
  __shared__ Down down[kMostSegments];
  const int size = p.D * p.E, head = blockIdx.x, b = head / p.H, h = head - b * p.H, which = blockIdx.z;
  const int n = length_of(p.lengths, b, p.L);
  const float w = decay_of(p.log_decay, h);
  for (int s = threadIdx.x; s < p.segments; s += 256) {
    const int rows = max(0, min(n - s * p.segment, p.segment)) + (s == 0 ? p.ahead - 1 : 0);
    down[s] = down_of(expf(w * rows), expm1f(w * rows));
  }
  __syncthreads();
  const int i = (blockIdx.y * 256 + threadIdx.x) * V;
  if (i >= size) return;
  float x[V];
  const float* first = which ? p.tfirst : p.first;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int d = (i + v) / p.E, e = i + v - d * p.E;
    x[v] = first ? p.first_scale * first[(long long)head * size + d * p.first_stride[0] + e * p.first_stride[1]] : 0.f;
  }
  float* at = (which ? p.tstates : p.states) + (long long)head * p.segments * size + i;
  constexpr int AHEAD = 8;  // loads under way at once
  for (int s0 = 0; s0 < p.segments; s0 += AHEAD, at += AHEAD * (long long)size) {
    Entries<V> own[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (s0 + k + 1 < p.segments) own[k] = *reinterpret_cast<const Entries<V>*>(at + k * (long long)size);  // (the last one's is nobody's)
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (s0 + k >= p.segments) break;
      Entries<V> begin;
#pragma unroll
      for (int v = 0; v < V; ++v) begin.x[v] = x[v];
      *reinterpret_cast<Entries<V>*>(at + k * (long long)size) = begin;
      if (s0 + k + 1 < p.segments) {
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = fmaf(x[v], down[s0 + k].by, fmaf(x[v], down[s0 + k].keep, own[k].x[v]));
      }
    }
  }
}

// Rows of a segment and segments (1: no workspace).
void cut(Scan& s) {
  // Rounds of as many CTAs as SMs hold at once, each of a segment's rows, and the states that a segment costs, about 3/1000 of a sequence; no
  // segment below 128 rows.  (us by segments, those of the rule marked: bf16 B4 H16 L2048 D64 with tangents and gradients 4* / 6 / 8 / 11: 407 / 550 / 431 /
  // 467; L8192 D128 forward and backward 4 / 6 / 8 / 9* / 16: 1587 / 1714 / 1615 / 1533 / 1510; fp32 B2 H8 L1023 D128 with tangents 4 / 6 / 8*: 363 / 281 / 218;
  // B4 H16 L2048 D64 with tangents and gradients 4 / 6 / 11 / 16*: 2202 / 2461 / 2110 / 2041, without tangents 4 / 6* / 8 / 11: 715 / 687 / 698 / 670.)
  const int heads = s.B * s.H, width = s.D > s.E ? s.D : s.E, chunk = s.dtype == JVPFA_FP32 && width > 64 ? 32 : 64;
  const int room = kSMs * (s.dtype == JVPFA_FP32 ? scan_ctas(s) : s.dtype == JVPFA_BF16 ? chunk_ctas<__nv_bfloat16>(s) : chunk_ctas<__half>(s));
  s.segments = 1, s.segment = s.L;
  double least = 1e30;
  for (int n = 1; n <= kMostSegments; ++n) {
    const int rows = ((s.L + n - 1) / n + chunk - 1) / chunk * chunk, segments = (s.L + rows - 1) / rows;
    if (n > 1 && rows < 128) break;
    const long long rounds = ((long long)heads * segments + room - 1) / room;
    const double cost = (double)rounds * rows + 0.003 * s.L * segments;
    if (cost < least) least = cost, s.segments = segments, s.segment = segments > 1 ? rows : s.L;
  }
}

// `found`: the segments' states are there already.
int launch(const Scan& s, cudaStream_t stream, bool found = false) {
  if (s.segments > 1 && !found) {
    const int rc = launch_of_type(s, false, stream);
    if (rc) return rc;
    const bool wide = s.D * s.E % 4 == 0;  // (the workspace begins on 16 bytes)
    const int each = wide ? 1024 : 256;
    const dim3 grid((unsigned)(s.B * s.H), (unsigned)((s.D * s.E + each - 1) / each), s.dual ? 2 : 1);
    if (wide)
      join_kernel<4><<<grid, 256, 0, stream>>>(s);
    else
      join_kernel<1><<<grid, 256, 0, stream>>>(s);
  }
  return launch_of_type(s, true, stream);
}

// ---- one more token ------------------------------------------------------------------------------------------------------
// S = l S + k v^T and o = scale S^T q, a CTA for `cols` columns of one head's state, V of them a thread.  Memory-bound: the state is read and
// written once, in 16-byte pieces, eight of a thread under way: B256 H16 D128 (537 MB) 84 us, 6.4 TB/s.
constexpr int kStepThreads = 256;

__device__ __forceinline__ float load_as(const void* p, long long at, int dtype) {
  if (dtype == JVPFA_FP32) return static_cast<const float*>(p)[at];
  return dtype == JVPFA_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]) : __half2float(static_cast<const __half*>(p)[at]);
}

template <int V>
__global__ void __launch_bounds__(kStepThreads) step_kernel(const __grid_constant__ jvpfa_linear_step_args a, const int cols) {
  __shared__ float sq[128], sk[128], part[kStepThreads * 4];
  const int tid = threadIdx.x, b = blockIdx.x / a.H, h = blockIdx.x - b * a.H;
  const int lanes = cols / V, row_step = kStepThreads / lanes;  // threads along a row, rows at once
  const int row0 = tid / lanes, e = blockIdx.y * cols + tid % lanes * V;
  const bool live = row0 < row_step && e < a.E;
  for (int d = tid; d < a.D; d += kStepThreads) {
    sq[d] = a.scale * load_as(a.q, b * a.q_stride[0] + h * a.q_stride[1] + d, a.dtype);
    sk[d] = load_as(a.k, b * a.k_stride[0] + h * a.k_stride[1] + d, a.dtype);
  }
  const float w = decay_of(a.log_decay, h);
  const Down down = down_of(expf(w), expm1f(w));
  float v[V], o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    v[i] = live ? load_as(a.v, b * a.v_stride[0] + h * a.v_stride[1] + e + i, a.dtype) : 0.f;
    o[i] = 0.f;
  }
  __syncthreads();
  float* state = a.state + b * a.state_stride[0] + h * a.state_stride[1] + e;
  if (live) {
    constexpr int AHEAD = 8;
    for (int d0 = row0; d0 < a.D; d0 += AHEAD * row_step) {
      float s[AHEAD][V];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int d = d0 + j * row_step;
        if (d >= a.D) break;
        if constexpr (V == 4) {
          const float4 x = *reinterpret_cast<const float4*>(state + (long long)d * a.E);
          s[j][0] = x.x, s[j][1] = x.y, s[j][2] = x.z, s[j][3] = x.w;
        } else {
          s[j][0] = state[(long long)d * a.E];
        }
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int d = d0 + j * row_step;
        if (d >= a.D) break;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          s[j][i] = fmaf(s[j][i], down.by, fmaf(s[j][i], down.keep, sk[d] * v[i]));
          o[i] += sq[d] * s[j][i];
        }
        if constexpr (V == 4)
          *reinterpret_cast<float4*>(state + (long long)d * a.E) = make_float4(s[j][0], s[j][1], s[j][2], s[j][3]);
        else
          state[(long long)d * a.E] = s[j][0];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) part[tid * V + i] = o[i];
  __syncthreads();
  // part: [row0][column of the CTA]
  for (int c = tid; c < cols; c += kStepThreads) {
    const int col = blockIdx.y * cols + c;
    if (col >= a.E) continue;
    float s = 0.f;
    for (int r = 0; r < row_step; ++r) s += part[(r * lanes + c / V) * V + c % V];
    const long long at = ((long long)b * a.H + h) * a.E + col;
    if (a.dtype == JVPFA_FP32)
      static_cast<float*>(a.o)[at] = s;
    else if (a.dtype == JVPFA_BF16)
      static_cast<__nv_bfloat16*>(a.o)[at] = __float2bfloat16_rn(s);
    else
      static_cast<__half*>(a.o)[at] = __float2half_rn(s);
  }
}

// ---- checks --------------------------------------------------------------------------------------------------------------
bool bad_dtype(int dtype) { return dtype != JVPFA_BF16 && dtype != JVPFA_FP16 && dtype != JVPFA_FP32; }

int bad_sizes(const jvpfa_linear_args& a) {
  if (bad_dtype(a.dtype)) return JVPFA_ERR_DTYPE;
  if (a.B < 1 || a.H < 1 || a.L < 1 || a.D < 1 || a.E < 1 || a.D > 128 || a.E > 128) return JVPFA_ERR_SHAPE;
  return (long long)a.B * a.H > (1 << 24) || a.L > (1 << 30) ? JVPFA_ERR_TOO_LARGE : JVPFA_OK;  // (a chunk behind the last row is counted in 32 bits)
}

int check(const jvpfa_linear_args* a, bool backward) {
  if (!a) return JVPFA_ERR_NULL;
  if (a->struct_size != (int32_t)sizeof(jvpfa_linear_args)) return JVPFA_ERR_STRUCT;
  if (const int rc = bad_sizes(*a)) return rc;
  // (backwards, the cotangents of the last state are divided by the scale)
  if (!(fabsf(a->scale) <= 0x1p64f) || (backward && fabsf(a->scale) < 0x1p-64f && (a->gstate || a->gtstate))) return JVPFA_ERR_UNSUPPORTED;
  if (!a->q.p || !a->k.p || !a->v.p) return JVPFA_ERR_NULL;
  if (!a->dual && (a->tq.p || a->tk.p || a->tv.p || a->tstate || a->to.p || a->tstate_out || a->gto.p || a->gtstate || a->dtq.p || a->dtk.p || a->dtv.p || a->dtstate))
    return JVPFA_ERR_NULL;
  if (!backward && (!a->o.p || (a->dual && !a->to.p))) return JVPFA_ERR_NULL;
  if (backward && !a->state && a->dstate) return JVPFA_ERR_NULL;
  const uintptr_t size = a->dtype == JVPFA_FP32 ? 4 : 2;
  for (const jvpfa_linear_tensor* x : {&a->q, &a->k, &a->v, &a->tq, &a->tk, &a->tv, &a->o, &a->to, &a->go, &a->gto, &a->dq, &a->dk, &a->dv, &a->dtq, &a->dtk, &a->dtv}) {
    if (!x->p) continue;
    if (reinterpret_cast<uintptr_t>(x->p) % size) return JVPFA_ERR_ALIGN;
    for (int64_t st : x->stride)
      if (st < 0) return JVPFA_ERR_SHAPE;
  }
  for (const void* p : {(const void*)a->state, (const void*)a->tstate, (const void*)a->state_out, (const void*)a->tstate_out, (const void*)a->gstate,
                        (const void*)a->gtstate, (const void*)a->dstate, (const void*)a->dtstate, (const void*)a->log_decay, (const void*)a->lengths})
    if (reinterpret_cast<uintptr_t>(p) % 4) return JVPFA_ERR_ALIGN;
  return JVPFA_OK;
}

// A scan with the call's sizes; D and E are those of its a and c.  cut_dual: cut as a call with tangents, or without, is.
Scan scan_of(const jvpfa_linear_args& a, int D, int E, bool cut_dual) {
  Scan s{};
  s.dtype = a.dtype, s.B = a.B, s.H = a.H, s.L = a.L, s.D = D, s.E = E;
  s.scale = a.scale, s.dual = a.dual != 0;
  s.log_decay = a.log_decay, s.lengths = a.lengths;
  s.first_scale = s.last_scale = 1.f, s.ahead = 1;
  s.first_stride[0] = s.last_stride[0] = s.state_stride[0] = E, s.first_stride[1] = s.last_stride[1] = s.state_stride[1] = 1;
  s.dual = cut_dual;
  cut(s);
  s.dual = a.dual != 0;
  return s;
}
// Where the segments' states are; `transposed`: as those of the map with b and c changed for one another.
void put_states(Scan& s, void* at, bool transposed = false) {
  s.states = static_cast<float*>(at);
  s.tstates = s.states + (size_t)s.B * s.H * s.segments * s.D * s.E;
  if (transposed) s.state_stride[0] = 1, s.state_stride[1] = s.D;
}
int64_t states_of(const jvpfa_linear_args& a) { return state_bytes(scan_of(a, a.D, a.E, a.dual != 0)) * (a.dual ? 2 : 1); }
// What the forward needs is nothing where it keeps its states.
int64_t workspace_bytes(const jvpfa_linear_args& a, bool backward) { return !backward && a.kept ? 0 : states_of(a); }

}  // namespace
}  // namespace linear
}  // namespace jvpfa

using namespace jvpfa;

extern "C" {

int64_t jvpfa_linear_fwd_workspace(const jvpfa_linear_args* a) { return linear::check(a, false) == JVPFA_OK ? linear::workspace_bytes(*a, false) : 0; }
int64_t jvpfa_linear_bwd_workspace(const jvpfa_linear_args* a) { return linear::check(a, true) == JVPFA_OK ? linear::workspace_bytes(*a, true) : 0; }
int64_t jvpfa_linear_kept_bytes(const jvpfa_linear_args* a) {
  if (!a || a->struct_size != (int32_t)sizeof(jvpfa_linear_args) || linear::bad_sizes(*a) != JVPFA_OK) return 0;
  return linear::states_of(*a);
}

int jvpfa_linear_fwd(const jvpfa_linear_args* a, void* stream) {
  int rc = linear::check(a, false);
  if (rc) return rc;
  const int64_t need = linear::workspace_bytes(*a, false);
  if (need && (!a->workspace || a->workspace_bytes < need)) return JVPFA_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(a->workspace) | reinterpret_cast<uintptr_t>(a->kept)) % 16) return JVPFA_ERR_ALIGN;
  rc = check_arch();
  if (rc) return rc;
  linear::Scan s = linear::scan_of(*a, a->D, a->E, a->dual != 0);
  s.a = a->q, s.b = a->k, s.c = a->v, s.ta = a->tq, s.tb = a->tk, s.tc = a->tv, s.out = a->o, s.tout = a->to;
  s.first = a->state, s.tfirst = a->tstate, s.last = a->state_out, s.tlast = a->tstate_out;
  linear::put_states(s, a->kept ? a->kept : a->workspace);
  return linear::launch(s, static_cast<cudaStream_t>(stream));
}

int jvpfa_linear_bwd(const jvpfa_linear_args* a, void* stream) {
  int rc = linear::check(a, true);
  if (rc) return rc;
  const int64_t need = linear::workspace_bytes(*a, true);
  if (need && (!a->workspace || a->workspace_bytes < need)) return JVPFA_ERR_NULL;
  if (a->kept && a->dual && !a->kept_dual) return JVPFA_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(a->workspace) | reinterpret_cast<uintptr_t>(a->kept)) % 16) return JVPFA_ERR_ALIGN;
  rc = check_arch();
  if (rc) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // With tangents the maps' value has gto for its cotangent and gives the tangents' gradients, and their tangent has go and gives the others.
  const bool dual = a->dual != 0;
  const jvpfa_linear_tensor none{}, &g = dual ? a->gto : a->go, &tg = dual ? a->go : none;
  auto value = [&](const jvpfa_linear_tensor& d, const jvpfa_linear_tensor& dt) -> const jvpfa_linear_tensor& { return dual ? dt : d; };
  auto tangent = [&](const jvpfa_linear_tensor& d) -> const jvpfa_linear_tensor& { return dual ? d : none; };
  if (a->dq.p || a->dtq.p) {
    linear::Scan s = linear::scan_of(*a, a->E, a->D, a->kept ? a->kept_dual != 0 : dual);
    s.a = g, s.ta = tg, s.b = a->v, s.tb = a->tv, s.c = a->k, s.tc = a->tk;
    s.out = value(a->dq, a->dtq), s.tout = tangent(a->dq);
    s.first = a->state, s.tfirst = a->tstate, s.first_stride[0] = 1, s.first_stride[1] = a->E;
    linear::put_states(s, a->kept ? a->kept : a->workspace, a->kept != nullptr);  // (the forward's are those of (k, v))
    rc = linear::launch(s, st, a->kept != nullptr);
    if (rc) return rc;
  }
  // Backwards, M begins with the cotangent of the last state, which the scale does not go with.
  const float* first = dual ? a->gtstate : a->gstate;
  const float* tfirst = dual ? a->gstate : nullptr;
  const float unscaled = first || tfirst ? 1.f / a->scale : 1.f;
  const bool keys = a->dk.p || a->dtk.p || a->dstate || a->dtstate;
  if (keys) {
    linear::Scan s = linear::scan_of(*a, a->E, a->D, dual);
    s.reversed = true, s.ahead = 0, s.last_ahead = 1, s.first_scale = unscaled, s.last_scale = a->scale;
    s.a = a->v, s.ta = a->tv, s.b = g, s.tb = tg, s.c = a->q, s.tc = a->tq;
    s.out = value(a->dk, a->dtk), s.tout = tangent(a->dk);
    s.first = first, s.tfirst = tfirst, s.first_stride[0] = 1, s.first_stride[1] = a->E;
    s.last = dual ? a->dtstate : a->dstate, s.tlast = dual ? a->dstate : nullptr, s.last_stride[0] = 1, s.last_stride[1] = a->E;
    linear::put_states(s, a->workspace);
    rc = linear::launch(s, st);
    if (rc) return rc;
  }
  if (a->dv.p || a->dtv.p) {
    linear::Scan s = linear::scan_of(*a, a->D, a->E, dual);
    s.reversed = true, s.ahead = 0, s.first_scale = unscaled;
    s.a = a->k, s.ta = a->tk, s.b = a->q, s.tb = a->tq, s.c = g, s.tc = tg;
    s.out = value(a->dv, a->dtv), s.tout = tangent(a->dv);
    s.first = first, s.tfirst = tfirst;
    linear::put_states(s, a->workspace, keys);  // (the keys' are those of (go, q))
    rc = linear::launch(s, st, keys);
    if (rc) return rc;
  }
  return JVPFA_OK;
}

int jvpfa_linear_step(const jvpfa_linear_step_args* a, void* stream) {
  if (!a) return JVPFA_ERR_NULL;
  if (a->struct_size != (int32_t)sizeof(jvpfa_linear_step_args)) return JVPFA_ERR_STRUCT;
  if (linear::bad_dtype(a->dtype)) return JVPFA_ERR_DTYPE;
  if (a->B < 1 || a->H < 1 || a->D < 1 || a->E < 1 || a->D > 128 || a->E > 128) return JVPFA_ERR_SHAPE;
  if ((long long)a->B * a->H > (1 << 24)) return JVPFA_ERR_TOO_LARGE;
  if (!a->q || !a->k || !a->v || !a->o || !a->state) return JVPFA_ERR_NULL;
  const uintptr_t size = a->dtype == JVPFA_FP32 ? 4 : 2;
  for (const void* p : {a->q, a->k, a->v, (const void*)a->o})
    if (reinterpret_cast<uintptr_t>(p) % size) return JVPFA_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(a->state) % 4 || reinterpret_cast<uintptr_t>(a->log_decay) % 4) return JVPFA_ERR_ALIGN;
  for (const int64_t* st : {a->q_stride, a->k_stride, a->v_stride, a->state_stride})
    if (st[0] < 0 || st[1] < 0) return JVPFA_ERR_SHAPE;
  // two heads of one state would race
  const int64_t one = (int64_t)a->D * a->E;
  const int64_t sb = a->state_stride[0], sh = a->state_stride[1];
  if ((a->H > 1 && sh < one) || (a->B > 1 && sb < one) || (a->B > 1 && a->H > 1 && (sb > sh ? sb < (a->H - 1) * sh + one : sh < (a->B - 1) * sb + one)))
    return JVPFA_ERR_SHAPE;
  const int rc = check_arch();
  if (rc) return rc;
  uint64_t all = reinterpret_cast<uint64_t>(a->state) | (uint64_t)a->E * 4;
  if (a->B > 1) all |= (uint64_t)sb * 4;
  if (a->H > 1) all |= (uint64_t)sh * 4;
  const bool wide = all % 16 == 0;
  // columns of a CTA: all, or 32 where the heads do not fill the SMs
  const int padded = (a->E + 3) / 4 * 4;
  const int cols = a->B * a->H < linear::kSMs && padded > 32 ? 32 : padded;
  const dim3 grid((unsigned)(a->B * a->H), (unsigned)((a->E + cols - 1) / cols));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (wide)
    linear::step_kernel<4><<<grid, linear::kStepThreads, 0, s>>>(*a, cols);
  else
    linear::step_kernel<1><<<grid, linear::kStepThreads, 0, s>>>(*a, cols);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "step_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
}

}  // extern "C"

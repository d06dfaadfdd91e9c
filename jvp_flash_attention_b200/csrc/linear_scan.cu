// The map of linear_common.cuh for float32, on TF32 instructions: entries and what is formed of them are split in two (common.cuh).
//
// A CTA takes a segment of one head's rows, chunk by chunk.  Warp w keeps columns 16 w .. 16 w + 15 of M in registers, transposed (rows of the
// accumulator are columns of M), which as it stands is the second operand of a M.  The weighted products of a chunk go through shared
// memory, since every warp needs all of them.
// What bounds it: with tangents three products of three instructions each.  B2 H8 L1023 D128 with tangents takes 223 us in 8 segments, the outputs' tensor
// pipe 35 % busy and issue slots 24 % (two warps a scheduler: 255 registers, one CTA on an SM).  Beside the products it is the splitting of operands, which each warp does for itself.
#include "linear_common.cuh"

namespace jvpfa {
namespace linear {

namespace {

// Two TF32 numbers that add up to an operand.
struct Part {
  uint32_t hi, lo;
  __device__ __forceinline__ void set(float x) { split_tf32(x, hi, lo); }
};
// x = a b, from nothing.
__device__ __forceinline__ void mma_fresh(float x[4], const uint32_t a[4], const uint32_t b[2]) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
}
// c += a b.  The tensor cores truncate what they add to an accumulator, always towards zero: over the thousand steps of a long sequence that
// is 2e-6 of a state.  So each step's product is formed from nothing and added here, rounded to nearest (4 additions for up to three
// instructions; the state of 8192 rows is then off by 1e-7, the same sequence's results in float32 by 3e-7 instead of 4e-6).
__device__ __forceinline__ void mul(float c[4], const Part (&a)[4], const Part (&b)[2]) {
  const uint32_t ah[4] = {a[0].hi, a[1].hi, a[2].hi, a[3].hi}, al[4] = {a[0].lo, a[1].lo, a[2].lo, a[3].lo};
  const uint32_t bh[2] = {b[0].hi, b[1].hi}, bl[2] = {b[0].lo, b[1].lo};
  float x[4];
  mma_fresh(x, al, bh);
  mma_1688_tf32(x, ah, bl);
  mma_1688_tf32(x, ah, bh);
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] += x[i];
}

// Rows row0 .. row0 + ROWS - 1 (of `n` in all, `back`: counted from the end) of a head into shared memory, zeros behind the last one and behind
// the width, and for an absent tensor.
template <int ROWS, int DT, int LD, int NT>
__device__ __forceinline__ void stage(float* to, const jvpfa_linear_tensor& x, long long head, int width, int row0, int rows, int n, bool back, bool wide) {
  constexpr int V = 4;
  const float* from = static_cast<const float*>(x.p) + head;
  for (int i = threadIdx.x; i < ROWS * (DT / V); i += NT) {
    const int r = i / (DT / V), col = i % (DT / V) * V;
    const long long at = (long long)(back ? n - 1 - row0 - r : row0 + r) * x.stride[2] + col;
    float* d = to + r * LD + col;
    const bool live = x.p && r < rows && col < width;
    if (!live) {
      *reinterpret_cast<uint4*>(d) = make_uint4(0, 0, 0, 0);
    } else if (wide) {
      cp_async16(d, from + at, 16);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = col + j < width ? from[at + j] : 0.f;
    }
  }
}

template <int DT>
struct ScanShape {
  static constexpr int CH = DT == 128 ? 32 : 64;  // rows of a chunk
  static constexpr int NW = DT / 16, NT = 32 * NW;
  static constexpr int LD = DT + 4, LP = CH + 4;
  static constexpr size_t bytes(bool dual, bool outs) {
    return (dual ? 2 : 1) * (sizeof(float) * (size_t)CH * LD * (outs ? 3 : 2) + (outs ? sizeof(float) * (size_t)CH * LP : 0));
  }
  // CTAs of an SM: as its shared memory has room for (2 KB of each are the system's and the powers), one with D = 128, which takes all registers.
  static constexpr int ctas(bool dual) { return DT == 128 ? 1 : (int)(227 * 1024 / (bytes(dual, true) + 2048)); }
};

// OUT: the outputs, from the states that the segments begin with; else the states that their rows leave, from nothing.
template <int DT, bool DUAL, bool OUT>
__global__ void __launch_bounds__(2 * DT, ScanShape<DT>::ctas(DUAL)) scan_kernel(const __grid_constant__ Scan p, const uint32_t wide) {
  using S = ScanShape<DT>;
  constexpr int CH = S::CH, NT = S::NT, LD = S::LD, LP = S::LP, ND = DT / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float power[CH + 2], less1[CH + 2];  // l^j and l^j - 1
  float* sB = reinterpret_cast<float*>(smem);
  float* sC = sB + CH * LD;
  float* stB = sC + CH * LD;
  float* stC = stB + (DUAL ? CH * LD : 0);
  float* sA = stC + (DUAL ? CH * LD : 0);
  float* stA = sA + CH * LD;
  float* sP = reinterpret_cast<float*>(stA + (DUAL ? CH * LD : 0));
  float* stP = sP + CH * LP;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int segment = blockIdx.x % p.segments, head = blockIdx.x / p.segments, b = head / p.H, h = head - b * p.H;
  const int n = length_of(p.lengths, b, p.L), row_begin = segment * p.segment, row_end = min(n, row_begin + p.segment);
  if (!OUT && segment + 1 == p.segments) return;  // nobody begins with what the last one leaves
  const float w = decay_of(p.log_decay, h);
  for (int j = tid; j < CH + 2; j += NT) {
    power[j] = expf(w * j);  // (in 64 bits a CTA would wait 2 us for them; what w * j loses is at most 2^-24 |w j| e^(w j) of a result)
    less1[j] = expm1f(w * j);
  }
  auto of_head = [&](const jvpfa_linear_tensor& x) { return b * x.stride[0] + h * x.stride[1]; };
  const int e0 = warp * 16;
  const long long size = (long long)p.D * p.E;

  float M[ND][4], tM[DUAL ? ND : 1][4];
  auto each = [&](auto f) {  // (d tile, entry, row d and column e of M)
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) f(i, j, i * 8 + 2 * t + (j & 1), e0 + g + (j >> 1) * 8);
  };
  each([&](int i, int j, int d, int e) {
    float x = 0.f, y = 0.f;
    if (OUT && d < p.D && e < p.E) {
      if (p.segments > 1) {
        const long long at = ((long long)head * p.segments + segment) * size + d * p.state_stride[0] + e * p.state_stride[1];
        x = p.states[at];
        if (DUAL) y = p.tstates[at];
      } else {
        const long long at = head * size + d * p.first_stride[0] + e * p.first_stride[1];
        if (p.first) x = p.first_scale * p.first[at];
        if (DUAL && p.tfirst) y = p.first_scale * p.tfirst[at];
      }
    }
    M[i][j] = x;
    if (DUAL) tM[i][j] = y;
  });
  // The given state is l^ahead away from the first row, what the rows leave l^1.
  int shift = OUT && segment == 0 ? p.ahead - 1 : 0;

  for (int row0 = row_begin; row0 < row_end; row0 += CH, shift = 0) {
    const int rows = min(CH, row_end - row0);
    __syncthreads();  // the tiles have been read (and the powers written)
    stage<CH, DT, LD, NT>(sB, p.b, of_head(p.b), p.D, row0, rows, n, p.reversed, wide & 1);
    stage<CH, DT, LD, NT>(sC, p.c, of_head(p.c), p.E, row0, rows, n, p.reversed, wide & 2);
    if (OUT) stage<CH, DT, LD, NT>(sA, p.a, of_head(p.a), p.D, row0, rows, n, p.reversed, wide & 4);
    if (DUAL) {
      stage<CH, DT, LD, NT>(stB, p.tb, of_head(p.tb), p.D, row0, rows, n, p.reversed, wide & 8);
      stage<CH, DT, LD, NT>(stC, p.tc, of_head(p.tc), p.E, row0, rows, n, p.reversed, wide & 16);
      if (OUT) stage<CH, DT, LD, NT>(stA, p.ta, of_head(p.ta), p.D, row0, rows, n, p.reversed, wide & 32);
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    if constexpr (OUT) {
      // the chunk's products, 16 rows and 8 columns at a time
      constexpr int TM = CH / 16, TN = CH / 8;
      for (int tile = warp; tile < TM * TN; tile += S::NW) {
        const int r0 = tile / TN * 16, s0 = tile % TN * 8;
        float x[4] = {}, y[4] = {};
        if (s0 < r0 + 16) {
#pragma unroll 4
          for (int k = 0; k < DT; k += 8) {
            Part fa[4], fb[2];
            auto load_rows = [&](Part(&f)[4], const float* s) {
#pragma unroll
              for (int i = 0; i < 4; ++i) f[i].set(s[(r0 + g + (i & 1) * 8) * LD + k + t + (i >> 1) * 4]);
            };
            auto load_cols = [&](Part(&f)[2], const float* s) {
#pragma unroll
              for (int i = 0; i < 2; ++i) f[i].set(s[(s0 + g) * LD + k + t + i * 4]);
            };
            load_rows(fa, sA), load_cols(fb, sB);
            mul(x, fa, fb);
            if constexpr (DUAL) {
              Part fta[4], ftb[2];
              load_rows(fta, stA), load_cols(ftb, stB);
              mul(y, fta, fb), mul(y, fa, ftb);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = r0 + g + (i >> 1) * 8, s = s0 + 2 * t + (i & 1);
          sP[r * LP + s] = s <= r ? x[i] * power[r - s] : 0.f;
          if (DUAL) stP[r * LP + s] = s <= r ? y[i] * power[r - s] : 0.f;
        }
      }
      __syncthreads();
      // out of the chunk's own rows and of M
      for (int r0 = 0; r0 < rows; r0 += 16) {
        float own[2][4] = {}, past[2][4] = {}, town[2][4] = {}, tpast[2][4] = {};
        for (int k = 0; k < r0 + 16; k += 8) {
          auto load_p = [&](Part(&f)[4], const float* s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i].set(s[(r0 + g + (i & 1) * 8) * LP + k + t + (i >> 1) * 4]);
          };
          auto times = [&](float(&acc)[2][4], const Part(&f)[4], const float* s) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              Part fc[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) fc[i].set(s[(k + t + i * 4) * LD + e0 + j * 8 + g]);
              mul(acc[j], f, fc);
            }
          };
          Part fp[4];
          load_p(fp, sP);
          times(own, fp, sC);
          if constexpr (DUAL) {
            times(town, fp, stC);
            load_p(fp, stP);
            times(town, fp, sC);
          }
        }
#pragma unroll
        for (int k = 0; k < ND; ++k) {
          // slots t and t + 4 of the contraction are entries 2 t and 2 t + 1, as M's accumulators have them
          auto load_rows = [&](Part(&f)[4], const float* s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i].set(s[(r0 + g + (i & 1) * 8) * LD + k * 8 + 2 * t + (i >> 1)]);
          };
          auto times = [&](float(&acc)[2][4], const Part(&f)[4], const float(&m)[4]) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              Part fm[2];
              fm[0].set(m[2 * j]), fm[1].set(m[2 * j + 1]);
              mul(acc[j], f, fm);
            }
          };
          Part fa[4];
          load_rows(fa, sA);
          times(past, fa, M[k]);
          if constexpr (DUAL) {
            times(tpast, fa, tM[k]);
            load_rows(fa, stA);
            times(tpast, fa, M[k]);
          }
        }
        float* out = static_cast<float*>(const_cast<void*>(p.out.p));
        float* tout = static_cast<float*>(const_cast<void*>(p.tout.p));
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = r0 + g + (i >> 1) * 8, e = e0 + j * 8 + 2 * t + (i & 1);
            if (r >= rows || e >= p.E) continue;
            const long long row = p.reversed ? n - 1 - row0 - r : row0 + r;
            const float f = power[r + 1 + shift];
            if (out) out[of_head(p.out) + row * p.out.stride[2] + e] = p.scale * (own[j][i] + f * past[j][i]);
            if (DUAL && tout) tout[of_head(p.tout) + row * p.tout.stride[2] + e] = p.scale * (town[j][i] + f * tpast[j][i]);
          }
      }
    }
    // M = l^rows M + sum of l^(rows - 1 - s) b_s c_s^T
    const Down down = down_of(power[rows + shift], less1[rows + shift]);
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        M[i][j] = fmaf(M[i][j], down.by, M[i][j] * down.keep);
        if (DUAL) tM[i][j] = fmaf(tM[i][j], down.by, tM[i][j] * down.keep);
      }
    for (int k = 0; k < rows; k += 8) {
      auto load_c = [&](Part(&f)[4], const float* s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = k + t + (i >> 1) * 4;
          f[i].set(r < rows ? s[r * LD + e0 + g + (i & 1) * 8] * power[rows - 1 - r] : 0.f);
        }
      };
      Part fc[4], ftc[4];
      load_c(fc, sC);
      if constexpr (DUAL) load_c(ftc, stC);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        auto load_b = [&](Part(&f)[2], const float* s) {
#pragma unroll
          for (int i = 0; i < 2; ++i) f[i].set(s[(k + t + i * 4) * LD + d * 8 + g]);
        };
        Part fb[2];
        load_b(fb, sB);
        mul(M[d], fc, fb);
        if constexpr (DUAL) {
          mul(tM[d], ftc, fb);
          load_b(fb, stB);
          mul(tM[d], fc, fb);
        }
      }
    }
  }

  if constexpr (!OUT) {
    each([&](int i, int j, int d, int e) {
      if (d >= p.D || e >= p.E) return;
      const long long at = ((long long)head * p.segments + segment) * size + d * p.state_stride[0] + e * p.state_stride[1];
      p.states[at] = M[i][j];
      if (DUAL) p.tstates[at] = tM[i][j];
    });
  } else {
    // rows behind the sequence's last one are zero
    for (int which = 0; which < (DUAL ? 2 : 1); ++which) {
      const jvpfa_linear_tensor& x = which ? p.tout : p.out;
      if (!x.p) continue;
      float* out = static_cast<float*>(const_cast<void*>(x.p)) + of_head(x);
      const int to = min(p.L, row_begin + p.segment);
      for (int row = max(n, row_begin) + warp; row < to; row += NT / 32)
        for (int e = lane; e < p.E; e += 32) out[row * x.stride[2] + e] = 0.f;
    }
    if (n == 0 ? segment == 0 : row_begin < n && row_begin + p.segment >= n) {
      const float f = n == 0 ? p.last_scale : p.last_scale * power[p.last_ahead];
      each([&](int i, int j, int d, int e) {
        if (d >= p.D || e >= p.E) return;
        const long long at = head * size + d * p.last_stride[0] + e * p.last_stride[1];
        if (p.last) p.last[at] = f * M[i][j];
        if (DUAL && p.tlast) p.tlast[at] = f * tM[i][j];
      });
    }
  }
}

template <int DT, bool DUAL, bool OUT>
int launch(const Scan& s, cudaStream_t stream) {
  static SmemOptIn opt;
  const auto kernel = scan_kernel<DT, DUAL, OUT>;
  constexpr size_t bytes = ScanShape<DT>::bytes(DUAL, OUT);
  static_assert(bytes <= 227 * 1024 - 1024, "an SM's shared memory");
  if (!opt.ensure(reinterpret_cast<const void*>(kernel), bytes)) return JVPFA_ERR_CUDA;
  uint32_t wide = 0;
  const jvpfa_linear_tensor* tensors[6] = {&s.b, &s.c, &s.a, &s.tb, &s.tc, &s.ta};
  for (int i = 0; i < 6; ++i)
    if (wide_tensor<float>(*tensors[i], s, i % 3 == 1 ? s.E : s.D)) wide |= 1u << i;
  kernel<<<(unsigned)((long long)s.B * s.H * s.segments), ScanShape<DT>::NT, bytes, stream>>>(s, wide);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "scan_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
}

template <bool OUT>
int launch(const Scan& s, cudaStream_t stream) {
  const int width = s.D > s.E ? s.D : s.E;
  if (width <= 32) return s.dual ? launch<32, true, OUT>(s, stream) : launch<32, false, OUT>(s, stream);
  if (width <= 64) return s.dual ? launch<64, true, OUT>(s, stream) : launch<64, false, OUT>(s, stream);
  return s.dual ? launch<128, true, OUT>(s, stream) : launch<128, false, OUT>(s, stream);
}

}  // namespace

int scan_ctas(const Scan& s) {
  const int width = s.D > s.E ? s.D : s.E;
  return width <= 32 ? ScanShape<32>::ctas(s.dual) : width <= 64 ? ScanShape<64>::ctas(s.dual) : ScanShape<128>::ctas(s.dual);
}

int launch_scan(const Scan& s, bool outputs, cudaStream_t stream) { return outputs ? launch<true>(s, stream) : launch<false>(s, stream); }

}  // namespace linear
}  // namespace jvpfa

// The map of linear_common.cuh for bfloat16, on the 16-bit instructions.
//
// A CTA takes a segment of one head's rows in chunks of 64.  Warp w keeps columns 16 w .. 16 w + 15 of M in registers, transposed: as they
// stand the accumulators are the second operand of a M, and the columns of c that the warp multiplies the chunk's products by are, loaded
// once, also the first operand of what the chunk adds to M.  A chunk is
//   products (a_t . b_s) l^(t-s), 16 x 16 blocks shared out among the warps, through shared memory;   a M, while they are under way;
//   one barrier;   products times c;   M = l^64 M + (c l^(63-s))^T b.
// What is formed in 32 bits and multiplied again (the weighted products, M, the weighted c) is split into bfloat16 numbers of 8 bits each,
// two, and three of the weighted c where the state itself is answered: two leave 2^-17 of an entry, well below what a result is rounded to,
// one would double its error.  What a chunk adds to M is formed apart and added rounded to nearest, since the tensor cores truncate.
// What bounds it: the tensor cores' 16-bit rate, with D = E = 128 5.2 million products a chunk (2 for each of a M, c^T b and the inner ones).
#include "linear_common.cuh"

namespace jvpfa {
namespace linear {

namespace {

using T = __nv_bfloat16;
constexpr int CH = 64, LP = CH + 8;

// Addresses in shared memory are 32-bit numbers here: what is added to a lane's own is part of the instruction then.
__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldmatrix(uint32_t r[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix_t(uint32_t r[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float low(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float high(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
// Two values as pairs of bfloat16 numbers, each the rounding of what the ones before it left.
template <int PARTS>
__device__ __forceinline__ void split(float x, float y, uint32_t (&part)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    part[i] = Elem<T>::pack(x, y);
    if (i + 1 < PARTS) {
      const float2 left = __ffma2_rn(make_float2(low(part[i]), high(part[i])), make_float2(-1.f, -1.f), make_float2(x, y));
      x = left.x, y = left.y;
    }
  }
}

// Rows row0 .. row0 + 63 (`back`: counted from the end of n) of a head into shared memory, zeros behind the last and behind the width, and for an
// absent tensor.
template <int DT, int NT>
__device__ __forceinline__ void stage(T* to, const jvpfa_linear_tensor& x, long long head, int width, int row0, int rows, int n, bool back, bool wide) {
  // (a loop of few instructions: the kernels' code is long, and what does not fit the instruction caches waits)
  constexpr int LD = DT + 8, PIECES = DT / 8, AT_ONCE = NT / PIECES;
  static_assert(AT_ONCE == 16, "four rows of a thread");
  const int col = threadIdx.x % PIECES * 8, r0 = threadIdx.x / PIECES;
  const T* from = static_cast<const T*>(x.p) + head + (long long)(back ? n - 1 - row0 - r0 : row0 + r0) * x.stride[2] + col;
  const long long step = back ? -AT_ONCE * x.stride[2] : AT_ONCE * x.stride[2];
  T* d = to + r0 * LD + col;
  const int live = x.p && col < width ? rows : 0;
#pragma unroll 1
  for (int r = r0; r < CH; r += AT_ONCE, from += step, d += AT_ONCE * LD) {
    if (r >= live) {
      *reinterpret_cast<uint4*>(d) = make_uint4(0, 0, 0, 0);
    } else if (wide) {
      cp_async16(d, from, 16);
    } else {
#pragma unroll 1
      for (int j = 0; j < 8; ++j) d[j] = col + j < width ? from[j] : Elem<T>::from_float(0.f);
    }
  }
}

// Shared memory of a CTA: two tiles of b (and of its tangent), which a chunk reads to its end, and one of c and one of a, which are free behind the
// products' barrier and take the next chunk's rows then; the products.  States alone: two tiles of b and c.
template <int DT, bool DUAL, bool OUT>
struct ChunkShape {
  static constexpr int LD = DT + 8, NT = 2 * DT, SIDES = DUAL ? 2 : 1, TILE = CH * LD;
  static constexpr int CTAS = DT == 32 ? (DUAL ? 2 : 4) : DT == 64 ? (DUAL ? 2 : 3) : DUAL ? 1 : 2;
  static constexpr size_t bytes() { return sizeof(T) * SIDES * (4 * (size_t)TILE + (OUT ? 2 * (size_t)CH * LP : 0)); }
};

// OUT: the outputs, from the states that the segments begin with; else the states that their rows leave, from nothing.
template <int DT, bool DUAL, bool OUT, int PARTS>
__global__ void __launch_bounds__(2 * DT, ChunkShape<DT, DUAL, OUT>::CTAS) chunk_kernel(const __grid_constant__ Scan p, const uint32_t wide) {
  using S = ChunkShape<DT, DUAL, OUT>;
  constexpr int NT = S::NT, LD = S::LD, ND = DT / 8, KD = DT / 16, NW = DT / 16, SIDES = DUAL ? 2 : 1;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float power[CH + 2], less1[CH + 2];  // l^j and l^j - 1
  constexpr int TILE = S::TILE;
  T* tiles_b = reinterpret_cast<T*>(smem);     // two times b and its tangent
  T* tiles_c = tiles_b + 2 * SIDES * TILE;     // c and its tangent (states alone: two times)
  T* tiles_a = tiles_c + SIDES * TILE;         // a and its tangent
  T* sP = tiles_a + SIDES * TILE;              // products in two parts, then their tangents
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
  auto each = [&](auto f) {  // (d tile, entry, row d and column e of M)
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) f(i, j, i * 8 + 2 * t + (j & 1), e0 + g + (j >> 1) * 8);
  };

  float M[SIDES][ND][4];
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
    M[0][i][j] = x;
    if (DUAL) M[SIDES - 1][i][j] = y;
  });
  // The given state is l^ahead away from the first row, what the rows leave l^1.
  int shift = OUT && segment == 0 ? p.ahead - 1 : 0;

  auto fetch_b = [&](int half, int row0) {
    const int rows = min(CH, row_end - row0);
    T* to = tiles_b + half * SIDES * TILE;
    stage<DT, NT>(to, p.b, of_head(p.b), p.D, row0, rows, n, p.reversed, wide & 1);
    if (DUAL) stage<DT, NT>(to + TILE, p.tb, of_head(p.tb), p.D, row0, rows, n, p.reversed, wide & 8);
  };
  auto fetch_c = [&](int half, int row0) {
    const int rows = min(CH, row_end - row0);
    T* to = tiles_c + (OUT ? 0 : half * SIDES * TILE);
    stage<DT, NT>(to, p.c, of_head(p.c), p.E, row0, rows, n, p.reversed, wide & 2);
    if (DUAL) stage<DT, NT>(to + TILE, p.tc, of_head(p.tc), p.E, row0, rows, n, p.reversed, wide & 16);
  };
  auto fetch_a = [&](int row0) {
    const int rows = min(CH, row_end - row0);
    stage<DT, NT>(tiles_a, p.a, of_head(p.a), p.D, row0, rows, n, p.reversed, wide & 4);
    if (DUAL) stage<DT, NT>(tiles_a + TILE, p.ta, of_head(p.ta), p.D, row0, rows, n, p.reversed, wide & 32);
  };
  // where a lane of ldmatrix reads: first operand and transposed second one (rows 0-7, 8-15, then columns 8-15), second one (columns 8-15, then rows 8-15)
  const int lane_row = lane & 15, lane_col = lane >> 4 << 3;
  const int lane_row_n = (lane & 7) + (lane >> 4 << 3), lane_col_n = lane >> 3 & 1 ? 8 : 0;
  constexpr uint32_t SZ = sizeof(T), ROWS16 = 16 * LD * SZ, P16 = 16 * LP * SZ, PART = CH * LP * SZ, SIDE = (SIDES - 1) * TILE * SZ;
  const uint32_t at_first = (lane_row * LD + lane_col) * SZ;  // of a first operand, or a transposed second one
  const uint32_t at_second = (lane_row_n * LD + lane_col_n) * SZ;
  const uint32_t lane_a = shared_address(tiles_a) + at_first, lane_p = shared_address(sP) + (lane_row * LP + lane_col) * SZ;

  int now = 0;
  if (row_begin < row_end) {
    fetch_b(0, row_begin), fetch_c(0, row_begin);
    if (OUT) fetch_a(row_begin);
    cp_async_commit();
  }
  for (int row0 = row_begin; row0 < row_end; row0 += CH, shift = 0, now ^= 1) {
    const int rows = min(CH, row_end - row0);
    const bool more = row0 + CH < row_end;
    cp_async_wait<0>();
    __syncthreads();  // this chunk has arrived, the one before has been read
    if (more) {
      fetch_b(now ^ 1, row0 + CH);
      if (!OUT) fetch_c(now ^ 1, row0 + CH);
      cp_async_commit();
    }
    const uint32_t tile_b = shared_address(tiles_b + now * SIDES * TILE), lane_b = tile_b + at_first;
    const uint32_t lane_c = shared_address(tiles_c + (OUT ? 0 : now * SIDES * TILE)) + at_first + e0 * SZ;
    uint32_t fc[SIDES][4][4];  // columns e0 .. e0 + 15 of c: 16 rows each; second operand's halves (0, 1) and (2, 3)
    if constexpr (OUT) {
      // the chunk's products
#pragma unroll 1
      for (int block = warp; block < 10; block += NW) {
        const int i = block < 1 ? 0 : block < 3 ? 1 : block < 6 ? 2 : 3, j = block - i * (i + 1) / 2;
        float x[SIDES][2][4] = {};
        if (i * 16 < rows) {
#pragma unroll
          for (int k = 0; k < KD; ++k) {
            uint32_t fa[4], fb[4];
            ldmatrix(fa, lane_a + i * ROWS16 + k * 32);
            ldmatrix(fb, tile_b + at_second + j * ROWS16 + k * 32);
            mma(x[0][0], fa, fb[0], fb[1]), mma(x[0][1], fa, fb[2], fb[3]);
            if constexpr (DUAL) {
              uint32_t fta[4], ftb[4];
              ldmatrix(fta, lane_a + SIDE + i * ROWS16 + k * 32);
              ldmatrix(ftb, tile_b + at_second + SIDE + j * ROWS16 + k * 32);
              mma(x[1][0], fta, fb[0], fb[1]), mma(x[1][1], fta, fb[2], fb[3]);
              mma(x[1][0], fa, ftb[0], ftb[1]), mma(x[1][1], fa, ftb[2], ftb[3]);
            }
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int r = i * 16 + g + u * 8, s = j * 16 + half * 8 + 2 * t;
            const float w0 = s <= r ? power[r - s] : 0.f, w1 = s + 1 <= r ? power[r - s - 1] : 0.f;
#pragma unroll
            for (int side = 0; side < SIDES; ++side) {
              uint32_t part[2];
              // (selected, not multiplied by zero: an entry right of the diagonal may be infinite)
              split(s <= r ? x[side][half][2 * u] * w0 : 0.f, s + 1 <= r ? x[side][half][2 * u + 1] * w1 : 0.f, part);
              *reinterpret_cast<uint32_t*>(sP + (2 * side) * CH * LP + r * LP + s) = part[0];
              *reinterpret_cast<uint32_t*>(sP + (2 * side + 1) * CH * LP + r * LP + s) = part[1];
            }
          }
      }
      // what is before the chunk, and its own rows
      // 16 rows from i * 16 on, in accumulators
      auto answer = [&](int i, const float (&tile)[SIDES][2][4]) {
#pragma unroll
        for (int side = 0; side < SIDES; ++side) {
          const jvpfa_linear_tensor& x = side ? p.tout : p.out;
          if (!x.p) continue;
          T* out = static_cast<T*>(const_cast<void*>(x.p)) + of_head(x);
          uint32_t v[4];  // (row g or g + 8, columns 0-7 or 8-15) of the tile, two entries
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j) v[2 * u + j] = Elem<T>::pack(p.scale * tile[side][j][2 * u], p.scale * tile[side][j][2 * u + 1]);
          auto row_of = [&](int r) { return (long long)(p.reversed ? n - 1 - row0 - r : row0 + r) * x.stride[2]; };
          if (wide >> (6 + side) & 1) {
            // four lanes hold two rows of 32 bytes, a word of each half row in each: they are turned so that each holds 16 successive bytes
            uint32_t s;
            s = __shfl_xor_sync(0xffffffffu, t & 1 ? v[0] : v[1], 1), (t & 1 ? v[0] : v[1]) = s;
            s = __shfl_xor_sync(0xffffffffu, t & 1 ? v[2] : v[3], 1), (t & 1 ? v[2] : v[3]) = s;
            s = __shfl_xor_sync(0xffffffffu, t & 2 ? v[0] : v[2], 2), (t & 2 ? v[0] : v[2]) = s;
            s = __shfl_xor_sync(0xffffffffu, t & 2 ? v[1] : v[3], 2), (t & 2 ? v[1] : v[3]) = s;
            const int r = i * 16 + g + (t >> 1) * 8, e = e0 + (t & 1) * 8;
            if (r < rows && e < p.E) *reinterpret_cast<uint4*>(out + row_of(r) + e) = make_uint4(v[0], v[1], v[2], v[3]);
          } else {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int r = i * 16 + g + u * 8, e = e0 + j * 8 + 2 * t;
                const __nv_bfloat162 two = *reinterpret_cast<const __nv_bfloat162*>(&v[2 * u + j]);
                if (r < rows && e < p.E) out[row_of(r) + e] = two.x;
                if (r < rows && e + 1 < p.E) out[row_of(r) + e + 1] = two.y;
              }
          }
        }
      };
      if constexpr (DT <= 64) {
        // M in two parts, once for all rows; then 16 rows after the other
        uint32_t m[SIDES][KD][2][2][2];  // side, step, columns 0-7 or 8-15, rows 0-7 or 8-15, part
#pragma unroll
        for (int side = 0; side < SIDES; ++side)
#pragma unroll
          for (int k = 0; k < KD; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int u = 0; u < 2; ++u) split(M[side][2 * k + u][2 * j], M[side][2 * k + u][2 * j + 1], m[side][k][j][u]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          ldmatrix_t(fc[0][k], lane_c + k * ROWS16);
          if (DUAL) ldmatrix_t(fc[SIDES - 1][k], lane_c + SIDE + k * ROWS16);
        }
        __syncthreads();  // the products are there, and nobody reads c again
        if (more) {
          fetch_c(0, row0 + CH);
          cp_async_commit();
        }
#pragma unroll 1
        for (int i = 0; i * 16 < rows; ++i) {
          float acc[SIDES][2][4] = {}, low_acc[2][4] = {};  // (two chains without tangents: an accumulator's next product is four instructions away)
#pragma unroll
          for (int k = 0; k < KD; ++k) {
            uint32_t fa[4], fta[4];
            ldmatrix(fa, lane_a + i * ROWS16 + k * 32);
            if (DUAL) ldmatrix(fta, lane_a + SIDE + i * ROWS16 + k * 32);
#pragma unroll
            for (int part = 1; part >= 0; --part)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                mma(!DUAL && part ? low_acc[j] : acc[0][j], fa, m[0][k][j][0][part], m[0][k][j][1][part]);
                if (DUAL) mma(acc[SIDES - 1][j], fa, m[SIDES - 1][k][j][0][part], m[SIDES - 1][k][j][1][part]);
                if (DUAL) mma(low_acc[j], fta, m[0][k][j][0][part], m[0][k][j][1][part]);
              }
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float f = power[min(i * 16 + g + u * 8, rows - 1) + 1 + shift];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int v = 2 * u; v < 2 * u + 2; ++v) {
                acc[SIDES - 1][j][v] = (acc[SIDES - 1][j][v] + low_acc[j][v]) * f;
                if (DUAL) acc[0][j][v] *= f;
              }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k > i) break;
#pragma unroll
            for (int part = 1; part >= 0; --part) {
              uint32_t fp[4], ftp[4];
              ldmatrix(fp, lane_p + part * PART + i * P16 + k * 32);
              if (DUAL) ldmatrix(ftp, lane_p + (2 + part) * PART + i * P16 + k * 32);
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                mma(acc[0][j], fp, fc[0][k][2 * j], fc[0][k][2 * j + 1]);
                if (DUAL) mma(acc[SIDES - 1][j], fp, fc[SIDES - 1][k][2 * j], fc[SIDES - 1][k][2 * j + 1]);
              }
              if constexpr (DUAL) {
#pragma unroll
                for (int j = 0; j < 2; ++j) mma(acc[1][j], ftp, fc[0][k][2 * j], fc[0][k][2 * j + 1]);
              }
            }
          }
          answer(i, acc);
        }
        __syncthreads();  // nobody reads a again
        if (more) {
          fetch_a(row0 + CH);
          cp_async_commit();
        }
      } else {
      float acc[SIDES][4][2][4] = {};
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        uint32_t m[SIDES][2][2][2];  // side, columns 0-7 or 8-15, rows 0-7 or 8-15, part
#pragma unroll
        for (int side = 0; side < SIDES; ++side)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) split(M[side][2 * k + u][2 * j], M[side][2 * k + u][2 * j + 1], m[side][j][u]);
        // (an accumulator's next product is eight instructions away, or four with tangents)
#pragma unroll
        for (int h2 = 0; h2 < 4; h2 += DUAL ? 2 : 4) {
          constexpr int TILES_AT_ONCE = DUAL ? 2 : 4;
          uint32_t fa[TILES_AT_ONCE][4];
#pragma unroll
          for (int i = 0; i < TILES_AT_ONCE; ++i) ldmatrix(fa[i], lane_a + (h2 + i) * ROWS16 + k * 32);
#pragma unroll
          for (int part = 1; part >= 0; --part)
#pragma unroll
            for (int i = 0; i < TILES_AT_ONCE; ++i)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                mma(acc[0][h2 + i][j], fa[i], m[0][j][0][part], m[0][j][1][part]);
                if (DUAL) mma(acc[SIDES - 1][h2 + i][j], fa[i], m[SIDES - 1][j][0][part], m[SIDES - 1][j][1][part]);
              }
          if constexpr (DUAL) {
#pragma unroll
            for (int i = 0; i < TILES_AT_ONCE; ++i) ldmatrix(fa[i], lane_a + SIDE + (h2 + i) * ROWS16 + k * 32);
#pragma unroll
            for (int part = 1; part >= 0; --part)
#pragma unroll
              for (int i = 0; i < TILES_AT_ONCE; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) mma(acc[1][h2 + i][j], fa[i], m[0][j][0][part], m[0][j][1][part]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float f = power[min(i * 16 + g + u * 8, rows - 1) + 1 + shift];
#pragma unroll
          for (int side = 0; side < SIDES; ++side)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[side][i][j][2 * u] *= f, acc[side][i][j][2 * u + 1] *= f;
        }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        ldmatrix_t(fc[0][k], lane_c + k * ROWS16);
        if (DUAL) ldmatrix_t(fc[SIDES - 1][k], lane_c + SIDE + k * ROWS16);
      }
      __syncthreads();  // the products are there, and nobody reads a and c again
      if (more) {
        fetch_c(0, row0 + CH), fetch_a(row0 + CH);
        cp_async_commit();
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i * 16 >= rows) break;
#pragma unroll
        for (int k = 0; k <= i; ++k) {
#pragma unroll
          for (int part = 1; part >= 0; --part) {
            uint32_t fp[4];
            ldmatrix(fp, lane_p + part * PART + i * P16 + k * 32);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              mma(acc[0][i][j], fp, fc[0][k][2 * j], fc[0][k][2 * j + 1]);
              if (DUAL) mma(acc[SIDES - 1][i][j], fp, fc[SIDES - 1][k][2 * j], fc[SIDES - 1][k][2 * j + 1]);
            }
            if constexpr (DUAL) {
              ldmatrix(fp, lane_p + (2 + part) * PART + i * P16 + k * 32);
#pragma unroll
              for (int j = 0; j < 2; ++j) mma(acc[1][i][j], fp, fc[0][k][2 * j], fc[0][k][2 * j + 1]);
            }
          }
        }
        float tile[SIDES][2][4];
#pragma unroll
        for (int side = 0; side < SIDES; ++side)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) tile[side][j][v] = acc[side][i][j][v];
        answer(i, tile);
      }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        ldmatrix_t(fc[0][k], lane_c + k * ROWS16);
        if (DUAL) ldmatrix_t(fc[SIDES - 1][k], lane_c + SIDE + k * ROWS16);
      }
    }
    // M = l^rows M + sum of l^(rows - 1 - s) b_s c_s^T; the factor by its distance from 1, which keeps the digits of slow decays.  As a first operand the
    // words of c are (0, 2, 1, 3).
    uint32_t wc[SIDES][4][4][PARTS];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int s = k * 16 + u * 8 + 2 * t;
        const float w0 = s < rows ? power[rows - 1 - s] : 0.f, w1 = s + 1 < rows ? power[rows - 2 - s] : 0.f;
#pragma unroll
        for (int side = 0; side < SIDES; ++side)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t x = fc[side][k][2 * j + u];
            const float2 y = __fmul2_rn(make_float2(low(x), high(x)), make_float2(w0, w1));
            split(y.x, y.y, wc[side][k][2 * u + j]);
          }
      }
    const float down = less1[rows + shift];
#pragma unroll
    for (int d = 0; d < ND; d += 2) {
      float x[SIDES][2][4] = {};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t fb[4];
        ldmatrix_t(fb, lane_b + k * ROWS16 + d * 16);
#pragma unroll
        for (int part = PARTS - 1; part >= 0; --part) {
          const uint32_t fa[4] = {wc[0][k][0][part], wc[0][k][1][part], wc[0][k][2][part], wc[0][k][3][part]};
          mma(x[0][0], fa, fb[0], fb[1]), mma(x[0][1], fa, fb[2], fb[3]);
          if constexpr (DUAL) {
            const uint32_t fta[4] = {wc[1][k][0][part], wc[1][k][1][part], wc[1][k][2][part], wc[1][k][3][part]};
            mma(x[1][0], fta, fb[0], fb[1]), mma(x[1][1], fta, fb[2], fb[3]);
          }
        }
        if constexpr (DUAL) {
          ldmatrix_t(fb, lane_b + SIDE + k * ROWS16 + d * 16);
#pragma unroll
          for (int part = PARTS - 1; part >= 0; --part) {
            const uint32_t fa[4] = {wc[0][k][0][part], wc[0][k][1][part], wc[0][k][2][part], wc[0][k][3][part]};
            mma(x[1][0], fa, fb[0], fb[1]), mma(x[1][1], fa, fb[2], fb[3]);
          }
        }
      }
#pragma unroll
      for (int side = 0; side < SIDES; ++side)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            float* m = &M[side][d + u][j];
            const float2 old = make_float2(m[0], m[1]);
            const float2 sum = __fadd2_rn(__ffma2_rn(old, make_float2(down, down), old), make_float2(x[side][u][j], x[side][u][j + 1]));
            m[0] = sum.x, m[1] = sum.y;
          }
    }
  }

  if constexpr (!OUT) {
    each([&](int i, int j, int d, int e) {
      if (d >= p.D || e >= p.E) return;
      const long long at = ((long long)head * p.segments + segment) * size + d * p.state_stride[0] + e * p.state_stride[1];
      p.states[at] = M[0][i][j];
      if (DUAL) p.tstates[at] = M[SIDES - 1][i][j];
    });
  } else {
    // rows behind the sequence's last one are zero
    for (int side = 0; side < SIDES; ++side) {
      const jvpfa_linear_tensor& x = side ? p.tout : p.out;
      if (!x.p) continue;
      T* out = static_cast<T*>(const_cast<void*>(x.p)) + of_head(x);
      const int from = max(n, row_begin), to = min(p.L, row_begin + p.segment);
      for (long long i = tid; i < (long long)(to - from) * p.E; i += NT) out[(from + i / p.E) * x.stride[2] + i % p.E] = Elem<T>::from_float(0.f);
    }
    if (n == 0 ? segment == 0 : row_begin < n && row_begin + p.segment >= n) {
      const float f = n == 0 ? p.last_scale : p.last_scale * power[p.last_ahead];
      each([&](int i, int j, int d, int e) {
        if (d >= p.D || e >= p.E) return;
        const long long at = head * size + d * p.last_stride[0] + e * p.last_stride[1];
        if (p.last) p.last[at] = f * M[0][i][j];
        if (DUAL && p.tlast) p.tlast[at] = f * M[SIDES - 1][i][j];
      });
    }
  }
}

bool wide_tensor(const jvpfa_linear_tensor& x, const Scan& s, int width) {
  uint64_t all = (uint64_t)width * sizeof(T) | reinterpret_cast<uint64_t>(x.p);
  const int counts[3] = {s.B, s.H, s.L};
  for (int d = 0; d < 3; ++d)
    if (counts[d] > 1) all |= (uint64_t)x.stride[d] * sizeof(T);
  return all % 16 == 0;
}

template <int DT, bool DUAL, bool OUT, int PARTS>
int launch(const Scan& s, cudaStream_t stream) {
  static SmemOptIn opt;
  const auto kernel = chunk_kernel<DT, DUAL, OUT, PARTS>;
  constexpr size_t bytes = ChunkShape<DT, DUAL, OUT>::bytes();
  static_assert(bytes * ChunkShape<DT, DUAL, OUT>::CTAS <= 227 * 1024 - ChunkShape<DT, DUAL, OUT>::CTAS * 2048, "an SM's shared memory");
  if (!opt.ensure(reinterpret_cast<const void*>(kernel), bytes)) return JVPFA_ERR_CUDA;
  uint32_t wide = 0;
  const jvpfa_linear_tensor* tensors[8] = {&s.b, &s.c, &s.a, &s.tb, &s.tc, &s.ta, &s.out, &s.tout};
  for (int i = 0; i < 8; ++i)
    if (wide_tensor(*tensors[i], s, i % 3 == 1 || i >= 6 ? s.E : s.D)) wide |= 1u << i;
  kernel<<<(unsigned)((long long)s.B * s.H * s.segments), ChunkShape<DT, DUAL, OUT>::NT, bytes, stream>>>(s, wide);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "chunk_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
}

template <int DT, bool OUT>
int launch(const Scan& s, cudaStream_t stream) {
  const bool exact = s.last || s.tlast;  // the state is a result of 32 bits
  if (s.dual) return exact ? launch<DT, true, OUT, 3>(s, stream) : launch<DT, true, OUT, 2>(s, stream);
  return exact ? launch<DT, false, OUT, 3>(s, stream) : launch<DT, false, OUT, 2>(s, stream);
}

template <bool OUT>
int launch(const Scan& s, cudaStream_t stream) {
  const int width = s.D > s.E ? s.D : s.E;
  return width <= 32 ? launch<32, OUT>(s, stream) : width <= 64 ? launch<64, OUT>(s, stream) : launch<128, OUT>(s, stream);
}

}  // namespace

int launch_chunks(const Scan& s, bool outputs, cudaStream_t stream) { return outputs ? launch<true>(s, stream) : launch<false>(s, stream); }

}  // namespace linear
}  // namespace jvpfa

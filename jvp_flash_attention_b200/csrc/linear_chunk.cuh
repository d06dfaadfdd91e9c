// The map of linear_common.cuh for the 16-bit types.
//
// A CTA takes a segment of one head's rows in chunks of 64.  Warp w keeps columns 16 w .. 16 w + 15 of M in registers, transposed: as they
// stand the accumulators are the second operand of a M, and the columns of c that the warp multiplies the chunk's products by are, loaded
// once, also the first operand of what the chunk adds to M.  A chunk is
//   products (a_t . b_s) l^(t-s), 16 x 16 blocks shared out among the warps, through shared memory;   a M;   products times c;
//   M = l^64 M + (c l^(63-s))^T b.
// Entries are multiplied as they are.  What is formed in 32 bits and multiplied again (weighted products, M, weighted c) keeps its exponent, so that no
// decay, row or entry takes digits from another (float16 numbers with a power of two for each tile did: keys in a chunk's first row alone, decayed by
// e^-0.5 a row, left a state of zero).  For bfloat16 it is two bfloat16 numbers (2^-17 of it is lost, 2^-8 of what a result is rounded to), three of the
// weighted c where the state is answered.  For float16, whose 11 bits fit a TF32 number whole, it is a TF32 number and what that left, as a bfloat16
// number (2^-19), of the weighted c where the state is answered as a TF32 number too (2^-22).  Products of entries are on each type's own instructions.  What a
// chunk adds to M is formed apart and added rounded to nearest, since the tensor cores truncate.
// What bounds it: latencies, with two to four warps a scheduler.  bf16 B4 H16 L8192 D128 takes 313 us for a map (tensor pipe 41 % busy, issue slots
// 34 %), fp16 499 (38 %, 40 %); B4 H16 L2048 D64 with tangents 84 (38 %, 28 %) and 133 (35 %, 30 %: 1.2 cycles an instruction it waits for
// instructions).  64 rows, since products within a chunk cost 64 (D + E) / 2 a row and M 2 D E; M in registers, since it is read and written
// every chunk.  Registers set the warps: 128 a thread for D = 128 twice on an SM, 168 for D = 64 three times, 255 with tangents.
#pragma once
#include <type_traits>

#include "linear_common.cuh"

namespace jvpfa {
namespace linear {

namespace {

constexpr int CH = 64, LP = CH + 8;

// Addresses in shared memory are 32-bit numbers here: what is added to a lane's own is part of the instruction then.
__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldmatrix(uint32_t r[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix_t(uint32_t r[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// c += a b, 16 x 16 entries and 16 x 8.
template <typename T>
__device__ __forceinline__ void mma(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float2 of_halves(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
// Two entries of a tensor.
template <typename T>
__device__ __forceinline__ float2 of_word(uint32_t w) {
  if constexpr (std::is_same_v<T, __half>)
    return of_halves(w);
  else
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Two neighbouring values of a contraction that were formed in 32 bits, as they are multiplied.  bfloat16: PARTS pairs of bfloat16 numbers, each the
// rounding of what the ones before it left.
template <typename T, int PARTS>
struct Formed {
  uint32_t part[PARTS];
  __device__ __forceinline__ void set(float2 x) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      part[i] = Elem<T>::pack(x.x, x.y);
      if (i + 1 < PARTS) x = __ffma2_rn(of_word<T>(part[i]), make_float2(-1.f, -1.f), x);
    }
  }
};
// float16: a TF32 number of each, which goes into slots t and t + 4 of a contraction over 8 (2 t and 2 t + 1 of the entries' order), and what it left: as a
// bfloat16 number, which meets the entries in bfloat16 too (together 2^-19 of the product is lost; on the 16-bit instructions, at half the time), or with PARTS = 3 as
// a TF32 number (2^-22).
template <int PARTS>
struct Formed<__half, PARTS> {
  uint32_t hi[2], lo[PARTS == 3 ? 2 : 1];
  __device__ __forceinline__ void set(float2 x) {
    uint32_t rest[2];
    split_tf32(x.x, hi[0], rest[0]), split_tf32(x.y, hi[1], rest[1]);
    if constexpr (PARTS == 3)
      lo[0] = rest[0], lo[1] = rest[1];
    else
      lo[0] = Elem<__nv_bfloat16>::pack(x.x - __uint_as_float(hi[0]), x.y - __uint_as_float(hi[1]));
  }
};
__device__ __forceinline__ uint32_t as_bfloat16(float2 x) { return Elem<__nv_bfloat16>::pack(x.x, x.y); }
// c += a b, a entries and b formed: of the contraction's first half and second half.
template <typename T, int PARTS>
__device__ __forceinline__ void mma_formed(float c[4], const uint32_t (&a)[4], const Formed<T, PARTS>& b0, const Formed<T, PARTS>& b1) {
  if constexpr (std::is_same_v<T, __half>) {
    const float2 x[4] = {of_halves(a[0]), of_halves(a[1]), of_halves(a[2]), of_halves(a[3])};
    if constexpr (PARTS == 2) {
      const uint32_t f[4] = {as_bfloat16(x[0]), as_bfloat16(x[1]), as_bfloat16(x[2]), as_bfloat16(x[3])};
      mma<__nv_bfloat16>(c, f, b0.lo[0], b1.lo[0]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t f[4] = {__float_as_uint(x[2 * k].x), __float_as_uint(x[2 * k + 1].x), __float_as_uint(x[2 * k].y), __float_as_uint(x[2 * k + 1].y)};
      if constexpr (PARTS == 3) mma_1688_tf32(c, f, (k ? b1 : b0).lo);
      mma_1688_tf32(c, f, (k ? b1 : b0).hi);
    }
  } else {
#pragma unroll
    for (int part = PARTS - 1; part >= 0; --part) mma<T>(c, a, b0.part[part], b1.part[part]);
  }
}
// c += a b, a formed and b entries.
template <typename T, int PARTS>
__device__ __forceinline__ void mma_formed(float c[4], const Formed<T, PARTS> (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>) {
    if constexpr (PARTS == 2) {
      const uint32_t f[4] = {a[0].lo[0], a[1].lo[0], a[2].lo[0], a[3].lo[0]};
      mma<__nv_bfloat16>(c, f, as_bfloat16(of_halves(b0)), as_bfloat16(of_halves(b1)));
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float2 x = of_halves(k ? b1 : b0);
      const uint32_t f[2] = {__float_as_uint(x.x), __float_as_uint(x.y)};
      if constexpr (PARTS == 3) {
        const uint32_t lo[4] = {a[2 * k].lo[0], a[2 * k + 1].lo[0], a[2 * k].lo[1], a[2 * k + 1].lo[1]};
        mma_1688_tf32(c, lo, f);
      }
      const uint32_t hi[4] = {a[2 * k].hi[0], a[2 * k + 1].hi[0], a[2 * k].hi[1], a[2 * k + 1].hi[1]};
      mma_1688_tf32(c, hi, f);
    }
  } else {
#pragma unroll
    for (int part = PARTS - 1; part >= 0; --part) {
      const uint32_t f[4] = {a[0].part[part], a[1].part[part], a[2].part[part], a[3].part[part]};
      mma<T>(c, f, b0, b1);
    }
  }
}
// Weighted entries of c between their forming and their use: in their parts, or for float16 as they are (its parts take twice the registers).
template <typename T, int PARTS>
struct Weighted {
  Formed<T, PARTS> x;
  __device__ __forceinline__ void set(float2 v) { x.set(v); }
  __device__ __forceinline__ Formed<T, PARTS> get() const { return x; }
};
template <int PARTS>
struct Weighted<__half, PARTS> {
  float2 x;
  __device__ __forceinline__ void set(float2 v) { x = v; }
  __device__ __forceinline__ Formed<__half, PARTS> get() const {
    Formed<__half, PARTS> f;
    f.set(x);
    return f;
  }
};

// Rows row0 .. row0 + 63 (`back`: counted from the end of n) of a head into shared memory, zeros behind the last and behind the width, and for an
// absent tensor.
template <typename T, int DT, int NT>
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

// Shared memory of a CTA: two tiles of b (and of its tangent), which a chunk reads to its end, and of a where there is room and a chunk reads it to its
// end, else one that takes the next rows once it is free; one of c, which is free behind the products' barrier; the products (bfloat16 in two parts,
// float16 in 32 bits).  States alone: two tiles of b and c.
template <typename T, int DT, bool DUAL, bool OUT>
struct ChunkShape {
  static constexpr bool HALF = std::is_same_v<T, __half>;
  static constexpr int LD = DT + 8, NT = 2 * DT, SIDES = DUAL ? 2 : 1, TILE = CH * LD;
  static constexpr int CTAS = DT == 32 ? (DUAL ? 2 : 4) : DT == 64 ? (DUAL ? 2 : 3) : DUAL ? 1 : 2;
  // LOOP: M in its parts once for all rows, then 16 rows after the other in one loop (its code stays in the instruction caches); else M's parts step by step, for
  // all rows together, as the registers do not hold them all.
  static constexpr bool LOOP = !HALF && DT <= 64;
  static constexpr size_t bytes_with(int tiles) { return SIDES * (2 * tiles * (size_t)TILE + (OUT ? 4 * (size_t)CH * LP : 0)); }
  static constexpr bool fits(size_t bytes) { return bytes * CTAS <= 227 * 1024 - CTAS * 2048; }
  static constexpr bool TWO_A = OUT && LOOP && fits(bytes_with(5));
  static constexpr size_t bytes = bytes_with(TWO_A ? 5 : 4);
};

// OUT: the outputs, from the states that the segments begin with; else the states that their rows leave, from nothing.  PW: parts of the weighted c.
template <typename T, int DT, bool DUAL, bool OUT, int PW>
__global__ void __launch_bounds__(2 * DT, ChunkShape<T, DT, DUAL, OUT>::CTAS) chunk_kernel(const __grid_constant__ Scan p, const uint32_t wide) {
  using S = ChunkShape<T, DT, DUAL, OUT>;
  using Two = Formed<T, 2>;
  constexpr int NT = S::NT, LD = S::LD, ND = DT / 8, KD = DT / 16, NW = DT / 16, SIDES = DUAL ? 2 : 1;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float power[CH + 2], less1[CH + 2];  // l^j and l^j - 1
  constexpr int TILE = S::TILE;
  T* tiles_b = reinterpret_cast<T*>(smem);     // two times b and its tangent
  T* tiles_c = tiles_b + 2 * SIDES * TILE;     // c and its tangent (states alone: two times)
  T* tiles_a = tiles_c + SIDES * TILE;         // a and its tangent, TWO_A: twice
  T* sP = tiles_a + (S::TWO_A ? 2 : 1) * SIDES * TILE;  // products in two parts, then their tangents
  float* sP32 = reinterpret_cast<float*>(sP);           // float16: in 32 bits
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
    stage<T, DT, NT>(to, p.b, of_head(p.b), p.D, row0, rows, n, p.reversed, wide & 1);
    if (DUAL) stage<T, DT, NT>(to + TILE, p.tb, of_head(p.tb), p.D, row0, rows, n, p.reversed, wide & 8);
  };
  auto fetch_c = [&](int half, int row0) {
    const int rows = min(CH, row_end - row0);
    T* to = tiles_c + (OUT ? 0 : half * SIDES * TILE);
    stage<T, DT, NT>(to, p.c, of_head(p.c), p.E, row0, rows, n, p.reversed, wide & 2);
    if (DUAL) stage<T, DT, NT>(to + TILE, p.tc, of_head(p.tc), p.E, row0, rows, n, p.reversed, wide & 16);
  };
  auto fetch_a = [&](int half, int row0) {
    const int rows = min(CH, row_end - row0);
    T* to = tiles_a + (S::TWO_A ? half * SIDES * TILE : 0);
    stage<T, DT, NT>(to, p.a, of_head(p.a), p.D, row0, rows, n, p.reversed, wide & 4);
    if (DUAL) stage<T, DT, NT>(to + TILE, p.ta, of_head(p.ta), p.D, row0, rows, n, p.reversed, wide & 32);
  };
  // where a lane of ldmatrix reads: first operand and transposed second one (rows 0-7, 8-15, then columns 8-15), second one (columns 8-15, then rows 8-15)
  const int lane_row = lane & 15, lane_col = lane >> 4 << 3;
  const int lane_row_n = (lane & 7) + (lane >> 4 << 3), lane_col_n = lane >> 3 & 1 ? 8 : 0;
  constexpr uint32_t SZ = 2, ROWS16 = 16 * LD * SZ, P16 = 16 * LP * SZ, PART = CH * LP * SZ, SIDE = (SIDES - 1) * TILE * SZ;
  const uint32_t at_first = (lane_row * LD + lane_col) * SZ;  // of a first operand, or a transposed second one
  const uint32_t at_second = (lane_row_n * LD + lane_col_n) * SZ;
  const uint32_t lane_p = shared_address(sP) + (lane_row * LP + lane_col) * SZ;

  int now = 0;
  if (row_begin < row_end) {
    fetch_b(0, row_begin), fetch_c(0, row_begin);
    if (OUT) fetch_a(0, row_begin);
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
      if (S::TWO_A) fetch_a(now ^ 1, row0 + CH);
      cp_async_commit();
    }
    const uint32_t tile_b = shared_address(tiles_b + now * SIDES * TILE), lane_b = tile_b + at_first;
    const uint32_t lane_a = shared_address(tiles_a + (S::TWO_A ? now * SIDES * TILE : 0)) + at_first;
    const uint32_t lane_c = shared_address(tiles_c + (OUT ? 0 : now * SIDES * TILE)) + at_first + e0 * SZ;
    uint32_t fc[SIDES][4][4];  // columns e0 .. e0 + 15 of c: 16 rows each; second operand's halves (0, 1) and (2, 3)
    auto load_c = [&] {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        ldmatrix_t(fc[0][k], lane_c + k * ROWS16);
        if (DUAL) ldmatrix_t(fc[SIDES - 1][k], lane_c + SIDE + k * ROWS16);
      }
    };
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
            mma<T>(x[0][0], fa, fb[0], fb[1]), mma<T>(x[0][1], fa, fb[2], fb[3]);
            if constexpr (DUAL) {
              uint32_t fta[4], ftb[4];
              ldmatrix(fta, lane_a + SIDE + i * ROWS16 + k * 32);
              ldmatrix(ftb, tile_b + at_second + SIDE + j * ROWS16 + k * 32);
              mma<T>(x[1][0], fta, fb[0], fb[1]), mma<T>(x[1][1], fta, fb[2], fb[3]);
              mma<T>(x[1][0], fa, ftb[0], ftb[1]), mma<T>(x[1][1], fa, ftb[2], ftb[3]);
            }
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int r = i * 16 + g + u * 8, s = j * 16 + half * 8 + 2 * t;
            const float w0 = power[max(0, r - s)], w1 = power[max(0, r - s - 1)];
#pragma unroll
            for (int side = 0; side < SIDES; ++side) {
              // (selected, not multiplied by zero: an entry right of the diagonal may be infinite)
              const float2 y = make_float2(s <= r ? x[side][half][2 * u] * w0 : 0.f, s + 1 <= r ? x[side][half][2 * u + 1] * w1 : 0.f);
              if constexpr (S::HALF) {
                *reinterpret_cast<float2*>(sP32 + side * CH * LP + r * LP + s) = y;
              } else {
                Two f;
                f.set(y);
                *reinterpret_cast<uint32_t*>(sP + (2 * side) * CH * LP + r * LP + s) = f.part[0];
                *reinterpret_cast<uint32_t*>(sP + (2 * side + 1) * CH * LP + r * LP + s) = f.part[1];
              }
            }
          }
      }
      // products of 16 rows from i * 16 on with 16 rows of c, or their tangents, as a first operand
      auto load_p = [&](Two (&f)[4], int side, int i, int k) {
        if constexpr (S::HALF) {
          const float* at = sP32 + side * CH * LP + (i * 16 + g) * LP + k * 16 + 2 * t;
#pragma unroll
          for (int v = 0; v < 4; ++v) f[v].set(*reinterpret_cast<const float2*>(at + (v & 1) * 8 * LP + (v >> 1) * 8));
        } else {
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            uint32_t r[4];
            ldmatrix(r, lane_p + (2 * side + part) * PART + i * P16 + k * 32);
#pragma unroll
            for (int v = 0; v < 4; ++v) f[v].part[part] = r[v];
          }
        }
      };
      // acc += products times c, with tangents products times tc and their tangents times c
      auto add_own = [&](float (&value)[2][4], float (&tangent)[2][4], int i, int k) {
        Two fp[4];
        load_p(fp, 0, i, k);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mma_formed(value[j], fp, fc[0][k][2 * j], fc[0][k][2 * j + 1]);
          if (DUAL) mma_formed(tangent[j], fp, fc[SIDES - 1][k][2 * j], fc[SIDES - 1][k][2 * j + 1]);
        }
        if constexpr (DUAL) {
          load_p(fp, 1, i, k);
#pragma unroll
          for (int j = 0; j < 2; ++j) mma_formed(tangent[j], fp, fc[0][k][2 * j], fc[0][k][2 * j + 1]);
        }
      };
      auto part_of_m = [&](Two& f, int side, int k, int j, int u) { f.set(make_float2(M[side][2 * k + u][2 * j], M[side][2 * k + u][2 * j + 1])); };
      // 16 rows from i * 16 on, in accumulators.  Four lanes hold two rows of 32 bytes, a word of each half row in each: they are turned so that each
      // holds 16 successive bytes of row g or g + 8.
      T* mine[SIDES];
      long long step[SIDES];
#pragma unroll
      for (int side = 0; side < SIDES; ++side) {
        const jvpfa_linear_tensor& x = side ? p.tout : p.out;
        const int r = g + (t >> 1) * 8;
        mine[side] = static_cast<T*>(const_cast<void*>(x.p)) + of_head(x) + (long long)(p.reversed ? n - 1 - row0 - r : row0 + r) * x.stride[2] + e0 + (t & 1) * 8;
        step[side] = (p.reversed ? -16 : 16) * x.stride[2];
      }
      auto answer = [&](int i, const float (&tile)[SIDES][2][4]) {
#pragma unroll
        for (int side = 0; side < SIDES; ++side) {
          const jvpfa_linear_tensor& x = side ? p.tout : p.out;
          uint32_t v[4];  // (row g or g + 8, columns 0-7 or 8-15) of the tile, two entries
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j) v[2 * u + j] = Elem<T>::pack(p.scale * tile[side][j][2 * u], p.scale * tile[side][j][2 * u + 1]);
          uint32_t s;
          s = __shfl_xor_sync(0xffffffffu, t & 1 ? v[0] : v[1], 1), (t & 1 ? v[0] : v[1]) = s;
          s = __shfl_xor_sync(0xffffffffu, t & 1 ? v[2] : v[3], 1), (t & 1 ? v[2] : v[3]) = s;
          s = __shfl_xor_sync(0xffffffffu, t & 2 ? v[0] : v[2], 2), (t & 2 ? v[0] : v[2]) = s;
          s = __shfl_xor_sync(0xffffffffu, t & 2 ? v[1] : v[3], 2), (t & 2 ? v[1] : v[3]) = s;
          const int e = e0 + (t & 1) * 8;
          if (x.p && i * 16 + g + (t >> 1) * 8 < rows && e < p.E) {
            if (wide >> (6 + side) & 1) {
              *reinterpret_cast<uint4*>(mine[side]) = make_uint4(v[0], v[1], v[2], v[3]);
            } else {
#pragma unroll 1
              for (int j = 0; j < 8 && e + j < p.E; ++j) {
                const uint32_t w = j < 2 ? v[0] : j < 4 ? v[1] : j < 6 ? v[2] : v[3];
                const uint16_t bits = (uint16_t)(w >> (j % 2 * 16));
                mine[side][j] = *reinterpret_cast<const T*>(&bits);
              }
            }
          }
          mine[side] += step[side];
        }
      };
      // what is before the chunk, and its own rows
      if constexpr (S::LOOP) {
        Two m[SIDES][KD][2][2];  // side, step, columns 0-7 or 8-15, rows 0-7 or 8-15
#pragma unroll
        for (int side = 0; side < SIDES; ++side)
#pragma unroll
          for (int k = 0; k < KD; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int u = 0; u < 2; ++u) part_of_m(m[side][k][j][u], side, k, j, u);
        load_c();
        __syncthreads();  // the products are there, and nobody reads c again
        if (more) {
          fetch_c(0, row0 + CH);
          cp_async_commit();
        }
#pragma unroll 1
        for (int i = 0; i * 16 < rows; ++i) {
          float acc[SIDES][2][4] = {}, other[2][4] = {};  // a M, with tangents a tM and ta M
#pragma unroll
          for (int k = 0; k < KD; ++k) {
            uint32_t fa[4], fta[4];
            ldmatrix(fa, lane_a + i * ROWS16 + k * 32);
            if (DUAL) ldmatrix(fta, lane_a + SIDE + i * ROWS16 + k * 32);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              mma_formed(acc[0][j], fa, m[0][k][j][0], m[0][k][j][1]);
              if (DUAL) mma_formed(acc[SIDES - 1][j], fa, m[SIDES - 1][k][j][0], m[SIDES - 1][k][j][1]);
              if (DUAL) mma_formed(other[j], fta, m[0][k][j][0], m[0][k][j][1]);
            }
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float f = power[min(i * 16 + g + u * 8, rows - 1) + 1 + shift];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int v = 2 * u; v < 2 * u + 2; ++v) {
                acc[0][j][v] *= f;
                if (DUAL) acc[SIDES - 1][j][v] = (acc[SIDES - 1][j][v] + other[j][v]) * f;
              }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k > i) break;
            add_own(acc[0], acc[SIDES - 1], i, k);
          }
          answer(i, acc);
        }
        if constexpr (!S::TWO_A) {
          __syncthreads();  // nobody reads a again
          if (more) {
            fetch_a(0, row0 + CH);
            cp_async_commit();
          }
        }
      } else {
        float acc[4][SIDES][2][4] = {};
#pragma unroll
        for (int k = 0; k < KD; ++k) {
          Two m[SIDES][2][2];  // side, columns 0-7 or 8-15, rows 0-7 or 8-15
#pragma unroll
          for (int side = 0; side < SIDES; ++side)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int u = 0; u < 2; ++u) part_of_m(m[side][j][u], side, k, j, u);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t fa[4];
            ldmatrix(fa, lane_a + i * ROWS16 + k * 32);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              mma_formed(acc[i][0][j], fa, m[0][j][0], m[0][j][1]);
              if (DUAL) mma_formed(acc[i][SIDES - 1][j], fa, m[SIDES - 1][j][0], m[SIDES - 1][j][1]);
            }
            if constexpr (DUAL) {
              ldmatrix(fa, lane_a + SIDE + i * ROWS16 + k * 32);
#pragma unroll
              for (int j = 0; j < 2; ++j) mma_formed(acc[i][1][j], fa, m[0][j][0], m[0][j][1]);
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
              for (int j = 0; j < 2; ++j) acc[i][side][j][2 * u] *= f, acc[i][side][j][2 * u + 1] *= f;
          }
        load_c();
        __syncthreads();  // the products are there, and nobody reads a and c again
        if (more) {
          fetch_c(0, row0 + CH), fetch_a(0, row0 + CH);
          cp_async_commit();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i * 16 >= rows) break;
#pragma unroll
          for (int k = 0; k <= i; ++k) add_own(acc[i][0], acc[i][SIDES - 1], i, k);
          answer(i, acc[i]);
        }
      }
    } else {
      load_c();
    }
    // M = l^rows M + sum of l^(rows - 1 - s) b_s c_s^T.  As a first operand the words of c are (0, 2, 1, 3).
    Weighted<T, PW> wc[SIDES][4][4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int s = k * 16 + u * 8 + 2 * t;
        const float2 by = make_float2(s < rows ? power[rows - 1 - s] : 0.f, s + 1 < rows ? power[rows - 2 - s] : 0.f);
#pragma unroll
        for (int side = 0; side < SIDES; ++side)
#pragma unroll
          for (int j = 0; j < 2; ++j) wc[side][k][2 * u + j].set(__fmul2_rn(of_word<T>(fc[side][k][2 * j + u]), by));
      }
    const Down down = down_of(power[rows + shift], less1[rows + shift]);
#pragma unroll
    for (int d = 0; d < ND; d += 2) {
      float x[SIDES][2][4] = {};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t fb[4];
        ldmatrix_t(fb, lane_b + k * ROWS16 + d * 16);
        Formed<T, PW> fa[4] = {wc[0][k][0].get(), wc[0][k][1].get(), wc[0][k][2].get(), wc[0][k][3].get()};
        mma_formed(x[0][0], fa, fb[0], fb[1]), mma_formed(x[0][1], fa, fb[2], fb[3]);
        if constexpr (DUAL) {
          const Formed<T, PW> fta[4] = {wc[1][k][0].get(), wc[1][k][1].get(), wc[1][k][2].get(), wc[1][k][3].get()};
          mma_formed(x[1][0], fta, fb[0], fb[1]), mma_formed(x[1][1], fta, fb[2], fb[3]);
          ldmatrix_t(fb, lane_b + SIDE + k * ROWS16 + d * 16);
          mma_formed(x[1][0], fa, fb[0], fb[1]), mma_formed(x[1][1], fa, fb[2], fb[3]);
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
            const float2 sum = __ffma2_rn(old, make_float2(down.by, down.by),
                                          __ffma2_rn(old, make_float2(down.keep, down.keep), make_float2(x[side][u][j], x[side][u][j + 1])));
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
      const int to = min(p.L, row_begin + p.segment);
      for (int row = max(n, row_begin) + warp; row < to; row += NT / 32)
        for (int e = lane; e < p.E; e += 32) out[row * x.stride[2] + e] = Elem<T>::from_float(0.f);
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

template <typename T, int DT, bool DUAL, bool OUT, int PW>
int launch(const Scan& s, cudaStream_t stream) {
  static SmemOptIn opt;
  using S = ChunkShape<T, DT, DUAL, OUT>;
  const auto kernel = chunk_kernel<T, DT, DUAL, OUT, PW>;
  constexpr size_t bytes = S::bytes;
  static_assert(S::fits(bytes), "an SM's shared memory");
  if (!opt.ensure(reinterpret_cast<const void*>(kernel), bytes)) return JVPFA_ERR_CUDA;
  uint32_t wide = 0;
  const jvpfa_linear_tensor* tensors[8] = {&s.b, &s.c, &s.a, &s.tb, &s.tc, &s.ta, &s.out, &s.tout};
  for (int i = 0; i < 8; ++i)
    if (wide_tensor<T>(*tensors[i], s, i % 3 == 1 || i >= 6 ? s.E : s.D)) wide |= 1u << i;
  kernel<<<(unsigned)((long long)s.B * s.H * s.segments), S::NT, bytes, stream>>>(s, wide);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "chunk_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
}

template <typename T, int DT, bool OUT>
int launch(const Scan& s, cudaStream_t stream) {
  if (s.last || s.tlast) return s.dual ? launch<T, DT, true, OUT, 3>(s, stream) : launch<T, DT, false, OUT, 3>(s, stream);
  return s.dual ? launch<T, DT, true, OUT, 2>(s, stream) : launch<T, DT, false, OUT, 2>(s, stream);
}

template <typename T, bool OUT>
int launch(const Scan& s, cudaStream_t stream) {
  const int width = s.D > s.E ? s.D : s.E;
  return width <= 32 ? launch<T, 32, OUT>(s, stream) : width <= 64 ? launch<T, 64, OUT>(s, stream) : launch<T, 128, OUT>(s, stream);
}

template <typename T, int DT>
int ctas_of(const Scan& s) {
  return s.dual ? ChunkShape<T, DT, true, true>::CTAS : ChunkShape<T, DT, false, true>::CTAS;
}

}  // namespace

template <typename T>
int chunk_ctas(const Scan& s) {
  const int width = s.D > s.E ? s.D : s.E;
  return width <= 32 ? ctas_of<T, 32>(s) : width <= 64 ? ctas_of<T, 64>(s) : ctas_of<T, 128>(s);
}

template <typename T>
int launch_chunks(const Scan& s, bool outputs, cudaStream_t stream) {
  return outputs ? launch<T, true>(s, stream) : launch<T, false>(s, stream);
}

}  // namespace linear
}  // namespace jvpfa

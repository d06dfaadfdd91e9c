// The map of linear_common.cuh for the 16-bit types, on float16 instructions.
//
// A CTA takes a segment of one head's rows in chunks of 64.  Warp w keeps columns 16 w .. 16 w + 15 of M in registers, transposed: as they
// stand the accumulators are the second operand of a M, and the columns of c that the warp multiplies the chunk's products by are, loaded
// once, also the first operand of what the chunk adds to M.  A chunk is
//   the tiles of a, b and c in float16, each with a power of two of its own;   products (a_t . b_s) l^(t-s), 16 x 16 blocks shared out among the
//   warps, through shared memory;   for 16 rows after the other a M and products times c;   M = l^64 M + (c l^(63-s))^T b.
// float16 has 11 bits where bfloat16 has 8: a bfloat16 entry fits it exactly within 30 powers of two of its tile's largest (what is below is
// 2^-39 of that), and what is formed in 32 bits and multiplied again (products, M, weighted c) takes one instruction for bfloat16 results, which it
// leaves at 1.0 of their own rounding, where bfloat16 parts take two.  float16 tensors take two parts, and the weighted c where the state is
// answered.  Each of these has a power of two as well (a block's, a warp's), so that nothing passes 65504 or falls below 2^-14 that counts.  What a
// chunk adds to M, or a block to a result, is formed apart and added rounded to nearest, since the tensor cores truncate.
// What bounds it: latencies, with two to four warps a scheduler.  bf16 B4 H16 L8192 D128 takes 304 us for a map, 78 of them at the rate of mma.sync (2.8
// million products a chunk; tensor pipe 26 % busy, issue slots 42 %), fp16 407; B4 H16 L2048 D64 with tangents 89, 21 % and 33 % (a third of the waits
// for a result, a fifth for instructions).  64 rows, since products within a chunk cost 64 (D + E) / 2 a row and M 2 D E; M in registers, since it is
// read and written every chunk.  Registers set the warps: 128 a thread for D = 64 four times on an SM and D = 128 twice, 255 with tangents.
#pragma once
#include <type_traits>

#include "linear_common.cuh"

namespace jvpfa {
namespace linear {

namespace {

constexpr int CH = 64, LP = CH + 8;
constexpr int kBlocks = 10;  // of 16 x 16 products on and left of the diagonal

// Addresses in shared memory are 32-bit numbers here: what is added to a lane's own is part of the instruction then.
__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldmatrix(uint32_t r[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix_t(uint32_t r[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float two_to(int k) { return __int_as_float((min(max(k, -126), 127) + 127) << 23); }
// The power of two that brings numbers up to `largest` (the bits of a float that is not negative) below 2^15.
__device__ __forceinline__ int room_for(uint32_t largest) { return largest == 0 ? 0 : min(14 - ((int)(largest >> 23) - 127), 126); }
constexpr uint32_t kInfinite = 0x7f800000u;
__device__ __forceinline__ uint32_t larger_finite(uint32_t most, float x) {
  const uint32_t bits = __float_as_uint(fabsf(x));
  return bits < kInfinite && bits > most ? bits : most;
}
__device__ __forceinline__ uint32_t halves(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 of_halves(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
// Two values as pairs of float16 numbers, each the rounding of what the ones before it left.
template <int PARTS>
__device__ __forceinline__ void split(float2 x, uint32_t (&part)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    part[i] = halves(x.x, x.y);
    if (i + 1 < PARTS) x = __ffma2_rn(of_halves(part[i]), make_float2(-1.f, -1.f), x);
  }
}
// Two entries of a tensor.
template <typename T>
__device__ __forceinline__ float2 of_word(uint32_t w) {
  if constexpr (std::is_same_v<T, __half>)
    return of_halves(w);
  else
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
struct Two;
template <>
struct Two<__half> { using type = __half2; };
template <>
struct Two<__nv_bfloat16> { using type = __nv_bfloat162; };

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

// A thread's own pieces of a tile that has arrived: their largest finite magnitude (bits of a float), and all of them in float16, times 2^k.
constexpr int kOwn = CH / 16;
template <typename T, int DT>
__device__ __forceinline__ T* own_place(T* tile, int r) {
  constexpr int LD = DT + 8, PIECES = DT / 8;
  return tile + (threadIdx.x / PIECES + r * 16) * LD + threadIdx.x % PIECES * 8;
}
template <typename T, int DT>
__device__ __forceinline__ void own(uint4 (&v)[kOwn], T* tile) {
#pragma unroll
  for (int r = 0; r < kOwn; ++r) v[r] = *reinterpret_cast<const uint4*>(own_place<T, DT>(tile, r));
}
template <typename T>
__device__ __forceinline__ uint32_t largest_of(const uint4 (&v)[kOwn]) {
  using W = typename Two<T>::type;
  W m;
  *reinterpret_cast<uint32_t*>(&m) = 0u;
#pragma unroll
  for (int r = 0; r < kOwn; ++r)
#pragma unroll
    for (const uint32_t w : {v[r].x, v[r].y, v[r].z, v[r].w}) m = __hmax2(m, __habs2(*reinterpret_cast<const W*>(&w)));  // (a NaN is passed over)
  const float2 both = of_word<T>(*reinterpret_cast<const uint32_t*>(&m));
  uint32_t most = __float_as_uint(fmaxf(both.x, both.y));
  if (most >= kInfinite) {  // the others' largest
    most = 0;
#pragma unroll
    for (int r = 0; r < kOwn; ++r)
#pragma unroll
      for (const uint32_t w : {v[r].x, v[r].y, v[r].z, v[r].w}) most = larger_finite(larger_finite(most, of_word<T>(w).x), of_word<T>(w).y);
  }
  return most;
}
template <typename T, int DT>
__device__ __forceinline__ void convert(T* tile, const uint4 (&v)[kOwn], int k) {
  const float2 by = make_float2(two_to(k), two_to(k));
  auto half_of = [&](uint32_t w) {
    const float2 x = __fmul2_rn(of_word<T>(w), by);
    return halves(x.x, x.y);
  };
#pragma unroll
  for (int r = 0; r < kOwn; ++r) *reinterpret_cast<uint4*>(own_place<T, DT>(tile, r)) = make_uint4(half_of(v[r].x), half_of(v[r].y), half_of(v[r].z), half_of(v[r].w));
}

// Shared memory of a CTA: two tiles of b (and of its tangent), which a chunk reads to its end, and of a where there is room, else one that takes the
// next rows behind the chunk's end; one of c, which is free behind the products' barrier; the products.  States alone: two tiles of b and c.
template <int DT, bool DUAL, bool OUT, int PP>
struct ChunkShape {
  static constexpr int LD = DT + 8, NT = 2 * DT, SIDES = DUAL ? 2 : 1, TILE = CH * LD;
  static constexpr int CTAS = DT == 32 ? (DUAL ? 2 : 4) : DT == 64 ? (DUAL ? 2 : 4) : DUAL ? 1 : 2;
  static constexpr size_t bytes_with(int tiles) { return 2 * SIDES * (tiles * (size_t)TILE + (OUT ? PP * (size_t)CH * LP : 0)); }
  static constexpr bool fits(size_t bytes) { return bytes * CTAS <= 227 * 1024 - CTAS * 2048; }
  static constexpr bool TWO_A = OUT && fits(bytes_with(5)), KEEP = DT <= 64;  // KEEP: a thread has registers for its pieces of all tiles
  static constexpr size_t bytes = bytes_with(TWO_A ? 5 : 4);
};

// OUT: the outputs, from the states that the segments begin with; else the states that their rows leave, from nothing.  PP: parts of products and
// of M, PW: of the weighted c.
template <typename T, int DT, bool DUAL, bool OUT, int PP, int PW>
__global__ void __launch_bounds__(2 * DT, ChunkShape<DT, DUAL, OUT, PP>::CTAS) chunk_kernel(const __grid_constant__ Scan p, const uint32_t wide) {
  using S = ChunkShape<DT, DUAL, OUT, PP>;
  constexpr int NT = S::NT, LD = S::LD, ND = DT / 8, KD = DT / 16, NW = DT / 16, SIDES = DUAL ? 2 : 1;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float power[CH + 2], less1[CH + 2];  // l^j and l^j - 1
  __shared__ uint32_t largest[6][8];               // of each tile, by warp
  __shared__ float block_unit[2][kBlocks];         // what the products' blocks are in units of
  constexpr int TILE = S::TILE;
  T* tiles_b = reinterpret_cast<T*>(smem);     // two times b and its tangent
  T* tiles_c = tiles_b + 2 * SIDES * TILE;     // c and its tangent (states alone: two times)
  T* tiles_a = tiles_c + SIDES * TILE;         // a and its tangent, TWO_A: twice
  T* sP = tiles_a + (S::TWO_A ? 2 : 1) * SIDES * TILE;  // products in their parts, then their tangents
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
    // b, its tangent, c, its tangent, a, its tangent
    T* const arrived[6] = {tiles_b + now * SIDES * TILE, tiles_b + now * SIDES * TILE + TILE, tiles_c + (OUT ? 0 : now * SIDES * TILE),
                           tiles_c + (OUT ? 0 : now * SIDES * TILE) + TILE, tiles_a + (S::TWO_A ? now * SIDES * TILE : 0),
                           tiles_a + (S::TWO_A ? now * SIDES * TILE : 0) + TILE};
    auto there = [&](int i) { return (DUAL || i % 2 == 0) && (OUT || i < 4); };
    uint4 mine_of[6][kOwn];
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      if (!there(i)) continue;
      own<T, DT>(mine_of[i], arrived[i]);
      const uint32_t m = __reduce_max_sync(0xffffffffu, largest_of<T>(mine_of[i]));
      if (lane == 0) largest[i][warp] = m;
    }
    __syncthreads();  // the largest are there, and the chunk before has been read
    if (more) {
      fetch_b(now ^ 1, row0 + CH);
      if (!OUT) fetch_c(now ^ 1, row0 + CH);
      if (S::TWO_A) fetch_a(now ^ 1, row0 + CH);
      cp_async_commit();
    }
    int room[6];
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      if (!there(i)) continue;
      room[i] = room_for(__reduce_max_sync(0xffffffffu, lane < NW ? largest[i][lane] : 0u));
      if (!S::KEEP) own<T, DT>(mine_of[i], arrived[i]);
      convert<T, DT>(arrived[i], mine_of[i], room[i]);
    }
    __syncthreads();  // everything is float16
    // what the tiles are in units of (1 of those that are zero, so that no zero meets an infinite unit)
    auto unit_of = [&](int i) { return there(i) ? two_to(-room[i]) : 0.f; };
    const float ub = unit_of(0), utb = unit_of(1), uc = unit_of(2), utc = unit_of(3), ua = unit_of(4), uta = unit_of(5);
    const uint32_t tile_b = shared_address(tiles_b + now * SIDES * TILE), lane_b = tile_b + at_first;
    const uint32_t lane_a = shared_address(arrived[4]) + at_first;
    const uint32_t lane_c = shared_address(tiles_c + (OUT ? 0 : now * SIDES * TILE)) + at_first + e0 * SZ;
    uint32_t fc[SIDES][4][4];  // columns e0 .. e0 + 15 of c: 16 rows each; second operand's halves (0, 1) and (2, 3)
    if constexpr (OUT) {
      // the chunk's products
#pragma unroll 1
      for (int block = warp; block < 10; block += NW) {
        const int i = block < 1 ? 0 : block < 3 ? 1 : block < 6 ? 2 : 3, j = block - i * (i + 1) / 2;
        float x[SIDES][2][4] = {}, z[2][4] = {};
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
              mma(z[0], fa, ftb[0], ftb[1]), mma(z[1], fa, ftb[2], ftb[3]);
            }
          }
        }
        // what they stand for, weighted (selected, not multiplied by zero: an entry right of the diagonal may be infinite)
        const float f = ua * ub, ft = uta * ub, fz = ua * utb;
        float most[SIDES] = {};
        // left of the diagonal block l^(r - c) = l^(r - 16 i) l^(16 i - c), no exponent below zero
        const float of_row[2] = {power[g], power[g + 8]};
        float of_col[2][2];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int v = 0; v < 2; ++v) of_col[half][v] = power[max(0, (i - j) * 16 - half * 8 - 2 * t - v)];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int r = i * 16 + g + (v >> 1) * 8, c = j * 16 + half * 8 + 2 * t + (v & 1);
            float by = of_row[v >> 1] * of_col[half][v & 1];
            if (i == j) by = power[max(0, r - c)];
            x[0][half][v] = c <= r ? x[0][half][v] * (by * f) : 0.f;
            most[0] = fmaxf(most[0], fabsf(x[0][half][v]));
            if constexpr (DUAL) {
              x[1][half][v] = c <= r ? (x[1][half][v] * ft + z[half][v] * fz) * by : 0.f;
              most[1] = fmaxf(most[1], fabsf(x[1][half][v]));
            }
          }
#pragma unroll
        for (int side = 0; side < SIDES; ++side) {
          uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most[side]));
          if (bits >= kInfinite) {  // what is not finite has no say for the others
            uint32_t m = 0;
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int v = 0; v < 4; ++v) m = larger_finite(m, x[side][half][v]);
            bits = __reduce_max_sync(0xffffffffu, m);
          }
          const int k = room_for(bits);
          if (lane == 0) block_unit[side][block] = two_to(-k);
          const float2 by = make_float2(two_to(k), two_to(k));
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int r = i * 16 + g + u * 8, c = j * 16 + half * 8 + 2 * t;
              uint32_t part[PP];
              split(__fmul2_rn(make_float2(x[side][half][2 * u], x[side][half][2 * u + 1]), by), part);
#pragma unroll
              for (int q = 0; q < PP; ++q) *reinterpret_cast<uint32_t*>(sP + (PP * side + q) * CH * LP + r * LP + c) = part[q];
            }
        }
      }
      // what is before the chunk, and its own rows
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
            for (int j = 0; j < 2; ++j) v[2 * u + j] = Elem<T>::pack(tile[side][j][2 * u], tile[side][j][2 * u + 1]);
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
      // M in its parts, once for all rows; then 16 rows after the other
      uint32_t m[SIDES][KD][2][2][PP];  // side, step, columns 0-7 or 8-15, rows 0-7 or 8-15, part
      float um[SIDES];
#pragma unroll
      for (int side = 0; side < SIDES; ++side) {
        float most = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int v = 0; v < 4; ++v) most = fmaxf(most, fabsf(M[side][d][v]));
        uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
        if (bits >= kInfinite) {
          uint32_t m_ = 0;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int v = 0; v < 4; ++v) m_ = larger_finite(m_, M[side][d][v]);
          bits = __reduce_max_sync(0xffffffffu, m_);
        }
        const int k_m = room_for(bits);
        um[side] = two_to(-k_m);
        const float2 by = make_float2(two_to(k_m), two_to(k_m));
#pragma unroll
        for (int k = 0; k < KD; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) split(__fmul2_rn(make_float2(M[side][2 * k + u][2 * j], M[side][2 * k + u][2 * j + 1]), by), m[side][k][j][u]);
      }
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
        float acc[SIDES][2][4] = {}, other[2][4] = {};  // a M, with tangents a tM and ta M
#pragma unroll
        for (int k = 0; k < KD; ++k) {
          uint32_t fa[4], fta[4];
          ldmatrix(fa, lane_a + i * ROWS16 + k * 32);
          if (DUAL) ldmatrix(fta, lane_a + SIDE + i * ROWS16 + k * 32);
#pragma unroll
          for (int part = PP - 1; part >= 0; --part)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              mma(acc[0][j], fa, m[0][k][j][0][part], m[0][k][j][1][part]);
              if (DUAL) mma(acc[SIDES - 1][j], fa, m[SIDES - 1][k][j][0][part], m[SIDES - 1][k][j][1][part]);
              if (DUAL) mma(other[j], fta, m[0][k][j][0][part], m[0][k][j][1][part]);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float f = p.scale * power[min(i * 16 + g + u * 8, rows - 1) + 1 + shift];
          const float f0 = f * (ua * um[0]), f1 = f * (ua * um[SIDES - 1]), f2 = f * (uta * um[0]);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 2 * u; v < 2 * u + 2; ++v) {
              if (DUAL) acc[SIDES - 1][j][v] = acc[SIDES - 1][j][v] * f1 + other[j][v] * f2;
              else
                acc[0][j][v] *= f0;
              if (DUAL) acc[0][j][v] *= f0;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (k > i) break;
          float x[SIDES][2][4] = {}, z[2][4] = {};  // products times c, with tangents products times tc and their tangents times c
#pragma unroll
          for (int part = PP - 1; part >= 0; --part) {
            uint32_t fp[4], ftp[4];
            ldmatrix(fp, lane_p + part * PART + i * P16 + k * 32);
            if (DUAL) ldmatrix(ftp, lane_p + (PP + part) * PART + i * P16 + k * 32);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              mma(x[0][j], fp, fc[0][k][2 * j], fc[0][k][2 * j + 1]);
              if (DUAL) mma(x[SIDES - 1][j], fp, fc[SIDES - 1][k][2 * j], fc[SIDES - 1][k][2 * j + 1]);
              if (DUAL) mma(z[j], ftp, fc[0][k][2 * j], fc[0][k][2 * j + 1]);
            }
          }
          const int block = i * (i + 1) / 2 + k;
          const float up = p.scale * block_unit[0][block], f0 = up * uc, f1 = up * utc, f2 = DUAL ? p.scale * block_unit[1][block] * uc : 0.f;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              if (DUAL) acc[SIDES - 1][j][v] += x[SIDES - 1][j][v] * f1 + z[j][v] * f2;
              acc[0][j][v] += x[0][j][v] * f0;
            }
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
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        ldmatrix_t(fc[0][k], lane_c + k * ROWS16);
        if (DUAL) ldmatrix_t(fc[SIDES - 1][k], lane_c + SIDE + k * ROWS16);
      }
    }
    // M = l^rows M + sum of l^(rows - 1 - s) b_s c_s^T.  As a first operand the words of c are (0, 2, 1, 3).
    uint32_t wc[SIDES][4][4][PW];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int s = k * 16 + u * 8 + 2 * t;
        const float2 by = make_float2(s < rows ? power[rows - 1 - s] : 0.f, s + 1 < rows ? power[rows - 2 - s] : 0.f);
#pragma unroll
        for (int side = 0; side < SIDES; ++side)
#pragma unroll
          for (int j = 0; j < 2; ++j) split(__fmul2_rn(of_halves(fc[side][k][2 * j + u]), by), wc[side][k][2 * u + j]);
      }
    const Down down = down_of(power[rows + shift], less1[rows + shift]);
    const float f0 = uc * ub, f1 = utc * ub, f2 = uc * utb;
#pragma unroll
    for (int d = 0; d < ND; d += 2) {
      float x[SIDES][2][4] = {}, z[2][4] = {};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t fb[4], ftb[4];
        ldmatrix_t(fb, lane_b + k * ROWS16 + d * 16);
        if (DUAL) ldmatrix_t(ftb, lane_b + SIDE + k * ROWS16 + d * 16);
#pragma unroll
        for (int part = PW - 1; part >= 0; --part) {
          const uint32_t fa[4] = {wc[0][k][0][part], wc[0][k][1][part], wc[0][k][2][part], wc[0][k][3][part]};
          mma(x[0][0], fa, fb[0], fb[1]), mma(x[0][1], fa, fb[2], fb[3]);
          if constexpr (DUAL) {
            const uint32_t fta[4] = {wc[1][k][0][part], wc[1][k][1][part], wc[1][k][2][part], wc[1][k][3][part]};
            mma(x[1][0], fta, fb[0], fb[1]), mma(x[1][1], fta, fb[2], fb[3]);
            mma(z[0], fa, ftb[0], ftb[1]), mma(z[1], fa, ftb[2], ftb[3]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          auto take_on = [&](float* to, float2 add) {
            const float2 old = make_float2(to[0], to[1]);
            const float2 sum = __ffma2_rn(old, make_float2(down.by, down.by), __ffma2_rn(old, make_float2(down.keep, down.keep), add));
            to[0] = sum.x, to[1] = sum.y;
          };
          take_on(&M[0][d + u][j], __fmul2_rn(make_float2(x[0][u][j], x[0][u][j + 1]), make_float2(f0, f0)));
          if constexpr (DUAL)
            take_on(&M[1][d + u][j], __ffma2_rn(make_float2(z[u][j], z[u][j + 1]), make_float2(f2, f2), __fmul2_rn(make_float2(x[1][u][j], x[1][u][j + 1]), make_float2(f1, f1))));
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
  constexpr int PP = std::is_same_v<T, __half> ? 2 : 1;
  const auto kernel = chunk_kernel<T, DT, DUAL, OUT, PP, PW>;
  constexpr size_t bytes = ChunkShape<DT, DUAL, OUT, PP>::bytes;
  static_assert(ChunkShape<DT, DUAL, OUT, PP>::fits(bytes), "an SM's shared memory");
  if (!opt.ensure(reinterpret_cast<const void*>(kernel), bytes)) return JVPFA_ERR_CUDA;
  uint32_t wide = 0;
  const jvpfa_linear_tensor* tensors[8] = {&s.b, &s.c, &s.a, &s.tb, &s.tc, &s.ta, &s.out, &s.tout};
  for (int i = 0; i < 8; ++i)
    if (wide_tensor<T>(*tensors[i], s, i % 3 == 1 || i >= 6 ? s.E : s.D)) wide |= 1u << i;
  kernel<<<(unsigned)((long long)s.B * s.H * s.segments), ChunkShape<DT, DUAL, OUT, PP>::NT, bytes, stream>>>(s, wide);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "chunk_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
}

template <typename T, int DT, bool OUT>
int launch(const Scan& s, cudaStream_t stream) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>)  // (else the weighted c has two parts anyway)
    if (!s.last && !s.tlast) return s.dual ? launch<T, DT, true, OUT, 1>(s, stream) : launch<T, DT, false, OUT, 1>(s, stream);
  return s.dual ? launch<T, DT, true, OUT, 2>(s, stream) : launch<T, DT, false, OUT, 2>(s, stream);
}

template <typename T, bool OUT>
int launch(const Scan& s, cudaStream_t stream) {
  const int width = s.D > s.E ? s.D : s.E;
  return width <= 32 ? launch<T, 32, OUT>(s, stream) : width <= 64 ? launch<T, 64, OUT>(s, stream) : launch<T, 128, OUT>(s, stream);
}

}  // namespace

template <typename T>
int launch_chunks(const Scan& s, bool outputs, cudaStream_t stream) {
  return outputs ? launch<T, true>(s, stream) : launch<T, false>(s, stream);
}

}  // namespace linear
}  // namespace jvpfa

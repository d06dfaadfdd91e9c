// The matrix products of the gated projection on the fifth-generation tensor cores, two SMs to a tile.
//
// A cluster of two CTAs computes 256 rows x 256 columns: every instruction (tcgen05.mma.cta_group::2, M = N = 256, K = 16) takes 128 rows
// of A and 128 columns of B from either CTA's shared memory, so an operand byte that a CTA loads serves twice the products that it
// would alone: 32 KB for each 512 cycles of products, where one CTA's 128 x 256 tiles ask for 48 KB, more than L2 delivers to all SMs.
//
// Forward (kPairGated): the columns are 128 features of wg (CTA 0's) beside the same 128 of wu (CTA 1's), so that g and u of a feature
// end up in one lane of one CTA and the gate is applied on the way out.  With tangents (kPairGatedDual) a CTA's 128 rows
// are 64 of x and the same 64 of tx: all four products of a (row, feature) are in one CTA, and of every 32 features the warp that has a
// row's value finishes 16 and the one that has its tangent the others, for which they hand each other what they hold through shared memory.
// Backward: products over the features (kPairDx: weights read across the contraction) and over the rows (kPairDw: both operands are).
//
// Sums are fp32 accumulators in TMEM, two of them (2 x 256 columns), so that a tile is written while the next is computed.  The tensor cores
// round a sum towards zero at every step of 16; fp32 results, whose products are six each of bf16 parts, are taken up in registers
// every 4 k-blocks and summed there to nearest (every 16: an error of 2.6e-6 of the norm at K = 768).
//
// Roles: warp 0 loads (TMA), warp 1 of CTA 0 issues the products, warp 2 owns TMEM, warps 4 to 11 write results.  Persistent: each cluster
// takes every (clusters)-th tile, in bands of tile rows, so that what runs at once shares its operands in L2.  Tiles of the last,
// partly empty round are cut along their depth into as many pieces as there are clusters for; the pieces' sums go through the workspace and
// join_kernel adds them in their order (plan_pair).
//
// Measured on a B200, short runs (1641 TFLOP/s is what a library product of 8192^3 reaches in one): bf16 M8192 K4096 F11008 forward 949 us = 1.56
// PFLOP/s, dx 952 us, dw 1033 us; value and tangent of M8192 K2048 F5464 474 us = 1.55; of K1024 F2736, where 16 k-blocks hardly hide the writing of
// a tile, 130 us = 1.41, and 149 us where a backward's 269 MB are kept.  In long runs the power limit sets the clock: the same forward takes 1050 us
// where the library's plain product of that size, without the gate, takes 1073.  Bound by the tensor cores' rate, or power.
#include "gated_common.cuh"

namespace jvpfa {
namespace tc5 {

namespace {

constexpr int kPairThreads = 384;
template <typename T, int KIND>
constexpr int kPairStages = sizeof(T) == 4 || KIND == kPairGated ? 5 : 6;  // (5: more room for what warps write through)
constexpr int kStageBytes = 32768;  // of a CTA: A 128 x 64, B 128 x 64
constexpr int kExchangeBytes = 32768;  // 4 pairs of warps x two directions x 2 x 16 features x 32 rows
constexpr int kMinPieceSteps = 4;
constexpr int kMinSavedSteps = 24, kMinSavedGated = 36;  // 7 us: a join's launch and its way through memory take 5 to 7, with the gate 6 to 10
constexpr int kAbortPairFull = 14, kAbortPairEmpty = 15, kAbortPairAcc = 16, kAbortPairAccEmpty = 17;

struct PairBarriers {
  uint64_t full[6], empty[6], acc_full[2], acc_empty[2];
  uint32_t tmem;
  int abort_flag;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of CTA 0's copy of a shared variable.
__device__ __forceinline__ uint32_t in_leader(const void* p) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
// What it tells is that TMEM has been read (tcgen05.wait::ld, tcgen05.fence), nothing that was written: a release at cluster scope would wait for
// every store of the thread on its way to memory first (half of the time of the fp32 kernels, which arrive once for 4 k-blocks).
__device__ __forceinline__ void arrive_in_leader(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A load into this CTA's shared memory whose bytes CTA 0's barrier counts.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(0), "r"(bar)
      : "memory");
}
// Arrives at this barrier of both CTAs when the products issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
               "h"((uint16_t)3)
               : "memory");
}
__device__ __forceinline__ void umma_pair(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %4, p;\n\t}"
      ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Tile t of the launch: the row of tiles (over all groups) and the column, in bands of p.band rows.
__device__ __forceinline__ void tile_at(const PairArgs& p, int t, int& mt, int& nt) {
  const int band = t / (p.band * p.tiles_n), r = t - band * p.band * p.tiles_n;
  const int high = min(p.band, p.tiles_m * p.groups - band * p.band);
  nt = r / high;
  mt = band * p.band + r - nt * high;
}

// A result warp's wait, which is long: it looks every 100 ns and leaves the issue slots and the power to the others.
__device__ __forceinline__ bool wait_for_sums(uint64_t* bar, uint32_t parity, const AbortState& ab) {
  return __all_sync(0xffffffffu, mbar_wait_backoff<100>(bar, parity, ab, kAbortPairAcc));
}

// What cluster `cluster` takes up as its `i`-th: a tile and the k-blocks of it, [begin, end); piece -1: all of them.
struct Item {
  int mt, nt, begin, end, piece;
};
__device__ __forceinline__ Item item_at(const PairArgs& p, int i) {
  Item r;
  int t = i;
  r.begin = 0, r.end = p.steps, r.piece = -1;
  if (i >= p.whole) {
    r.piece = i - p.whole;
    const int rest = r.piece / p.cut;
    t = p.whole + rest;
    r.begin = (r.piece - rest * p.cut) * p.piece;
    r.end = min(p.steps, r.begin + p.piece);
  }
  tile_at(p, t, r.mt, r.nt);
  return r;
}

// Results leave through the warp's own shared memory, 32 rows (a lane has a row) of N entries, so that lanes that write at once write next to
// each other.  put: 16 entries of a lane's row, from entry `first` on.
template <typename T, int N>
constexpr int kRowsBytes = 32 * (N * (int)sizeof(T) + 16);
template <typename T, int N>
__device__ __forceinline__ void put(uint8_t* mine, int lane, int first, const float (&v)[16]) {
  constexpr int E = 16 / sizeof(T), pitch = N * sizeof(T) + 16;
#pragma unroll
  for (int k = 0; k < 16 / E; ++k) {
    uint4 x;
    if constexpr (sizeof(T) == 4)
      x = make_uint4(__float_as_uint(v[k * 4]), __float_as_uint(v[k * 4 + 1]), __float_as_uint(v[k * 4 + 2]), __float_as_uint(v[k * 4 + 3]));
    else
      x = make_uint4(Elem<T>::pack(v[k * 8], v[k * 8 + 1]), Elem<T>::pack(v[k * 8 + 2], v[k * 8 + 3]),
                     Elem<T>::pack(v[k * 8 + 4], v[k * 8 + 5]), Elem<T>::pack(v[k * 8 + 6], v[k * 8 + 7]));
    *reinterpret_cast<uint4*>(mine + lane * pitch + first * sizeof(T) + k * 16) = x;
  }
}
// ... and from there to a row-major matrix, from its column c on: whole 16-byte pieces, or rows that begin anywhere.
template <typename T, int N, int M>
__device__ __forceinline__ void write_pieces(T* out, const PairArgs& p, int row0, int c, int lane, const uint8_t* mine) {
  constexpr int E = 16 / sizeof(T), U = M / E, pitch = N * sizeof(T) + 16;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int r = (i * 32 + lane) / U, k = (i * 32 + lane) % U;
    if (row0 + r < p.rows && c + k * E < p.cols)
      *reinterpret_cast<uint4*>(out + (size_t)(row0 + r) * p.cols + c + k * E) = *reinterpret_cast<const uint4*>(mine + r * pitch + k * 16);
  }
}
template <typename T, int N>
__device__ __forceinline__ void write_entries(T* out, const PairArgs& p, int row0, int c, int lane, const uint8_t* mine) {
  constexpr int pitch = N * sizeof(T) + 16;
  if constexpr (sizeof(T) == 2) {
    // Two at a time where a word begins; the lane that has none of a row beginning between words, its ends.
    uint16_t* const base = reinterpret_cast<uint16_t*>(out);
#pragma unroll 4
    for (int i = 0; i < N / 2; ++i) {
      const int r = (i * 32 + lane) / (N / 2), k = (i * 32 + lane) % (N / 2) * 2;
      const size_t at = (size_t)(row0 + r) * p.cols + c;
      const uint16_t* const e = reinterpret_cast<const uint16_t*>(mine + r * pitch);
      if (row0 + r >= p.rows) continue;
      const int odd = (int)((reinterpret_cast<uintptr_t>(base) / 2 + at) & 1);
      if (!odd || k + 2 < N) {
        if (c + k + odd + 1 < p.cols)
          *reinterpret_cast<uint32_t*>(base + at + k + odd) = e[k + odd] | (uint32_t)e[k + odd + 1] << 16;
        else if (c + k + odd < p.cols)
          base[at + k + odd] = e[k + odd];
      } else {
        if (c < p.cols) base[at] = e[0];
        if (c + N - 1 < p.cols) base[at + N - 1] = e[N - 1];
      }
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < N; ++i) {
      const int r = (i * 32 + lane) / N, k = (i * 32 + lane) % N;
      if (row0 + r < p.rows && c + k < p.cols) out[(size_t)(row0 + r) * p.cols + c + k] = reinterpret_cast<const T*>(mine + r * pitch)[k];
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void write_rows(T* out, const PairArgs& p, int row0, int c, int lane, const uint8_t* mine) {
  __syncwarp();
  if (p.aligned)
    write_pieces<T, N, N>(out, p, row0, c, lane, mine);
  else
    write_entries<T, N>(out, p, row0, c, lane, mine);
  __syncwarp();
}

// The gate, for 16 features from c on of 32 rows: what a backward reads, h in place of g and th in place of tg.
template <typename T, bool DUAL>
__device__ __forceinline__ void finish_gated(const PairArgs& p, int row0, int c, int lane, float (&g)[16], float (&u)[16], float (&tg)[16],
                                             float (&tu)[16]) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int N = 16;
  if (p.kept && row0 < p.rows && c < p.cols) {
    uint8_t* block = p.kept + (size_t)((row0 >> 5) * ((p.cols + 31) >> 5) + (c >> 5)) * (DUAL ? 4 : 2) * Kept<T>::kBlock;
    keep<T>(block, lane, c & 31, g);
    keep<T>(block + Kept<T>::kBlock, lane, c & 31, u);
    if constexpr (DUAL) {
      keep<T>(block + 2 * Kept<T>::kBlock, lane, c & 31, tg);
      keep<T>(block + 3 * Kept<T>::kBlock, lane, c & 31, tu);
    }
  }
  with_activation(p.activation, [&](auto kind) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const Activated y = activate<decltype(kind)::value, EXACT>(g[j]);
      if constexpr (DUAL) tg[j] = y.d1 * tg[j] * u[j] + y.a * tu[j];
      g[j] = y.a * u[j];
    }
  });
}
// h and th of finish_gated on their way out.
template <typename T>
__device__ __forceinline__ void write_dual(const PairArgs& p, int row0, int c, int lane, uint8_t* mine, const float (&h)[16], const float (&th)[16]) {
  put<T, 16>(mine, lane, 0, h);
  write_rows<T, 16>(static_cast<T*>(p.h), p, row0, c, lane, mine);
  put<T, 16>(mine, lane, 0, th);
  write_rows<T, 16>(static_cast<T*>(p.th), p, row0, c, lane, mine);
}

// A thread's b-th 16 sums of its piece.
__device__ __forceinline__ float4* partial_at(const PairArgs& p, int piece, int rank, int warp, int b, int lane) {
  return reinterpret_cast<float4*>(p.partial + ((((size_t)piece * 2 + rank) * 8 + warp) * 8 + b) * 512) + lane;
}

template <typename T>
struct Operand {
  using type = T;
  static constexpr bool kParts = false;
};
template <>
struct Operand<float> {
  using type = __nv_bfloat16;
  static constexpr bool kParts = true;
};

// Entries of a row that a warp has room for.
template <typename T, int KIND>
constexpr int kAtOnce = KIND == kPairGated && sizeof(T) == 2 ? 64 : 32;
template <typename T, int KIND>
constexpr int kThroughBytes = KIND == kPairGatedDual ? kExchangeBytes : 8 * kRowsBytes<T, kAtOnce<T, KIND>>;

template <typename T, int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    pair_kernel(const __grid_constant__ PairArgs p, const __grid_constant__ PairMaps maps) {
  constexpr bool GATED = KIND <= kPairGatedDual, DUAL = KIND == kPairGatedDual, A_MN = KIND == kPairDw, B_MN = KIND >= kPairDx;
  constexpr bool PARTS = Operand<T>::kParts;
  constexpr int STAGES = kPairStages<T, KIND>, AT_ONCE = kAtOnce<T, KIND>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint8_t* through = smem + STAGES * kStageBytes;  // for the warps that write
  PairBarriers& bar = *reinterpret_cast<PairBarriers*>(through + kThroughBytes<T, KIND>);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;

  if (threadIdx.x == 32) {
    for (int i = 0; i < 4; ++i) prefetch_tmap(&maps.a[i]);
    for (int i = 0; i < 2; ++i) prefetch_tmap(&maps.b[i]);
  }
  if (threadIdx.x == 0) {
    const int before = *reinterpret_cast<volatile int*>(p.status);
    bar.abort_flag = before;
    for (int i = 0; i < STAGES; ++i) mbar_init(&bar.full[i], 1), mbar_init(&bar.empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bar.acc_full[i], 1), mbar_init(&bar.acc_empty[i], 16);
    fence_mbar_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&bar.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the other CTA's barriers exist
  tc_fence_after();
  const uint32_t tmem = bar.tmem;
  const AbortState ab{&bar.abort_flag, p.status};
  const bool refused = bar.abort_flag != 0;

  if (warp == 0) {
    if (lane == 0 && !refused) {
      const int rows_of_tile = DUAL ? 128 : 256;
      int n = 0;  // k-blocks so far
      bool ok = true;
      for (int i = cluster; i < p.items && ok; i += clusters) {
        const Item it = item_at(p, i);
        const int group = it.mt / p.tiles_m, m0 = (it.mt - group * p.tiles_m) * rows_of_tile + (int)rank * (rows_of_tile / 2);
        const int n0 = GATED ? it.nt * 128 : it.nt * 256 + (int)rank * 128;
        int segment = it.begin / p.kblocks, kb = it.begin - segment * p.kblocks, source = segment / p.pairs, pair = segment - source * p.pairs;
        for (int step = it.begin; step < it.end; ++step, ++n) {
          const CUtensorMap* ma = &maps.a[GATED ? 0 : 2 * group + source];
          const CUtensorMap* mb = &maps.b[GATED ? rank : source];
          const int pa = PARTS ? 0x850 >> (2 * pair) & 3 : 0, pb = PARTS ? 0x244 >> (2 * pair) & 3 : 0;
          const int stage = n % STAGES;
          ok = mbar_wait(&bar.empty[stage], (n / STAGES & 1) ^ 1, ab, kAbortPairEmpty);
          if (!ok) break;
          if (rank == 0) mbar_expect_tx(&bar.full[stage], 2 * kStageBytes);
          const uint32_t full = in_leader(&bar.full[stage]), to = smem_u32(smem + stage * kStageBytes);
          if constexpr (A_MN) {
            tma_load_pair(to, ma, full, m0, kb * 64, pa);
            tma_load_pair(to + 8192, ma, full, m0 + 64, kb * 64, pa);
          } else {
            tma_load_pair(to, ma, full, kb * 64, m0, pa);
            if constexpr (DUAL) tma_load_pair(to + 8192, &maps.a[1], full, kb * 64, m0, pa);
          }
          if constexpr (B_MN) {
            tma_load_pair(to + 16384, mb, full, n0, kb * 64, pb);
            tma_load_pair(to + 16384 + 8192, mb, full, n0 + 64, kb * 64, pb);
          } else {
            tma_load_pair(to + 16384, mb, full, kb * 64, n0, pb);
          }
          if (++kb == p.kblocks) {
            kb = 0;
            if (++pair == p.pairs) pair = 0, ++source;
          }
        }
      }
      // What the products have still to say to this CTA's barriers arrives before it ends.
      for (int i = 0; i < STAGES && ok; ++i, ++n)
        ok = mbar_wait(&bar.empty[n % STAGES], (n / STAGES & 1) ^ 1, ab, kAbortPairEmpty);
    }
  } else if (warp == 1) {
    if (rank == 0 && !refused) {
      constexpr uint32_t idesc = make_idesc(Fmt<typename Operand<T>::type>::kIdesc, 256, 256, A_MN, B_MN);
      constexpr uint32_t lbo = (8192 >> 4) << 16;
      constexpr uint32_t step_a = A_MN ? 128 : 2, step_b = B_MN ? 128 : 2;  // 16 of the contraction, in 16 bytes
      int n = 0, acc = 0;
      bool ok = true;
      for (int i = cluster; i < p.items && ok; i += clusters) {
        const Item it = item_at(p, i);
        for (int done = it.begin; done < it.end && ok; ++acc) {
          const int upto = min(it.end, done + p.chunk), buf = acc & 1;
          ok = mbar_wait_warp(&bar.acc_empty[buf], (acc >> 1 & 1) ^ 1, ab, kAbortPairAccEmpty);
          if (!ok) break;
          tc_fence_after();
          for (bool first = true; done < upto; ++done, ++n) {
            const int stage = n % STAGES;
            ok = mbar_wait_warp(&bar.full[stage], n / STAGES & 1, ab, kAbortPairFull);
            if (!ok) break;
            tc_fence_after();
            const uint32_t a = (smem_u32(smem + stage * kStageBytes) & 0x3ffff) >> 4, b = a + (16384 >> 4);
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_pair(tmem + buf * 256, (A_MN ? lbo : kDescLo) | (a + k * step_a), (B_MN ? lbo : kDescLo) | (b + k * step_b), idesc,
                          !first || k > 0);
              commit_pair(&bar.empty[stage]);
            }
            __syncwarp();
            first = false;
          }
          if (ok && elect_one()) commit_pair(&bar.acc_full[buf]);
          __syncwarp();
        }
      }
    }
  } else if (warp >= 4) {
    const int e = warp - 4, q = warp & 3, half = e >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    uint8_t* const mine = through + (DUAL ? ((half * 2 + (q & 1)) * 2 + (q >> 1)) * 4096 : e * kRowsBytes<T, AT_ONCE>);
    int acc = 0;
    bool ok = !refused;
    for (int i = cluster; i < p.items; i += clusters) {
      const Item it = item_at(p, i);
      const int group = it.mt / p.tiles_m, m = it.mt - group * p.tiles_m;
      const int row0 = DUAL ? m * 128 + (int)rank * 64 + (q & 1) * 32 : m * 256 + (int)rank * 128 + q * 32;
      auto release = [&](int buf) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_in_leader(in_leader(&bar.acc_empty[buf]));
      };
      // this thread's 128 accumulators: gated 64 of g and the 64 of u that belong to them, else 128 columns
      uint32_t col = 0;
      auto column = [&](int c) { return col + (GATED ? (c >> 6) * 128 + half * 64 + (c & 63) : half * 128 + c); };
      if constexpr (PARTS) {
        float sum[8][16];
#pragma unroll
        for (int b = 0; b < 8; ++b)
#pragma unroll
          for (int j = 0; j < 16; ++j) sum[b][j] = 0.f;
        for (int done = it.begin; done < it.end; done += p.chunk) {
          const int buf = acc & 1;
          ok = ok && wait_for_sums(&bar.acc_full[buf], acc >> 1 & 1, ab);
          if (!ok) break;
          tc_fence_after();
          col = lanes + buf * 256;
#pragma unroll
          for (int b = 0; b < 8; ++b) {
            uint32_t r[16];
            tmem_ld16(column(b * 16), r);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) sum[b][j] += __uint_as_float(r[j]);
          }
          if (done + p.chunk < it.end) release(acc++ & 1);
        }
        // The sums go back where the last of their terms came from, so that what follows can go through them in a loop.
        if (ok) {
#pragma unroll
          for (int b = 0; b < 8; ++b) tmem_st16(column(b * 16), reinterpret_cast<const uint32_t(&)[16]>(sum[b]));
          tmem_wait_st();
        }
      } else {
        ok = ok && wait_for_sums(&bar.acc_full[acc & 1], acc >> 1 & 1, ab);
        if (ok) tc_fence_after();
        col = lanes + (acc & 1) * 256;
      }
      // Neighbouring accumulators of this thread (to be waited for), NaN after a wait that gave up.
      auto take16 = [&](int c, float (&v)[16]) {
        if (ok) {
          tmem_ld16(column(c), reinterpret_cast<uint32_t(&)[16]>(v));
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = poison_f32();
        }
      };
      auto taken = [&](bool last) {
        if (!ok) return;
        tmem_wait_ld();
        if (last) release(acc & 1);
      };
      // (Loops that stay loops: a CTA of a short call goes through this once, and the time of straight-line code is that of fetching it.)
      if (it.piece >= 0) {
#pragma unroll 1
        for (int b = 0; b < 8; ++b) {
          float v[16];
          take16(b * 16, v);
          taken(b == 7);
          float4* to = partial_at(p, it.piece, (int)rank, e, b, lane);
#pragma unroll
          for (int j = 0; j < 4; ++j) to[j * 32] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
      } else if constexpr (DUAL) {
        // Of 32 features the warp of the value finishes 0 to 15, that of the tangent the others.
        const bool tangent = q >= 2;
        const int pair_id = half * 2 + (q & 1);
        float* const to = reinterpret_cast<float*>(mine) + lane;
        const float* const from = reinterpret_cast<const float*>(through + (pair_id * 2 + (tangent ? 0 : 1)) * 4096) + lane;
#pragma unroll 1
        for (int b = 0; b < 2; ++b) {
          float g[16], u[16], tg[16], tu[16];  // first what is handed over, of the other's 16 features, then one's own
          take16(b * 32 + (tangent ? 0 : 16), tg);
          take16(64 + b * 32 + (tangent ? 0 : 16), tu);
          take16(b * 32 + (tangent ? 16 : 0), g);
          take16(64 + b * 32 + (tangent ? 16 : 0), u);
          taken(b == 1);
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 16; ++j) to[j * 32] = tg[j], to[(16 + j) * 32] = tu[j];
          asm volatile("bar.sync %0, 64;" ::"r"(1 + pair_id) : "memory");
#pragma unroll
          for (int j = 0; j < 16; ++j) tg[j] = from[j * 32], tu[j] = from[(16 + j) * 32];
          asm volatile("bar.sync %0, 64;" ::"r"(1 + pair_id) : "memory");
          if (tangent) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float x = g[j], y = u[j];
              g[j] = tg[j], u[j] = tu[j], tg[j] = x, tu[j] = y;
            }
          }
          const int c = it.nt * 128 + half * 64 + b * 32 + (tangent ? 16 : 0);
          finish_gated<T, true>(p, row0, c, lane, g, u, tg, tu);
          write_dual<T>(p, row0, c, lane, mine, g, tg);
        }
      } else if constexpr (GATED) {
#pragma unroll 1
        for (int b = 0; b < 4; ++b) {
          float g[16], u[16];
          take16(b * 16, g);
          take16(64 + b * 16, u);
          taken(b == 3);
          // Whole pieces leave 32 entries at a time; rows that begin anywhere 64, whole lines of which most sectors are (fp16 M3990 K1024
          // F2731: 55 -> 49 us; whole pieces of F2736 42 by 32, 44 by 64).
          const int span = p.aligned ? 32 : AT_ONCE, c = it.nt * 128 + half * 64 + b * 16, first = b * 16 % span;
          finish_gated<T, false>(p, row0, c, lane, g, u, g, u);
          put<T, AT_ONCE>(mine, lane, first, g);
          if (first + 16 == span) {
            __syncwarp();
            if (p.aligned)
              write_pieces<T, AT_ONCE, 32>(static_cast<T*>(p.h), p, row0, c - first, lane, mine);
            else
              write_entries<T, AT_ONCE>(static_cast<T*>(p.h), p, row0, c - first, lane, mine);
            __syncwarp();
          }
        }
      } else {
#pragma unroll 1
        for (int b = 0; b < 4; ++b) {
          float v[16], w[16];
          take16(b * 32, v);
          take16(b * 32 + 16, w);
          taken(b == 3);
          put<T, 32>(mine, lane, 0, v);
          put<T, 32>(mine, lane, 16, w);
          write_rows<T, 32>(static_cast<T*>(p.out[group]), p, row0, it.nt * 256 + half * 128 + b * 32, lane, mine);
        }
      }
      ++acc;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (bar.abort_flag != 0) {
    // Something gave up: copies and products that may still be in flight get time to land before shared memory and TMEM go.
    const long long t0 = clock64();
    while (clock64() - t0 < (1ll << 22)) {
    }
  }
  cluster_sync();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
  cluster_sync();
}

// The sums of a cut tile's pieces, in their order, and what becomes of them.  A warp takes 32 rows x 16 columns, as one of pair_kernel's did.
constexpr int kJoinWarps = 4;
template <typename T, int KIND>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ PairArgs p) {
  constexpr bool GATED = KIND <= kPairGatedDual, DUAL = KIND == kPairGatedDual;
  constexpr int kBlocks = GATED ? 4 : 8, kQ = DUAL ? 2 : 4;  // tasks: tile, rank, half, q, block
  constexpr int kBytes = kRowsBytes<T, 16>;
  __shared__ __align__(16) uint8_t through[kJoinWarps * kBytes];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int task = blockIdx.x * kJoinWarps + warp;
  const int b = task % kBlocks, q = task / kBlocks % kQ, half = task / (kBlocks * kQ) % 2, rank = task / (kBlocks * kQ * 2) % 2;
  const int rest = task / (kBlocks * kQ * 4);
  if (rest * p.cut >= p.items - p.whole) return;
  uint8_t* const mine = through + warp * kBytes;
  int mt, nt;
  tile_at(p, p.whole + rest, mt, nt);
  const int group = mt / p.tiles_m, m = mt - group * p.tiles_m;
  const int row0 = DUAL ? m * 128 + rank * 64 + q * 32 : m * 256 + rank * 128 + q * 32;
  const int c = GATED ? nt * 128 + half * 64 + b * 16 : nt * 256 + half * 128 + b * 16;
  if (row0 >= p.rows || c >= p.cols) return;
  auto add_up = [&](int q_, int b_, float (&v)[16]) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = 0.f;
#pragma unroll 2
    for (int k = 0; k < p.cut; ++k) {
      const float4* from = partial_at(p, rest * p.cut + k, rank, half * 4 + q_, b_, lane);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 x = from[j * 32];
        v[4 * j] += x.x, v[4 * j + 1] += x.y, v[4 * j + 2] += x.z, v[4 * j + 3] += x.w;
      }
    }
  };
  if constexpr (GATED) {
    float g[16], u[16], tg[DUAL ? 16 : 1], tu[DUAL ? 16 : 1];
    add_up(q, b, g);
    add_up(q, b + 4, u);
    if constexpr (DUAL) {
      add_up(q + 2, b, tg);
      add_up(q + 2, b + 4, tu);
      finish_gated<T, true>(p, row0, c, lane, g, u, tg, tu);
      write_dual<T>(p, row0, c, lane, mine, g, tg);
    } else {
      finish_gated<T, false>(p, row0, c, lane, g, u, g, u);
      put<T, 16>(mine, lane, 0, g);
      write_rows<T, 16>(static_cast<T*>(p.h), p, row0, c, lane, mine);
    }
  } else {
    float v[16];
    add_up(q, b, v);
    put<T, 16>(mine, lane, 0, v);
    write_rows<T, 16>(static_cast<T*>(p.out[group]), p, row0, c, lane, mine);
  }
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return JVPFA_OK;
  set_last_cuda_error(e, what);
  return JVPFA_ERR_CUDA;
}

template <typename T, int KIND>
int launch_kind(const PairArgs& p, const PairMaps& maps, cudaStream_t s) {
  constexpr size_t smem = kPairStages<T, KIND> * kStageBytes + kThroughBytes<T, KIND> + sizeof(PairBarriers) + 1024;
  static_assert(smem <= 232448, "shared memory of a CTA");
  auto kern = pair_kernel<T, KIND>;
  static SmemOptIn opt_in;
  if (!opt_in.ensure(reinterpret_cast<const void*>(kern), smem)) return JVPFA_ERR_CUDA;
  const int pairs = device_sms() / 2;
  kern<<<2 * (p.items < pairs ? p.items : pairs), kPairThreads, smem, s>>>(p, maps);
  const int rc = launched("gated pair_kernel");
  if (rc || p.items == p.whole) return rc;
  constexpr int tasks = KIND <= kPairGated ? 4 * 4 * 4 : KIND == kPairGatedDual ? 4 * 2 * 4 : 8 * 4 * 4;  // of a tile
  join_kernel<T, KIND><<<(p.items - p.whole) / p.cut * (tasks / kJoinWarps), kJoinWarps * 32, 0, s>>>(p);
  return launched("gated join_kernel");
}

template <typename T>
int launch_type(int kind, const PairArgs& p, const PairMaps& maps, cudaStream_t s) {
  switch (kind) {
    case kPairGated: return launch_kind<T, kPairGated>(p, maps, s);
    case kPairGatedDual: return launch_kind<T, kPairGatedDual>(p, maps, s);
    case kPairDx: return launch_kind<T, kPairDx>(p, maps, s);
    default: return launch_kind<T, kPairDw>(p, maps, s);
  }
}

}  // namespace

int device_sms() {
  static int cached[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  n = __atomic_load_n(&cached[dev], __ATOMIC_RELAXED);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 2) n = 148;
    __atomic_store_n(&cached[dev], n, __ATOMIC_RELAXED);
  }
  return n;
}

bool encode_matrix(CUtensorMap* m, int dtype, const void* ptr, int rows, int cols, int64_t stride, int planes, int box_rows) {
  const int64_t plane = (int64_t)rows * stride, st[3] = {plane * planes, plane, stride};
  const CUtensorMapDataType dt = dtype == JVPFA_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode_map4d(m, dt, ptr, cols, rows, planes, 1, st, box_rows);
}

int plan_pair(int dtype, int kind, PairArgs& p) {
  const bool gated = kind <= kPairGatedDual;
  const int rows = kind == kPairGatedDual ? 128 : 256, cols = gated ? 128 : 256;
  p.kblocks = (p.depth + 63) / 64;
  p.pairs = dtype == JVPFA_FP32 ? 6 : 1;
  const long long steps = (long long)p.sources * p.pairs * p.kblocks;
  p.tiles_m = (p.rows + rows - 1) / rows;
  p.tiles_n = (p.cols + cols - 1) / cols;
  const long long tiles = (long long)p.groups * p.tiles_m * p.tiles_n;
  // (what a CTA counts, k-blocks of its tiles and tiles of a band, stays in 32 bits)
  if (steps > 2147483647LL || tiles > 2147483647LL - 1024 || steps * (tiles / 64 + 1) > 2147483647LL) return JVPFA_ERR_TOO_LARGE;
  // A tile's sum is one wait of the warps that write it, and waits are bounded: 2^20 k-blocks (67 million rows for dw) take some 0.4 seconds.
  if (dtype != JVPFA_FP32 && steps > kMaxSteps) return JVPFA_ERR_TOO_LARGE;
  p.steps = (int)steps;
  p.chunk = dtype == JVPFA_FP32 ? 4 : p.steps;
  // 74 tiles at once read band + 74 / band panels of their operands.  8 is the fewest, and best for the backward's, whose panels are as deep as the
  // features or the rows are many; the forward's are shallow enough that a band of 16 stays in L2 while all columns go by (M8192
  // K4096 F11008, sustained: forward 1092 -> 1051 us; all three products at 16 instead of 8 differ by less than they do between runs).
  p.band = gated ? 16 : 8;
  p.aligned = p.cols % (dtype == JVPFA_FP32 ? 4 : 8) == 0;
  // The tiles of the last round are cut into as many pieces as there are clusters for, where that saves more than a launch and the way
  // through memory cost.
  const int clusters = device_sms() / 2, rest = (int)(tiles % clusters);
  p.whole = p.items = (int)tiles;
  p.cut = 1, p.piece = p.steps;
  if (rest > 0) {
    int cut = clusters / rest;
    if (cut > p.steps / kMinPieceSteps) cut = p.steps / kMinPieceSteps;
    if (cut > 1) {
      const int piece = (p.steps + cut - 1) / cut;
      cut = (p.steps + piece - 1) / piece;
      if (cut > 1 && p.steps - piece >= (gated ? kMinSavedGated : kMinSavedSteps)) {
        p.whole = (int)tiles - rest;
        p.cut = cut, p.piece = piece;
        p.items = p.whole + rest * cut;
      }
    }
  }
  return JVPFA_OK;
}

int64_t pair_workspace(const PairArgs& p) { return (int64_t)(p.items - p.whole) * 256 * 256 * 4; }

int launch_pair(int dtype, int kind, const PairArgs& planned, const PairMaps& maps, cudaStream_t s) {
  PairArgs p = planned;
  p.status = tc5_status_device_ptr();
  if (!p.status) {
    set_last_cuda_error(cudaErrorUnknown, "status word address");
    return JVPFA_ERR_CUDA;
  }
  if (dtype == JVPFA_BF16) return launch_type<__nv_bfloat16>(kind, p, maps, s);
  if (dtype == JVPFA_FP16) return launch_type<__half>(kind, p, maps, s);
  return launch_type<float>(kind, p, maps, s);
}

}  // namespace tc5
}  // namespace jvpfa

// The matrix products of the gated projection on the fifth-generation tensor cores, two SMs to a tile.
//
// A cluster of two CTAs computes 256 rows x 256 columns: every instruction (tcgen05.mma.cta_group::2, M = N = 256, K = 16) takes 128 rows
// of A and 128 columns of B from either CTA's shared memory, so an operand byte that a CTA loads serves twice the products that it
// would alone: 32 KB for each 512 cycles of products, where one CTA's 128 x 256 tiles ask for 48 KB, more than L2 delivers to all SMs.
//
// Forward (kPairGated): the columns are 128 features of wg (CTA 0's) beside the same 128 of wu (CTA 1's), so that g and u of a feature
// end up in one lane of one CTA and the gate is applied on the way out.  With tangents (kPairGatedDual) a CTA's 128 rows
// are 64 of x and the same 64 of tx: all four products of a (row, feature) are in one CTA, and the lanes of the value hand a'(g) u and a(g)
// to those of the tangent through shared memory.
// Backward: products over the features (kPairDx: weights read across the contraction) and over the rows (kPairDw: both operands are).
//
// Sums are fp32 accumulators in TMEM, two of them (2 x 256 columns), so that a tile is written while the next is computed.  The tensor cores
// round a sum towards zero at every step of 16; fp32 results, whose products are six each of bf16 parts, are taken up in registers
// every 16 k-blocks and summed there to nearest.
//
// Roles: warp 0 loads (TMA), warp 1 of CTA 0 issues the products, warp 2 owns TMEM, warps 4 to 11 write results.  Persistent: each cluster
// takes every (clusters)-th tile, in bands of 8 tiles of rows so that what runs at once shares its operands in L2.
#include "gated_common.cuh"

namespace jvpfa {
namespace tc5 {

namespace {

constexpr int kPairThreads = 384;
constexpr int kPairStages = 6;
constexpr int kStageBytes = 32768;  // of a CTA: A 128 x 64, B 128 x 64
constexpr int kBand = 8;
constexpr int kExchangeBytes = 32768;
constexpr int kAbortPairFull = 14, kAbortPairEmpty = 15, kAbortPairAcc = 16, kAbortPairAccEmpty = 17;

struct PairBarriers {
  uint64_t full[kPairStages], empty[kPairStages], acc_full[2], acc_empty[2];
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
__device__ __forceinline__ void arrive_in_leader(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
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

// Tile t of the launch: the row of tiles (over all groups) and the column.
__device__ __forceinline__ void tile_at(const PairArgs& p, int t, int& mt, int& nt) {
  const int band = t / (kBand * p.tiles_n), r = t - band * kBand * p.tiles_n;
  const int high = min(kBand, p.tiles_m * p.groups - band * kBand);
  nt = r / high;
  mt = band * kBand + r - nt * high;
}

// 32 neighbouring entries of a row.
template <typename T>
__device__ __forceinline__ void store32(T* row, int c, int n, bool pieces, const float (&v)[32]) {
  if (pieces && c + 32 <= n) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(row + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 32; j += 8)
        *reinterpret_cast<uint4*>(row + c + j) = make_uint4(Elem<T>::pack(v[j], v[j + 1]), Elem<T>::pack(v[j + 2], v[j + 3]),
                                                            Elem<T>::pack(v[j + 4], v[j + 5]), Elem<T>::pack(v[j + 6], v[j + 7]));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (c + j < n) row[c + j] = Elem<T>::from_float(v[j]);
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

template <typename T, int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    pair_kernel(const __grid_constant__ PairArgs p, const __grid_constant__ PairMaps maps) {
  constexpr bool GATED = KIND <= kPairGatedDual, DUAL = KIND == kPairGatedDual, A_MN = KIND == kPairDw, B_MN = KIND >= kPairDx;
  constexpr bool PARTS = Operand<T>::kParts;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  float* exchange = reinterpret_cast<float*>(smem + kPairStages * kStageBytes);
  PairBarriers& bar = *reinterpret_cast<PairBarriers*>(smem + kPairStages * kStageBytes + (DUAL ? kExchangeBytes : 0));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    const int before = *reinterpret_cast<volatile int*>(p.status);
    bar.abort_flag = before;
    for (int i = 0; i < kPairStages; ++i) mbar_init(&bar.full[i], 1), mbar_init(&bar.empty[i], 1);
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
      for (int t = cluster; t < p.tiles && ok; t += clusters) {
        int mt, nt;
        tile_at(p, t, mt, nt);
        const int group = mt / p.tiles_m, m0 = (mt - group * p.tiles_m) * rows_of_tile + (int)rank * (rows_of_tile / 2);
        const int n0 = GATED ? nt * 128 : nt * 256 + (int)rank * 128;
        for (int s = 0; s < p.sources && ok; ++s) {
          const CUtensorMap* ma = &maps.a[GATED ? 0 : 2 * group + s];
          const CUtensorMap* mb = &maps.b[GATED ? rank : s];
          for (int pair = 0; pair < p.pairs && ok; ++pair) {
            const int pa = PARTS ? 0x850 >> (2 * pair) & 3 : 0, pb = PARTS ? 0x244 >> (2 * pair) & 3 : 0;
            for (int kb = 0; kb < p.kblocks; ++kb, ++n) {
              const int stage = n % kPairStages;
              ok = mbar_wait(&bar.empty[stage], (n / kPairStages & 1) ^ 1, ab, kAbortPairEmpty);
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
            }
          }
        }
      }
      // What the products have still to say to this CTA's barriers arrives before it ends.
      for (int i = 0; i < kPairStages && ok; ++i, ++n)
        ok = mbar_wait(&bar.empty[n % kPairStages], (n / kPairStages & 1) ^ 1, ab, kAbortPairEmpty);
    }
  } else if (warp == 1) {
    if (rank == 0 && !refused) {
      constexpr uint32_t idesc = make_idesc(Fmt<typename Operand<T>::type>::kIdesc, 256, 256, A_MN, B_MN);
      constexpr uint32_t lbo = (8192 >> 4) << 16;
      constexpr uint32_t step_a = A_MN ? 128 : 2, step_b = B_MN ? 128 : 2;  // 16 of the contraction, in 16 bytes
      int n = 0, acc = 0;
      bool ok = true;
      for (int t = cluster; t < p.tiles && ok; t += clusters) {
        for (int done = 0; done < p.steps && ok; ++acc) {
          const int upto = min(p.steps, done + p.chunk), buf = acc & 1;
          ok = mbar_wait_warp(&bar.acc_empty[buf], (acc >> 1 & 1) ^ 1, ab, kAbortPairAccEmpty);
          if (!ok) break;
          tc_fence_after();
          for (bool first = true; done < upto; ++done, ++n) {
            const int stage = n % kPairStages;
            ok = mbar_wait_warp(&bar.full[stage], n / kPairStages & 1, ab, kAbortPairFull);
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
    const int q = warp & 3, half = (warp - 4) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    constexpr int kPieces = 16 / sizeof(T);
    const bool pieces = p.cols % kPieces == 0;
    int acc = 0;
    bool ok = !refused;
    for (int t = cluster; t < p.tiles; t += clusters) {
      int mt, nt;
      tile_at(p, t, mt, nt);
      const int group = mt / p.tiles_m, m = mt - group * p.tiles_m;
      const int row = DUAL ? m * 128 + (int)rank * 64 + (q & 1) * 32 + lane : m * 256 + (int)rank * 128 + q * 32 + lane;
      const bool inside = row < p.rows;
      const size_t at = (size_t)row * p.cols;
      float sum[PARTS ? 4 : 1][32];
      uint32_t col = 0;
      // this thread's 4 x 32 accumulators: gated g, g, u, u of 2 x 32 features, else 128 columns
      auto column = [&](int b) { return col + (GATED ? (b >> 1) * 128 + half * 64 + (b & 1) * 32 : half * 128 + b * 32); };
      auto release = [&](int buf) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_in_leader(in_leader(&bar.acc_empty[buf]));
      };
      if constexpr (PARTS) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[b][j] = 0.f;
        for (int done = 0; done < p.steps; done += p.chunk, ++acc) {
          const int buf = acc & 1;
          ok = ok && mbar_wait_warp(&bar.acc_full[buf], acc >> 1 & 1, ab, kAbortPairAcc);
          if (!ok) continue;
          tc_fence_after();
          col = lanes + buf * 256;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            uint32_t r[32];
            tmem_ld32(column(b), r);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[b][j] += __uint_as_float(r[j]);
          }
          release(buf);
        }
      } else {
        ok = ok && mbar_wait_warp(&bar.acc_full[acc & 1], acc >> 1 & 1, ab, kAbortPairAcc);
        if (ok) tc_fence_after();
        col = lanes + (acc & 1) * 256;
      }
      // 32 accumulators of this thread
      auto take = [&](int b, float (&v)[32]) {
        if constexpr (PARTS) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = sum[b][j];
        } else if (ok) {
          tmem_ld32(column(b), reinterpret_cast<uint32_t(&)[32]>(v));
        }
      };
      if constexpr (GATED) {
        const bool tangent = DUAL && q >= 2;
        T* const out = static_cast<T*>(tangent ? p.th : p.h) + at;
        T* const save_g = static_cast<T*>(tangent ? p.tg : p.g);
        T* const save_u = static_cast<T*>(tangent ? p.tu : p.u);
        float* const ex = exchange + half * (kExchangeBytes / 8) + (q & 1) * 32 + lane;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int c = nt * 128 + half * 64 + b * 32;
          float g[32], u[32], o[32];
          take(b, g);
          take(b + 2, u);
          if (!PARTS && ok) {
            tmem_wait_ld();
            if (b == 1) release(acc & 1);
          }
          if (!tangent) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const Activated y = activate<PARTS>(p.activation, g[j]);
              o[j] = y.a * u[j];
              if constexpr (DUAL) ex[j * 64] = y.d1 * u[j], ex[(32 + j) * 64] = y.a;
            }
          }
          if constexpr (DUAL) {
            asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
            if (tangent) {
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = ex[j * 64] * g[j] + ex[(32 + j) * 64] * u[j];
            }
            asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
          }
          if (inside && ok) {
            store32(out, c, p.cols, pieces, o);
            if (save_g) store32(save_g + at, c, p.cols, pieces, g), store32(save_u + at, c, p.cols, pieces, u);
          }
          __syncwarp();
        }
        if (!ok && inside && nt * 128 + half * 64 < p.cols) out[nt * 128 + half * 64] = Elem<T>::from_float(poison_f32());
      } else {
        T* const out = static_cast<T*>(p.out[group]) + at;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          float v[32];
          take(b, v);
          if (!PARTS && ok) {
            tmem_wait_ld();
            if (b == 3) release(acc & 1);
          }
          if (inside && ok) store32(out, nt * 256 + half * 128 + b * 32, p.cols, pieces, v);
          __syncwarp();
        }
        if (!ok && inside && nt * 256 + half * 128 < p.cols) out[nt * 256 + half * 128] = Elem<T>::from_float(poison_f32());
      }
      if constexpr (!PARTS) ++acc;
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

template <typename T, int KIND>
int launch_kind(const PairArgs& p, const PairMaps& maps, cudaStream_t s) {
  constexpr size_t smem = kPairStages * kStageBytes + (KIND == kPairGatedDual ? kExchangeBytes : 0) + sizeof(PairBarriers) + 1024;
  static_assert(smem <= 232448, "shared memory of a CTA");
  auto kern = pair_kernel<T, KIND>;
  static SmemOptIn opt_in;
  if (!opt_in.ensure(reinterpret_cast<const void*>(kern), smem)) return JVPFA_ERR_CUDA;
  const int pairs = device_sms() / 2;
  kern<<<2 * (p.tiles < pairs ? p.tiles : pairs), kPairThreads, smem, s>>>(p, maps);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "gated pair_kernel");
    return JVPFA_ERR_CUDA;
  }
  return JVPFA_OK;
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

bool encode_matrix(CUtensorMap* m, int dtype, const void* ptr, int rows, int cols, int64_t stride, int planes, int box_rows) {
  const int64_t plane = (int64_t)rows * stride, st[3] = {plane * planes, plane, stride};
  const CUtensorMapDataType dt = dtype == JVPFA_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode_map4d(m, dt, ptr, cols, rows, planes, 1, st, box_rows);
}

int launch_pair(int dtype, int kind, PairArgs& p, const PairMaps& maps, cudaStream_t s) {
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
  p.steps = (int)steps;
  p.tiles = (int)tiles;
  p.chunk = dtype == JVPFA_FP32 ? 16 : p.steps;
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

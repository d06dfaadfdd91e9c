// The gated projection's products for few rows (up to 128, value and tangent together): what counts is how quickly the weights arrive.
//
// The roles of rows and columns are exchanged: a tile of 128 weight rows (or columns, for dx) is the instruction's M, the rows of x are
// its N, so nothing is computed for rows that are not there beyond the next multiple of 16.
//   kFewGated  64 features: 64 rows of wg beside the same 64 of wu, contraction over K; then the gate
//   kFewDx     128 columns of dx: the weights across the contraction, which runs over the features of wg and then of wu
// A cluster of 1 to 8 CTAs shares a tile, a part of the depth each, so that all SMs have a part of the weights under way also where there are few
// tiles; the parts' sums meet in the CTAs' shared memory and are added in their order, each CTA finishing a part of the tile.
//
// fp32 weights are read once, as they are: 16 warps load them, split them into three bf16 parts and lay these down for the tensor cores
// (a copy of the parts in memory would be written and read again, four times the bytes).  The tensor cores round towards zero at every
// step of 16, so those warps take the sums up in registers every 4 k-blocks, while the next go to another accumulator; and the five lesser
// products of parts have accumulators of their own, where what is rounded away is that much smaller.
//
// Bound by memory, the weights read once.  Measured on a B200: one row of bf16 K4096 F11008 35 us = 5.2 TB/s, 32 rows 39, 100 rows 46; 24 rows with
// tangent of fp16 K1024 F2736 9.4 us (two CTAs of 108 KB of stages an SM; one of 216 KB: 55 and 14.9 us).  fp32 one row of K4096 F11008
// 106 us = 3.4 TB/s, 100 rows 120: 24 products and a splitting to a k-block keep the shared-memory port busy (all tiles cut alike, in five rounds: 148).
#include "gated_common.cuh"

namespace jvpfa {
namespace tc5 {

namespace {

// Warps 0: TMA, 1: products, 2: TMEM, from 4 on: fp32 weights, results
template <typename T>
constexpr int kFewThreads = sizeof(T) == 4 ? 640 : 384;
template <typename T>
constexpr int kFewResident = sizeof(T) == 4 ? 1 : 3;  // CTAs that plan_few counts on an SM's registers for: 56 a thread in 16 bits
constexpr int kSplitThreads = 512, kUnits = 1024 / kSplitThreads;  // fp32: a k-block's 1024 pieces of eight entries
constexpr int kAbortFewFull = 18, kAbortFewEmpty = 19, kAbortFewAcc = 20, kAbortFewAccEmpty = 21;
constexpr int kTakeUp = 4;   // fp32: k-blocks between two looks at the accumulators
constexpr int kTile = 16384;  // 128 x 64 weights, 16 bits

struct FewBarriers {
  uint64_t full[8], empty[8], acc[2], acc_empty[2];
  uint32_t tmem;
  int abort_flag;
};

template <typename T>
struct FewOperand {
  using type = T;
  static constexpr int kParts = 1;
};
template <>
struct FewOperand<float> {
  using type = __nv_bfloat16;
  static constexpr int kParts = 3;
};

__device__ __forceinline__ uint32_t few_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void few_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A word of another CTA's shared memory.
__device__ __forceinline__ float remote(uint32_t address, int rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(address), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// fp32 weights of k-block `step`: this thread's pieces of eight neighbouring entries (zeros beyond the matrix).
template <int KIND>
struct Piece8 {
  float v[kUnits][8];
  __device__ __forceinline__ static void place(const FewArgs& p, int tile, int step, int unit, const float*& row, int& c, bool& inside) {
    if constexpr (KIND == kFewGated) {
      const int r = unit >> 3, f = tile * 64 + (r & 63);
      inside = f < p.features;
      row = static_cast<const float*>(r < 64 ? p.wg : p.wu) + (size_t)f * (r < 64 ? p.wg_stride : p.wu_stride);
      c = step * 64 + (unit & 7) * 8;
    } else {
      const int up = step >= p.kblocks, f = (step - (up ? p.kblocks : 0)) * 64 + (unit >> 4);
      inside = f < p.features;
      row = static_cast<const float*>(up ? p.wu : p.wg) + (size_t)f * (up ? p.wu_stride : p.wg_stride);
      c = tile * 128 + (unit & 15) * 8;
    }
  }
  __device__ __forceinline__ void load(const FewArgs& p, int tile, int step, int tid) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const float* row;
      int c;
      bool inside;
      place(p, tile, step, i * kSplitThreads + tid, row, c, inside);
      const int left = inside ? p.width - c : 0;
      if (p.pieces && left >= 8) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(row + c)), b = __ldg(reinterpret_cast<const float4*>(row + c) + 1);
        v[i][0] = a.x, v[i][1] = a.y, v[i][2] = a.z, v[i][3] = a.w, v[i][4] = b.x, v[i][5] = b.y, v[i][6] = b.z, v[i][7] = b.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = j < left ? __ldg(row + c + j) : 0.f;
      }
    }
  }
  // ... as three parts, in the 128-byte-swizzled form of a tile contiguous along the contraction, or across it.
  __device__ __forceinline__ void store(uint8_t* stage, int tid) const {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int unit = i * kSplitThreads + tid;
      const int r = KIND == kFewGated ? unit >> 3 : unit >> 4, ch = KIND == kFewGated ? unit & 7 : unit & 15;
      uint8_t* at = stage + (ch >> 3) * 8192 + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
      uint32_t w[3][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // Cut, not rounded (24 bits are 8 + 8 + 8 that way too): conversions run at an eighth of the rate of these, and would take longer
        // than the weights need to arrive.  What the six products leave out is at most 2^-21 of one, 2^-24 on average.
        float a = v[i][2 * j], b = v[i][2 * j + 1];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          w[k][j] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
          a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u), b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
        }
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(at + k * kTile) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
    }
  }
};

// BIG: more than 64 columns (fp32: a thread holds 32 sums, and has one k-block less under way).
template <typename T, int KIND, bool BIG>
__global__ void __launch_bounds__(kFewThreads<T>, kFewResident<T>) few_kernel(const __grid_constant__ FewArgs p, const __grid_constant__ FewMaps maps) {
  constexpr int PARTS = FewOperand<T>::kParts;
  constexpr bool SPLIT = PARTS > 1, GATED = KIND == kFewGated;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  const int N = p.padded * p.groups, rows_bytes = N * 128;
  const int stage_bytes = PARTS * (kTile + rows_bytes);  // weights, then rows, part by part
  FewBarriers& bar = *reinterpret_cast<FewBarriers*>(smem + p.stages * stage_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.cluster > 1 ? (int)few_rank() : 0, tile = p.first + (int)blockIdx.x / p.cluster;
  const int begin = (int)((long long)p.steps * rank / p.cluster), end = (int)((long long)p.steps * (rank + 1) / p.cluster);

  if (threadIdx.x == 0) {
    bar.abort_flag = *reinterpret_cast<volatile int*>(p.status);
    for (int i = 0; i < p.stages; ++i) mbar_init(&bar.full[i], SPLIT ? 1 + kSplitThreads / 32 : 1), mbar_init(&bar.empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bar.acc[i], 1), mbar_init(&bar.acc_empty[i], kSplitThreads / 32);
    fence_mbar_init();
  }
  if (warp == 2) {
    tmem_alloc(&bar.tmem, p.tmem_columns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar.tmem;
  const AbortState ab{&bar.abort_flag, p.status};
  bool ok = bar.abort_flag == 0;

  if (warp == 0) {
    if (lane == 0) {
      for (int step = begin, n = 0; step < end && ok; ++step, ++n) {
        const int stage = n % p.stages;
        ok = mbar_wait(&bar.empty[stage], (n / p.stages & 1) ^ 1, ab, kAbortFewEmpty);
        if (!ok) break;
        uint8_t* to = smem + stage * stage_bytes;
        mbar_expect_tx(&bar.full[stage], PARTS * rows_bytes + (SPLIT ? 0 : kTile));
        const int source = !GATED && step >= p.kblocks, kb = step - source * p.kblocks;
        if constexpr (!SPLIT) {
          if constexpr (GATED) {
            tma_load_4d(to, &maps.w[0], &bar.full[stage], kb * 64, tile * 64, 0, 0);
            tma_load_4d(to + 8192, &maps.w[1], &bar.full[stage], kb * 64, tile * 64, 0, 0);
          } else {
            tma_load_4d(to, &maps.w[source], &bar.full[stage], tile * 128, kb * 64, 0, 0);
            tma_load_4d(to + 8192, &maps.w[source], &bar.full[stage], tile * 128 + 64, kb * 64, 0, 0);
          }
        }
        for (int part = 0; part < PARTS; ++part)
          for (int g = 0; g < p.groups; ++g)
            tma_load_4d(to + PARTS * kTile + part * rows_bytes + g * p.padded * 128, &maps.rows[GATED ? g : 2 * g + source], &bar.full[stage], kb * 64,
                        0, part, 0);
      }
    }
  } else if (warp == 1) {
    const uint32_t idesc = make_idesc(Fmt<typename FewOperand<T>::type>::kIdesc, 128, 0, !GATED, 0) | (uint32_t)(N >> 3) << 17;
    constexpr uint32_t a_form = GATED ? kDescLo : (8192u >> 4) << 16, step_a = GATED ? 2 : 128;
    for (int step = begin, n = 0; step < end && ok; ++step, ++n) {
      const int stage = n % p.stages;
      ok = mbar_wait_warp(&bar.full[stage], n / p.stages & 1, ab, kAbortFewFull);
      if (!ok) break;
      tc_fence_after();
      const uint32_t a = (smem_u32(smem + stage * stage_bytes) & 0x3ffff) >> 4, b = a + PARTS * (kTile >> 4);
      if constexpr (SPLIT) {
        const int chunk = n / kTakeUp, buf = chunk & 1;
        const uint32_t d = tmem + buf * 2 * N;  // the leading products' accumulator, and the others'
        const bool first = n % kTakeUp == 0;
        if (first) {
          ok = mbar_wait_warp(&bar.acc_empty[buf], (chunk >> 1 & 1) ^ 1, ab, kAbortFewAccEmpty);
          if (!ok) break;
          tc_fence_after();
        }
        if (elect_one()) {
#pragma unroll
          for (int pair = 0; pair < 6; ++pair) {
            const int pa = 0x850 >> (2 * pair) & 3, pb = 0x244 >> (2 * pair) & 3;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_ss_lo_dyn(pair ? d + N : d, a_form | (a + pa * (kTile >> 4) + k * step_a), kDescLo | (b + pb * (rows_bytes >> 4) + k * 2), idesc,
                             !first || pair > 1 || k > 0);
          }
          tc_commit(&bar.empty[stage]);
          if (n % kTakeUp == kTakeUp - 1 || step + 1 == end) tc_commit(&bar.acc[buf]);
        }
      } else if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_ss_lo_dyn(tmem, a_form | (a + k * step_a), kDescLo | (b + k * 2), idesc, n > 0 || k > 0);
        tc_commit(&bar.empty[stage]);
        if (step + 1 == end) tc_commit(&bar.acc[0]);
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    const int tid = threadIdx.x - 128, q = warp & 3, set = (warp >> 2) - 1;
    constexpr int kSets = kFewThreads<T> / 128 - 1;  // of four warps, which have 16 columns in turn
    constexpr int kRun = SPLIT ? (BIG ? 2 : 1) : 1, kAhead = BIG ? 1 : 2;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    float run[kRun][16];
    if constexpr (SPLIT) {
#pragma unroll
      for (int c = 0; c < kRun; ++c)
#pragma unroll
        for (int j = 0; j < 16; ++j) run[c][j] = 0.f;
      int taken = 0;
      auto take_up = [&]() {
        const int buf = taken & 1;
        ok = ok && mbar_wait_warp(&bar.acc[buf], taken >> 1 & 1, ab, kAbortFewAcc);
        if (!ok) return;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < kRun; ++c) {
          const int column = (c * kSets + set) * 16;
          if (column >= N) break;
          uint32_t r[16];
          tmem_ld16(lanes + (buf * 2 + 1) * N + column, r);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) run[c][j] += __uint_as_float(r[j]);
          tmem_ld16(lanes + buf * 2 * N + column, r);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) run[c][j] += __uint_as_float(r[j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.acc_empty[buf]);
        ++taken;
      };
      // One or two k-blocks are under way while another is split: up to 64 KB of each SM's, which is what memory's latency asks for.
      Piece8<KIND> piece[kAhead + 1];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (begin + i < end) piece[i].load(p, tile, begin + i, tid);
      for (int first = 0; begin + first < end && ok; first += kAhead + 1) {
#pragma unroll
        for (int i = 0; i <= kAhead; ++i) {
          const int n = first + i, step = begin + n;
          if (step >= end || !ok) break;
          if (step + kAhead < end) piece[(i + kAhead) % (kAhead + 1)].load(p, tile, step + kAhead, tid);
          const int stage = n % p.stages;
          ok = mbar_wait_warp(&bar.empty[stage], (n / p.stages & 1) ^ 1, ab, kAbortFewEmpty);
          if (!ok) break;
          piece[i].store(smem + stage * stage_bytes, tid);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.full[stage]);
          if (n % kTakeUp == kTakeUp - 1 && n >= kTakeUp) take_up();  // what the k-blocks before these four gave
        }
      }
      const int all = (end - begin + kTakeUp - 1) / kTakeUp;
      while (ok && taken < all) take_up();
    } else {
      ok = ok && mbar_wait_warp(&bar.acc[0], 0, ab, kAbortFewAcc);
      if (ok) tc_fence_after();
    }
    // All products are done (by every warp's account): the stages' memory takes the sums, column by column.
    float* const sums = reinterpret_cast<float*>(smem);
    for (int c = 0; (c * kSets + set) * 16 < N; ++c) {
      const int column = (c * kSets + set) * 16;
      float v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = poison_f32();
      if constexpr (SPLIT) {
#pragma unroll
        for (int k = 0; k < kRun; ++k)
          if (ok && k == c) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = run[k][j];
          }
      } else if (ok) {
        tmem_ld16(lanes + column, reinterpret_cast<uint32_t(&)[16]>(v));
        tmem_wait_ld();
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) sums[(column + j) * 128 + q * 32 + lane] = v[j];
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
  if (p.cluster > 1) few_cluster_sync();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, p.tmem_columns);
  }

  // This CTA's part of the tile.
  const uint32_t sums = smem_u32(smem);
  auto add_up = [&](int column, int line) {
    const int at = (column * 128 + line) * 4;
    if (p.cluster == 1) return *reinterpret_cast<const float*>(smem + at);
    float v = 0.f;
    for (int r = 0; r < p.cluster; ++r) v += remote(sums + at, r);
    return v;
  };
  constexpr int kLines = GATED ? 64 : 128;  // of the tile: features, or columns of dx
  const int total = kLines * p.rows * (GATED ? 1 : p.groups);
  const int from = (int)((long long)total * rank / p.cluster), to = (int)((long long)total * (rank + 1) / p.cluster);
  if constexpr (GATED) {
    with_activation(p.activation, [&](auto kind) {
      for (int i = from + (int)threadIdx.x; i < to; i += kFewThreads<T>) {
        const int row = i / kLines, line = i % kLines, f = tile * 64 + line;
        if (f >= p.features) continue;
        const float g = add_up(row, line), u = add_up(row, 64 + line);
        const Activated y = activate<decltype(kind)::value, sizeof(T) == 4>(g);
        static_cast<T*>(p.h)[(size_t)row * p.features + f] = Elem<T>::from_float(y.a * u);
        float v[4] = {g, u, 0.f, 0.f};
        if (p.groups > 1) {
          v[2] = add_up(p.padded + row, line), v[3] = add_up(p.padded + row, 64 + line);
          static_cast<T*>(p.th)[(size_t)row * p.features + f] = Elem<T>::from_float(y.d1 * v[2] * u + y.a * v[3]);
        }
        if (p.kept) {
          uint8_t* block = p.kept + (size_t)((row >> 5) * ((p.features + 31) >> 5) + (f >> 5)) * (2 * p.groups) * Kept<T>::kBlock;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < 2 * p.groups) keep_entry<T>(block + k * Kept<T>::kBlock, row & 31, f & 31, v[k]);
        }
      }
    });
  } else {
    for (int i = from + (int)threadIdx.x; i < to; i += kFewThreads<T>) {
      const int line = i % kLines, g = i / kLines / p.rows, row = i / kLines - g * p.rows, c = tile * 128 + line;
      if (c < p.width) static_cast<T*>(p.out[g])[(size_t)row * p.width + c] = Elem<T>::from_float(add_up(g * p.padded + row, line));
    }
  }
  if (p.cluster > 1) {
    __syncwarp();
    few_cluster_sync();  // the others have read what is here
  }
}

template <typename T, int KIND, bool BIG>
int launch_tiles(const FewArgs& p, const FewMaps& maps, cudaStream_t s) {
  constexpr int PARTS = FewOperand<T>::kParts;
  const size_t smem = (size_t)p.stages * PARTS * (kTile + p.padded * p.groups * 128) + sizeof(FewBarriers) + 1024;
  auto kern = few_kernel<T, KIND, BIG>;
  static SmemOptIn opt_in;
  if (!opt_in.ensure(reinterpret_cast<const void*>(kern), 232448)) return JVPFA_ERR_CUDA;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(p.tiles * p.cluster));
  config.blockDim = dim3(kFewThreads<T>);
  config.dynamicSmemBytes = smem;
  config.stream = s;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = (unsigned)p.cluster;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = p.cluster > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&config, kern, p, maps);
  if (e == cudaSuccess) return JVPFA_OK;
  (void)cudaGetLastError();
  set_last_cuda_error(e, "gated few_kernel");
  return JVPFA_ERR_CUDA;
}

template <typename T, int KIND>
int launch_kind(const FewArgs& planned, const FewMaps& maps, cudaStream_t s) {
  auto launch = [&](int first, int tiles, int cluster) {
    FewArgs p = planned;
    p.first = first, p.tiles = tiles, p.cluster = cluster;
    if constexpr (sizeof(T) == 4)
      if (p.padded * p.groups > 64) return launch_tiles<T, KIND, true>(p, maps, s);
    return launch_tiles<T, KIND, false>(p, maps, s);
  };
  int rc = planned.whole ? launch(0, planned.whole, 1) : JVPFA_OK;
  if (!rc && planned.tiles > planned.whole) rc = launch(planned.whole, planned.tiles - planned.whole, planned.cluster);
  return rc;
}

}  // namespace

bool plan_few(int dtype, int kind, FewArgs& p) {
  const int parts = dtype == JVPFA_FP32 ? 3 : 1;
  if (p.rows > 128) return false;
  p.padded = p.groups == 1 ? (p.rows + 15) / 16 * 16 : (p.rows + 7) / 8 * 8;
  const int N = p.padded * p.groups;
  if (N > 128) return false;
  const int depth = kind == kFewGated ? p.width : p.features;
  p.kblocks = (depth + 63) / 64;
  if (p.kblocks > kMaxSteps / 2) return false;
  p.steps = kind == kFewGated ? p.kblocks : 2 * p.kblocks;
  p.tiles = kind == kFewGated ? (p.features + 63) / 64 : (p.width + 127) / 128;
  // CTAs of a tile: as many as find room at once.  fp32, where a CTA has an SM to itself: tiles by whole rounds of the SMs first, in a launch of
  // their own, so that a last round of few does not take as long as one of all.
  const int at_once = parts > 1 ? device_sms() : 2 * device_sms();
  p.first = 0;
  p.whole = parts > 1 ? p.tiles / at_once * at_once : 0;
  const int rest = p.tiles - p.whole;
  p.cluster = 1;
  while (p.cluster < 8 && rest * 2 * p.cluster <= at_once && 4 * p.cluster <= p.steps) p.cluster *= 2;
  // Room for stages: fp32 one CTA an SM, whose registers hold what is under way; else two CTAs, or three, with less under way each, where they take
  // the tiles in fewer rounds.  us of bf16 K2048 with two and with three, 1 row / 32 / 100, values and tangents alike: F11008 (172 tiles) 19.2, 20.5, 26.1
  // and 20.2, 22.6, 30.6; F20000 (313) 40.4, 43.0, 49.0 and 31.4, 32.7, 38.5; F28672 (448, two rounds of either) 43.2, 45.8, 55.0 and 47.2, 51.4, 66.7;
  // F40000 (625) 63.3, 68.0, 79.4 and 55.1, 60.3, 73.0; dx of K40960 F1024 (320) 38.7, 42.2, 54.3 and 26.7, 29.6, 42.9.  The sums take the stages' place
  // at the end.
  const auto rounds = [&](int ctas) { return (p.tiles + ctas * device_sms() - 1) / (ctas * device_sms()); };
  const int stage = parts * (kTile + N * 128), room = parts > 1 ? 224 * 1024 : rounds(3) < rounds(2) ? 74 * 1024 : 108 * 1024;
  p.stages = room / stage < 8 ? room / stage : 8;
  if (p.stages * stage < N * 512) return false;
  p.tmem_columns = 32;
  while (p.tmem_columns < (parts > 1 ? 4 : 1) * N) p.tmem_columns *= 2;
  return true;
}

int launch_few(int dtype, int kind, const FewArgs& planned, const FewMaps& maps, cudaStream_t s) {
  FewArgs p = planned;
  p.status = tc5_status_device_ptr();
  if (!p.status) {
    set_last_cuda_error(cudaErrorUnknown, "status word address");
    return JVPFA_ERR_CUDA;
  }
  const bool gated = kind == kFewGated;
  if (dtype == JVPFA_BF16) return gated ? launch_kind<__nv_bfloat16, kFewGated>(p, maps, s) : launch_kind<__nv_bfloat16, kFewDx>(p, maps, s);
  if (dtype == JVPFA_FP16) return gated ? launch_kind<__half, kFewGated>(p, maps, s) : launch_kind<__half, kFewDx>(p, maps, s);
  return gated ? launch_kind<float, kFewGated>(p, maps, s) : launch_kind<float, kFewDx>(p, maps, s);
}

}  // namespace tc5
}  // namespace jvpfa

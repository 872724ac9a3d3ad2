// Block-scaled GEMM for one CTA per tile, with the weight's rows as the MMA's M and the tokens as its
// N, and K split over a cluster:  out[m, n] = alpha * sum_k A[m, k] W[n, k] + bias[n].
//
// With few tokens the product is bound by the weight's bytes (0.56 per element with nvfp4).  The
// codes need no conversion on the way: TMA brings them to shared memory and the MMA reads them
// there, with the scales in tensor memory.  A CTA streams 128 weight rows against up to 128 tokens;
// where the tiles leave SMs idle, the CTAs of a cluster take a share of K each and add their fp32
// partial tiles through distributed shared memory in rank order (the same result every time).
// 6 warps: 0-3 epilogue, 4 TMA producer, 5 MMA and scale copies.
//
// For a few tokens the kernel can take the activations as they are: the epilogue warps, idle until
// the end, quantise each stage's columns of the tokens into shared memory, in the layout that TMA would
// have written.  Every CTA does so for its share of K; the work is small next to 128 weight rows, and
// a launch and the wait for it are saved.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mx_gemm.cuh"

namespace svdq {

int make_code_map(CUtensorMap* map, const void* codes, int fmt, bool spread, int rows, int k_pad, int box_rows) {
  const uint64_t row_bytes = (uint64_t)mx_row_bytes(fmt, k_pad);
  if (spread)  // 16 codes of 8 bytes become 16 bytes of shared memory; coordinates count codes
    return make_tma_2d(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, codes, (uint64_t)k_pad, (uint64_t)rows, row_bytes,
                       128, (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
  return make_tma_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, row_bytes, (uint64_t)rows, row_bytes, 128,
                     (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

int make_scale_map(CUtensorMap* map, const void* scales, int fmt, int rows, int k_pad, int box_tiles, int box_blocks) {
  const uint64_t tiles = (uint64_t)k_pad / mx_block(fmt) / 4;
  const uint64_t dims[3] = {128, tiles, (uint64_t)mx_rows_pad(rows) / 128};
  const uint64_t strides[2] = {512, tiles * 512};
  const uint32_t box[3] = {128, (uint32_t)box_tiles, (uint32_t)box_blocks};
  return make_tma(map, CU_TENSOR_MAP_DATA_TYPE_INT32, scales, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

namespace {

constexpr int kRows = 128;       // weight rows per tile
constexpr int kMaxStages = 12;
constexpr int kSplitThreads = 192;
constexpr int kMaxSplit = 8;
constexpr int kRoomTwo = 108 * 1024, kRoomOne = 216 * 1024;  // bytes of a ring with two CTAs or one to an SM

struct SplitBars {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t done;
  uint32_t tmem_base;
  int abort_flag;
};

constexpr int kExtra = sizeof(SplitBars) + 1024;

struct SplitArgs {
  MxOutput o;
  MxInput in;
  int k;
  int steps;    // stages of K in all
  int split;    // CTAs of the cluster, a share of K each
  int stages;   // ring depth
  int n_tiles;  // tiles along the weight's rows
  bool early_weight;
  int* err;
};

enum : int { kWaitSplitEmpty = 0x501, kWaitSplitFull = 0x511, kWaitSplitDone = 0x512, kWaitSplitEpi = 0x521,
             kWaitSplitQuant = 0x531 };

__device__ __forceinline__ void mbar_arrive_cta(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Warps' worth of 16-column pieces in a stage of M tokens.
template <int MODE>
__host__ __device__ constexpr int fused_groups(int M) { return (M * (MxMode<MODE>::kStageCols / 16) + 31) / 32; }

template <int MODE, int TN>
struct SplitShape {
  static constexpr int kScale = MxMode<MODE>::kScaleTiles * 512;
  static constexpr int kTok = kRows * 128;            // offset of the tokens' codes in a stage
  static constexpr int kScaleW = kTok + TN * 128;
  static constexpr int kScaleT = kScaleW + kScale;
  static constexpr int kBytes = kScaleT + kScale;
  // a spread box counts the bytes of its codes, not the padding that it skips
  static constexpr int kTx = kBytes - (MODE == kModeW4A8 ? kRows * 64 : 0);
  static constexpr int kStage = (kBytes + 1023) / 1024 * 1024;
  static constexpr int kSfw = TN < 32 ? 32 : TN;       // columns of tensor memory
  static constexpr int kSft = kSfw + 4 * MxMode<MODE>::kScaleTiles;
  // bytes that TMA brings where the activations are quantised here
  static constexpr int kTxFused = kTx - TN * 128 - kScale;
  static constexpr int kCols = kSft + 4 * MxMode<MODE>::kScaleTiles <= 64 ? 64 : kSft + 16 <= 128 ? 128 : 256;
};

// The activations of stages s0 .. s1 - 1, quantised by warps 0-3.  A lane takes 16 columns of a token;
// `groups` warps' worth of them make a stage, and the warps take the groups of all stages in turn, each
// with its next group's columns on the way while it works on one.
template <int MODE, typename T>
__device__ __forceinline__ void quantize_stages(const SplitArgs& a, SplitBars* bars, uint8_t* ring, int stage_bytes,
                                                int tok, int scale, Nvfp4Unit* units, int s0, int s1,
                                                volatile int* abort_flag) {
  constexpr int kFmt = MODE == kModeNvfp4 ? kNvfp4 : MODE == kModeMxfp4 ? kMxfp4 : kMxfp8;
  constexpr int kChunks = MxMode<MODE>::kStageCols / 16;  // per token and stage
  constexpr int kLanes = kFmt == kNvfp4 ? 4 : 8;          // per word of scales
  using Codes = typename CodeWord<kFmt>::type;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = fused_groups<MODE>(a.o.M);
  const float g = kFmt == kNvfp4 && a.o.a_scale ? *a.o.a_scale : 1.0f;
  auto load = [&](int s, int group, T (&x)[16]) {
    const int item = group * 32 + lane, m = item / kChunks;
    const int c = m < a.o.M && s < s1 ? s * MxMode<MODE>::kStageCols + item % kChunks * 16 : a.k;
    const T* row = static_cast<const T*>(a.in.x) + (m < a.o.M ? (size_t)m * a.in.ldx : 0);
    if (!a.in.vec) {
      load_shifted(row, c, a.k, x);
    } else if (c < a.k) {
      load_vec(row + c, x);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = from_float<T>(0.0f);
    }
  };
  alignas(32) T x[16];
  load(s0 + warp / groups, warp % groups, x);
  if constexpr (kFmt == kNvfp4) {
    units[threadIdx.x] = nvfp4_unit<significant_bits<T>()>(threadIdx.x, g);
    asm volatile("bar.sync 1, 128;" ::: "memory");  // warps 0-3
  }
  for (int q = warp; q < (s1 - s0) * groups; q += 4) {
    alignas(32) T next[16];
    load(s0 + (q + 4) / groups, (q + 4) % groups, next);
    uint32_t byte;
    const Codes codes = encode_chunk<T, kFmt>(x, g, units, byte);
    const uint32_t word = scale_word<kFmt>(byte);
    const int turn = q / groups, stage = turn % a.stages;
    const uint32_t phase = (uint32_t)(turn / a.stages) & 1u;
    if (!warp_spin_wait(smem_u32(&bars->empty[stage]), phase ^ 1u, abort_flag, a.err, kWaitSplitQuant)) break;
    uint8_t* at = ring + (size_t)stage * stage_bytes;
    const int item = q % groups * 32 + lane, m = item / kChunks, c = item % kChunks;
    if (m < a.o.M) {
      // 128-byte rows in 16-byte pieces, piece p of row m at p ^ (m % 8) (the 128-byte swizzle)
      const int off = c * (int)sizeof(Codes);
      *reinterpret_cast<Codes*>(at + tok + m * 128 + ((((off >> 4) ^ (m & 7)) << 4) | (off & 15))) = codes;
      if (c % kLanes == 0) *reinterpret_cast<uint32_t*>(at + scale + (c / kLanes) * 512 + m * 16) = word;
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive_cta(smem_u32(&bars->full[stage]));
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = next[j];
  }
}

// X: the activations' type where they are quantised here, void where they come as codes and scales.
template <int MODE, int TN, typename X>
__global__ void __launch_bounds__(kSplitThreads)
    mx_gemm_split_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap t_map,
                         const __grid_constant__ CUtensorMap sw_map, const __grid_constant__ CUtensorMap st_map,
                         const __grid_constant__ SplitArgs a) {
  using S = SplitShape<MODE, TN>;
  using Mode = MxMode<MODE>;
  constexpr bool kFused = !std::is_void<X>::value;
  __shared__ __align__(16) Nvfp4Unit units[kFused && MODE == kModeNvfp4 ? 128 : 1];
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw & 1023u)) & 1023u;
  const uint32_t base = raw + pad;
  SplitBars* bars = reinterpret_cast<SplitBars*>(smem_raw + pad + (size_t)a.stages * S::kStage);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = a.split > 1 ? (int)cluster_ctarank() : 0;
  const int tile = blockIdx.x / a.split;
  const int n0 = (tile % a.n_tiles) * kRows, m0 = (tile / a.n_tiles) * TN;
  const int s0 = (int)((int64_t)a.steps * rank / a.split), s1 = (int)((int64_t)a.steps * (rank + 1) / a.split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      // the producer, and the groups of activations that are quantised here
      mbar_init(smem_u32(&bars->full[s]), 1 + (kFused ? fused_groups<MODE>(a.o.M) : 0));
      mbar_init(smem_u32(&bars->empty[s]), 1);
    }
    mbar_init(smem_u32(&bars->done), 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 4 && lane == 0) {
    prefetch_tma_desc(&w_map);
    prefetch_tma_desc(&sw_map);
    if (!kFused) {
      prefetch_tma_desc(&t_map);
      prefetch_tma_desc(&st_map);
    }
  }
  if (warp == 5) {
    tmem_alloc_1(smem_u32(&bars->tmem_base), S::kCols);
    tmem_relinquish_1();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  auto load_weight = [&](int s, int stage) {
    const uint32_t bar = smem_u32(&bars->full[stage]), at = base + (uint32_t)(stage * S::kStage);
    mbar_arrive_expect_tx(bar, kFused ? S::kTxFused : S::kTx);
    tma_load_2d(at, &w_map, bar, s * 128, n0);
    tma_load_3d(at + S::kScaleW, &sw_map, bar, 0, s * Mode::kScaleTiles, n0 / 128);
  };
  // Stages whose weight is on its way before the wait for the launch before this one.  That launch is the
  // quantisation of this call's activations; it has itself waited for everything before it when
  // this one begins, so a weight that an earlier launch wrote is in memory.
  const int early = !kFused && a.early_weight ? min(a.stages, s1 - s0) : 0;
  if (warp == 4 && early > 0) {
    if (elect_one())
      for (int i = 0; i < early; ++i) load_weight(s0 + i, i);
    __syncwarp();
  }
  pdl_wait();
  pdl_trigger();

  // producer and MMA roles: the whole warp runs the loop, one lane issues
  if (warp == 4) {
    int stage = 0;
    uint32_t phase = 0, filled = early > 0 ? (1u << early) - 1u : 0u, par = 0;
    bool ok = true;
    for (int s = s0; s < s1; ++s) {
      if (!(ok = warp_spin_wait(smem_u32(&bars->empty[stage]), phase ^ 1u, abort_flag, a.err, kWaitSplitEmpty))) break;
      const uint32_t bar = smem_u32(&bars->full[stage]), at = base + (uint32_t)(stage * S::kStage);
      if (elect_one()) {
        if (s - s0 >= early) load_weight(s, stage);
        if (!kFused) {
          tma_load_2d(at + S::kTok, &t_map, bar, s * 128, m0);
          tma_load_3d(at + S::kScaleT, &st_map, bar, 0, s * Mode::kScaleTiles, m0 / 128);
        }
      }
      __syncwarp();
      filled |= 1u << stage;
      par = (par & ~(1u << stage)) | (phase << stage);
      if (++stage == a.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (!ok && lane == 0)  // copies in flight land before the CTA exits
      for (int s = 0; s < a.stages; ++s)
        if (filled & (1u << s)) mbar_wait_drain(smem_u32(&bars->full[s]), (par >> s) & 1u, 100000000ull);
  } else if (warp == 5) {
    int stage = 0;
    uint32_t phase = 0;
    for (int s = s0; s < s1; ++s) {
      if (!warp_spin_wait(smem_u32(&bars->full[stage]), phase, abort_flag, a.err, kWaitSplitFull)) break;
      tc_fence_after();
      const uint32_t at = base + (uint32_t)(stage * S::kStage);
      const uint64_t dw = desc_k_sw128(at), dt = desc_k_sw128(at + S::kTok);
      if (elect_one()) {
#pragma unroll
        for (int t = 0; t < Mode::kScaleTiles; ++t) {
          copy_scale_tile<false>(tmem + S::kSfw + 4 * t, at + S::kScaleW + 512 * t);
          copy_scale_tile<false>(tmem + S::kSft + 4 * t, at + S::kScaleT + 512 * t);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          umma_mx<MODE, false>(tmem, dw + (uint64_t)(2 * j), dt + (uint64_t)(2 * j),
                               mx_idesc<MODE>(kRows, TN, true, Mode::byte_of(j)), tmem + S::kSfw + 4 * Mode::tile_of(j),
                               tmem + S::kSft + 4 * Mode::tile_of(j), (s > s0 || j > 0) ? 1u : 0u);
        umma_commit_1(smem_u32(&bars->empty[stage]));
      }
      __syncwarp();
      if (++stage == a.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (elect_one()) {
      umma_commit_1(smem_u32(&bars->done));  // also after an abort: MMAs end before TMEM is freed
      if (!mbar_wait_drain(smem_u32(&bars->done), 0, 1000000000ull)) {
        *abort_flag = 1;
        atomicCAS(a.err, 0, kWaitSplitDone);
      }
    }
    __syncwarp();
  }
  if constexpr (kFused) {
    if (warp < 4)
      quantize_stages<MODE, X>(a, bars, smem_raw + pad, S::kStage, S::kTok, S::kScaleT, units, s0, s1, abort_flag);
    __syncwarp();
  }
  // epilogue: warp w holds weight rows 32 w .. 32 w + 31, one per lane, and every token's column
  const int row = warp * 32 + lane, n = n0 + row;
  bool ok = true;
  if (warp < 4) {
    ok = warp_spin_wait(smem_u32(&bars->done), 0, abort_flag, a.err, kWaitSplitEpi);
    ok = __all_sync(0xffffffffu, ok && !*abort_flag);
    tc_fence_after();
  }
  const float alpha = mx_alpha(a.o);
  const float bias = a.o.bias && warp < 4 && n < a.o.N ? __bfloat162float(a.o.bias[n]) : 0.0f;
  if (warp < 4) {
#pragma unroll
    for (int c = 0; c < TN; c += 16) {
      if (m0 + c >= a.o.M) break;
      uint32_t v[16];
      tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)c, v);
      tmem_ld_wait_regs16(v);
      if (!ok) continue;
      if (a.split > 1) {  // the ring is idle: the partial tile, one token after the other
        float* part = reinterpret_cast<float*>(smem_raw + pad);
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(c + i) * kRows + row] = __uint_as_float(v[i]);
      } else if (n < a.o.N) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (m0 + c + i < a.o.M) store_one(a.o, m0 + c + i, n, fmaf(alpha, __uint_as_float(v[i]), bias));
      }
    }
  }
  if (a.split > 1) {
    // a share of the tokens each: a thread adds 4 rows of one token over the ranks, in rank order
    if (!ok) *abort_flag = 1;
    cluster_sync();
    const int per = (TN + a.split - 1) / a.split;
    const int t1 = min(min(TN, (rank + 1) * per), a.o.M - m0);
    const int r4 = lane * 4, nn = n0 + r4;
    const bool good = *abort_flag == 0;
    float b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = a.o.bias && nn + i < a.o.N ? __bfloat162float(a.o.bias[nn + i]) : 0.0f;
    for (int t = rank * per + warp; t < t1; t += kSplitThreads / 32) {
      float4 p[kMaxSplit];
#pragma unroll
      for (int r = 0; r < kMaxSplit; ++r)
        if (r < a.split)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(p[r].x), "=f"(p[r].y), "=f"(p[r].z), "=f"(p[r].w)
                       : "r"(mapa_shared(base + (uint32_t)(t * kRows + r4) * 4, (uint32_t)r))
                       : "memory");
      float v[4] = {p[0].x, p[0].y, p[0].z, p[0].w};
#pragma unroll
      for (int r = 1; r < kMaxSplit; ++r)
        if (r < a.split) {
          v[0] += p[r].x;
          v[1] += p[r].y;
          v[2] += p[r].z;
          v[3] += p[r].w;
        }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (good && nn + i < a.o.N) store_one(a.o, m0 + t, nn + i, fmaf(alpha, v[i], b[i]));
    }
    cluster_sync();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc_1(tmem, S::kCols);
  }
}

// Clusters of `split` CTAs with an SM to each CTA that run at once on the current device: an
// occupancy query per cluster size, cached.  (GPCs of 16 to 18 SMs: 74 pairs, 45 clusters of 3, 33
// of 4, 26 of 5, 22 of 6, 15 of 7 or 8 on a B200.)
int resident_clusters(const void* kern, int split, size_t smem) {
  static std::atomic<int> cache[64][kMaxSplit + 1];
  int dev = 0;
  cudaGetDevice(&dev);
  std::atomic<int>* slot = dev >= 0 && dev < 64 ? &cache[dev][split] : nullptr;
  int n = slot ? slot->load(std::memory_order_relaxed) : 0;
  if (n > 0) return n;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)split, 1, 1);
  cfg.blockDim = dim3(kSplitThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    n = num_sms() / split;
  }
  if (slot) slot->store(n, std::memory_order_relaxed);
  return n;
}

// How a call would run here, and about how long (us past the fixed cost of a launch).
struct SplitPlan {
  int steps, n_tiles, tiles, split, stages;
  float us;
};

// us per stage of one CTA, [mode][TN]: a stage is 19 to 37 KB through L2 at some 80 GB/s to an SM;
// nvfp4 at 128 tokens is bound by its scale copies.  Measured at N 6144, K 6144 with one CTA a tile.
constexpr float kStageUs[3][4] = {{.30f, .33f, .44f, .64f}, {.26f, .28f, .38f, .50f}, {.24f, .26f, .36f, .43f}};

template <int MODE, int TN, typename X>
int plan_split(const MxGemm& g, SplitPlan* p) {
  using S = SplitShape<MODE, TN>;
  auto kern = mx_gemm_split_kernel<MODE, TN, X>;
  cudaError_t ce = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRoomOne + kExtra);
  if (ce == cudaSuccess)
    ce = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (ce != cudaSuccess) return check_cuda(ce, "svdq_mx_gemm: shared memory attribute");
  // two CTAs to an SM where the ring is deep enough at half the memory
  const int per_sm = S::kStage * 4 <= kRoomTwo ? 2 : 1;
  p->stages = std::min(kMaxStages, (per_sm == 2 ? kRoomTwo : kRoomOne) / S::kStage);
  p->steps = (g.k_pad + MxMode<MODE>::kStageCols - 1) / MxMode<MODE>::kStageCols;
  p->n_tiles = (g.o.N + kRows - 1) / kRows;
  p->tiles = p->n_tiles * ((g.o.M + TN - 1) / TN);
  // K is split as far as all clusters still run at once, down to two stages each: one round more
  // cost more than the deeper split saved at every size measured (N 6144, K 16384, 16 tokens, mxfp8
  // on mxfp4: 14.0 us split 5 ways, 22.1 in 6)
  p->split = 1;
  const void* k = reinterpret_cast<const void*>(kern);
  for (int s = kMaxSplit; s > 1 && p->split == 1; --s)
    if (2 * s <= p->steps && p->tiles <= per_sm * resident_clusters(k, s, kRoomOne + kExtra)) p->split = s;
  const int ctas = p->tiles * p->split, sms = num_sms();
  const int rounds = (ctas + per_sm * sms - 1) / (per_sm * sms);
  const float share = ctas > sms && per_sm == 2 ? 1.5f : 1.0f;  // two CTAs of an SM share its bandwidth
  p->us = rounds * share * (float)((p->steps + p->split - 1) / p->split) * kStageUs[MODE][TN == 16 ? 0 : TN == 32 ? 1 : TN == 64 ? 2 : 3] +
          (p->split > 1 ? TN / 64.0f : 0.0f);
  return SVDQ_OK;
}

template <int MODE, int TN, typename X>
int launch_split(const MxGemm& g, const SplitPlan& p) {
  using S = SplitShape<MODE, TN>;
  CUtensorMap w, t, sw, st;
  int e;
  const bool spread = MODE == kModeW4A8;
  if ((e = make_code_map(&w, g.w_codes, g.w_fmt, spread, g.o.N, g.k_pad, kRows))) return e;
  if ((e = make_scale_map(&sw, g.w_scales, g.w_fmt, g.o.N, g.k_pad, MxMode<MODE>::kScaleTiles, 1))) return e;
  if (std::is_void<X>::value) {
    if ((e = make_code_map(&t, g.a_codes, g.a_fmt, false, g.o.M, g.k_pad, TN))) return e;
    if ((e = make_scale_map(&st, g.a_scales, g.a_fmt, g.o.M, g.k_pad, MxMode<MODE>::kScaleTiles, 1))) return e;
  } else {  // not read
    t = w;
    st = sw;
  }
  SplitArgs a{};
  a.o = g.o;
  a.in = g.in;
  a.k = g.k;
  a.err = g.err;
  a.steps = p.steps;
  a.n_tiles = p.n_tiles;
  a.early_weight = g.early_weight;
  a.split = p.split;
  a.stages = p.stages;
  return launch_pdl("svdq_mx_gemm launch", mx_gemm_split_kernel<MODE, TN, X>, dim3((unsigned)(p.tiles * p.split)),
                    dim3(kSplitThreads), (size_t)a.stages * S::kStage + kExtra, g.stream, a.split, w, t, sw, st, a);
}

// One product: the pair kernel or this one, whichever is estimated to end first.  A tile of the pair
// kernel costs 0.42 (nvfp4), 0.40 (mxfp4) or 0.36 us (mxfp8 x mxfp4) per stage.  At N 6144, K 6144,
// mxfp8 on mxfp4: 128 tokens 16.2 us here against 21.2 on pairs, 256 tokens 25.8 against 21.4.  Both timed for 204 calls
// (8 to 4352 tokens, four weights, three modes, weight out of L2), the estimate's choice was slower by more than 1%
// in one, by 3%.
template <int MODE, int TN>
int choose(const MxGemm& g) {
  constexpr float kPairUs[3] = {.42f, .40f, .36f};
  SplitPlan p;
  const int e = plan_split<MODE, TN, void>(g, &p);
  if (e) return e;
  const int pairs = num_sms() / 2, tiles = ((g.o.M + 255) / 256) * ((g.o.N + 255) / 256);
  const float us = (float)((tiles + pairs - 1) / pairs) * p.steps * kPairUs[MODE];
  return us < p.us ? launch_mx_gemm_pair(g) : launch_split<MODE, TN, void>(g, p);
}
template <int MODE, typename X>
int launch_fused(const MxGemm& g) {
  SplitPlan p;
  const int e = plan_split<MODE, 16, X>(g, &p);
  return e ? e : launch_split<MODE, 16, X>(g, p);
}
template <int MODE>
int choose_tokens(const MxGemm& g) {
  if (g.in.x)
    return g.in.dtype == SVDQ_BF16   ? launch_fused<MODE, __nv_bfloat16>(g)
           : g.in.dtype == SVDQ_FP16 ? launch_fused<MODE, __half>(g)
                                     : launch_fused<MODE, float>(g);
  if (g.o.M <= 16) return choose<MODE, 16>(g);
  if (g.o.M <= 32) return choose<MODE, 32>(g);
  if (g.o.M <= 64) return choose<MODE, 64>(g);
  return choose<MODE, 128>(g);
}

// Checks a product's arguments (the activations as codes and scales, or g.in) and runs it.
int mx_product(MxGemm& g, int K) {
  const int M = g.o.M, N = g.o.N;
  SVDQ_REQUIRE((g.a_fmt == g.w_fmt && (g.a_fmt == kNvfp4 || g.a_fmt == kMxfp4)) ||
                   (g.a_fmt == kMxfp8 && g.w_fmt == kMxfp4),
               "svdq_mx_gemm: operands are nvfp4 x nvfp4, mxfp4 x mxfp4 or mxfp8 x mxfp4 (activations x weight)");
  SVDQ_REQUIRE(dtype_ok(g.o.out_dtype), "svdq_mx_gemm: out must be bf16, fp16 or fp32");
  SVDQ_REQUIRE(M >= 0 && N > 0 && K > 0 && g.o.ldo >= N, "svdq_mx_gemm: bad M/N/K/ldo");
  SVDQ_REQUIRE((!g.o.a_scale && !g.o.w_scale) || g.a_fmt == kNvfp4, "svdq_mx_gemm: only nvfp4 operands have tensor scales");
  if (M == 0) return SVDQ_OK;
  SVDQ_REQUIRE((g.in.x || (g.a_codes && g.a_scales)) && g.w_codes && g.w_scales && g.o.out, "svdq_mx_gemm: null pointer");
  SVDQ_REQUIRE(((reinterpret_cast<uintptr_t>(g.a_codes) | reinterpret_cast<uintptr_t>(g.a_scales) |
                 reinterpret_cast<uintptr_t>(g.w_codes) | reinterpret_cast<uintptr_t>(g.w_scales)) & 31u) == 0,
               "svdq_mx_gemm: codes and scales must be 32-byte aligned");
  SVDQ_REQUIRE(element_aligned(g.o.out, dtype_bytes(g.o.out_dtype)) && element_aligned(g.o.bias, 2) &&
                   element_aligned(g.o.a_scale, 4) && element_aligned(g.o.w_scale, 4),
               "svdq_mx_gemm: out, bias and tensor scales must be aligned to their elements");
  if (M > (1 << 24) || N > (1 << 24) || K > (1 << 28))
    return set_error(SVDQ_ERR_UNSUPPORTED, "svdq_mx_gemm: M and N up to 2^24, K up to 2^28");
  g.mode = g.a_fmt == kNvfp4 ? kModeNvfp4 : g.a_fmt == kMxfp4 ? kModeMxfp4 : kModeW4A8;
  g.k = K;
  g.k_pad = mx_k_pad(K);
  g.err = device_error_word();
  if (!g.err) return set_error(SVDQ_ERR_CUDA, "svdq_mx_gemm: device error word unavailable");
  if (g.mode == kModeNvfp4) return choose_tokens<kModeNvfp4>(g);
  return g.mode == kModeMxfp4 ? choose_tokens<kModeMxfp4>(g) : choose_tokens<kModeW4A8>(g);
}

// Workspace of svdq_mx_linear: the codes, then the scales from the next 256-byte boundary.
size_t mx_code_bytes(int M, int K, int fmt) { return ((size_t)M * mx_row_bytes(fmt, mx_k_pad(K)) + 255) / 256 * 256; }

}  // namespace
}  // namespace svdq

extern "C" int svdq_mx_gemm(const void* a_codes, const void* a_scales, int a_format, const float* a_tensor_scale,
                            const void* w_codes, const void* w_scales, int w_format, const float* w_tensor_scale,
                            const void* bias, void* out, int out_dtype, int64_t ldo, int M, int N, int K,
                            cudaStream_t stream) {
  using namespace svdq;
  MxGemm g{};
  g.a_codes = a_codes;
  g.a_scales = a_scales;
  g.a_fmt = a_format;
  g.w_codes = w_codes;
  g.w_scales = w_scales;
  g.w_fmt = w_format;
  g.o = MxOutput{a_tensor_scale, w_tensor_scale, static_cast<const __nv_bfloat16*>(bias), out, ldo, out_dtype, M, N};
  g.stream = stream;
  return mx_product(g, K);
}

extern "C" size_t svdq_mx_linear_workspace_bytes(int M, int K, int a_format) {
  using namespace svdq;
  if (M <= kMaxFusedTokens || K <= 0 || !mx_format_ok(a_format) || M > (1 << 30) || K > (1 << 30)) return 0;
  return mx_code_bytes(M, K, a_format) + svdq_mx_scale_bytes(M, K, a_format);
}

extern "C" int svdq_mx_linear(const void* x, int64_t ldx, int dtype, int a_format, const float* a_tensor_scale,
                              const void* w_codes, const void* w_scales, int w_format, const float* w_tensor_scale,
                              const void* bias, void* out, int out_dtype, int64_t ldo, int M, int N, int K,
                              void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  using namespace svdq;
  SVDQ_REQUIRE(mx_format_ok(a_format), "svdq_mx_linear: unknown activation format");
  SVDQ_REQUIRE(dtype_ok(dtype), "svdq_mx_linear: x must be bf16, fp16 or fp32");
  SVDQ_REQUIRE(M >= 0 && K > 0 && ldx >= K, "svdq_mx_linear: bad M/K/ldx");
  SVDQ_REQUIRE(x || M == 0, "svdq_mx_linear: null pointer");
  SVDQ_REQUIRE(element_aligned(x, dtype_bytes(dtype)), "svdq_mx_linear: x must be aligned to its elements");
  MxGemm g{};
  g.a_fmt = a_format;
  g.w_codes = w_codes;
  g.w_scales = w_scales;
  g.w_fmt = w_format;
  g.o = MxOutput{a_tensor_scale, w_tensor_scale, static_cast<const __nv_bfloat16*>(bias), out, ldo, out_dtype, M, N};
  g.stream = stream;
  if (M <= kMaxFusedTokens) {  // one launch
    g.in = MxInput{x, ldx, dtype, K % 16 == 0 && rows_aligned(x, ldx, dtype_bytes(dtype), 32)};
    return mx_product(g, K);
  }
  SVDQ_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0 &&
                   workspace_bytes >= svdq_mx_linear_workspace_bytes(M, K, a_format),
               "svdq_mx_linear: workspace must be 256-byte aligned and hold svdq_mx_linear_workspace_bytes()");
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  uint8_t* scales = codes + mx_code_bytes(M, K, a_format);
  g.a_codes = codes;
  g.a_scales = scales;
  g.early_weight = true;
  const int st = svdq_mx_quantize(x, ldx, dtype, M, K, a_format, a_tensor_scale, codes, scales, stream);
  return st ? st : mx_product(g, K);
}

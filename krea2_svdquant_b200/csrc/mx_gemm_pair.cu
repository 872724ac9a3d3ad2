// Block-scaled GEMM on CTA pairs, for batches that fill 256 x 256 tiles:
//   out[m, n] = alpha * sum_k A[m, k] W[n, k] + bias[n].
//
// Persistent kernel, clusters of two CTAs.  A pair owns one 256 x 256 tile at a time: the even CTA
// issues cta_group::2 MMAs whose 256 token rows and 256 weight rows are split between the two CTAs'
// shared memory, so an operand byte crosses L2 once per pair.  12 warps per CTA:
//   warp 0      TMA producer (both CTAs): codes of its 128 token rows and 128 weight rows, scale tiles
//               of its token rows and of all 256 weight rows, counted on the even CTA's barrier
//   warp 1      TMEM (both CTAs); in the even CTA scale copies and MMAs
//   warps 4-11  epilogue (both CTAs): two warpgroups, 32-column chunks in turn
//
// Tensor memory has 512 columns, and the scales need some, so two accumulators of 256 columns do not
// fit beside them.  They overlap by 64 columns instead: columns 0-255 and 192-447, scales from 448.
// The epilogue reads the shared columns first, and the next tile's MMAs wait for that alone.
#include <algorithm>

#include "mx_gemm.cuh"

namespace svdq {
namespace {

constexpr int BM = 128;  // token rows and weight rows per CTA
constexpr int BN = 256;
constexpr int kPairThreads = 384;
constexpr int kAccShift = 192;  // column of the second accumulator
constexpr int kScaleCol = 448;
constexpr int kMaxStages = 6;

struct PairBars {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t acc_full[2];
  uint64_t acc_free;  // the columns that the accumulators share have been read (16 warps)
  uint64_t done;
  uint32_t tmem_base;
  int abort_flag;
  float turn[8][32 * 33];  // a 32 x 32 chunk per epilogue warp, rows padded against bank conflicts
};

struct PairArgs {
  MxOutput o;
  int steps;
  int m_blocks, n_blocks, tiles, group;
  int* err;
};

enum : int {
  kWaitPairEmpty = 0x601,
  kWaitPairFull = 0x611,
  kWaitPairAcc = 0x612,
  kWaitPairDone = 0x613,
  kWaitPairEpi = 0x621
};

template <int MODE>
struct PairShape {
  static constexpr int kTiles = MxMode<MODE>::kScaleTiles;
  static constexpr int kB = BM * 128;
  static constexpr int kSfa = 2 * BM * 128;
  static constexpr int kSfb = kSfa + kTiles * 512;
  static constexpr int kBytes = kSfb + 2 * kTiles * 512;
  // of one CTA; a spread box counts the bytes of its codes
  static constexpr int kTx = kBytes - (MODE == kModeW4A8 ? BM * 64 : 0);
  static constexpr int kStage = (kBytes + 1023) / 1024 * 1024;
  static constexpr int kRing = 227 * 1024 - 1024 - (int)sizeof(PairBars);
  static constexpr int kStages = kRing / kStage < kMaxStages ? kRing / kStage : kMaxStages;
  static constexpr size_t kSmem = (size_t)kStages * kStage + sizeof(PairBars) + 1024;
};

// Arrive on an mbarrier of either CTA after reads of tensor memory (completed, and ordered by a
// tcgen05 fence).  Release at CTA scope: at cluster scope the arrival waits for this thread's output
// stores of the tile before to be performed, over 1000 cycles in which the next tile cannot start.
__device__ __forceinline__ void mbar_arrive_after_tmem(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y,
                                                 int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Row blocks advance along N in groups of a.group, so that the tiles of one moment share operands in
// L2.  A group's activations stay there while the weight streams past once, so groups are as large as
// kGroupBytes allow (and even).  nvfp4 K 6144 (0.9 MB a block): groups of 24 ran 5% faster than of 8
// (M 4352, N 16384: 188 us against 198); mxfp8 K 16384 (4.3 MB a block): groups of 16 ran 5% slower.
constexpr int64_t kGroupBytes = 28 << 20;
__device__ __forceinline__ void tile_of(int t, const PairArgs& a, int& mb, int& nb) {
  const int per_group = a.group * a.n_blocks;
  const int first = (t / per_group) * a.group;
  const int r = t % per_group;
  const int gm = min(a.m_blocks - first, a.group);
  mb = first + r % gm;
  nb = r / gm;
}

__device__ __forceinline__ uint32_t pack2(int dtype, float a, float b) {
  if (dtype == SVDQ_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// 32 x 32 outputs from the accumulator: lane l holds row m0 + l, columns n .. n + 31.  Where the
// rows allow it each lane writes its row in 32-byte pieces (through shared memory and TMA stores
// instead, M 4352, N 16384, nvfp4: 50 us against 49 at K 1024, 194 against 160 at K 6144; a short K is
// bound by writing the output); otherwise (N or the output's address
// is not a multiple of 32 bytes, or columns are missing) the chunk is turned in shared memory and
// each row leaves as 32 neighbouring elements.
__device__ __forceinline__ void store_chunk(const MxOutput& o, int m0, int lane, int n, const uint32_t (&acc)[32],
                                            float alpha, bool wide, float* turn) {
  if (m0 >= o.M || n >= o.N) return;
  if (wide && n + 32 <= o.N) {
    if (m0 + lane >= o.M) return;
    float v[32];
    if (o.bias) {
      const uint4* b = reinterpret_cast<const uint4*>(o.bias + n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 w = __ldg(b + i);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[8 * i + 2 * j] = fmaf(alpha, __uint_as_float(acc[8 * i + 2 * j]), __uint_as_float(ww[j] << 16));
          v[8 * i + 2 * j + 1] =
              fmaf(alpha, __uint_as_float(acc[8 * i + 2 * j + 1]), __uint_as_float(ww[j] & 0xFFFF0000u));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = alpha * __uint_as_float(acc[i]);
    }
    const size_t at = (size_t)(m0 + lane) * o.ldo + n;
    if (o.out_dtype == SVDQ_FP32) {
      float* p = static_cast<float*>(o.out) + at;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(v[8 * i + j]);
        store32(p + 8 * i, w);
      }
    } else {
      uint16_t* p = static_cast<uint16_t*>(o.out) + at;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = pack2(o.out_dtype, v[16 * i + 2 * j], v[16 * i + 2 * j + 1]);
        store32(p + 16 * i, w);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) turn[lane * 33 + i] = __uint_as_float(acc[i]);
  __syncwarp();
  if (n + lane < o.N) {
    const float bias = o.bias ? __bfloat162float(o.bias[n + lane]) : 0.0f;
    const int rows = min(32, o.M - m0);
#pragma unroll 8
    for (int r = 0; r < rows; ++r) store_one(o, m0 + r, n + lane, fmaf(alpha, turn[r * 33 + lane], bias));
  }
  __syncwarp();
}

template <int MODE>
__global__ void __launch_bounds__(kPairThreads, 1)
    mx_gemm_pair_kernel(const __grid_constant__ CUtensorMap t_map, const __grid_constant__ CUtensorMap w_map,
                        const __grid_constant__ CUtensorMap st_map, const __grid_constant__ CUtensorMap sw_map,
                        const __grid_constant__ PairArgs a) {
  using S = PairShape<MODE>;
  using Mode = MxMode<MODE>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw & 1023u)) & 1023u;
  const uint32_t base = raw + pad;
  PairBars* bars = reinterpret_cast<PairBars*>(smem_raw + pad + (size_t)S::kStages * S::kStage);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(smem_u32(&bars->full[s]), 1);
      mbar_init(smem_u32(&bars->empty[s]), 1);
    }
    mbar_init(smem_u32(&bars->acc_full[0]), 1);
    mbar_init(smem_u32(&bars->acc_full[1]), 1);
    mbar_init(smem_u32(&bars->acc_free), 16);
    mbar_init(smem_u32(&bars->done), 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tma_desc(&t_map);
    prefetch_tma_desc(&w_map);
    prefetch_tma_desc(&st_map);
    prefetch_tma_desc(&sw_map);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&bars->tmem_base), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before either signals the other
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  pdl_wait();
  pdl_trigger();

  // producer and MMA roles: the whole warp runs the loop, one lane issues
  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0, filled = 0, par = 0;
    bool ok = true;
    for (int t = pair; ok && t < a.tiles; t += pairs) {
      int mb, nb;
      tile_of(t, a, mb, nb);
      const int m0 = mb * 2 * BM + (int)rank * BM, n0 = nb * BN + (int)rank * BM;
      for (int s = 0; s < a.steps; ++s) {
        if (!(ok = warp_spin_wait(smem_u32(&bars->empty[stage]), phase ^ 1u, abort_flag, a.err, kWaitPairEmpty))) break;
        const uint32_t full = mapa_shared(smem_u32(&bars->full[stage]), 0);
        const uint32_t at = base + (uint32_t)(stage * S::kStage);
        if (elect_one()) {
          if (leader) mbar_arrive_expect_tx(smem_u32(&bars->full[stage]), 2 * S::kTx);
          tma_load_2d_pair(at, &t_map, full, s * 128, m0);
          tma_load_2d_pair(at + S::kB, &w_map, full, s * 128, n0);
          tma_load_3d_pair(at + S::kSfa, &st_map, full, 0, s * S::kTiles, m0 / 128);
          tma_load_3d_pair(at + S::kSfb, &sw_map, full, 0, s * S::kTiles, nb * 2);
        }
        __syncwarp();
        filled |= 1u << stage;
        par = (par & ~(1u << stage)) | (phase << stage);
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok && leader && lane == 0)  // copies in flight land before the CTA exits
      for (int s = 0; s < S::kStages; ++s)
        if (filled & (1u << s)) mbar_wait_drain(smem_u32(&bars->full[s]), (par >> s) & 1u, 100000000ull);
  } else if (warp == 1) {
    if (leader) {
      int stage = 0, j = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t sfa = tmem + kScaleCol, sfb = sfa + 4 * S::kTiles;
      for (int t = pair; ok && t < a.tiles; t += pairs, ++j) {
        if (j > 0 && !(ok = warp_spin_wait(smem_u32(&bars->acc_free), (uint32_t)(j - 1) & 1u, abort_flag, a.err,
                                           kWaitPairAcc)))
          break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)((j & 1) * kAccShift);
        for (int s = 0; s < a.steps; ++s) {
          if (!(ok = warp_spin_wait(smem_u32(&bars->full[stage]), phase, abort_flag, a.err, kWaitPairFull))) break;
          tc_fence_after();
          const uint32_t at = base + (uint32_t)(stage * S::kStage);
          const uint64_t da = desc_k_sw128(at), db = desc_k_sw128(at + S::kB);
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < S::kTiles; ++i) {
              copy_scale_tile<true>(sfa + 4 * i, at + S::kSfa + 512 * i);
              copy_scale_tile<true>(sfb + 8 * i, at + S::kSfb + 512 * i);
              copy_scale_tile<true>(sfb + 8 * i + 4, at + S::kSfb + 512 * (S::kTiles + i));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              umma_mx<MODE, true>(d, da + (uint64_t)(2 * i), db + (uint64_t)(2 * i),
                                  mx_idesc<MODE>(2 * BM, BN, false, Mode::byte_of(i)), sfa + 4 * Mode::tile_of(i),
                                  sfb + 8 * Mode::tile_of(i), (s > 0 || i > 0) ? 1u : 0u);
            umma_commit_pair(smem_u32(&bars->empty[stage]));
          }
          __syncwarp();
          if (++stage == S::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok && elect_one()) umma_commit_pair(smem_u32(&bars->acc_full[j & 1]));
        __syncwarp();
      }
      if (elect_one()) {
        umma_commit_pair_local(smem_u32(&bars->done));  // every MMA ends before TMEM is freed or a CTA exits
        if (!mbar_wait_drain(smem_u32(&bars->done), 0, 1000000000ull)) {
          *abort_flag = 1;
          atomicCAS(a.err, 0, kWaitPairDone);
        }
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    const int half = (warp - 4) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t free_bar = mapa_shared(smem_u32(&bars->acc_free), 0);
    const float alpha = mx_alpha(a.o);
    const int esz = a.o.out_dtype == SVDQ_FP32 ? 4 : 2;
    const bool wide = ((reinterpret_cast<uintptr_t>(a.o.out) | (uintptr_t)(a.o.ldo * esz)) & 31u) == 0 &&
                      (reinterpret_cast<uintptr_t>(a.o.bias) & 15u) == 0;
    int j = 0;
    for (int t = pair; t < a.tiles; t += pairs, ++j) {
      int mb, nb;
      tile_of(t, a, mb, nb);
      const int m0 = mb * 2 * BM + (int)rank * BM + (warp & 3) * 32, n0 = nb * BN;
      const int first = (j & 1) ? half : 6 + half;  // the chunk in the columns that the accumulators share
      const uint32_t acc = lanes + (uint32_t)((j & 1) * kAccShift);
      if (!warp_spin_wait(smem_u32(&bars->acc_full[j & 1]), (uint32_t)(j >> 1) & 1u, abort_flag, a.err, kWaitPairEpi))
        break;
      tc_fence_after();
      uint32_t va[32], vb[32];
      tmem_ld32(acc + (uint32_t)(first * 32), va);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t (&cur)[32] = (c & 1) ? vb : va;
        uint32_t (&nxt)[32] = (c & 1) ? va : vb;
        tmem_ld_wait_regs(cur);
        if (c == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_after_tmem(free_bar);
        }
        if (c < 3) tmem_ld32(acc + (uint32_t)(((first + 2 * (c + 1)) & 7) * 32), nxt);
        store_chunk(a.o, m0, lane, n0 + ((first + 2 * c) & 7) * 32, cur, alpha, wide, bars->turn[warp - 4]);
      }
    }
  }
  // neither CTA exits or frees TMEM while the pair's MMAs can touch its memory
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

template <int MODE>
int launch_pair(const MxGemm& g) {
  using S = PairShape<MODE>;
  CUtensorMap t, w, st, sw;
  int e;
  if ((e = make_code_map(&t, g.a_codes, g.a_fmt, false, g.o.M, g.k_pad, BM))) return e;
  if ((e = make_code_map(&w, g.w_codes, g.w_fmt, MODE == kModeW4A8, g.o.N, g.k_pad, BM))) return e;
  if ((e = make_scale_map(&st, g.a_scales, g.a_fmt, g.o.M, g.k_pad, S::kTiles, 1))) return e;
  if ((e = make_scale_map(&sw, g.w_scales, g.w_fmt, g.o.N, g.k_pad, S::kTiles, 2))) return e;
  PairArgs a{};
  a.o = g.o;
  a.err = g.err;
  a.steps = (g.k_pad + MxMode<MODE>::kStageCols - 1) / MxMode<MODE>::kStageCols;
  a.m_blocks = (g.o.M + 2 * BM - 1) / (2 * BM);
  a.n_blocks = (g.o.N + BN - 1) / BN;
  a.tiles = a.m_blocks * a.n_blocks;
  const int64_t block = (int64_t)2 * BM * (mx_row_bytes(g.a_fmt, g.k_pad) + g.k_pad / mx_block(g.a_fmt));
  const int most_m = (int)std::max<int64_t>(1, std::min<int64_t>(kGroupBytes / block, a.m_blocks));
  const int groups = (a.m_blocks + most_m - 1) / most_m;
  a.group = (a.m_blocks + groups - 1) / groups;
  auto kern = mx_gemm_pair_kernel<MODE>;
  const cudaError_t ce = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem);
  if (ce != cudaSuccess) return check_cuda(ce, "svdq_mx_gemm: shared memory attribute");
  const int most = num_sms() / 2;
  const int pairs = a.tiles < most ? a.tiles : most;
  return launch_pdl("svdq_mx_gemm launch", kern, dim3(2 * pairs), dim3(kPairThreads), S::kSmem, g.stream, 2, t, w, st,
                    sw, a);
}

}  // namespace

int launch_mx_gemm_pair(const MxGemm& g) {
  if (g.mode == kModeNvfp4) return launch_pair<kModeNvfp4>(g);
  if (g.mode == kModeMxfp4) return launch_pair<kModeMxfp4>(g);
  return launch_pair<kModeW4A8>(g);
}

}  // namespace svdq

// What the block-scaled GEMM kernels share: the operand modes, MMA and scale-copy instructions, and
// the output arithmetic.
#pragma once

#include "mx_common.cuh"

namespace svdq {

// Operand modes.  Every stage row is 128 bytes of shared memory in the 128-byte swizzle, and one MMA
// takes 32 bytes of K, so a stage is four MMAs whatever the types.
//   kModeNvfp4  4-bit x 4-bit, e4m3 scales per 16: a stage is 256 columns
//   kModeMxfp4  4-bit x 4-bit, e8m0 scales per 32: a stage is 256 columns
//   kModeW4A8   8-bit activations x 4-bit weight, e8m0 scales per 32: a stage is 128 columns, the
//               4-bit codes spread by TMA to 16 codes in 16 bytes (8 bytes of codes, 8 of padding)
enum : int { kModeNvfp4 = 0, kModeMxfp4 = 1, kModeW4A8 = 2 };

template <int MODE>
struct MxMode {
  static constexpr int kStageCols = MODE == kModeW4A8 ? 128 : 256;  // columns of K per stage
  // 512-byte scale tiles (128 rows x 4 blocks) per stage: 64 columns each for nvfp4, 128 for the others
  static constexpr int kScaleTiles = MODE == kModeNvfp4 ? 4 : MODE == kModeMxfp4 ? 2 : 1;
  static constexpr int kStepCols = kStageCols / 4;                  // columns of K per MMA
  // the scale tile and the byte of its words that MMA j of a stage starts at
  __device__ static constexpr int tile_of(int j) { return MODE == kModeNvfp4 ? j : MODE == kModeMxfp4 ? j / 2 : 0; }
  __device__ static constexpr int byte_of(int j) { return MODE == kModeNvfp4 ? 0 : MODE == kModeMxfp4 ? 2 * (j & 1) : j; }
};

// Instruction descriptor of a block-scaled MMA: B scale byte [4,6), A type [7,10), B type [10,13),
// N >> 3 [17,23), scale type [23] (0 e4m3, 1 e8m0), M >> 4 [24,29), A scale byte [29,31).
// Types: e2m1 is 1 where both operands are 4-bit, 5 beside 8-bit ones; e4m3 is 0.
template <int MODE>
__device__ constexpr uint32_t mx_idesc(int m, int n, bool weight_is_a, int scale_byte) {
  const uint32_t w = MODE == kModeW4A8 ? 5u : 1u, t = MODE == kModeW4A8 ? 0u : 1u;
  return ((uint32_t)scale_byte << 4) | ((weight_is_a ? w : t) << 7) | ((weight_is_a ? t : w) << 10) |
         ((uint32_t)(n >> 3) << 17) | ((MODE == kModeNvfp4 ? 0u : 1u) << 23) | ((uint32_t)(m >> 4) << 24) |
         ((uint32_t)scale_byte << 29);
}

// D (+)= A * B with block scales, one CTA (PAIR false) or a CTA pair.
template <int MODE, bool PAIR>
__device__ __forceinline__ void umma_mx(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t accumulate) {
#define SVDQ_MX_MMA(GROUP, KIND, VEC)                                                                              \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                                   \
               "tcgen05.mma.cta_group::" GROUP ".kind::" KIND ".block_scale.scale_vec::" VEC                       \
               " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),                                                  \
               "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                                     \
               : "memory")
  if constexpr (MODE == kModeNvfp4) {
    if constexpr (PAIR) SVDQ_MX_MMA("2", "mxf4nvf4", "4X");
    else SVDQ_MX_MMA("1", "mxf4nvf4", "4X");
  } else if constexpr (MODE == kModeMxfp4) {
    if constexpr (PAIR) SVDQ_MX_MMA("2", "mxf4", "2X");
    else SVDQ_MX_MMA("1", "mxf4", "2X");
  } else {
    if constexpr (PAIR) SVDQ_MX_MMA("2", "mxf8f6f4", "1X");
    else SVDQ_MX_MMA("1", "mxf8f6f4", "1X");
  }
#undef SVDQ_MX_MMA
}

// One 512-byte scale tile from shared memory to 4 columns of tensor memory (row r of the tile to
// lane r % 32, column r / 32; repeated for the four lane quarters).  Runs in order with the MMAs
// that the same thread issues before and after it.
template <bool PAIR>
__device__ __forceinline__ void copy_scale_tile(uint32_t taddr, uint32_t smem) {
  // unswizzled, K-major: 8-row groups of 16-byte rows, 128 bytes apart
  const uint64_t desc = (uint64_t)((smem >> 4) & 0x3FFFu) | ((uint64_t)(128u >> 4) << 16) |
                        ((uint64_t)(128u >> 4) << 32) | ((uint64_t)1u << 46);
  if constexpr (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// out = alpha * sum + bias, stored as out_dtype; alpha = the product of the operands' tensor scales.
struct MxOutput {
  const float* a_scale;  // tensor scales, or null
  const float* w_scale;
  const __nv_bfloat16* bias;
  void* out;
  int64_t ldo;
  int out_dtype;
  int M, N;
};
__device__ __forceinline__ float mx_alpha(const MxOutput& o) {
  float v = 1.0f;
  if (o.a_scale) v = *o.a_scale;
  if (o.w_scale) v *= *o.w_scale;
  return v;
}
__device__ __forceinline__ void store_one(const MxOutput& o, int m, int n, float v) {
  const size_t at = (size_t)m * o.ldo + n;
  if (o.out_dtype == SVDQ_BF16) static_cast<__nv_bfloat16*>(o.out)[at] = __float2bfloat16_rn(v);
  else if (o.out_dtype == SVDQ_FP16) static_cast<__half*>(o.out)[at] = __float2half_rn(v);
  else static_cast<float*>(o.out)[at] = v;
}

// Tensor maps of an operand's codes (2-D) and scale tiles (3-D: 128 words, tiles along K, 128-row blocks).
int make_code_map(CUtensorMap* map, const void* codes, int fmt, bool spread, int rows, int k_pad, int box_rows);
int make_scale_map(CUtensorMap* map, const void* scales, int fmt, int rows, int k_pad, int box_tiles, int box_blocks);

// Activations that a GEMM quantises itself.
struct MxInput {
  const void* x;  // null: the activations come as codes and scales
  int64_t ldx;
  int dtype;
  bool vec;  // rows on 32-byte boundaries and K a multiple of 16
};
// Up to 4 tokens: 128 columns or more of each, a warp's work or two per stage.  Each CTA quantises its share of
// K again, so more tokens cost more the more tiles of weight rows there are.  us against a quantisation before
// (weight out of L2):
//                              4 tokens       5              8
//   nvfp4  bf16  N 16384 K 6144  12.8 / 14.9   15.4 / 15.1   18.4 / 15.5
//   nvfp4  bf16  N 1536  K 6144   5.5 / 7.0     6.6 / 6.9     6.7 / 7.0
//   mxfp8  bf16  N 16384 K 6144  13.5 / 15.4   16.4 / 15.3   17.1 / 15.9
//   mxfp4  fp32  N 6144  K 16384 13.6 / 14.4   15.8 / 14.4   18.5 / 14.5
// From fp32 to nvfp4, whose units cost most, 3 and 4 tokens are up to 11% slower at N 16384 or K 16384 (17.4 / 15.8)
// and 8% faster at N 1536; they keep the limit of the others, as the workspace's size does not know the type.
constexpr int kMaxFusedTokens = 4;

// One checked GEMM call.
struct MxGemm {
  int mode;
  MxInput in;
  bool early_weight;  // the launch before this one is this call's own and does not write the weight
  int k;
  const void *a_codes, *a_scales, *w_codes, *w_scales;
  int a_fmt, w_fmt;
  int k_pad;
  MxOutput o;
  int* err;
  cudaStream_t stream;
};
int launch_mx_gemm_pair(const MxGemm& g);

}  // namespace svdq

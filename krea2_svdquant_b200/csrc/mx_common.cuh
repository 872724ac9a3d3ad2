// Block-scaled floating-point formats (nvfp4, mxfp4, mxfp8): layouts, block quantisation and the
// launch helper shared by the kernels that write or read them.
//
//   nvfp4   e2m1 codes, blocks of 16 columns, e4m3 scales, one fp32 scale per tensor
//   mxfp4   e2m1 codes, blocks of 32 columns, e8m0 scales (powers of two)
//   mxfp8   e4m3 codes, blocks of 32 columns, e8m0 scales
//
// Codes are rows of K_pad = round_up(K, 128) columns, zero past K; 4-bit codes lie two to a byte,
// the even column in the low half.  Scale bytes lie in 512-byte tiles of 128 rows x 4 blocks:
// byte (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4 of tile (row / 128, block / 4), which is
// what one tcgen05.cp of 32 rows x 128 bits moves into tensor memory as the scale operand of a
// block-scaled MMA.  Rows past the last one hold zero bytes.
#pragma once

#include "svdq_common.cuh"

namespace svdq {

enum : int { kNvfp4 = SVDQ_MX_NVFP4, kMxfp4 = SVDQ_MX_MXFP4, kMxfp8 = SVDQ_MX_MXFP8 };

constexpr int kMxKAlign = 128;  // columns of a code row are padded to this many
__host__ __device__ constexpr int mx_k_pad(int K) { return (K + kMxKAlign - 1) / kMxKAlign * kMxKAlign; }
__host__ __device__ constexpr int mx_block(int fmt) { return fmt == kNvfp4 ? 16 : 32; }
__host__ __device__ constexpr int mx_row_bytes(int fmt, int k_pad) { return fmt == kMxfp8 ? k_pad : k_pad / 2; }
__host__ __device__ constexpr int mx_rows_pad(int M) { return (M + 127) / 128 * 128; }

// Offset of the 32-bit word that holds the scales of `row` for blocks 4 * word .. 4 * word + 3.
__device__ __forceinline__ size_t mx_scale_word(int row, int word, int words_per_row) {
  return ((size_t)(row >> 7) * words_per_row + word) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)byte));
  return __half2float(__ushort_as_half((uint16_t)h2));
}
__device__ __forceinline__ uint32_t e4m3x2_satfinite(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Eight values as e2m1 codes, value i in bits 4i..4i+3.
__device__ __forceinline__ uint32_t e2m1x8_satfinite(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// 2^(byte - 127) as fp32 (byte 0 is a subnormal, byte 255 is NaN).
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}

// Scale byte of an mx block from the bits of its largest magnitude: 2^(floor(log2 amax) - emax),
// emax the exponent of the largest code (2 for e2m1, 8 for e4m3), clamped to 2^-127; a block with
// an infinity or a NaN has the NaN byte.
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
  constexpr int emax = FMT == kMxfp4 ? 2 : 8;
  const int field = (int)(amax_bits >> 23);
  return field == 255 ? 255u : (uint32_t)max(field - emax, 0);
}
// The factor 2^-e that brings a block to its codes' range.  Products with it are exact except
// where they underflow, far below the smallest code.
__device__ __forceinline__ float mx_inverse_scale(uint32_t byte) {
  return byte == 255 ? 0.0f : __uint_as_float((254u - byte) << 23);
}

// nvfp4 scale byte: e4m3(amax / (6 g)), correctly rounded.  The quotient is taken in 64 bits, where
// a value that is not halfway between two e4m3 values stays off it, and reaches 32 bits rounded to
// odd (truncated, with the last bit set when anything was cut off), which keeps it off too.
// NaN (0x7F) where amax or the quotient is not finite or the tensor scale is not positive.
__device__ __forceinline__ uint32_t nvfp4_scale_byte(uint32_t amax_bits, float g) {
  const double t = (double)__uint_as_float(amax_bits) / (6.0 * (double)g);
  if (amax_bits >= 0x7F800000u || !(t >= 0.0) || !(g > 0.0f && g <= 3.402823466e38f)) return 0x7Fu;
  const float f = __double2float_rz(t);
  const float odd = (double)f == t ? f : __uint_as_float(__float_as_uint(f) | 1u);
  return e4m3x2_satfinite(odd, 0.0f) & 0xFFu;
}
// e2m1 code of q, ties to even, from comparisons (the rare path below).
__device__ __forceinline__ uint32_t e2m1_of(double q) {
  const double a = fabs(q);
  const uint32_t c = (a > 0.25) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0);
  return c | (signbit(q) ? 8u : 0u);
}
// 16 values of an nvfp4 block as codes e2m1(x / (sf g)) of the exact quotient.  d = fl32(sf g) and
// x / d is formed correctly rounded from the reciprocal (Markstein's correction, P. Markstein, IBM
// J. R&D 34(1), 1990).  That decides every code unless the rounded quotient lands on a border
// between two codes without being there: impossible when sf g has at most 16 significant bits and
// x at most 11 (x - border * d is then zero or above 2^-19 of x); otherwise such blocks are redone
// in 64 bits, as are blocks whose d or quotients leave the range the correction needs.
template <bool SHORT_X>
__device__ __forceinline__ uint2 nvfp4_codes(const float (&x)[16], uint32_t amax_bits, uint32_t sf_byte, float g) {
  const float sf = e4m3_value(sf_byte);
  if (sf_byte == 0u || sf_byte == 0x7Fu) return make_uint2(0u, 0u);
  const float d = sf * g;
  const float dl = fmaf(sf, g, -d);
  bool redo = !(d >= 8.0e-28f && d <= 1.0e30f && __uint_as_float(amax_bits) <= d * 65536.0f);
  const float y = __frcp_rn(d);
  float q[16];
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const uint64_t xx = f2_pack(x[i], x[i + 1]);
    const uint64_t yy = f2_pack(y, y), nd = f2_pack(-d, -d);
    const uint64_t q0 = f2_mul(xx, yy);
    const uint64_t qq = f2_fma(f2_fma(q0, nd, xx), yy, q0);
    q[i] = f2_lo(qq);
    q[i + 1] = f2_hi(qq);
  }
  if (!SHORT_X || dl != 0.0f || (__float_as_uint(d) & 0xFFu) != 0u) {
#pragma unroll
    for (int i = 0; i < 16; ++i) redo |= (__float_as_uint(q[i]) << 11) == 0u && q[i] != 0.0f;
  }
  if (redo) {
    const double dd = (double)sf * (double)g;
    uint2 w = make_uint2(0u, 0u);
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      float a = 0.f, b = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j == i) {
          a = x[j];
          b = x[8 + j];
        }
      }
      w.x |= e2m1_of((double)a / dd) << (4 * i);
      w.y |= e2m1_of((double)b / dd) << (4 * i);
    }
    return w;
  }
  return make_uint2(e2m1x8_satfinite(q), e2m1x8_satfinite(q + 8));
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N values of a row from column c: 16-byte loads where the row allows them and all N columns
// exist, element by element up to K otherwise (zero past it).
template <typename T, int N>
__device__ __forceinline__ void load_cols(const T* row, int c, int K, bool vec, T (&v)[N]) {
  if (vec && c + N <= K) {
    constexpr int W = N * (int)sizeof(T) / 16;
    const uint4* p = reinterpret_cast<const uint4*>(row + c);
#pragma unroll
    for (int i = 0; i < W; ++i) reinterpret_cast<uint4*>(v)[i] = p[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = c + i < K ? row[c + i] : from_float<T>(0.0f);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_cols(T* row, int c, int K, bool vec, const T (&v)[N]) {
  if (vec && c + N <= K) {
    constexpr int W = N * (int)sizeof(T) / 16;
    uint4* p = reinterpret_cast<uint4*>(row + c);
#pragma unroll
    for (int i = 0; i < W; ++i) p[i] = reinterpret_cast<const uint4*>(v)[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i < K) row[c + i] = v[i];
  }
}

// Rows of a matrix start on 16-byte boundaries.
inline bool rows_aligned16(const void* p, int64_t ld, int elem_bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * elem_bytes) % 16 == 0;
}
inline int dtype_bytes(int dtype) { return dtype == SVDQ_FP32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == SVDQ_BF16 || dtype == SVDQ_FP16 || dtype == SVDQ_FP32; }
inline bool mx_format_ok(int fmt) { return fmt == kNvfp4 || fmt == kMxfp4 || fmt == kMxfp8; }

// A launch that may begin while the launch before it on the stream drains (its kernel waits with
// pdl_wait before it touches memory).
template <typename... P, typename... A>
inline int launch_pdl(const char* what, void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                      int cluster, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return check_cuda(e, what);
  }
  return SVDQ_OK;
}

}  // namespace svdq

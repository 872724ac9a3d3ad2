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

// The correctly rounded quotient q = x / h, moved to odd: where x / (h + l) is not exactly q, the
// neighbour of q on its side, or q itself, whose last bit is set.  Rounding that to a type with at
// least two bits fewer gives the rounding of the exact quotient.
__device__ __forceinline__ float to_odd(float q, float x, float h, float l) {
  const float r = fmaf(-q, l, fmaf(-q, h, x));  // x - q (h + l): the inner difference is exact
  const uint32_t u = __float_as_uint(q);
  const int side = ((int)(__float_as_uint(r) ^ u) >> 31) | 1;  // the exact quotient is larger (1) or smaller (-1)
  return r != 0.0f && (u & 1u) == 0u ? __uint_as_float(u + (uint32_t)side) : q;
}
// x / h, correctly rounded, from y = the rounded reciprocal of h (P. Markstein, IBM J. R&D 34(1), 1990),
// while neither h, x nor the quotient is near the ends of fp32's range.
__device__ __forceinline__ float quotient(float x, float h, float y) {
  const float q = x * y;
  return fmaf(fmaf(-q, h, x), y, q);
}

// nvfp4 scale byte: e4m3(amax / (6 g)) of the exact quotient, through a quotient rounded to odd (in 64
// bits at the ends of the range).  NaN (0x7F) where amax is not finite or the tensor scale is not a
// positive number.
__device__ __forceinline__ uint32_t nvfp4_scale_byte(uint32_t amax_bits, float g) {
  const float amax = __uint_as_float(amax_bits);
  const float h = 6.0f * g, l = fmaf(6.0f, g, -h);
  float t;
  if (h >= 1.0e-25f && h <= 1.0e25f && amax <= h * 65536.0f) {
    t = to_odd(quotient(amax, h, __frcp_rn(h)), amax, h, l);
  } else {
    const double d = (double)amax / (6.0 * (double)g);
    if (!(amax_bits < 0x7F800000u && g > 0.0f && __float_as_uint(g) < 0x7F800000u)) return 0x7Fu;
    t = __double2float_rz(d);
    if ((double)t != d) t = __uint_as_float(__float_as_uint(t) | 1u);
  }
  return e4m3x2_satfinite(t, 0.0f) & 0xFFu;
}
// e2m1 code of q, ties to even, from comparisons.
__device__ __forceinline__ uint32_t e2m1_of(double q) {
  const double a = fabs(q);
  const uint32_t c = (a > 0.25) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0);
  return c | (signbit(q) ? 8u : 0u);
}
// An nvfp4 block whose scale or values are near the ends of fp32's range, in 64 bits.
static __device__ __noinline__ uint2 nvfp4_codes_wide(const float* x, float sf, float g) {
  const double d = (double)sf * (double)g;
  uint32_t w[2] = {0u, 0u};
#pragma unroll 1
  for (int i = 0; i < 16; ++i) w[i >> 3] |= e2m1_of((double)x[i] / d) << (4 * (i & 7));
  return make_uint2(w[0], w[1]);
}
// 16 values of an nvfp4 block as codes e2m1(x / (sf g)) of the exact quotient.  d = fl32(sf g) and x / d
// is formed correctly rounded.  That decides every code unless the rounded quotient lands on a
// border between two codes without being there: impossible when d = sf g has at most 16
// significant bits and x at most 11 (x - border * d is then zero or above 2^-19 of x).  Otherwise a
// block with a quotient of at most 3 significant bits, as borders are, moves its quotients to odd.
// Takes -x: with q0 = (-x)(-y), r = q0 d - x and q = q0 - r y a zero keeps its sign.
template <bool SHORT_X>
__device__ __forceinline__ uint2 nvfp4_codes(const float (&nx)[16], uint32_t amax_bits, uint32_t sf_byte, float g) {
  const float sf = e4m3_value(sf_byte);
  if (sf_byte == 0u || sf_byte == 0x7Fu) return make_uint2(0u, 0u);
  const float d = sf * g;
  const float dl = fmaf(sf, g, -d);
  if (!(d >= 8.0e-28f && d <= 1.0e30f && __uint_as_float(amax_bits) <= d * 65536.0f)) {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = -nx[i];
    return nvfp4_codes_wide(v, sf, g);
  }
  const float y = __frcp_rn(d);
  const uint64_t ny = f2_pack(-y, -y), dd = f2_pack(d, d);
  float q[16];
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const uint64_t xx = f2_pack(nx[i], nx[i + 1]);
    const uint64_t q0 = f2_mul(xx, ny);
    const uint64_t qq = f2_fma(f2_fma(q0, dd, xx), ny, q0);
    q[i] = f2_lo(qq);
    q[i + 1] = f2_hi(qq);
  }
  if (!SHORT_X || dl != 0.0f || (__float_as_uint(d) & 0xFFu) != 0u) {
    bool near_border = false;
#pragma unroll
    for (int i = 0; i < 16; ++i) near_border |= (__float_as_uint(q[i]) & 0x1FFFFFu) == 0u;
    if (near_border) {
#pragma unroll
      for (int i = 0; i < 16; ++i) q[i] = to_odd(q[i], -nx[i], d, dl);
    }
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

// Bits of the largest magnitude of N values; a NaN is larger than every number.
template <int N>
__device__ __forceinline__ uint32_t amax_bits_of(const float (&v)[N]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(m), "f"(fabsf(v[i])));
  return __float_as_uint(m);
}

// N values of a row from column c (N elements are 16, 32 or 64 bytes) where all of them exist and the
// row is aligned to them (up to 32 bytes).
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, T (&v)[N]) {
  constexpr int kBytes = N * (int)sizeof(T);
  if constexpr (kBytes % 32 == 0) {
#pragma unroll
    for (int i = 0; i < kBytes / 32; ++i) {
      uint32_t* w = reinterpret_cast<uint32_t*>(v) + 8 * i;
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(reinterpret_cast<const uint8_t*>(p) + 32 * i)
                   : "memory");
    }
  } else {
    *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const T (&v)[N]) {
  constexpr int kBytes = N * (int)sizeof(T);
  if constexpr (kBytes % 32 == 0) {
#pragma unroll
    for (int i = 0; i < kBytes / 32; ++i) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(v) + 8 * i;
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<uint8_t*>(p) + 32 * i),
                   "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                   : "memory");
    }
  } else {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
  }
}
// The same for rows that are not aligned or end inside: lane l of the warp owns columns c .. c + N - 1
// of the row at `row`, and the warp goes over all of its elements 32 at a time, neighbouring lanes at
// neighbouring columns, through `stage` (32 N elements of shared memory of this warp, 16-byte
// aligned).  Columns from K on read as zero and are not written.  Every lane takes part.
template <typename T, int N>
__device__ __forceinline__ void load_warp(const T* row, int c, int K, T* stage, T (&v)[N]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int e = j * 32 + lane;
    const T* p = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), e / N));
    const int col = __shfl_sync(0xffffffffu, c, e / N) + e % N;
    stage[e] = col < K ? p[col] : from_float<T>(0.0f);
  }
  __syncwarp();
  constexpr int W = N * (int)sizeof(T) / 16;
#pragma unroll
  for (int i = 0; i < W; ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(stage + lane * N)[i];
  __syncwarp();
}
template <typename T, int N>
__device__ __forceinline__ void store_warp(T* row, int c, int K, T* stage, const T (&v)[N]) {
  const int lane = threadIdx.x & 31;
  constexpr int W = N * (int)sizeof(T) / 16;
#pragma unroll
  for (int i = 0; i < W; ++i) reinterpret_cast<uint4*>(stage + lane * N)[i] = reinterpret_cast<const uint4*>(v)[i];
  __syncwarp();
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int e = j * 32 + lane;
    T* p = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), e / N));
    const int col = __shfl_sync(0xffffffffu, c, e / N) + e % N;
    if (col < K) p[col] = stage[e];
  }
  __syncwarp();
}

// Rows of a matrix start on boundaries of `align` bytes.
inline bool rows_aligned(const void* p, int64_t ld, int elem_bytes, int align) {
  return reinterpret_cast<uintptr_t>(p) % align == 0 && (ld * elem_bytes) % align == 0;
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

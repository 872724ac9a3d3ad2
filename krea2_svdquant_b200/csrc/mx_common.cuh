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

// A quotient q within a hair more than half a step of x / (h + l), moved to odd: where x / (h + l) is not exactly
// q, the neighbour of q on its side, or q itself, whose last bit is set.  Rounding that to a type with at
// least two bits fewer gives the rounding of the exact quotient.
__device__ __forceinline__ float to_odd(float q, float x, float h, float l) {
  const float r = fmaf(-q, l, fmaf(-q, h, x));  // x - q (h + l): the inner difference is exact
  const uint32_t u = __float_as_uint(q);
  const int side = ((int)(__float_as_uint(r) ^ u) >> 31) | 1;  // the exact quotient is larger (1) or smaller (-1)
  return r != 0.0f && (u & 1u) == 0u ? __uint_as_float(u + (uint32_t)side) : q;
}
// Such a quotient from y = the rounded reciprocal of h (P. Markstein, IBM J. R&D 34(1), 1990), with the
// divisor's rest l in the correction: x / h alone, correctly rounded, can be a step and a half from x / (h + l), on
// the other side of a border.  While neither h, x nor the quotient is near the ends of fp32's range.
__device__ __forceinline__ float quotient(float x, float h, float l, float y) {
  const float q = x * y;
  return fmaf(fmaf(-q, l, fmaf(-q, h, x)), y, q);
}

// nvfp4 scale byte: e4m3(amax / (6 g)) of the exact quotient, through a quotient rounded to odd (in 64
// bits at the ends of the range).  NaN (0x7F) where amax is not finite or the tensor scale is not a
// positive number.
__device__ __forceinline__ uint32_t nvfp4_scale_byte(uint32_t amax_bits, float g) {
  const float amax = __uint_as_float(amax_bits);
  const float h = 6.0f * g, l = fmaf(6.0f, g, -h);
  float t;
  if (h >= 1.0e-25f && h <= 1.0e25f && amax <= h * 65536.0f) {
    t = to_odd(quotient(amax, h, l, __frcp_rn(h)), amax, h, l);
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
// An nvfp4 block whose scale or values are near the ends of fp32's range, in 64 bits.  Rare: one element
// at a time, picked out of registers, so that it costs the usual path neither registers nor a stack.
__device__ __forceinline__ uint2 nvfp4_codes_wide(const float (&x)[16], float sf, float g) {
  const double d = (double)sf * (double)g;
  uint2 w = make_uint2(0u, 0u);
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    float v = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j == i) v = x[j];
    const uint32_t c = e2m1_of((double)v / d) << (4 * (i & 7));
    if (i < 8) w.x |= c;
    else w.y |= c;
  }
  return w;
}

// What the quotients of an nvfp4 block need, by its scale byte.  A launch has one tensor scale g, so a
// CTA works this out once per byte.
enum : uint32_t { kTimesY = 0, kQuotient = 1, kQuotientOdd = 2 };
struct Nvfp4Unit {
  float d;        // fl32(sf g)
  float y;        // kTimesY: the factor that stands for 1 / (sf g); otherwise 1 / d, rounded
  float limit;    // magnitudes up to this take fp32 (below 0: none)
  uint32_t how;
};

// Codes are e2m1(x / (sf g)) of the exact quotient, ties to even.  For x of P significant bits (8 in
// bf16, 11 in fp16) few x matter: a border b between two codes has the significand m / 4, m = 4 .. 7,
// and only x_m 2^k, x_m = m sf g rounded to P bits, can come close to b sf g.  All x_m 2^k of one m lie on
// the same side of their borders, and where they lie on them, ties to even go down for m = 4 and 5
// and up for 6 and 7.  So where the x_m that come within 2^-20 of their borders all want one side, and the
// others keep 2^-17 away, x times the reciprocal of sf g moved by 2^-19 to that side decides every
// code (its rounding errors are below 2^-22).  Otherwise the correctly rounded quotient x / d does,
// unless d is not sf g or an x_m is close to its border without being on it; then, and for fp32 (P = 24),
// quotients that have at most 3 significant bits, as borders do, are moved to odd one by one.
// (Sides matter often: g = amax / 2688 = amax / (7 * 384) with a short amax brings every 7 sf g next to
// a short number, and g = 1 puts every x_m on its border.  4352 x 6144 bf16: 16.5 us with one product,
// 18.0 with the quotient.)
template <int P>
__device__ __forceinline__ Nvfp4Unit nvfp4_unit(uint32_t byte, float g) {
  const float sf = e4m3_value(byte);
  const float d = sf * g, dl = fmaf(sf, g, -d);
  Nvfp4Unit u{d, 0.0f, -1.0f, kQuotientOdd};
  if (!(d >= 8.0e-28f && d <= 1.0e30f)) return u;  // 64 bits
  u.limit = d * 65536.0f;
  u.y = __frcp_rn(d);
  if constexpr (P < 24) {
    bool up = false, down = false, between = false, beside = dl != 0.0f;
#pragma unroll
    for (int m = 4; m <= 7; ++m) {
      constexpr uint32_t drop = 24 - P;
      const float xm = __uint_as_float((__float_as_uint((float)m * d) + (1u << (drop - 1))) & ~((1u << drop) - 1u));
      const float delta = fmaf((float)m, d, -xm) + (float)m * dl;
      const float off = fabsf(delta);
      if (off < xm * 0x1p-20f) {
        const bool to_down = delta != 0.0f ? delta > 0.0f : m < 6;
        up |= !to_down;
        down |= to_down;
        beside |= delta != 0.0f;
      } else {
        between |= off < xm * 0x1p-17f;
      }
    }
    if (!(up && down) && !((up || down) && between)) {
      u.how = kTimesY;
      if (up) u.y *= 1.0f + 0x1p-19f;
      if (down) u.y *= 1.0f - 0x1p-19f;
    } else if (!beside) {
      u.how = kQuotient;
    }
  }
  return u;
}

// 16 values of an nvfp4 block as codes.
__device__ __forceinline__ uint2 nvfp4_codes(const float (&x)[16], uint32_t amax_bits, uint32_t byte,
                                             const Nvfp4Unit& u, float g) {
  if (byte == 0u || byte == 0x7Fu) return make_uint2(0u, 0u);
  if (!(__uint_as_float(amax_bits) <= u.limit)) return nvfp4_codes_wide(x, e4m3_value(byte), g);
  float q[16];
  if (u.how == kTimesY) {
    const uint64_t yy = f2_pack(u.y, u.y);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const uint64_t p = f2_mul(f2_pack(x[i], x[i + 1]), yy);
      q[i] = f2_lo(p);
      q[i + 1] = f2_hi(p);
    }
  } else {
    // Markstein's correction with -x: q0 = (-x)(-y), r = q0 (d + dl) - x, q = q0 - r y, so that a zero keeps its sign
    const float dl = fmaf(e4m3_value(byte), g, -u.d);
    const uint64_t ny = f2_pack(-u.y, -u.y), dd = f2_pack(u.d, u.d), ll = f2_pack(dl, dl);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const uint64_t xx = f2_pack(-x[i], -x[i + 1]);
      const uint64_t q0 = f2_mul(xx, ny);
      const uint64_t p = f2_fma(f2_fma(q0, ll, f2_fma(q0, dd, xx)), ny, q0);
      q[i] = f2_lo(p);
      q[i + 1] = f2_hi(p);
    }
    if (u.how == kQuotientOdd) {
      bool near_border = false;
#pragma unroll
      for (int i = 0; i < 16; ++i) near_border |= (__float_as_uint(q[i]) & 0x1FFFFFu) == 0u;
      if (near_border) {
#pragma unroll
        for (int i = 0; i < 16; ++i) q[i] = to_odd(q[i], x[i], u.d, dl);
      }
    }
  }
  return make_uint2(e2m1x8_satfinite(q), e2m1x8_satfinite(q + 8));
}

// Multiplies by a power of two (an mx block's 2^-e), two values an instruction.
template <int N>
__device__ __forceinline__ void scale_all(float (&v)[N], float f) {
  const uint64_t ff = f2_pack(f, f);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const uint64_t p = f2_mul(f2_pack(v[i], v[i + 1]), ff);
    v[i] = f2_lo(p);
    v[i + 1] = f2_hi(p);
  }
}
template <int N>
__device__ __forceinline__ void e4m3_words(const float (&v)[N], uint32_t (&w)[N / 4]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    w[i] = e4m3x2_satfinite(v[4 * i], v[4 * i + 1]) | e4m3x2_satfinite(v[4 * i + 2], v[4 * i + 3]) << 16;
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

// Bits (fp32) of the largest magnitude of N values; a NaN is larger than every number.
template <int N>
__device__ __forceinline__ uint32_t amax_bits_of(const float (&v)[N]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(m), "f"(fabsf(v[i])));
  return __float_as_uint(m);
}
template <int N>
__device__ __forceinline__ uint32_t amax_bits_of(const __nv_bfloat16 (&v)[N]) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(v);
  __nv_bfloat162 m = __habs2(p[0]);
#pragma unroll
  for (int i = 1; i < N / 2; ++i) m = __hmax2_nan(m, __habs2(p[i]));
  return __float_as_uint(__bfloat162float(__hmax_nan(m.x, m.y)));
}
template <int N>
__device__ __forceinline__ uint32_t amax_bits_of(const __half (&v)[N]) {
  const __half2* p = reinterpret_cast<const __half2*>(v);
  __half2 m = __habs2(p[0]);
#pragma unroll
  for (int i = 1; i < N / 2; ++i) m = __hmax2_nan(m, __habs2(p[i]));
  return __float_as_uint(__half2float(__hmax_nan(__low2half(m), __high2half(m))));
}
template <typename T>
__host__ __device__ constexpr int significant_bits();
template <>
constexpr int significant_bits<float>() { return 24; }
template <>
constexpr int significant_bits<__half>() { return 11; }
template <>
constexpr int significant_bits<__nv_bfloat16>() { return 8; }

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
// The same for a row of any alignment that may end inside: columns from K on are zero.  Reads the
// aligned 16-byte words that hold a byte of the row (so never a word that is not partly the row's), one
// more than aligned columns take, and shifts.  A row's shift is the same for all its columns.
template <typename T, int N>
__device__ __forceinline__ void load_shifted(const T* row, int c, int K, T (&v)[N]) {
  constexpr int kWords = N * (int)sizeof(T) / 4;
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + c), end = reinterpret_cast<uintptr_t>(row + K);
  const uintptr_t first = at & ~(uintptr_t)15;
  uint32_t w[kWords + 4];
#pragma unroll
  for (int i = 0; i <= kWords / 4; ++i) {
    uint4 q = make_uint4(0u, 0u, 0u, 0u);
    if (c < K && first + 16 * i < end) q = *reinterpret_cast<const uint4*>(first + 16 * i);
    w[4 * i] = q.x;
    w[4 * i + 1] = q.y;
    w[4 * i + 2] = q.z;
    w[4 * i + 3] = q.w;
  }
  const uint32_t shift = (uint32_t)(at & 15);
  if (shift & 8) {
#pragma unroll
    for (int i = 0; i < kWords + 2; ++i) w[i] = w[i + 2];
  }
  if (shift & 4) {
#pragma unroll
    for (int i = 0; i < kWords + 1; ++i) w[i] = w[i + 1];
  }
  uint32_t* out = reinterpret_cast<uint32_t*>(v);
#pragma unroll
  for (int i = 0; i < kWords; ++i) out[i] = sizeof(T) == 4 ? w[i] : __funnelshift_r(w[i], w[i + 1], 8 * (shift & 2));
  if (c + N > K) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i >= K) v[i] = from_float<T>(0.0f);
  }
}
// The way back, by a warp whose lane l has columns c .. c + N - 1 of the row at `row`: the warp writes
// its elements 32 at a time, neighbouring lanes at neighbouring columns, through `stage` (32 N
// elements of shared memory of this warp, 16-byte aligned).  Columns from K on are not written.
// Every lane takes part.
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

// 16 codes: 8 bytes of 4-bit ones or 16 of 8-bit ones.
template <int FMT>
struct CodeWord {
  using type = uint2;
};
template <>
struct CodeWord<kMxfp8> {
  using type = uint4;
};

// The codes of 16 columns of an mx block from its scale byte.
template <typename T, int FMT>
__device__ __forceinline__ typename CodeWord<FMT>::type mx_codes(const T (&x)[16], uint32_t byte) {
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = to_float(x[i]);
  if (byte == 255u) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.0f;
  }
  scale_all(v, mx_inverse_scale(byte));
  if constexpr (FMT == kMxfp4) {
    return make_uint2(e2m1x8_satfinite(v), e2m1x8_satfinite(v + 8));
  } else {
    uint32_t w[4];
    e4m3_words(v, w);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// The codes of 16 columns and their block's scale byte.  An mx block is shared with
// the neighbouring lane (lane ^ 1), so every lane of the warp takes part.
template <typename T, int FMT>
__device__ __forceinline__ typename CodeWord<FMT>::type encode_chunk(const T (&x)[16], float g, const Nvfp4Unit* units,
                                                                     uint32_t& byte) {
  uint32_t amax = amax_bits_of(x);
  if constexpr (FMT == kNvfp4) {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = to_float(x[i]);
    byte = nvfp4_scale_byte(amax, g);
    return nvfp4_codes(v, amax, byte, units[byte], g);
  } else {
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    byte = mx_scale_byte<FMT>(amax);
    return mx_codes<T, FMT>(x, byte);
  }
}
// The four scale bytes of a word, from the 4 (nvfp4) or 8 (mx) neighbouring lanes that have them.
template <int FMT>
__device__ __forceinline__ uint32_t scale_word(uint32_t byte) {
  constexpr int kStep = FMT == kNvfp4 ? 1 : 2;  // lanes per block
  uint32_t word = byte << (8 * (((threadIdx.x & 31) / kStep) & 3));
  word |= __shfl_xor_sync(0xffffffffu, word, kStep);
  word |= __shfl_xor_sync(0xffffffffu, word, 2 * kStep);
  return word;
}

// Rows of a matrix start on boundaries of `align` bytes.
inline bool rows_aligned(const void* p, int64_t ld, int elem_bytes, int align) {
  return reinterpret_cast<uintptr_t>(p) % align == 0 && (ld * elem_bytes) % align == 0;
}
inline bool element_aligned(const void* p, int elem_bytes) { return reinterpret_cast<uintptr_t>(p) % elem_bytes == 0; }
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

// Root-mean-square norm with the residual's addition, written as mxfp8 (e4m3 codes, a power-of-two
// scale per 32 columns):
//   h = x + residual, rounded to its type and stored;   y = h * rsqrt(mean(h^2) + eps) * weight
//   scale = 2^(floor(log2 max|y|) - 8) per 32 columns,  code = e4m3(y / scale)
// The norm reads h as it is stored, so a residual stream read back later gives the same norm.
//
// Codes and scales are those of the exact y.  In fp32 y comes out within 7 2^-24 of it (relative), which
// decides every code but those with a border between y (1 - 2^-21) and y (1 + 2^-21), one in 10^5, and
// every scale but those whose largest y is that near a power of two.  Where a warp meets one, the CTA sums
// the row again in 64 bits and the warp works those columns out again from there.  So it does where fp32
// does not hold the squares, the root or h * weight: rows far from one, up to the ends of the type's
// range (a y past fp32's own is an infinity).  At 4352 x 6144 bf16 7% of the rows come to that, and all of it
// costs 1.5 us of 32.4 with a residual, 5 of 21.7 without (against y rounded to fp32 and then to its code).
#include "mx_common.cuh"

namespace svdq {
namespace {

struct NormArgs {
  const void* x;
  int64_t ldx;
  const void* residual;
  int64_t ldr;
  const void* weight;
  float eps;
  double per_column;  // 1 / H
  int M, H, h_pad;
  uint8_t* codes;
  uint8_t* scales;
  void* sum;
  int64_t lds;
};

constexpr float kNear = 0x1p-21f;

// d rounded to fp32, moved to odd: where fp32 does not hold d and the nearest value is even, the one on its
// other side.  Rounding that again, to at most 22 bits, gives the rounding of d.  Within 2^-46 d is taken for
// the fp32 value itself, so that a y that lies on a border (a row of equal elements, eps 0) is not moved
// off it by its last bits.
__device__ __forceinline__ float float_to_odd(double d) {
  const float f = __double2float_rn(d);
  const double r = d - (double)f;
  const uint32_t u = __float_as_uint(f);
  if ((u & 1u) != 0u || !(fabsf(f) < INFINITY) || !(fabs(r) > 0x1p-46 * fabs(d))) return f;
  return __uint_as_float((r > 0.0) == (d > 0.0) ? u + 1u : u - 1u);
}

// C = 32 bytes of a row's columns; zero from column H on.
template <bool VEC, typename T, int C>
__device__ __forceinline__ void load_columns(const T* row, int c, int H, T (&v)[C]) {
  if constexpr (!VEC) {
    load_shifted(row, c, H, v);
  } else if (c < H) {
    load_vec(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = from_float<T>(0.0f);
  }
}
// Bits of the largest magnitude of an mx block, from the 32 / C neighbouring lanes that have it.
template <int C>
__device__ __forceinline__ uint32_t block_max(const float (&y)[C]) {
  uint32_t amax = amax_bits_of(y);
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  if (C == 8) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  return amax;
}
template <int W>
__device__ __forceinline__ void store_codes(const NormArgs& a, int row, int c, const uint32_t (&q)[W], uint32_t byte) {
  constexpr int L = 8 / W;  // lanes per block
  const int lane = threadIdx.x & 31, words = a.h_pad / 128;
  uint32_t word = byte << (8 * ((lane / L) & 3));
  word |= __shfl_xor_sync(0xffffffffu, word, L);
  word |= __shfl_xor_sync(0xffffffffu, word, 2 * L);
  if (c < a.h_pad) {
    uint8_t* to = a.codes + (size_t)row * a.h_pad + c;
    if constexpr (W == 4) *reinterpret_cast<uint4*>(to) = make_uint4(q[0], q[1], q[2], q[3]);
    else *reinterpret_cast<uint2*>(to) = make_uint2(q[0], q[1]);
    if (lane % (4 * L) == 0) *reinterpret_cast<uint32_t*>(a.scales + mx_scale_word(row, c >> 7, words)) = word;
  }
}

// The codes of a warp's columns (c is the lane's) in 64 bits, from the row as it is stored.
template <typename T, bool VEC>
__device__ __forceinline__ void encode_exactly(const NormArgs& a, int row, const T* h_row, int c, double root) {
  constexpr int C = 32 / (int)sizeof(T);
  alignas(32) T h[C], w[C];
  load_columns<VEC>(h_row, c, a.H, h);
  if (a.weight) load_columns<VEC>(static_cast<const T*>(a.weight), c, a.H, w);
  if (c >= a.H) root = 0.0;  // a row's root can be infinite or NaN, the blocks that pad it hold zeros all the same
  float y[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    double d = (double)to_float(h[i]);
    if (a.weight) d *= (double)to_float(w[i]);
    y[i] = float_to_odd(d * root);
  }
  const uint32_t byte = mx_scale_byte<kMxfp8>(block_max(y));
  if (byte == 255u) {
#pragma unroll
    for (int i = 0; i < C; ++i) y[i] = 0.0f;
  }
  scale_all(y, mx_inverse_scale(byte));
  uint32_t q[C / 4];
  e4m3_words(y, q);
  store_codes(a, row, c, q, byte);
}

// One CTA per row.  A thread owns C columns of each C * THREADS (C = 16, or 8 in fp32: 32 bytes); the
// 32 / C neighbouring lanes of an mx block share its scale.  The row stays in registers between the
// two steps (the sum of squares, then the codes) for up to PASSES * C * THREADS columns; PASSES == 0
// reads it again instead.  Bound by HBM: 6 bytes read or written as bf16 and 1.03 as codes per
// element with a residual (4352 x 6144 bf16: 32.4 us, 5.8 TB/s; without one 21.7 us, 3.7 TB/s, where the
// instructions count for more).
template <typename T, int THREADS, int PASSES, bool VEC>
__global__ void __launch_bounds__(THREADS) rms_norm_mx_kernel(const NormArgs a) {
  constexpr int C = 32 / (int)sizeof(T);
  constexpr int kKeep = PASSES > 0 ? PASSES : 1;
  __shared__ double part[THREADS / 32];
  __shared__ __align__(16) T stage[VEC ? 1 : THREADS * C];
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  const int words = a.h_pad / 128;
  if (row >= a.M) {  // rows that only fill a tile of scales
    for (int w = tid; w < words; w += THREADS) *reinterpret_cast<uint32_t*>(a.scales + mx_scale_word(row, w, words)) = 0u;
    return;
  }
  const T* xr = static_cast<const T*>(a.x) + (size_t)row * a.ldx;
  const T* rr = a.residual ? static_cast<const T*>(a.residual) + (size_t)row * a.ldr : nullptr;
  T* sr = a.sum ? static_cast<T*>(a.sum) + (size_t)row * a.lds : nullptr;
  const T* weight = static_cast<const T*>(a.weight);
  const int passes = PASSES > 0 ? PASSES : (a.h_pad + C * THREADS - 1) / (C * THREADS);
  auto column = [&](int p) { return (p * THREADS + tid) * C; };
  auto load = [&](const T* p, int c, T (&v)[C]) { load_columns<VEC>(p, c, a.H, v); };
  alignas(32) T keep[kKeep][C];
  alignas(32) T res[kKeep][C];
  double ss = 0.0;
  auto pass_bit = [](int p) { return 1u << (PASSES > 0 || p < 31 ? p : 31); };  // the last one is of all the rest
  uint32_t some = 0;  // passes of which this thread has an element that is not zero
  auto add = [&](int p, T (&h)[C], const T (&r)[C]) {
    const int c = column(p);
    if (rr) {
#pragma unroll
      for (int i = 0; i < C; ++i) h[i] = from_float<T>(to_float(h[i]) + to_float(r[i]));
      if constexpr (!VEC) store_warp(sr, c, a.H, stage + (tid & ~31) * C, h);
      else if (c < a.H) store_vec(sr + c, h);
    }
    uint64_t s2[2] = {0, 0};  // C / 4 squares each, and 64 bits from there on: off by (C / 4 + 1) 2^-24 at most
#pragma unroll
    for (int i = 0; i < C; i += 2) {
      const uint64_t v = f2_pack(to_float(h[i]), to_float(h[i + 1]));
      s2[i / 2 % 2] = f2_fma(v, v, s2[i / 2 % 2]);
    }
    const uint64_t both = f2_add(s2[0], s2[1]);
    ss += (double)f2_lo(both) + (double)f2_hi(both);
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) bits |= reinterpret_cast<const uint32_t*>(h)[i];
    some |= (bits & (sizeof(T) == 2 ? 0x7FFF7FFFu : 0x7FFFFFFFu)) != 0u ? pass_bit(p) : 0u;
  };
  if constexpr (PASSES > 0) {  // every load first
#pragma unroll
    for (int p = 0; p < PASSES; ++p) load(xr, column(p), keep[p]);
    if (rr) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) load(rr, column(p), res[p]);
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) add(p, keep[p], res[p]);
  } else {
    for (int p = 0; p < passes; ++p) {
      load(xr, column(p), keep[0]);
      if (rr) load(rr, column(p), res[0]);
      add(p, keep[0], res[0]);
    }
  }
  auto over_row = [&](double t) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) part[tid >> 5] = t;
    __syncthreads();
    t = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) t += part[w];
    return t;
  };
  // Between 2^-60 and 2^60 no square was infinite, and what those below fp32's normal range lost does not count.
  const double v = fma(over_row(ss), a.per_column, (double)a.eps);
  const bool near_one = v >= 0x1p-60 && v <= 0x1p60;
  const float root = near_one ? 1.0f / sqrtf((float)v) : 1.0f;
  const uint64_t root2 = f2_pack(root, root);

  // In fp32.  The pass's bit where a code or the scale is not certain.
  auto encode = [&](int p, const T (&h)[C]) {
    const int c = column(p);
    alignas(32) T w[C];
    if (weight) load(weight, c, w);
    float y[C], z[C];
#pragma unroll
    for (int i = 0; i < C; i += 2) {
      uint64_t v2 = f2_pack(to_float(h[i]), to_float(h[i + 1]));
      if (weight) v2 = f2_mul(v2, f2_pack(to_float(w[i]), to_float(w[i + 1])));
      v2 = f2_mul(v2, root2);
      y[i] = z[i] = f2_lo(v2);
      y[i + 1] = z[i + 1] = f2_hi(v2);
    }
    const uint32_t amax = block_max(y);
    // From 2^-60 on a block's codes do not see what an h * weight below fp32's normal range lost (2^-150; in y
    // 2^-120); an infinite one, or a NaN, shows in amax.
    const bool unsure = !near_one || amax >= 0x7F800000u || (amax < 0x21800000u && (some & pass_bit(p)) != 0u) ||
                  ((amax + 8u) ^ (amax - 8u)) >> 23 != 0u && amax != 0u;
    const uint32_t byte = mx_scale_byte<kMxfp8>(amax);
    const float f = mx_inverse_scale(byte);
    uint32_t q[C / 4], r[C / 4];
    scale_all(y, f * (1.0f + kNear));
    scale_all(z, f * (1.0f - kNear));
    e4m3_words(y, q);
    e4m3_words(z, r);
    uint32_t differ = 0;
#pragma unroll
    for (int i = 0; i < C / 4; ++i) differ |= q[i] ^ r[i];
    store_codes(a, row, c, q, byte);
    return unsure || differ != 0u ? pass_bit(p) : 0u;
  };
  const T* h_row = sr ? sr : xr;  // the sums as this warp stored them
  uint32_t again = 0;             // passes that the warp works out again
  if constexpr (PASSES > 0) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) again |= encode(p, keep[p]);
  } else {
    for (int p = 0; p < passes; ++p) {
      if constexpr (!VEC) __syncwarp();
      load(h_row, column(p), keep[0]);
      again |= encode(p, keep[0]);
    }
  }
  again = __reduce_or_sync(0xffffffffu, again);
  if (!__syncthreads_or((int)again)) return;
  double t[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 1
  for (int p = 0; p < passes; ++p) {
    alignas(32) T h[C];
    load(h_row, column(p), h);
#pragma unroll
    for (int i = 0; i < C; ++i) t[i & 3] = fma((double)to_float(h[i]), (double)to_float(h[i]), t[i & 3]);
  }
  const double exact = 1.0 / sqrt(fma(over_row((t[0] + t[1]) + (t[2] + t[3])), a.per_column, (double)a.eps));
#pragma unroll 1
  for (int p = 0; p < passes; ++p)
    if (again & pass_bit(p)) encode_exactly<T, VEC>(a, row, h_row, column(p), exact);
}

template <typename T, bool VEC>
int launch_norm(const NormArgs& a, cudaStream_t stream) {
  constexpr int C = 32 / (int)sizeof(T);
  const dim3 grid(mx_rows_pad(a.M));
  const char* what = "svdq_rms_norm_mx launch";
  const int chunks = a.h_pad / C;
  if (chunks <= 128) return launch_pdl(what, rms_norm_mx_kernel<T, 128, 1, VEC>, grid, dim3(128), 0, stream, 1, a);
  if (chunks <= 256) return launch_pdl(what, rms_norm_mx_kernel<T, 128, 2, VEC>, grid, dim3(128), 0, stream, 1, a);
  if (chunks <= 384 && sizeof(T) == 2)  // three passes of fp32 do not fit the registers
    return launch_pdl(what, rms_norm_mx_kernel<T, 128, 3, VEC>, grid, dim3(128), 0, stream, 1, a);
  if (chunks <= 512) return launch_pdl(what, rms_norm_mx_kernel<T, 256, 2, VEC>, grid, dim3(256), 0, stream, 1, a);
  if (chunks <= 768) return launch_pdl(what, rms_norm_mx_kernel<T, 256, 3, VEC>, grid, dim3(256), 0, stream, 1, a);
  if (chunks <= 1024) return launch_pdl(what, rms_norm_mx_kernel<T, 256, 4, VEC>, grid, dim3(256), 0, stream, 1, a);
  if (chunks <= 2048) return launch_pdl(what, rms_norm_mx_kernel<T, 512, 4, VEC>, grid, dim3(512), 0, stream, 1, a);
  return launch_pdl(what, rms_norm_mx_kernel<T, 512, 0, VEC>, grid, dim3(512), 0, stream, 1, a);
}

}  // namespace
}  // namespace svdq

extern "C" int svdq_rms_norm_mx(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
                                int dtype, float eps, int M, int H, void* codes, void* scales, void* sum, int64_t lds,
                                cudaStream_t stream) {
  using namespace svdq;
  SVDQ_REQUIRE(dtype_ok(dtype), "svdq_rms_norm_mx: x must be bf16, fp16 or fp32");
  SVDQ_REQUIRE(M >= 0 && H > 0 && ldx >= H, "svdq_rms_norm_mx: bad M/H/ldx");
  SVDQ_REQUIRE(eps >= 0.0f, "svdq_rms_norm_mx: eps must not be negative");
  SVDQ_REQUIRE((residual == nullptr) == (sum == nullptr), "svdq_rms_norm_mx: residual and sum go together");
  SVDQ_REQUIRE(residual == nullptr || (ldr >= H && lds >= H), "svdq_rms_norm_mx: bad ldr/lds");
  if (M == 0) return SVDQ_OK;
  SVDQ_REQUIRE(x && codes && scales, "svdq_rms_norm_mx: null pointer");
  SVDQ_REQUIRE(((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15u) == 0,
               "svdq_rms_norm_mx: codes and scales must be 16-byte aligned");
  const int elem = dtype_bytes(dtype);
  SVDQ_REQUIRE(element_aligned(x, elem) && element_aligned(residual, elem) && element_aligned(weight, elem) &&
                   element_aligned(sum, elem),
               "svdq_rms_norm_mx: x, residual, weight and sum must be aligned to their elements");
  if (M > (1 << 30) || H > (1 << 30)) return set_error(SVDQ_ERR_UNSUPPORTED, "svdq_rms_norm_mx: matrix too large");
  NormArgs a{};
  a.x = x;
  a.ldx = ldx;
  a.residual = residual;
  a.ldr = ldr;
  a.weight = weight;
  a.eps = eps;
  a.per_column = 1.0 / H;
  a.M = M;
  a.H = H;
  a.h_pad = mx_k_pad(H);
  const bool vec = H % (32 / elem) == 0 && rows_aligned(x, ldx, elem, 32) &&
                   (!residual || (rows_aligned(residual, ldr, elem, 32) && rows_aligned(sum, lds, elem, 32))) &&
                   reinterpret_cast<uintptr_t>(weight) % 32 == 0;
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = static_cast<uint8_t*>(scales);
  a.sum = sum;
  a.lds = lds;
  if (dtype == SVDQ_BF16) return vec ? launch_norm<__nv_bfloat16, true>(a, stream) : launch_norm<__nv_bfloat16, false>(a, stream);
  if (dtype == SVDQ_FP16) return vec ? launch_norm<__half, true>(a, stream) : launch_norm<__half, false>(a, stream);
  return vec ? launch_norm<float, true>(a, stream) : launch_norm<float, false>(a, stream);
}

// Root-mean-square norm with the residual's addition, written as mxfp8 (e4m3 codes, a power-of-two
// scale per 32 columns):
//   h = x + residual, rounded to its type and stored;   y = h * rsqrt(mean(h^2) + eps) * weight
//   scale = 2^(floor(log2 max|y|) - 8) per 32 columns,  code = e4m3(y / scale)
// The norm reads h as it is stored, so a residual stream read back later gives the same norm.  Squares
// are summed in fp32 within a thread and in 64 bits over the row, the root is held as the sum of two
// fp32 values, and h * weight is exact in fp32 for 16-bit types: y is rounded to fp32 once before it
// is rounded to its code, so that hardly a code or a scale falls on the other side of a border.
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

// One CTA per row.  A thread owns C columns of each C * THREADS (C = 16, or 8 in fp32: 32 bytes); the
// 32 / C neighbouring lanes of an mx block share its scale.  The row stays in registers between the
// two steps (the sum of squares, then the codes) for up to PASSES * C * THREADS columns; PASSES == 0
// reads it again instead.  Bound by HBM: 6 bytes read or written as bf16 and 1.03 as codes per
// element with a residual.
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
  auto load = [&](const T* p, int c, T (&v)[C]) {
    if constexpr (!VEC) {
      load_shifted(p, c, a.H, v);
    } else if (c < a.H) {
      load_vec(p + c, v);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = from_float<T>(0.0f);
    }
  };
  alignas(32) T keep[kKeep][C];
  alignas(32) T res[kKeep][C];
  uint64_t ss2 = 0;  // two sums of squares
  auto add = [&](int c, T (&h)[C], const T (&r)[C]) {
    if (rr) {
#pragma unroll
      for (int i = 0; i < C; ++i) h[i] = from_float<T>(to_float(h[i]) + to_float(r[i]));
      if constexpr (!VEC) store_warp(sr, c, a.H, stage + (tid & ~31) * C, h);
      else if (c < a.H) store_vec(sr + c, h);
    }
#pragma unroll
    for (int i = 0; i < C; i += 2) {
      const uint64_t v = f2_pack(to_float(h[i]), to_float(h[i + 1]));
      ss2 = f2_fma(v, v, ss2);
    }
  };
  if constexpr (PASSES > 0) {  // every load first
#pragma unroll
    for (int p = 0; p < PASSES; ++p) load(xr, column(p), keep[p]);
    if (rr) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) load(rr, column(p), res[p]);
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) add(column(p), keep[p], res[p]);
  } else {
    for (int p = 0; p < passes; ++p) {
      load(xr, column(p), keep[0]);
      if (rr) load(rr, column(p), res[0]);
      add(column(p), keep[0], res[0]);
    }
  }
  double ss = (double)f2_lo(ss2) + (double)f2_hi(ss2);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) part[tid >> 5] = ss;
  __syncthreads();
  ss = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) ss += part[w];
  // 1 / sqrt(v) as hi + lo: hi = fp32 of it to a few ulp, lo = hi (1 - v hi^2) / 2 (a Newton step)
  const double v = fma(ss, a.per_column, (double)a.eps);
  const float hi = 1.0f / sqrtf((float)v);
  const float lo = 0.5f * hi * (float)fma(-v, (double)hi * (double)hi, 1.0);
  const uint64_t hi2 = f2_pack(hi, hi), lo2 = isfinite(hi) && hi != 0.0f ? f2_pack(lo, lo) : 0;
  auto encode = [&](int c, const T (&h)[C]) {
    alignas(32) T w[C];
    if (weight) load(weight, c, w);
    float y[C];
#pragma unroll
    for (int i = 0; i < C; i += 2) {
      uint64_t p = f2_pack(to_float(h[i]), to_float(h[i + 1]));
      if (weight) p = f2_mul(p, f2_pack(to_float(w[i]), to_float(w[i + 1])));
      p = f2_fma(p, hi2, f2_mul(p, lo2));
      y[i] = f2_lo(p);
      y[i + 1] = f2_hi(p);
    }
    uint32_t amax = amax_bits_of(y);
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    if (C == 8) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const uint32_t byte = mx_scale_byte<kMxfp8>(amax);
    if (byte == 255u) {
#pragma unroll
      for (int i = 0; i < C; ++i) y[i] = 0.0f;
    }
    scale_all(y, mx_inverse_scale(byte));
    uint32_t q[C / 4];
    e4m3_words(y, q);
    constexpr int L = 32 / C;  // lanes per block
    uint32_t word = byte << (8 * ((lane / L) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, L);
    word |= __shfl_xor_sync(0xffffffffu, word, 2 * L);
    if (c < a.h_pad) {
      uint8_t* to = a.codes + (size_t)row * a.h_pad + c;
      if constexpr (C == 16) *reinterpret_cast<uint4*>(to) = make_uint4(q[0], q[1], q[2], q[3]);
      else *reinterpret_cast<uint2*>(to) = make_uint2(q[0], q[1]);
      if (lane % (4 * L) == 0) *reinterpret_cast<uint32_t*>(a.scales + mx_scale_word(row, c >> 7, words)) = word;
    }
  };
  if constexpr (PASSES > 0) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) encode(column(p), keep[p]);
  } else {
    for (int p = 0; p < passes; ++p) {
      if constexpr (!VEC) __syncwarp();
      load(sr ? sr : xr, column(p), keep[0]);  // the sums as this warp stored them
      encode(column(p), keep[0]);
    }
  }
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

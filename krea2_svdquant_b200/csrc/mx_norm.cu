// Root-mean-square norm with the residual's addition, written as mxfp8 (e4m3 codes, a power-of-two
// scale per 32 columns):
//   h = x + residual, rounded to its type and stored;   y = h * rsqrt(mean(h^2) + eps) * weight
//   scale = 2^(floor(log2 max|y|) - 8) per 32 columns,  code = e4m3(y / scale)
// The mean and y stay in fp32: y is rounded once, to its code.  The norm reads h as it is stored, so
// a residual stream read back later gives the same norm.
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
  int M, H, h_pad;
  bool vec;       // rows of x, residual and sum, and weight, start on 16-byte boundaries
  uint8_t* codes;
  uint8_t* scales;
  void* sum;
  int64_t lds;
};

// One CTA per row.  A thread owns 8 columns of each 8 * THREADS; four neighbouring lanes share an
// mx block.  The row stays in registers between the two steps (the sum of squares, then the codes)
// for up to PASSES * 8 * THREADS columns; PASSES == 0 reads it again instead.  Bound by HBM: 6
// bytes read or written as bf16 and 1.03 as codes per element with a residual.
template <typename T, int THREADS, int PASSES>
__global__ void __launch_bounds__(THREADS) rms_norm_mx_kernel(const NormArgs a) {
  constexpr int kKeep = PASSES > 0 ? PASSES : 1;
  __shared__ float part[THREADS / 32];
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
  const int passes = (a.h_pad + 8 * THREADS - 1) / (8 * THREADS);
  T keep[kKeep][8];
  float ss = 0.0f;
  auto first = [&](int p, T (&h)[8]) {
    const int c = (p * THREADS + tid) * 8;
    load_cols<T, 8>(xr, c, a.H, a.vec, h);
    if (rr) {
      T r[8];
      load_cols<T, 8>(rr, c, a.H, a.vec, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = from_float<T>(to_float(h[i]) + to_float(r[i]));
      store_cols<T, 8>(sr, c, a.H, a.vec, h);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(to_float(h[i]), to_float(h[i]), ss);
  };
  if constexpr (PASSES > 0) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) first(p, keep[p]);
  } else {
    for (int p = 0; p < passes; ++p) first(p, keep[0]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) part[tid >> 5] = ss;
  __syncthreads();
  ss = 0.0f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) ss += part[w];
  const float inv = 1.0f / sqrtf(ss / (float)a.H + a.eps);
  auto second = [&](int p, const T (&h)[8]) {
    const int c = (p * THREADS + tid) * 8;
    T w[8];
    float y[8];
    if (a.weight) {
      load_cols<T, 8>(static_cast<const T*>(a.weight), c, a.H, a.vec, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = to_float(h[i]) * inv * to_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = to_float(h[i]) * inv;
    }
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(y[i]) & 0x7FFFFFFFu);
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const uint32_t byte = mx_scale_byte<kMxfp8>(amax);
    const float f = mx_inverse_scale(byte);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = byte == 255u ? 0.0f : y[i] * f;
    if (c < a.h_pad)
      *reinterpret_cast<uint2*>(a.codes + (size_t)row * a.h_pad + c) =
          make_uint2(e4m3x2_satfinite(y[0], y[1]) | e4m3x2_satfinite(y[2], y[3]) << 16,
                     e4m3x2_satfinite(y[4], y[5]) | e4m3x2_satfinite(y[6], y[7]) << 16);
    uint32_t word = byte << (8 * ((lane >> 2) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    if (c < a.h_pad && (lane & 15) == 0)
      *reinterpret_cast<uint32_t*>(a.scales + mx_scale_word(row, c >> 7, words)) = word;
  };
  if constexpr (PASSES > 0) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) second(p, keep[p]);
  } else {
    for (int p = 0; p < passes; ++p) {
      T h[8];
      // the sum as this thread stored it, or x itself
      load_cols<T, 8>(sr ? sr : xr, (p * THREADS + tid) * 8, a.H, a.vec, h);
      second(p, h);
    }
  }
}

template <typename T>
int launch_norm(const NormArgs& a, cudaStream_t stream) {
  const dim3 grid(mx_rows_pad(a.M));
  const char* what = "svdq_rms_norm_mx launch";
  if (a.h_pad <= 1024) return launch_pdl(what, rms_norm_mx_kernel<T, 128, 1>, grid, dim3(128), 0, stream, 1, a);
  if (a.h_pad <= 2048) return launch_pdl(what, rms_norm_mx_kernel<T, 256, 1>, grid, dim3(256), 0, stream, 1, a);
  if (a.h_pad <= 4096) return launch_pdl(what, rms_norm_mx_kernel<T, 256, 2>, grid, dim3(256), 0, stream, 1, a);
  if (a.h_pad <= 6144) return launch_pdl(what, rms_norm_mx_kernel<T, 256, 3>, grid, dim3(256), 0, stream, 1, a);
  if (a.h_pad <= 8192) return launch_pdl(what, rms_norm_mx_kernel<T, 256, 4>, grid, dim3(256), 0, stream, 1, a);
  if (a.h_pad <= 16384) return launch_pdl(what, rms_norm_mx_kernel<T, 512, 4>, grid, dim3(512), 0, stream, 1, a);
  return launch_pdl(what, rms_norm_mx_kernel<T, 512, 0>, grid, dim3(512), 0, stream, 1, a);
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
  if (M > (1 << 30) || H > (1 << 30)) return set_error(SVDQ_ERR_UNSUPPORTED, "svdq_rms_norm_mx: matrix too large");
  NormArgs a{};
  const int eb = dtype_bytes(dtype);
  a.x = x;
  a.ldx = ldx;
  a.residual = residual;
  a.ldr = ldr;
  a.weight = weight;
  a.eps = eps;
  a.M = M;
  a.H = H;
  a.h_pad = mx_k_pad(H);
  a.vec = rows_aligned16(x, ldx, eb) && (!residual || (rows_aligned16(residual, ldr, eb) && rows_aligned16(sum, lds, eb))) &&
          (reinterpret_cast<uintptr_t>(weight) & 15u) == 0;
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = static_cast<uint8_t*>(scales);
  a.sum = sum;
  a.lds = lds;
  if (dtype == SVDQ_BF16) return launch_norm<__nv_bfloat16>(a, stream);
  if (dtype == SVDQ_FP16) return launch_norm<__half>(a, stream);
  return launch_norm<float>(a, stream);
}

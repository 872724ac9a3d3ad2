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
  uint8_t* codes;
  uint8_t* scales;
  void* sum;
  int64_t lds;
};

// One CTA per row.  A thread owns 8 columns of each 8 * THREADS; four neighbouring lanes share an
// mx block.  The row and the weight stay in registers between the two steps (the sum of squares, then
// the codes) for up to PASSES * 8 * THREADS columns; PASSES == 0 reads them again instead.  Bound by
// HBM: 6 bytes read or written as bf16 and 1.03 as codes per element with a residual.
template <typename T, int THREADS, int PASSES, bool VEC>
__global__ void __launch_bounds__(THREADS) rms_norm_mx_kernel(const NormArgs a) {
  constexpr int kKeep = PASSES > 0 ? PASSES : 1;
  __shared__ float part[THREADS / 32];
  __shared__ __align__(16) T stage_all[VEC ? 1 : THREADS * 8];
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  const int words = a.h_pad / 128;
  if (row >= a.M) {  // rows that only fill a tile of scales
    for (int w = tid; w < words; w += THREADS) *reinterpret_cast<uint32_t*>(a.scales + mx_scale_word(row, w, words)) = 0u;
    return;
  }
  T* stage = stage_all + (VEC ? 0 : (tid & ~31) * 8);
  const T* xr = static_cast<const T*>(a.x) + (size_t)row * a.ldx;
  const T* rr = a.residual ? static_cast<const T*>(a.residual) + (size_t)row * a.ldr : nullptr;
  T* sr = a.sum ? static_cast<T*>(a.sum) + (size_t)row * a.lds : nullptr;
  const T* weight = static_cast<const T*>(a.weight);
  const int passes = PASSES > 0 ? PASSES : (a.h_pad + 8 * THREADS - 1) / (8 * THREADS);
  auto load = [&](const T* p, int c, T (&v)[8]) {
    if constexpr (VEC) {
      if (c < a.H) {
        load_vec(p + c, v);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = from_float<T>(0.0f);
      }
    } else {
      load_warp(p, c, a.H, stage, v);
    }
  };
  alignas(32) T keep[kKeep][8];
  alignas(32) T res[kKeep][8];
  alignas(32) T wt[kKeep][8];
  float ss = 0.0f;
  auto add = [&](int c, T (&h)[8], const T (&r)[8]) {
    if (rr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = from_float<T>(to_float(h[i]) + to_float(r[i]));
      if constexpr (VEC) {
        if (c < a.H) store_vec(sr + c, h);
      } else {
        store_warp(sr, c, a.H, stage, h);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(to_float(h[i]), to_float(h[i]), ss);
  };
  if constexpr (PASSES > 0) {  // every load first
#pragma unroll
    for (int p = 0; p < PASSES; ++p) load(xr, (p * THREADS + tid) * 8, keep[p]);
    if (rr) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) load(rr, (p * THREADS + tid) * 8, res[p]);
    }
    if (weight) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) load(weight, (p * THREADS + tid) * 8, wt[p]);
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) add((p * THREADS + tid) * 8, keep[p], res[p]);
  } else {
    for (int p = 0; p < passes; ++p) {
      const int c = (p * THREADS + tid) * 8;
      load(xr, c, keep[0]);
      if (rr) load(rr, c, res[0]);
      add(c, keep[0], res[0]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) part[tid >> 5] = ss;
  __syncthreads();
  ss = 0.0f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) ss += part[w];
  const float inv = 1.0f / sqrtf(ss / (float)a.H + a.eps);
  auto encode = [&](int c, const T (&h)[8], const T (&w)[8]) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = to_float(h[i]) * inv;
    if (weight) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= to_float(w[i]);
    }
    uint32_t amax = amax_bits_of(y);
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const uint32_t byte = mx_scale_byte<kMxfp8>(amax);
    const float f = mx_inverse_scale(byte);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= f;
    if (byte == 255u) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = 0.0f;
    }
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
    for (int p = 0; p < PASSES; ++p) encode((p * THREADS + tid) * 8, keep[p], wt[p]);
  } else {
    for (int p = 0; p < passes; ++p) {
      const int c = (p * THREADS + tid) * 8;
      if constexpr (!VEC) __syncwarp();  // the sums of this warp's columns, as its lanes stored them
      load(sr ? sr : xr, c, keep[0]);
      if (weight) load(weight, c, wt[0]);
      encode(c, keep[0], wt[0]);
    }
  }
}

template <typename T, bool VEC>
int launch_norm(const NormArgs& a, cudaStream_t stream) {
  const dim3 grid(mx_rows_pad(a.M));
  const char* what = "svdq_rms_norm_mx launch";
  if (a.h_pad <= 1024) return launch_pdl(what, rms_norm_mx_kernel<T, 128, 1, VEC>, grid, dim3(128), 0, stream, 1, a);
  if (a.h_pad <= 2048) return launch_pdl(what, rms_norm_mx_kernel<T, 256, 1, VEC>, grid, dim3(256), 0, stream, 1, a);
  if (a.h_pad <= 4096) return launch_pdl(what, rms_norm_mx_kernel<T, 256, 2, VEC>, grid, dim3(256), 0, stream, 1, a);
  if (a.h_pad <= 6144) return launch_pdl(what, rms_norm_mx_kernel<T, 256, 3, VEC>, grid, dim3(256), 0, stream, 1, a);
  if (a.h_pad <= 8192) return launch_pdl(what, rms_norm_mx_kernel<T, 256, 4, VEC>, grid, dim3(256), 0, stream, 1, a);
  if (a.h_pad <= 16384) return launch_pdl(what, rms_norm_mx_kernel<T, 512, 4, VEC>, grid, dim3(512), 0, stream, 1, a);
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
  const int al = 8 * eb;
  const bool vec = H % 8 == 0 && rows_aligned(x, ldx, eb, al) &&
                   (!residual || (rows_aligned(residual, ldr, eb, al) && rows_aligned(sum, lds, eb, al))) &&
                   reinterpret_cast<uintptr_t>(weight) % al == 0;
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = static_cast<uint8_t*>(scales);
  a.sum = sum;
  a.lds = lds;
  if (dtype == SVDQ_BF16) return vec ? launch_norm<__nv_bfloat16, true>(a, stream) : launch_norm<__nv_bfloat16, false>(a, stream);
  if (dtype == SVDQ_FP16) return vec ? launch_norm<__half, true>(a, stream) : launch_norm<__half, false>(a, stream);
  return vec ? launch_norm<float, true>(a, stream) : launch_norm<float, false>(a, stream);
}

// Quantisation to the block-scaled formats, reading them back, and the nvfp4 tensor scale.
#include "mx_common.cuh"

namespace svdq {
namespace {

constexpr int kThreads = 256;

// Quotient and remainder by a divisor that is fixed for a launch: floor(n / d) = (n * mul) >> 32 >>
// shift with mul = ceil(2^(32 + shift) / d), exact for n < 2^31 (T. Granlund, P. Montgomery,
// "Division by Invariant Integers using Multiplication", PLDI 1994).
struct FastDiv {
  uint32_t d, mul, shift;
};
FastDiv fast_div(uint32_t d) {
  uint32_t shift = 0;
  while ((1u << shift) < d) ++shift;
  const uint64_t mul = d == 1 ? 0 : (((uint64_t)1 << (31 + shift)) + d - 1) / d;
  return FastDiv{d, (uint32_t)mul, shift};
}
__device__ __forceinline__ uint32_t div_by(const FastDiv& f, uint32_t n) {
  return f.d == 1 ? n : __umulhi(n, f.mul) >> (f.shift - 1);
}

// Chunks of 16 elements that a thread reads back: 64 bytes written.
template <typename T>
__host__ __device__ constexpr int unroll_of() { return sizeof(T) == 2 ? 2 : 1; }
// Columns that a thread quantises: 64 bytes read.
template <typename T>
__host__ __device__ constexpr int columns_of() { return 64 / (int)sizeof(T); }

struct QuantArgs {
  const void* x;
  int64_t ldx;
  int M, K;
  uint32_t chunks;     // chunks of all rows with scales (M rounded up to 128)
  FastDiv per_row;     // chunks per row
  bool vec;
  const float* tensor_scale;
  uint8_t* codes;
  uint8_t* scales;
};

// A thread quantises 64 bytes of a row: 32 columns of a 16-bit type, which are two nvfp4 blocks or one
// mx block, or 16 columns in fp32, one nvfp4 block or half an mx block whose other half is the
// neighbouring lane's.  HBM moves 2 bytes in and 0.5 out per element from bf16 to a 4-bit format;
// the instructions for them are nearly as much work, so what is done once per thread is shared by as
// many columns as stay in registers.  4352 x 6144 from bf16: to mxfp4 13.0 us with 16 columns a thread,
// 11.6 us (5.8 TB/s) with 32; to nvfp4 17 us (4.0 TB/s), bound by the instructions.  The four scale
// bytes of a 32-bit word of the tile layout come from 2 to 8 neighbouring lanes and leave as one store.
//
// A CTA takes kThreads neighbouring chunks.  From fp32 to nvfp4 it stays for a share of the launch's
// chunks, with the loads of the next ones issued before the present ones are worked on, because its
// units cost as much as half a step (4352 x 6144: 21.6 us against 25.5); the others run faster one
// step to a CTA (from bf16 to nvfp4 18.1 us against 20.4 when that was tried).  VEC: rows on 32-byte
// boundaries and K a multiple of 16.
template <typename T, int FMT>
__host__ __device__ constexpr bool stays() { return FMT == kNvfp4 && sizeof(T) == 4; }
constexpr int kStayCtas = 3;  // per SM: 256 threads of up to 80 registers

template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(kThreads) mx_quantize_kernel(const QuantArgs a) {
  constexpr int C = columns_of<T>(), kPieces = C / 16;
  constexpr int kRowUnits = 128 / C;  // chunks per 128 columns
  using Codes = typename CodeWord<FMT>::type;
  __shared__ __align__(16) Nvfp4Unit units[FMT == kNvfp4 ? 128 : 1];
  pdl_wait();
  pdl_trigger();
  struct Place {
    uint32_t id;
    int row, chunk;
    bool live;
  };
  auto place = [&](uint32_t step) {
    Place p;
    p.id = step * kThreads + threadIdx.x;
    const uint32_t r = div_by(a.per_row, p.id);
    p.row = (int)r;
    p.chunk = (int)(p.id - r * a.per_row.d);
    p.live = p.id < a.chunks && p.row < a.M;
    return p;
  };
  auto load = [&](const Place& p, T (&x)[kPieces][16]) {
    const T* src = static_cast<const T*>(a.x) + (p.live ? (size_t)p.row * a.ldx : 0);
    const int c = p.live ? p.chunk * C : a.K;
    if constexpr (VEC) {
#pragma unroll
      for (int h = 0; h < kPieces; ++h) {
        if (c + 16 * h < a.K) {
          load_vec(src + c + 16 * h, x[h]);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[h][i] = from_float<T>(0.0f);
        }
      }
    } else {
      load_shifted(src, c, a.K, reinterpret_cast<T(&)[C]>(x));
    }
  };
  const uint32_t steps = (a.chunks + kThreads - 1) / kThreads;
  alignas(32) T x[kPieces][16];
  Place at = place(blockIdx.x);
  load(at, x);
  const float g = a.tensor_scale ? *a.tensor_scale : 1.0f;
  if constexpr (FMT == kNvfp4) {
    if (threadIdx.x < 128) units[threadIdx.x] = nvfp4_unit<significant_bits<T>()>(threadIdx.x, g);
    __syncthreads();
  }
  for (uint32_t step = blockIdx.x; step < steps; step += gridDim.x) {
    alignas(32) T next[kPieces][16];
    Place then{};
    if (stays<T, FMT>() && step + gridDim.x < steps) {
      then = place(step + gridDim.x);
      load(then, next);
    }
    Codes codes[kPieces];
    uint32_t word;
    if constexpr (FMT == kNvfp4) {
      uint32_t bytes = 0;
#pragma unroll
      for (int h = 0; h < kPieces; ++h) {
        uint32_t byte;
        codes[h] = encode_chunk<T, FMT>(x[h], g, units, byte);
        bytes |= byte << (8 * h);
      }
      if (!at.live) bytes = 0;
      word = bytes << (8 * kPieces * (threadIdx.x & (4 / kPieces - 1)));
      word |= __shfl_xor_sync(0xffffffffu, word, 1);
      if (kPieces == 1) word |= __shfl_xor_sync(0xffffffffu, word, 2);
    } else {
      uint32_t amax = 0;
#pragma unroll
      for (int h = 0; h < kPieces; ++h) amax = max(amax, amax_bits_of(x[h]));
      if (kPieces == 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      const uint32_t byte = mx_scale_byte<FMT>(amax);
#pragma unroll
      for (int h = 0; h < kPieces; ++h) codes[h] = mx_codes<T, FMT>(x[h], byte);
      constexpr int L = 2 / kPieces;  // lanes per block
      word = (at.live ? byte : 0u) << (8 * ((threadIdx.x / L) & 3));
      word |= __shfl_xor_sync(0xffffffffu, word, L);
      word |= __shfl_xor_sync(0xffffffffu, word, 2 * L);
    }
    if (at.live) {
      Codes* to = reinterpret_cast<Codes*>(a.codes + (size_t)at.row * mx_row_bytes(FMT, (int)a.per_row.d * C)) +
                  at.chunk * kPieces;
      if constexpr (kPieces == 2 && FMT != kMxfp8) {
        *reinterpret_cast<uint4*>(to) = make_uint4(codes[0].x, codes[0].y, codes[1].x, codes[1].y);
      } else {
#pragma unroll
        for (int h = 0; h < kPieces; ++h) to[h] = codes[h];
      }
    }
    constexpr int kLanes = (FMT == kNvfp4 ? 64 : 128) / C;  // lanes per word
    if (at.id < a.chunks && (threadIdx.x & (kLanes - 1)) == 0) {
      const int words = (int)a.per_row.d / kRowUnits * (FMT == kNvfp4 ? 2 : 1);
      *reinterpret_cast<uint32_t*>(a.scales + mx_scale_word(at.row, at.chunk / kLanes, words)) = word;
    }
    if (!stays<T, FMT>()) break;
    at = then;
#pragma unroll
    for (int h = 0; h < kPieces; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[h][i] = next[h][i];
  }
}

struct ReadArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  const float* tensor_scale;
  int M, K;
  uint32_t chunks;
  FastDiv per_row;
  bool vec;
  void* out;
  int64_t ldo;
};

// Reading back: one thread turns 16 codes into values, code * scale (* tensor scale) in fp32,
// rounded once to T.  Bound by HBM (0.56 bytes read, 2 written per element from nvfp4 to bf16).
template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(kThreads) mx_dequantize_kernel(const ReadArgs a) {
  constexpr int kUnroll = unroll_of<T>();
  __shared__ __align__(16) T stage[VEC ? 1 : kThreads * 16];
  pdl_wait();
  pdl_trigger();
  const int blocks = (int)a.per_row.d * 16 / mx_block(FMT);
  const float g = FMT == kNvfp4 && a.tensor_scale ? *a.tensor_scale : 1.0f;
  using Codes = typename CodeWord<FMT>::type;
  Codes w[kUnroll];
  uint32_t byte[kUnroll];
  int row[kUnroll], chunk[kUnroll];
  bool live[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t id = (blockIdx.x * kUnroll + u) * kThreads + threadIdx.x;
    const uint32_t r = div_by(a.per_row, id);
    row[u] = (int)r;
    chunk[u] = (int)(id - r * a.per_row.d);
    live[u] = id < a.chunks && chunk[u] * 16 < a.K;
    w[u] = Codes{};
    byte[u] = 0;
    if (live[u]) {
      const int block = chunk[u] * 16 / mx_block(FMT);
      byte[u] = a.scales[mx_scale_word(row[u], block >> 2, blocks >> 2) + (block & 3)];
      w[u] = reinterpret_cast<const Codes*>(a.codes + (size_t)row[u] * mx_row_bytes(FMT, (int)a.per_row.d * 16))[chunk[u]];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const float unit = FMT == kNvfp4 ? e4m3_value(byte[u]) * g : e8m0_value(byte[u]);
    const uint32_t* ww = reinterpret_cast<const uint32_t*>(&w[u]);
    alignas(32) T v[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t h2;
      if constexpr (FMT == kMxfp8) {
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)(ww[i >> 1] >> (16 * (i & 1)))));
      } else {  // the conversion takes the low byte; with other bits above it, it gave wrong values
        asm("{\n\t.reg .b8 b, c;\n\tmov.b16 {b, c}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}"
            : "=r"(h2)
            : "h"((uint16_t)((ww[i >> 2] >> (8 * (i & 3))) & 0xFFu)));
      }
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
      v[2 * i] = from_float<T>(f.x * unit);
      v[2 * i + 1] = from_float<T>(f.y * unit);
    }
    T* dst = static_cast<T*>(a.out) + (live[u] ? (size_t)row[u] * a.ldo : 0);
    if constexpr (VEC) {
      if (live[u]) store_vec(dst + chunk[u] * 16, v);
    } else {
      store_warp(dst, live[u] ? chunk[u] * 16 : a.K, a.K, stage + (threadIdx.x & ~31) * 16, v);
    }
  }
}

// Largest magnitude of a matrix as fp32 bits, by an integer maximum: any order gives the same
// result, and a NaN is larger than every number.
template <typename T>
__global__ void __launch_bounds__(kThreads) mx_amax_kernel(const T* x, int64_t ldx, uint32_t chunks, FastDiv per_row,
                                                           int K, bool vec, uint32_t* out) {
  uint32_t amax = 0;
  for (uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x; i < chunks; i += (uint64_t)gridDim.x * kThreads) {
    const uint32_t row = div_by(per_row, (uint32_t)i);
    const int c = (int)((uint32_t)i - row * per_row.d) * 16;
    if (vec) {
      if (c >= K) continue;
      alignas(32) T v[16];
      load_vec(x + (size_t)row * ldx + c, v);
      amax = max(amax, amax_bits_of(v));
    } else {
      alignas(32) T v[16];
      load_shifted(x + (size_t)row * ldx, c, K, v);
      amax = max(amax, amax_bits_of(v));
    }
  }
  amax = __reduce_max_sync(0xffffffffu, amax);
  if ((threadIdx.x & 31) == 0) atomicMax(out, amax);
}
// amax bits -> the tensor scale amax / (6 * 448), 1 for a matrix of zeros.  Below fp32's normal range it is
// rounded up: to nearest it can be 0, which is no scale, or so much too small that the largest elements saturate.
__global__ void mx_tensor_scale_kernel(float* out) {
  const float amax = *out;
  const float g = amax / 2688.0f;
  *out = amax == 0.0f ? 1.0f : g < 0x1p-126f ? __fdiv_ru(amax, 2688.0f) : g;
}

// chunks and per_row of a matrix of `rows` rows in chunks of C columns; false where a launch cannot hold it
bool chunk_grid(int rows, int K, int C, uint32_t* chunks, FastDiv* per_row) {
  const uint32_t per = (uint32_t)mx_k_pad(K) / C;
  const uint64_t n = (uint64_t)rows * per;
  if ((uint64_t)rows * mx_k_pad(K) >= (1ull << 35)) return false;
  *chunks = (uint32_t)n;
  *per_row = fast_div(per);
  return true;
}

template <typename T, bool VEC>
int launch_quantize(int fmt, const QuantArgs& a, cudaStream_t stream) {
  const uint32_t steps = (a.chunks + kThreads - 1) / kThreads, most = (uint32_t)num_sms() * kStayCtas;
  const dim3 grid(fmt == kNvfp4 && stays<T, kNvfp4>() && steps > most ? most : steps), block(kThreads);
  const char* what = "svdq_mx_quantize launch";
  if (fmt == kNvfp4) return launch_pdl(what, mx_quantize_kernel<T, kNvfp4, VEC>, grid, block, 0, stream, 1, a);
  if (fmt == kMxfp4) return launch_pdl(what, mx_quantize_kernel<T, kMxfp4, VEC>, grid, block, 0, stream, 1, a);
  return launch_pdl(what, mx_quantize_kernel<T, kMxfp8, VEC>, grid, block, 0, stream, 1, a);
}
template <typename T, bool VEC>
int launch_dequantize(int fmt, const ReadArgs& a, cudaStream_t stream) {
  const uint32_t per = kThreads * unroll_of<T>();
  const dim3 grid((a.chunks + per - 1) / per), block(kThreads);
  const char* what = "svdq_mx_dequantize launch";
  if (fmt == kNvfp4) return launch_pdl(what, mx_dequantize_kernel<T, kNvfp4, VEC>, grid, block, 0, stream, 1, a);
  if (fmt == kMxfp4) return launch_pdl(what, mx_dequantize_kernel<T, kMxfp4, VEC>, grid, block, 0, stream, 1, a);
  return launch_pdl(what, mx_dequantize_kernel<T, kMxfp8, VEC>, grid, block, 0, stream, 1, a);
}

}  // namespace
}  // namespace svdq

extern "C" size_t svdq_mx_scale_bytes(int rows, int K, int format) {
  using namespace svdq;
  if (rows <= 0 || K <= 0 || K > (1 << 30) || rows > (1 << 30) || !mx_format_ok(format)) return 0;
  return (size_t)mx_rows_pad(rows) * (mx_k_pad(K) / mx_block(format));
}

extern "C" int svdq_mx_quantize(const void* x, int64_t ldx, int dtype, int M, int K, int format,
                                const float* tensor_scale, void* codes, void* scales, cudaStream_t stream) {
  using namespace svdq;
  SVDQ_REQUIRE(mx_format_ok(format), "svdq_mx_quantize: unknown format");
  SVDQ_REQUIRE(dtype_ok(dtype), "svdq_mx_quantize: x must be bf16, fp16 or fp32");
  SVDQ_REQUIRE(M >= 0 && K > 0 && ldx >= K, "svdq_mx_quantize: bad M/K/ldx");
  SVDQ_REQUIRE(tensor_scale == nullptr || format == kNvfp4, "svdq_mx_quantize: only nvfp4 has a tensor scale");
  if (M == 0) return SVDQ_OK;
  SVDQ_REQUIRE(x && codes && scales, "svdq_mx_quantize: null pointer");
  SVDQ_REQUIRE(((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15u) == 0,
               "svdq_mx_quantize: codes and scales must be 16-byte aligned");
  SVDQ_REQUIRE(element_aligned(x, dtype_bytes(dtype)) && element_aligned(tensor_scale, 4),
               "svdq_mx_quantize: x and tensor_scale must be aligned to their elements");
  QuantArgs a{};
  if (M > (1 << 30) || K > (1 << 30) || !chunk_grid(mx_rows_pad(M), K, 64 / dtype_bytes(dtype), &a.chunks, &a.per_row))
    return set_error(SVDQ_ERR_UNSUPPORTED, "svdq_mx_quantize: more than 2^35 padded elements");
  a.x = x;
  a.ldx = ldx;
  a.M = M;
  a.K = K;
  a.vec = K % 16 == 0 && rows_aligned(x, ldx, dtype_bytes(dtype), 32);
  a.tensor_scale = tensor_scale;
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = static_cast<uint8_t*>(scales);
  if (dtype == SVDQ_BF16) return a.vec ? launch_quantize<__nv_bfloat16, true>(format, a, stream) : launch_quantize<__nv_bfloat16, false>(format, a, stream);
  if (dtype == SVDQ_FP16) return a.vec ? launch_quantize<__half, true>(format, a, stream) : launch_quantize<__half, false>(format, a, stream);
  return a.vec ? launch_quantize<float, true>(format, a, stream) : launch_quantize<float, false>(format, a, stream);
}

extern "C" int svdq_mx_dequantize(const void* codes, const void* scales, int format, const float* tensor_scale, int M,
                                  int K, void* out, int64_t ldo, int dtype, cudaStream_t stream) {
  using namespace svdq;
  SVDQ_REQUIRE(mx_format_ok(format), "svdq_mx_dequantize: unknown format");
  SVDQ_REQUIRE(dtype_ok(dtype), "svdq_mx_dequantize: out must be bf16, fp16 or fp32");
  SVDQ_REQUIRE(M >= 0 && K > 0 && ldo >= K, "svdq_mx_dequantize: bad M/K/ldo");
  SVDQ_REQUIRE(tensor_scale == nullptr || format == kNvfp4, "svdq_mx_dequantize: only nvfp4 has a tensor scale");
  if (M == 0) return SVDQ_OK;
  SVDQ_REQUIRE(codes && scales && out, "svdq_mx_dequantize: null pointer");
  SVDQ_REQUIRE(((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15u) == 0,
               "svdq_mx_dequantize: codes and scales must be 16-byte aligned");
  SVDQ_REQUIRE(element_aligned(out, dtype_bytes(dtype)) && element_aligned(tensor_scale, 4),
               "svdq_mx_dequantize: out and tensor_scale must be aligned to their elements");
  ReadArgs a{};
  if (M > (1 << 30) || K > (1 << 30) || !chunk_grid(M, K, 16, &a.chunks, &a.per_row))
    return set_error(SVDQ_ERR_UNSUPPORTED, "svdq_mx_dequantize: more than 2^35 padded elements");
  a.codes = static_cast<const uint8_t*>(codes);
  a.scales = static_cast<const uint8_t*>(scales);
  a.tensor_scale = tensor_scale;
  a.M = M;
  a.K = K;
  a.vec = K % 16 == 0 && rows_aligned(out, ldo, dtype_bytes(dtype), 32);
  a.out = out;
  a.ldo = ldo;
  if (dtype == SVDQ_BF16) return a.vec ? launch_dequantize<__nv_bfloat16, true>(format, a, stream) : launch_dequantize<__nv_bfloat16, false>(format, a, stream);
  if (dtype == SVDQ_FP16) return a.vec ? launch_dequantize<__half, true>(format, a, stream) : launch_dequantize<__half, false>(format, a, stream);
  return a.vec ? launch_dequantize<float, true>(format, a, stream) : launch_dequantize<float, false>(format, a, stream);
}

extern "C" int svdq_mx_tensor_scale(const void* x, int64_t ldx, int dtype, int M, int K, float* out,
                                    cudaStream_t stream) {
  using namespace svdq;
  SVDQ_REQUIRE(dtype_ok(dtype), "svdq_mx_tensor_scale: x must be bf16, fp16 or fp32");
  SVDQ_REQUIRE(M >= 0 && K > 0 && ldx >= K, "svdq_mx_tensor_scale: bad M/K/ldx");
  SVDQ_REQUIRE(out && (x || M == 0), "svdq_mx_tensor_scale: null pointer");
  SVDQ_REQUIRE(element_aligned(x, dtype_bytes(dtype)) && element_aligned(out, 4),
               "svdq_mx_tensor_scale: x and out must be aligned to their elements");
  int st = check_cuda(cudaMemsetAsync(out, 0, sizeof(float), stream), "svdq_mx_tensor_scale: clear");
  if (st) return st;
  uint32_t chunks = 0;
  FastDiv per_row{};
  if (M > (1 << 30) || K > (1 << 30) || !chunk_grid(M, K, 16, &chunks, &per_row))
    return set_error(SVDQ_ERR_UNSUPPORTED, "svdq_mx_tensor_scale: more than 2^35 padded elements");
  if (chunks > 0) {
    const bool vec = K % 16 == 0 && rows_aligned(x, ldx, dtype_bytes(dtype), 32);
    const uint32_t want = (chunks + kThreads - 1) / kThreads, most = (uint32_t)num_sms() * 8;
    const dim3 grid(want < most ? want : most), block(kThreads);
    uint32_t* bits = reinterpret_cast<uint32_t*>(out);
    if (dtype == SVDQ_BF16)
      mx_amax_kernel<<<grid, block, 0, stream>>>(static_cast<const __nv_bfloat16*>(x), ldx, chunks, per_row, K, vec, bits);
    else if (dtype == SVDQ_FP16)
      mx_amax_kernel<<<grid, block, 0, stream>>>(static_cast<const __half*>(x), ldx, chunks, per_row, K, vec, bits);
    else
      mx_amax_kernel<<<grid, block, 0, stream>>>(static_cast<const float*>(x), ldx, chunks, per_row, K, vec, bits);
    st = check_launch("svdq_mx_tensor_scale launch");
    if (st) return st;
  }
  mx_tensor_scale_kernel<<<1, 1, 0, stream>>>(out);
  return check_launch("svdq_mx_tensor_scale launch");
}

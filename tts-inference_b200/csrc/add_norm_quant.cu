// Residual addition, RMSNorm and 8-bit quantization of a row in one launch
// (qtts_add_rms_norm_quant): what stands between two W8A8 linears of a decoder
// layer (qtts/models/talker.py:249, 271 followed by qtts/quant/fp8.py:77-78 or
// int8.py:138-140 as separate ops).
//   h = x + residual;  y = w * (h * (1 / sqrt(mean(h^2) + eps)))
//   scale = max(max|y|, 1e-6) * fl32(1 / 448 or 1 / 127);  q = rne(y * (1 / scale))
// All of it in fp32 from the inputs to the codes: the stored residual is h
// rounded to its type, but the norm reads the unrounded sum and the quantizer
// the unrounded y, so one rounding (to 8 bits) separates the codes from the
// formula. A row that holds a NaN or an infinity gets a NaN scale, so that no
// finite codes stand for it.
//
// Bound by memory: 7 bytes an element (bf16 in, e4m3 out) are read or written once;
// 16384 rows of 2048 in 42 us, 5.6 TB/s (fp32 in: 69 us, 6.5 TB/s). One row of 2048:
// 1.6 us, a launch and two latencies.
// A row stays in registers between its load and its codes: a warp a row up to 512
// channels, 128 to 1024 threads up to 16384, one or two chunks of eight channels a
// thread; longer rows are read three times (2048 rows of 20000: 131 us). A launch has
// at most 1024 threads an SM, whose CTAs walk over the rows, and the next row's loads
// are under way while the two reductions of this one wait for their barriers. Loads and stores are 16 bytes
// even where rows are not: all arrays then have rows of the same displacement, and a
// thread takes whole aligned chunks of eight elements, only the two ends of a row
// element by element (and the weight, which is displaced otherwise in every row:
// 16384 rows of 2047 in 145 us).
#include <cuda_fp8.h>

#include <type_traits>

#include "kernels.h"
#include "prologue.cuh"

namespace qtts {
namespace {

constexpr int kAnThreads = 256;

template <bool kMax>
__device__ __forceinline__ float warp_reduce(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = kMax ? nan_max(v, w) : v + w;
  }
  return v;
}

// Over the kWarps warps that hold a row; every thread returns the same bits.
template <bool kMax, int kWarps>
__device__ __forceinline__ float row_reduce(float v, float* sh) {
  v = warp_reduce<kMax>(v);
  if constexpr (kWarps > 1) {
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) v = kMax ? nan_max(v, sh[i]) : v + sh[i];
  }
  return v;
}

// rne(y * inv_scale) as a code. int8: |y * inv_scale| <= 127 (1 + 2^-22), so adding 1.5 * 2^23
// leaves the rounded integer in the low byte.
template <bool kInt8>
__device__ __forceinline__ uint32_t to_codes2(float a, float b, float inv_scale) {
  a *= inv_scale, b *= inv_scale;
  if constexpr (kInt8) {
    return __byte_perm(__float_as_uint(a + 12582912.f), __float_as_uint(b + 12582912.f), 0x0040) & 0xFFFFu;
  } else {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  }
}

// Codes are products with the reciprocal of the scale, one IEEE division a row.
__device__ __forceinline__ float row_scale(float amax, bool int8) {
  return nan_max(amax, 1e-6f) * (int8 ? 1.0f / 127.0f : 1.0f / 448.0f);
}

// Eight elements as loaded: 16 bytes of a 16-bit type, 32 of fp32.
template <typename XT>
struct Raw8 {
  uint4 u[sizeof(XT) / 2];
};

template <typename XT>
__device__ __forceinline__ void unpack8(const Raw8<XT>& raw, float (&v)[8]) {
  const XT* e = reinterpret_cast<const XT*>(&raw);
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] = to_float(e[q]);
}

template <typename XT>
__device__ __forceinline__ void store8(XT* p, const float (&v)[8]) {
  Raw8<XT> raw;
  XT* e = reinterpret_cast<XT*>(&raw);
#pragma unroll
  for (int q = 0; q < 8; ++q) e[q] = from_float<XT>(v[q]);
#pragma unroll
  for (int q = 0; q < static_cast<int>(sizeof(XT) / 2); ++q) reinterpret_cast<uint4*>(p)[q] = raw.u[q];
}

// kWhole: no row is displaced and the width is a multiple of eight. Otherwise chunk c of row
// `row` is its elements [8 c - m, 8 c - m + 8), m its displacement, and a chunk that is not
// wholly inside the row is taken element by element.
template <typename XT, bool kInt8, int kTpr, int kChunks, bool kWhole>
__global__ void __launch_bounds__(kTpr == 32 ? 128 : kTpr) add_norm_quant_kernel(const AddNormQuantArgs a) {
  constexpr int kWarps = kTpr / 32;
  constexpr int kRows = kTpr == 32 ? 4 : 1;  // rows a CTA at a time
  __shared__ float sh[2][kWarps];
  pdl_launch_dependents();
  const int t = kTpr == 32 ? threadIdx.x & 31 : threadIdx.x;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + (kTpr == 32 ? threadIdx.x >> 5 : 0);
  if (row >= a.rows) return;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRows;
  pdl_wait();
  const bool add = a.residual != nullptr;
  const XT* w = static_cast<const XT*>(a.weight);

  Raw8<XT> xr[kChunks], rr[kChunks], wr[kChunks];
  const auto start = [&](int64_t r, int i) {  // first element of this thread's chunk i of row r
    return 8 * (t + i * kTpr) - (kWhole ? 0 : static_cast<int>((r * a.ldx) & 7));
  };
  const auto inside = [&](int e0) { return e0 >= 0 && e0 + 8 <= a.width; };
  const auto fetch = [&](int64_t r) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int e0 = start(r, i);
      xr[i] = rr[i] = Raw8<XT>{};
      if (inside(e0)) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const XT*>(a.x) + r * a.ldx + e0);
#pragma unroll
        for (int q = 0; q < static_cast<int>(sizeof(XT) / 2); ++q) xr[i].u[q] = __ldcs(p + q);
        if (add) {
          const uint4* p2 = reinterpret_cast<const uint4*>(static_cast<const XT*>(a.residual) + r * a.ldr + e0);
#pragma unroll
          for (int q = 0; q < static_cast<int>(sizeof(XT) / 2); ++q) rr[i].u[q] = __ldcs(p2 + q);
        }
      }
    }
  };
  if constexpr (kWhole) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      wr[i] = Raw8<XT>{};
      const int e0 = 8 * (t + i * kTpr);
      if (inside(e0)) {
#pragma unroll
        for (int q = 0; q < static_cast<int>(sizeof(XT) / 2); ++q) {
          wr[i].u[q] = __ldg(reinterpret_cast<const uint4*>(w + e0) + q);
        }
      }
    }
  }
  fetch(row);
  while (row < a.rows) {
    const XT* x = static_cast<const XT*>(a.x) + row * a.ldx;
    const XT* res = add ? static_cast<const XT*>(a.residual) + row * a.ldr : nullptr;
    XT* ro = add ? static_cast<XT*>(a.residual_out) + row * a.ldro : nullptr;
    float h[kChunks][8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int e0 = start(row, i);
      float v[8];
      unpack8<XT>(xr[i], h[i]);
      unpack8<XT>(rr[i], v);
#pragma unroll
      for (int q = 0; q < 8; ++q) h[i][q] += v[q];
      if (inside(e0)) {
        if (add) store8<XT>(ro + e0, h[i]);
      } else if (!kWhole && e0 < a.width && e0 + 8 > 0) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (e0 + q >= 0 && e0 + q < a.width) {
            h[i][q] = to_float(x[e0 + q]) + (add ? to_float(res[e0 + q]) : 0.f);
            if (add) ro[e0 + q] = from_float<XT>(h[i][q]);
          }
        }
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) ss = fmaf(h[i][q], h[i][q], ss);
    }
    const int64_t next = row + stride;
    if (next < a.rows) fetch(next);
    const float inv = rms_inv(row_reduce<false, kWarps>(ss, sh[0]), a.width, a.eps);
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int e0 = start(row, i);
      float v[8];
      if constexpr (kWhole) {
        unpack8<XT>(wr[i], v);
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = e0 + q >= 0 && e0 + q < a.width ? to_float(__ldg(w + e0 + q)) : 0.f;
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        h[i][q] = rms_apply(h[i][q], inv, v[q]);
        amax = nan_max(amax, fabsf(h[i][q]));
      }
    }
    const float scale = row_scale(row_reduce<true, kWarps>(amax, sh[1]), kInt8);
    const float inv_scale = __fdiv_rn(1.0f, scale);
    uint8_t* q8 = static_cast<uint8_t*>(a.q) + row * a.ldq;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int e0 = start(row, i);
      uint32_t c[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) c[q] = to_codes2<kInt8>(h[i][2 * q], h[i][2 * q + 1], inv_scale);
      if (inside(e0)) {
        *reinterpret_cast<uint2*>(q8 + e0) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
      } else if (!kWhole) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (e0 + q >= 0 && e0 + q < a.width) q8[e0 + q] = static_cast<uint8_t>(c[q / 2] >> (8 * (q & 1)));
        }
      }
    }
    if (t == 0) a.scale[row] = scale;
    row = next;
  }
}

// Rows longer than the registers, and arrays whose rows are displaced differently.
template <typename XT, bool kInt8>
__global__ void __launch_bounds__(kAnThreads) add_norm_quant_long_kernel(const AddNormQuantArgs a) {
  __shared__ float sh[2][kAnThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.x;
  const XT* x = static_cast<const XT*>(a.x) + row * a.ldx;
  const XT* r = a.residual != nullptr ? static_cast<const XT*>(a.residual) + row * a.ldr : nullptr;
  XT* ro = a.residual != nullptr ? static_cast<XT*>(a.residual_out) + row * a.ldro : nullptr;
  const XT* w = static_cast<const XT*>(a.weight);
  float ss = 0.f;
  for (int k = threadIdx.x; k < a.width; k += kAnThreads) {
    const float h = to_float(x[k]) + (r != nullptr ? to_float(r[k]) : 0.f);
    ss = fmaf(h, h, ss);
  }
  const float inv = rms_inv(row_reduce<false, kAnThreads / 32>(ss, sh[0]), a.width, a.eps);
  float amax = 0.f;
  for (int k = threadIdx.x; k < a.width; k += kAnThreads) {
    const float h = to_float(x[k]) + (r != nullptr ? to_float(r[k]) : 0.f);
    amax = nan_max(amax, fabsf(rms_apply(h, inv, to_float(w[k]))));
  }
  const float scale = row_scale(row_reduce<true, kAnThreads / 32>(amax, sh[1]), kInt8);
  const float inv_scale = __fdiv_rn(1.0f, scale);
  uint8_t* q = static_cast<uint8_t*>(a.q) + row * a.ldq;
  for (int k = threadIdx.x; k < a.width; k += kAnThreads) {
    // residual_out may be x or the residual: an element is written after its last reading, which
    // is this thread's.
    const float h = to_float(x[k]) + (r != nullptr ? to_float(r[k]) : 0.f);
    q[k] = static_cast<uint8_t>(to_codes2<kInt8>(rms_apply(h, inv, to_float(w[k])), 0.f, inv_scale));
    if (r != nullptr) ro[k] = from_float<XT>(h);
  }
  if (threadIdx.x == 0) a.scale[row] = scale;
}

template <typename XT, bool kInt8>
int launch_an(const AddNormQuantArgs& a, bool pdl, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  // Up to 1024 threads an SM; of 128-thread CTAs, at 91 registers, five of the eight are there at once and
  // the others follow. Two chunks a thread: 16384 rows of 2048 take 42 us (one chunk: 49; four: 40), one
  // row 1.6 (one or four chunks 0.1 to 0.3 more).
  const auto go = [&](auto kern, int threads, int rows_a_cta, int ctas_a_sm) {
    const int64_t need = (static_cast<int64_t>(a.rows) + rows_a_cta - 1) / rows_a_cta;
    const int64_t most = static_cast<int64_t>(kNumSMs) * ctas_a_sm;
    cfg.blockDim = dim3(threads);
    cfg.gridDim = dim3(static_cast<unsigned>(need < most ? need : most));
    return cudaLaunchKernelEx(&cfg, kern, a) == cudaSuccess ? QTTS_OK : QTTS_ERR_LAUNCH;
  };
  const auto pick = [&](auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    // Chunks of a row at its worst displacement.
    const int chunks = (a.width + (kWhole ? 0 : 7) + 7) / 8;
    if (chunks <= 64) return go(add_norm_quant_kernel<XT, kInt8, 32, 2, kWhole>, 128, 4, 8);
    if (chunks <= 256) return go(add_norm_quant_kernel<XT, kInt8, 128, 2, kWhole>, 128, 1, 8);
    if (chunks <= 512) return go(add_norm_quant_kernel<XT, kInt8, 256, 2, kWhole>, 256, 1, 4);
    if (chunks <= 1024) return go(add_norm_quant_kernel<XT, kInt8, 512, 2, kWhole>, 512, 1, 2);
    return go(add_norm_quant_kernel<XT, kInt8, 1024, 2, kWhole>, 1024, 1, 1);
  };
  if (a.vec && a.whole) {
    if (a.width <= 16384) return pick(std::true_type{});
  } else if (a.vec && a.width <= 16384 - 7) {
    return pick(std::false_type{});
  }
  cfg.gridDim = dim3(a.rows);
  cfg.blockDim = dim3(kAnThreads);
  return cudaLaunchKernelEx(&cfg, add_norm_quant_long_kernel<XT, kInt8>, a) == cudaSuccess ? QTTS_OK
                                                                                          : QTTS_ERR_LAUNCH;
}

}  // namespace

int launch_add_norm_quant(const AddNormQuantArgs& a, int dtype, int q_dtype, bool pdl, cudaStream_t stream) {
  const bool int8 = q_dtype == QTTS_INT8;
  switch (dtype) {
    case QTTS_BF16:
      return int8 ? launch_an<__nv_bfloat16, true>(a, pdl, stream) : launch_an<__nv_bfloat16, false>(a, pdl, stream);
    case QTTS_FP16:
      return int8 ? launch_an<__half, true>(a, pdl, stream) : launch_an<__half, false>(a, pdl, stream);
    case QTTS_FP32:
      return int8 ? launch_an<float, true>(a, pdl, stream) : launch_an<float, false>(a, pdl, stream);
    default:
      return QTTS_ERR_DTYPE;
  }
}

}  // namespace qtts

extern "C" int qtts_add_rms_norm_quant(const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                       const void* weight, float eps, void* residual_out, int64_t ldro, int dtype,
                                       void* q, int64_t ldq, int q_dtype, float* scale, int rows, int width,
                                       unsigned flags, void* stream) {
  using namespace qtts;
  if (rows < 0 || width < 1 || width > 65536) return QTTS_ERR_SHAPE;
  if (rows == 0) return QTTS_OK;
  if (x == nullptr || weight == nullptr || q == nullptr || scale == nullptr) return QTTS_ERR_NULL;
  if ((residual == nullptr) != (residual_out == nullptr)) return QTTS_ERR_NULL;
  if (dtype != QTTS_BF16 && dtype != QTTS_FP16 && dtype != QTTS_FP32) return QTTS_ERR_DTYPE;
  if (q_dtype != QTTS_E4M3 && q_dtype != QTTS_INT8) return QTTS_ERR_DTYPE;
  if (ldx < width || ldq < width || (residual != nullptr && (ldr < width || ldro < width))) return QTTS_ERR_SHAPE;
  const size_t sz = dtype == QTTS_FP32 ? 4 : 2;
  const auto al = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!al(x, sz) || !al(residual, sz) || !al(residual_out, sz) || !al(weight, sz) || !al(scale, 4)) {
    return QTTS_ERR_ALIGN;
  }
  const int dev_ok = check_device();
  if (dev_ok != QTTS_OK) return dev_ok;
  AddNormQuantArgs a{x, ldx, residual, ldr, weight, eps, residual_out, ldro, q, ldq, scale, rows, width, false, false};
  const auto same = [&](int64_t ld) { return rows == 1 || (ld - ldx) % 8 == 0; };
  a.vec = al(x, 16) && al(residual, 16) && al(residual_out, 16) && al(weight, 16) && al(q, 8) && same(ldq) &&
          (residual == nullptr || (same(ldr) && same(ldro)));
  a.whole = (rows == 1 || ldx % 8 == 0) && width % 8 == 0;
  return launch_add_norm_quant(a, dtype, q_dtype, (flags & QTTS_FLAG_PDL) != 0, static_cast<cudaStream_t>(stream));
}

// Residual addition, RMSNorm and 8-bit quantization of a row in one launch
// (qtts_add_rms_norm_quant): what stands between two W8A8 linears of a decoder
// layer (qtts/models/talker.py:249, 271 followed by qtts/quant/fp8.py:77-78 or
// int8.py:138-140 as separate ops).
//   h = x + residual;  y = w * (h * (1 / sqrt(mean(h^2) + eps)))
//   scale = max(max|y|, 1e-6) * fl32(1 / 448 or 1 / 127);  q = rne(y / scale)
// All of it in fp32 from the inputs to the codes: the stored residual is h
// rounded to its type, but the norm reads the unrounded sum and the quantizer
// the unrounded y, so one rounding (to 8 bits) separates the codes from the
// formula. A row that holds a NaN or an infinity gets a NaN scale, so that no
// finite codes stand for it.
#include <cuda_fp8.h>

#include "kernels.h"
#include "prologue.cuh"

namespace qtts {
namespace {

constexpr int kAnThreads = 256;

template <bool kMax>
__device__ __forceinline__ float block_reduce(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = kMax ? nan_max(v, w) : v + w;
  }
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = sh[0];
#pragma unroll
  for (int i = 1; i < kAnThreads / 32; ++i) r = kMax ? nan_max(r, sh[i]) : r + sh[i];
  __syncthreads();
  return r;
}

template <bool kInt8>
__device__ __forceinline__ uint8_t to_code(float y, float scale) {
  const float v = __fdiv_rn(y, scale);
  if constexpr (kInt8) {
    return static_cast<uint8_t>(static_cast<int8_t>(fminf(fmaxf(rintf(v), -127.f), 127.f)));
  } else {
    return static_cast<uint8_t>(__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3));
  }
}

template <typename XT, bool kInt8>
__global__ void __launch_bounds__(kAnThreads) add_norm_quant_kernel(const AddNormQuantArgs a) {
  __shared__ float sh[kAnThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x;
  const XT* x = static_cast<const XT*>(a.x) + row * a.ldx;
  const XT* r = a.residual != nullptr ? static_cast<const XT*>(a.residual) + row * a.ldr : nullptr;
  XT* ro = a.residual != nullptr ? static_cast<XT*>(a.residual_out) + row * a.ldro : nullptr;
  const XT* w = static_cast<const XT*>(a.weight);
  float ss = 0.f;
  for (int k = threadIdx.x; k < a.width; k += kAnThreads) {
    const float h = to_float(x[k]) + (r != nullptr ? to_float(r[k]) : 0.f);
    ss = fmaf(h, h, ss);
  }
  const float inv = rms_inv(block_reduce<false>(ss, sh), a.width, a.eps);
  float amax = 0.f;
  for (int k = threadIdx.x; k < a.width; k += kAnThreads) {
    const float h = to_float(x[k]) + (r != nullptr ? to_float(r[k]) : 0.f);
    amax = nan_max(amax, fabsf(rms_apply(h, inv, to_float(w[k]))));
  }
  const float scale = nan_max(block_reduce<true>(amax, sh), 1e-6f) * (kInt8 ? 1.0f / 127.0f : 1.0f / 448.0f);
  uint8_t* q = static_cast<uint8_t*>(a.q) + row * a.ldq;
  for (int k = threadIdx.x; k < a.width; k += kAnThreads) {
    const float h = to_float(x[k]) + (r != nullptr ? to_float(r[k]) : 0.f);
    q[k] = to_code<kInt8>(rms_apply(h, inv, to_float(w[k])), scale);
    if (r != nullptr) ro[k] = from_float<XT>(h);
  }
  if (threadIdx.x == 0) a.scale[row] = scale;
}

template <typename XT>
int launch_an(const AddNormQuantArgs& a, int q_dtype, bool pdl, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.rows);
  cfg.blockDim = dim3(kAnThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  const cudaError_t e = q_dtype == QTTS_INT8 ? cudaLaunchKernelEx(&cfg, add_norm_quant_kernel<XT, true>, a)
                                             : cudaLaunchKernelEx(&cfg, add_norm_quant_kernel<XT, false>, a);
  return e == cudaSuccess ? QTTS_OK : QTTS_ERR_LAUNCH;
}

}  // namespace

int launch_add_norm_quant(const AddNormQuantArgs& a, int dtype, int q_dtype, bool pdl, cudaStream_t stream) {
  switch (dtype) {
    case QTTS_BF16:
      return launch_an<__nv_bfloat16>(a, q_dtype, pdl, stream);
    case QTTS_FP16:
      return launch_an<__half>(a, q_dtype, pdl, stream);
    case QTTS_FP32:
      return launch_an<float>(a, q_dtype, pdl, stream);
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
  AddNormQuantArgs a{x, ldx, residual, ldr, weight, eps, residual_out, ldro, q, ldq, scale, rows, width, false};
  a.vec = width % 8 == 0 && al(x, 16) && al(residual, 16) && al(residual_out, 16) && al(weight, 16) && al(q, 8) &&
          (ldx * sz) % 16 == 0 && ldq % 8 == 0 &&
          (residual == nullptr || ((ldr * sz) % 16 == 0 && (ldro * sz) % 16 == 0));
  return launch_add_norm_quant(a, dtype, q_dtype, (flags & QTTS_FLAG_PDL) != 0, static_cast<cudaStream_t>(stream));
}

// Per-head RMSNorm, rotary positions with several axes and the 4-bit cache write
// of a fused projection's output, in one launch (qtts_rope_kv4_append).
//
// Input row of a token: [q heads | k heads | v heads], D channels each
// (MergedLinear's qkv order). Per head of q and k:
//   y = w * (x * (1 / sqrt(mean(x^2) + eps)))          (skipped without a weight)
//   (y[j], y[j + D/2]) turned by the angle of pair j    (skipped without tables)
// where the angle is the table's row for the position of the token along the axis
// that pair j belongs to (time, height, width for images and video; one axis for
// text). q is written in its own type, k and v as 4-bit groups (kv4.cuh). All of
// it in fp32 between the load and the one rounding of each output, each step of the
// formula rounded by itself (square root and divisions as IEEE has them, no product
// contracted with the sum that takes it) and the sum of squares in one fixed order:
// near the boundary between two codes a last bit decides, so the codes are those
// of the same steps as separate fp32 operations, bit for bit.
//
// D / 8 lanes hold one head row, eight neighbouring channels each: one 16-byte
// load, a pair's partner D / 16 lanes away, a group of 32 channels on four
// neighbouring lanes, and a lane's eight codes are exactly one 32-bit word of a
// key row or two 16-bit words of a value row.
//
// The projection's row is read once, q, codes and (where asked for) the stored
// values are written once: 8192 tokens of 16 + 2 x 8 heads of 128 channels, 145 MB,
// in 45 us (3.2 TB/s), which the instructions of norm, rotation and quantizer bound
// more than the memory does. (With an approximate root and weight, cosine and root
// folded into one factor it was 41 us, and codes near a boundary differed.) A lane's
// channels are the same in every head, so a warp takes several heads of one token and
// gathers its cosines and sines once; how many is chosen so that a short call still
// has a warp for every head pair and a long one few gathers. 28 such warps an SM, each
// with its next row under way, beat fewer with more registers (8192 tokens: 45 us; 24
// warps 47).
#include <type_traits>

#include "kernels.h"
#include "kv4.cuh"
#include "prologue.cuh"

namespace qtts {
namespace {

constexpr int kAhead = 1;  // passes whose rows are loaded ahead

// a / s for the s whose correctly rounded reciprocal is r: Markstein's correction of the
// product a * r by its remainder, which gives the correctly rounded quotient.
__device__ __forceinline__ float divide(float a, float s, float r) {
  const float q = a * r;
  return fmaf(fmaf(-q, s, a), r, q);
}

// Sum of squares of a head row, eight channels a lane; every lane of the row returns the same bits.
// One order, that of torch's mean over fp32: 128 channels as 32 sums of four neighbours, one after
// the other, 64 as they are; then the upper half is added to the lower until one sum is left. A
// step across lanes also shares out the sums that a lane holds, so that later steps have fewer.
template <int D>
__device__ __forceinline__ float row_sumsq(const float (&x)[8], int l) {
  const auto across = [](float v, int o) { return __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o)); };
  float p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] = __fmul_rn(x[i], x[i]);
  if constexpr (D == 128) {
    const float s0 = __fadd_rn(__fadd_rn(__fadd_rn(p[0], p[1]), p[2]), p[3]);
    const float s1 = __fadd_rn(__fadd_rn(__fadd_rn(p[4], p[5]), p[6]), p[7]);
    const bool up = (l & 8) != 0;
    float s = __fadd_rn(up ? s1 : s0, __shfl_xor_sync(0xffffffffu, up ? s0 : s1, 8));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) s = across(s, o);
    return across(s, 8);
  } else {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      const bool up = (l & o) != 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < o) {
          const float keep = up ? p[i + o] : p[i];
          p[i] = __fadd_rn(keep, __shfl_xor_sync(0xffffffffu, up ? p[i] : p[i + o], o));
        }
      }
    }
    float s = p[0];
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) s = across(s, o);
    return s;
  }
}

// The eight codes of a lane's channels; returns them one a nibble and gives the
// values that they stand for. lo/hi: minimum and maximum of the group.
__device__ __forceinline__ uint32_t quantize_group(const float (&y)[8], float lo, float hi, uint32_t& params,
                                                   float (&held)[8]) {
  const __nv_bfloat16 sb = __float2bfloat16_rn(divide(hi - lo, 15.0f, 1.0f / 15.0f));
  const __nv_bfloat16 zb = __float2bfloat16_rn(lo);
  params = static_cast<uint32_t>(__bfloat16_as_ushort(sb)) | (static_cast<uint32_t>(__bfloat16_as_ushort(zb)) << 16);
  const float s = __bfloat162float(sb), z = __bfloat162float(zb);
  // A scale below 2^-60 is divided by 2^64 times larger, as is what it divides, so that
  // reciprocal and remainder stay in range.
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = y[i] - z;
  float su = s;
  if (s < 0x1p-60f) {
    su *= 0x1p64f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= 0x1p64f;
  }
  const float r = s > 0.f ? __frcp_rn(su) : 0.f;
  float c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = fminf(fmaxf(divide(x[i], su, r), 0.f), 15.f);
    c[i] = (q + 12582912.f) - 12582912.f;  // 1.5 * 2^23: to the nearest whole number, ties to even
    held[i] = fmaf(c[i], s, z);            // c * s is exact
  }
  // Four codes at a time as one whole number below 2^16 in a float's low bits.
  const float a = fmaf(c[3], 4096.f, fmaf(c[2], 256.f, fmaf(c[1], 16.f, c[0])));
  const float b = fmaf(c[7], 4096.f, fmaf(c[6], 256.f, fmaf(c[5], 16.f, c[4])));
  return __byte_perm(__float_as_uint(a + 8388608.f), __float_as_uint(b + 8388608.f), 0x5410);
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&y)[8]) {
  uint4 o;
  T* r = reinterpret_cast<T*>(&o);
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = from_float<T>(y[i]);
  return o;
}

template <typename T, int D>
__global__ void __launch_bounds__(32, 28) rope_kv4_kernel(const RopeKv4Args a, int passes, int warps_a_token,
                                                           uint32_t token_inv, uint32_t page_inv) {
  constexpr int kLanes = D / 8;          // lanes a head row
  constexpr int kHeads = 32 / kLanes;    // head rows a pass of a warp
  constexpr int kGroups = D / kKv4Group;
  pdl_launch_dependents();
  pdl_wait();
  // One warp a CTA: token, passes and kinds are the CTA's, so every branch is uniform.
  const int lane = threadIdx.x;
  const int token = div_by(blockIdx.x, warps_a_token, token_inv);
  const int64_t t = token;
  const int l = lane % kLanes;
  const int sub = lane / kLanes;  // which of the pass's heads
  const int kvh = a.cache.kv_heads;
  // A pass takes kHeads heads of one kind: the q passes first, then k, then v.
  const int nq = (a.q_heads + kHeads - 1) / kHeads, nk = (kvh + kHeads - 1) / kHeads;
  const int p_first = (static_cast<int>(blockIdx.x) - token * warps_a_token) * passes;
  const int p_end = min(p_first + passes, nq + 2 * nk);
  const T* src = static_cast<const T*>(a.qkv) + t * a.ldqkv + 8 * l;

  // A token with a position outside the tables gives zeros and is not stored.
  bool ok = true;
  const int64_t slot = a.slots[t];
  int64_t pos[kMaxRopeAxes] = {};
  if (a.cos != nullptr) {
    // Axes that are not there read the last one: all loads at once, none under a condition.
#pragma unroll
    for (int x = 0; x < kMaxRopeAxes; ++x) pos[x] = a.positions[min(x, a.axes - 1) * a.ldpos + t];
#pragma unroll
    for (int x = 0; x < kMaxRopeAxes; ++x) {
      if (pos[x] < 0 || pos[x] >= a.table_len) {
        pos[x] = 0;
        ok = false;
      }
    }
    if (!ok && lane == 0) record_status(QTTS_ERR_SHAPE);
  }
  const bool inside = slot < a.cache.pages * a.cache.page_size;
  if (!inside && lane == 0) record_status(QTTS_ERR_SHAPE);
  const bool stored = ok && inside && slot >= 0;
  const int64_t page = !stored ? 0
                       : slot <= 0x7fffffff ? div_by(static_cast<int>(slot), a.cache.page_size, page_inv)
                                            : slot / a.cache.page_size;
  const int in_page = stored ? static_cast<int>(slot - page * a.cache.page_size) : 0;

  // Norm weights, cosines and signed sines of this lane's channels: gathered once for all heads of a
  // kind.
  uint4 fw = make_uint4(0u, 0u, 0u, 0u);
  float fa[8], fb[8];
  const auto factors = [&](const void* weight) {
    if (a.cos != nullptr) {
      const int j0 = 8 * (l % (kLanes / 2));  // first of this lane's pairs
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = j0 + i;
        const int axis = static_cast<int>(a.axis_of[j >> 5] >> (2 * (j & 31))) & 3;
        const int64_t at = (axis == 0 ? pos[0] : axis == 1 ? pos[1] : axis == 2 ? pos[2] : pos[3]) * (D / 2) + j;
        fa[i] = __ldg(a.cos + at);
        const float sn = __ldg(a.sin + at);
        fb[i] = l < kLanes / 2 ? -sn : sn;
      }
    }
    if (weight != nullptr) {
      fw = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(weight) + 8 * l));
    }
  };
  // Each step of the formula rounded once, none contracted with the next.
  const auto turn = [&](const uint4& raw, float(&y)[8], bool norm) {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = to_float(e[i]);
    if (norm) {
      const float inv = rms_inv(row_sumsq<D>(y, l), D, a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = rms_apply(y[i], inv, to_float(reinterpret_cast<const T*>(&fw)[i]));
    }
    if (a.cos != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float other = __shfl_xor_sync(0xffffffffu, y[i], kLanes / 2);
        y[i] = __fadd_rn(__fmul_rn(y[i], fa[i]), __fmul_rn(other, fb[i]));
      }
    }
  };
  // Codes, parameters and (where asked for) the values of a head row, through this lane's pointers.
  const auto quantize = [&](const float(&y)[8], bool live, uint8_t* codes, uint32_t* param, T* values, auto is_value) {
    float lo = y[0], hi = y[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) lo = nan_min(lo, y[i]), hi = nan_max(hi, y[i]);
#pragma unroll
    for (int o = 2; o > 0; o >>= 1) {
      lo = nan_min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = nan_max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    uint32_t params;
    float held[8];
    const uint32_t word = quantize_group(y, lo, hi, params, held);
    if (!live) return;
    if (a.k_values != nullptr) __stcs(reinterpret_cast<uint4*>(values), pack8<T>(held));
    if (stored) {
      if constexpr (decltype(is_value)::value) {
        *reinterpret_cast<uint16_t*>(codes) = static_cast<uint16_t>(word & 0xffffu);
        *reinterpret_cast<uint16_t*>(codes + 2 * kGroups) = static_cast<uint16_t>(word >> 16);
      } else {
        *reinterpret_cast<uint32_t*>(codes) = word;
      }
      if (l % 4 == 0) *param = params;
    }
  };

  // The passes of one kind that are this warp's, kAhead rows in flight. A lane beyond the kind's heads
  // loads the last one again and stores nothing. Everything that moves with the pass is a pointer.
  const auto run = [&](auto kind_c, int base, int count, const void* weight) {
    constexpr int kKind = decltype(kind_c)::value;
    const int kind_heads = kKind == 0 ? a.q_heads : kvh;
    const int from = max(p_first - base, 0), to = min(p_end - base, count);
    if (from >= to) return;
    const T* at = src + static_cast<int64_t>(kKind == 0 ? 0 : kKind == 1 ? a.q_heads : a.q_heads + kvh) * D;
    const auto fetch = [&](int p) {
      return __ldcs(reinterpret_cast<const uint4*>(at + min(min(p, to - 1) * kHeads + sub, kind_heads - 1) * D));
    };
    uint4 raw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) raw[u] = fetch(from + u);
    if constexpr (kKind < 2) factors(weight);
    const int h0 = from * kHeads + sub;
    T* out = nullptr;            // q, or the values
    uint8_t* codes = nullptr;    // this lane's place in the head's row
    uint32_t* params = nullptr;  // its group's
    int64_t codes_step = 0, params_step = 0;
    if constexpr (kKind == 0) {
      out = static_cast<T*>(a.q_out) + t * a.ldq + h0 * D + 8 * l;
    } else {
      out = static_cast<T*>(kKind == 1 ? a.k_values : a.v_values) + (t * kvh + h0) * D + 8 * l;
      const int64_t row = kv4_row(a.cache, page, h0, in_page);
      const int j = l / 4, c = l % 4;
      codes = (kKind == 1 ? a.cache.k_codes : a.cache.v_codes) + row * (D / 2) +
              (kKind == 1 ? 4 * (c * kGroups + j) : 2 * (2 * c * kGroups + j));
      params = (kKind == 1 ? a.cache.k_params : a.cache.v_params) + row * kGroups + j;
      codes_step = static_cast<int64_t>(kHeads) * a.cache.page_size * (D / 2);
      params_step = static_cast<int64_t>(kHeads) * a.cache.page_size * kGroups;
    }
    for (int p0 = from; p0 < to; p0 += kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int p = p0 + u;
        if (p < to) {
          const uint4 now = raw[u];
          if (p + kAhead < to) raw[u] = fetch(p + kAhead);
          const bool live = p * kHeads + sub < kind_heads;
          float y[8];
          if constexpr (kKind < 2) {
            turn(now, y, weight != nullptr);
          } else {
            const T* e = reinterpret_cast<const T*>(&now);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = to_float(e[i]);
          }
          if (!ok) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = 0.f;
          }
          if constexpr (kKind == 0) {
            if (live) *reinterpret_cast<uint4*>(out) = pack8<T>(y);
          } else {
            quantize(y, live, codes, params, out, std::integral_constant<bool, kKind == 2>{});
            codes += codes_step, params += params_step;
          }
          out += kHeads * D;
        }
      }
    }
  };
  run(std::integral_constant<int, 0>{}, 0, nq, a.q_norm);
  run(std::integral_constant<int, 1>{}, nq, nk, a.k_norm);
  run(std::integral_constant<int, 2>{}, nq + nk, nk, nullptr);
}

template <typename T, int D>
int launch_rk(const RopeKv4Args& a, bool pdl, cudaStream_t stream) {
  constexpr int kHeads = 32 / (D / 8);
  // Passes a token needs.
  const int total = (a.q_heads + kHeads - 1) / kHeads + 2 * ((a.cache.kv_heads + kHeads - 1) / kHeads);
  // A warp for every pass while that is less than 32 warps an SM, about as many as are resident;
  // then longer warps, which gather their angles once, up to 16 passes. A warp's passes follow
  // one another, so longer ones before the SMs are full only wait (from 4 | 16 | 32 warps an SM on:
  // 333 tokens of 16 + 2 x 8 heads of 128 channels 10.9 | 6.5 | 6.1 us, 1000 tokens 15.7 | 11.4 | 9.4,
  // 333 of 32 + 2 x 4 heads of 64 channels 6.2 | 5.6 | 5.3; 8192 tokens 45 each way).
  int passes = 1;
  while (passes < 16 && passes < total && static_cast<int64_t>(a.tokens) * total >= 32ll * kNumSMs * passes) passes *= 2;
  const int warps_a_token = (total + passes - 1) / passes;
  const int64_t warps = static_cast<int64_t>(a.tokens) * warps_a_token;
  cudaLaunchConfig_t cfg = {};
  if (warps > 0x7fffffff) return QTTS_ERR_SHAPE;
  cfg.gridDim = dim3(static_cast<unsigned>(warps));
  cfg.blockDim = dim3(32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, rope_kv4_kernel<T, D>, a, passes, warps_a_token,
                            0xffffffffu / static_cast<uint32_t>(warps_a_token),
                            0xffffffffu / static_cast<uint32_t>(a.cache.page_size)) == cudaSuccess
             ? QTTS_OK
             : QTTS_ERR_LAUNCH;
}

}  // namespace

int launch_rope_kv4(const RopeKv4Args& a, int dtype, int head_dim, bool pdl, cudaStream_t stream) {
  if (dtype == QTTS_BF16) {
    return head_dim == 128 ? launch_rk<__nv_bfloat16, 128>(a, pdl, stream)
                           : launch_rk<__nv_bfloat16, 64>(a, pdl, stream);
  }
  return head_dim == 128 ? launch_rk<__half, 128>(a, pdl, stream) : launch_rk<__half, 64>(a, pdl, stream);
}

}  // namespace qtts

extern "C" int qtts_rope_kv4_append(const void* qkv, int64_t ldqkv, int dtype, int tokens, int q_heads, int kv_heads,
                                    int head_dim, const void* q_norm, const void* k_norm, float eps,
                                    const float* cos, const float* sin, int64_t table_len, const int64_t* positions,
                                    int64_t ldpos, int axes, const int* sections, int interleaved,
                                    const int64_t* slots, void* q_out, int64_t ldq, uint8_t* k_codes, void* k_params,
                                    uint8_t* v_codes, void* v_params, int64_t pages, int page_size, void* k_values,
                                    void* v_values, unsigned flags, void* stream) {
  using namespace qtts;
  if (tokens < 0 || q_heads < 0 || kv_heads < 1 || q_heads > 4096 || kv_heads > 4096) return QTTS_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128) return QTTS_ERR_SHAPE;
  if (pages < 0 || page_size < 1) return QTTS_ERR_SHAPE;
  if (dtype != QTTS_BF16 && dtype != QTTS_FP16) return QTTS_ERR_DTYPE;
  if (tokens == 0) return QTTS_OK;
  if (qkv == nullptr || slots == nullptr || (q_heads > 0 && q_out == nullptr)) return QTTS_ERR_NULL;
  if (pages > 0 && (k_codes == nullptr || k_params == nullptr || v_codes == nullptr || v_params == nullptr)) {
    return QTTS_ERR_NULL;
  }
  if ((cos == nullptr) != (sin == nullptr) || (cos != nullptr && (positions == nullptr || sections == nullptr))) {
    return QTTS_ERR_NULL;
  }
  if ((k_values == nullptr) != (v_values == nullptr)) return QTTS_ERR_NULL;
  const int64_t width = static_cast<int64_t>(q_heads + 2 * kv_heads) * head_dim;
  if (ldqkv < width || ldq < static_cast<int64_t>(q_heads) * head_dim) return QTTS_ERR_SHAPE;
  const auto al = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!al(qkv, 16) || !al(q_out, 16) || !al(q_norm, 16) || !al(k_norm, 16) || !al(k_values, 16) ||
      !al(v_values, 16) || !al(k_codes, 16) || !al(v_codes, 16) || !al(k_params, 16) || !al(v_params, 16) ||
      ldqkv % 8 != 0 || ldq % 8 != 0 || !al(cos, 4) || !al(sin, 4) || !al(positions, 8) || !al(slots, 8)) {
    return QTTS_ERR_ALIGN;
  }
  RopeKv4Args a{};
  if (cos != nullptr) {
    if (axes < 1 || axes > kMaxRopeAxes || table_len < 1 || ldpos < tokens) return QTTS_ERR_SHAPE;
    int sum = 0;
    for (int x = 0; x < axes; ++x) {
      if (sections[x] < 0 || sections[x] > head_dim / 2) return QTTS_ERR_SHAPE;
      sum += sections[x];
    }
    if (sum != head_dim / 2) return QTTS_ERR_SHAPE;
    for (int j = 0; j < head_dim / 2; ++j) {
      int axis = 0;
      if (interleaved) {
        // 0 1 2 0 1 2 ...; an axis that has had its share leaves its turns to axis 0.
        axis = j % axes;
        if (j >= axes * sections[axis]) axis = 0;
      } else {
        for (int end = sections[0]; j >= end; end += sections[axis]) ++axis;
      }
      a.axis_of[j >> 5] |= static_cast<uint64_t>(axis) << (2 * (j & 31));
    }
  }
  const int dev_ok = check_device();
  if (dev_ok != QTTS_OK) return dev_ok;
  a.qkv = qkv;
  a.ldqkv = ldqkv;
  a.tokens = tokens;
  a.q_heads = q_heads;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.eps = eps;
  a.cos = cos;
  a.sin = sin;
  a.table_len = table_len;
  a.positions = positions;
  a.ldpos = ldpos;
  a.axes = axes;
  a.slots = slots;
  a.q_out = q_out;
  a.ldq = ldq;
  a.cache = Kv4Cache{k_codes, static_cast<uint32_t*>(k_params), v_codes, static_cast<uint32_t*>(v_params), pages,
                     page_size, kv_heads};
  a.k_values = k_values;
  a.v_values = v_values;
  return launch_rope_kv4(a, dtype, head_dim, (flags & QTTS_FLAG_PDL) != 0, static_cast<cudaStream_t>(stream));
}

// Attention over a paged key/value cache held in 4 bits (qtts_kv4_attention):
//   out[i, h] = sum_t softmax_t( scale * q[i, h] . k[t, h'] ) v[t, h'],  h' = h / (heads / kv_heads)
// over the tokens t that row i of its request sees: t <= len - n + i with `causal`
// (its n new tokens are the last of the len cached ones), t < len without. A row
// that sees nothing gives zeros.
//
// One CTA per (new token, head): tiles of 128 tokens, one token a thread for the
// scores, one channel a thread for the weighted sum, running maximum and sum.
#include "kernels.h"
#include "kv4.cuh"

namespace qtts {
namespace {

constexpr int kKaThreads = 128;

// First and number of new tokens of request b, checked against the arguments.
__device__ __forceinline__ bool request_rows(const Kv4AttnArgs& a, int b, int& start, int& n) {
  if (a.q_starts == nullptr) {
    start = b * a.max_q;
    n = a.max_q;
    return true;
  }
  start = a.q_starts[b];
  n = a.q_starts[b + 1] - start;
  return start >= 0 && n >= 0 && n <= a.max_q && start <= a.total_q - n;
}

template <typename T, int D>
__global__ void __launch_bounds__(kKaThreads) kv4_attention_kernel(const Kv4AttnArgs a) {
  constexpr int kGroups = D / kKv4Group;
  __shared__ float qs[D];
  __shared__ float ps[kKaThreads];
  __shared__ int64_t rows[kKaThreads];
  __shared__ float red[4];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x;
  const int b = blockIdx.z, i = blockIdx.x, head = blockIdx.y;
  int start, n;
  if (!request_rows(a, b, start, n)) {
    if (tid == 0) record_status(QTTS_ERR_SHAPE);
    return;
  }
  if (i >= n) return;
  int len = a.lengths[b];
  if (len < 0 || len > static_cast<int64_t>(a.table_cols) * a.cache.page_size) {
    if (tid == 0) record_status(QTTS_ERR_SHAPE);
    len = 0;
  }
  const int sees = a.causal ? max(0, len - n + i + 1) : len;
  const int kvh = head / (a.q_heads / a.cache.kv_heads);
  const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(start + i) * a.q_token_stride + head * a.q_head_stride;
  if (tid < D) qs[tid] = to_float(q[tid]);
  __syncthreads();
  float m = -INFINITY, sum = 0.f, acc = 0.f;
  for (int t0 = 0; t0 < sees; t0 += kKaThreads) {
    const int t = t0 + tid;
    float s = -INFINITY;
    int64_t row = -1;
    if (t < sees) {
      const int page = a.table[b * a.ld_table + t / a.cache.page_size];
      if (page < 0 || page >= a.cache.pages) {
        record_status(QTTS_ERR_SHAPE);
      } else {
        row = kv4_row(a.cache, page, kvh, t % a.cache.page_size);
        const uint32_t* w = reinterpret_cast<const uint32_t*>(a.cache.k_codes + row * (D / 2));
        s = 0.f;
        for (int ch = 0; ch < D; ++ch) {
          const uint32_t p = a.cache.k_params[row * kGroups + ch / 32];
          const uint32_t word = w[((ch % 32) / 8) * kGroups + ch / 32];
          s = fmaf(qs[ch], fmaf(static_cast<float>((word >> (4 * (ch % 8))) & 15u), kv4_scale(p), kv4_min(p)), s);
        }
        s *= a.scale;
      }
    }
    rows[tid] = row;
    float mt = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
    if ((tid & 31) == 0) red[tid >> 5] = mt;
    __syncthreads();
    const float mn = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
    const float safe = mn == -INFINITY ? 0.f : mn;
    const float f = expf(m - safe);
    ps[tid] = expf(s - safe);
    m = mn;
    __syncthreads();
    sum *= f;
    acc *= f;
    for (int u = 0; u < kKaThreads; ++u) {
      const int64_t r = rows[u];
      if (r < 0) continue;
      sum += ps[u];
      if (tid < D) {
        const uint32_t p = a.cache.v_params[r * kGroups + tid / 32];
        const uint16_t* w = reinterpret_cast<const uint16_t*>(a.cache.v_codes + r * (D / 2));
        const uint32_t code = (w[((tid % 32) / 4) * kGroups + tid / 32] >> (4 * (tid % 4))) & 15u;
        acc = fmaf(ps[u], fmaf(static_cast<float>(code), kv4_scale(p), kv4_min(p)), acc);
      }
    }
    __syncthreads();
  }
  if (tid < D) {
    static_cast<T*>(a.out)[static_cast<int64_t>(start + i) * a.out_token_stride + head * D + tid] =
        from_float<T>(sum > 0.f || sum != sum ? acc / sum : 0.f);
  }
}

template <typename T, int D>
int launch_ka(const Kv4AttnArgs& a, bool pdl, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.max_q, a.q_heads, a.batch);
  cfg.blockDim = dim3(kKaThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kv4_attention_kernel<T, D>, a) == cudaSuccess ? QTTS_OK : QTTS_ERR_LAUNCH;
}

}  // namespace

int launch_kv4_attention(const Kv4AttnArgs& a, int dtype, int head_dim, bool pdl, cudaStream_t stream) {
  if (dtype == QTTS_BF16) {
    return head_dim == 128 ? launch_ka<__nv_bfloat16, 128>(a, pdl, stream)
                           : launch_ka<__nv_bfloat16, 64>(a, pdl, stream);
  }
  return head_dim == 128 ? launch_ka<__half, 128>(a, pdl, stream) : launch_ka<__half, 64>(a, pdl, stream);
}

}  // namespace qtts

extern "C" int qtts_kv4_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype,
                                  const uint8_t* k_codes, const void* k_params, const uint8_t* v_codes,
                                  const void* v_params, int64_t pages, int page_size, const int32_t* block_table,
                                  int64_t ld_table, int table_cols, const int32_t* lengths, const int32_t* q_starts,
                                  int total_q, int max_q, int batch, int q_heads, int kv_heads, int head_dim,
                                  float scale, int causal, void* out, int64_t out_token_stride, unsigned flags,
                                  void* stream) {
  using namespace qtts;
  if (batch < 0 || batch > 65535 || total_q < 0 || max_q < 0 || max_q > total_q) return QTTS_ERR_SHAPE;
  if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0 || q_heads > 4096) return QTTS_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128) return QTTS_ERR_SHAPE;
  if (pages < 0 || page_size < 16 || page_size % 16 != 0 || table_cols < 0 || ld_table < table_cols) {
    return QTTS_ERR_SHAPE;
  }
  if (dtype != QTTS_BF16 && dtype != QTTS_FP16) return QTTS_ERR_DTYPE;
  if (batch == 0 || total_q == 0 || max_q == 0) return QTTS_OK;
  if (q_starts == nullptr && static_cast<int64_t>(batch) * max_q != total_q) return QTTS_ERR_SHAPE;
  if (static_cast<int64_t>(table_cols) * page_size > 0x7fffffff) return QTTS_ERR_SHAPE;
  if (q == nullptr || out == nullptr || lengths == nullptr) return QTTS_ERR_NULL;
  if (table_cols > 0 && block_table == nullptr) return QTTS_ERR_NULL;
  if (pages > 0 && (k_codes == nullptr || k_params == nullptr || v_codes == nullptr || v_params == nullptr)) {
    return QTTS_ERR_NULL;
  }
  if (q_head_stride < head_dim || q_token_stride < 0 ||
      out_token_stride < static_cast<int64_t>(q_heads) * head_dim) {
    return QTTS_ERR_SHAPE;
  }
  const auto al = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!al(q, 16) || !al(out, 16) || !al(k_codes, 16) || !al(k_params, 16) || !al(v_codes, 16) || !al(v_params, 16) ||
      q_token_stride % 8 != 0 || q_head_stride % 8 != 0 || out_token_stride % 8 != 0 || !al(block_table, 4) ||
      !al(lengths, 4) || !al(q_starts, 4)) {
    return QTTS_ERR_ALIGN;
  }
  const int dev_ok = check_device();
  if (dev_ok != QTTS_OK) return dev_ok;
  Kv4AttnArgs a{};
  a.q = q;
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.cache = Kv4Cache{const_cast<uint8_t*>(k_codes), static_cast<uint32_t*>(const_cast<void*>(k_params)),
                     const_cast<uint8_t*>(v_codes), static_cast<uint32_t*>(const_cast<void*>(v_params)), pages,
                     page_size, kv_heads};
  a.table = block_table;
  a.ld_table = ld_table;
  a.table_cols = table_cols;
  a.lengths = lengths;
  a.q_starts = q_starts;
  a.total_q = total_q;
  a.max_q = max_q;
  a.batch = batch;
  a.q_heads = q_heads;
  a.scale = scale;
  a.causal = causal;
  a.out = out;
  a.out_token_stride = out_token_stride;
  return launch_kv4_attention(a, dtype, head_dim, (flags & QTTS_FLAG_PDL) != 0, static_cast<cudaStream_t>(stream));
}

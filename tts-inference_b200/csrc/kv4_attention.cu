// Attention over a paged key/value cache held in 4 bits (qtts_kv4_attention):
//   out[i, h] = sum_t softmax_t( scale * q[i, h] . k[t, h'] ) v[t, h'],  h' = h / (heads / kv_heads)
// over the tokens t that row i of its request sees: t <= len - n + i with `causal`
// (its n new tokens are the last of the len cached ones), t < len without. A row
// that sees nothing gives zeros.
//
// Few rows a request (decode steps, short chunks). What bounds it is reading the
// cache once, 0.625 bytes an element, and almost as much the instructions that
// turn nibbles into matrix operands, so those are kept few:
//   * scores as S^T = K q^T with mma.sync m16n8k16: 16 tokens by 8 rows, a row
//     being a (new token, query head) pair that shares the key head. A nibble is
//     ORed into the mantissa of a power of two (128 + code in bf16, 1024 + code in
//     fp16: exact); the accumulator starts at minus that power times the sum of
//     the row's q over the group, so it ends as sum(q * code), and the group's
//     scale and minimum enter once per (token, row, group), in fp32;
//   * out^T = V^T P^T: two tokens' half-words are interleaved by a byte permute, so
//     a nibble mask again gives operand pairs. The probability times the value's
//     scale is what is rounded to bf16; sum p (code - 8) scale + p (minimum + 8 scale)
//     keeps the rounded part as small as the values themselves. The 128 + 8 is
//     taken out with one more product per group by a constant row of -136 with the
//     same rounded probabilities, exactly as it went in;
//   * every warp streams its own tiles of 32 tokens through a ring of bulk copies
//     and keeps its own running maximum and sum; the warps of a CTA meet in shared
//     memory, and where there are few (request, head) pairs a cluster of up to 16
//     CTAs splits one of them and meets in distributed shared memory: one launch,
//     no workspace, sums in a fixed order.
#include <type_traits>

#include "kernels.h"
#include "kv4.cuh"

namespace qtts {
namespace {

constexpr int kTile = 32;   // tokens a warp takes at a time
constexpr int kStages = 2;  // tiles in flight a warp

__device__ __forceinline__ uint32_t nib_pair(uint32_t w, int n, uint32_t magic) {
  return ((w >> (4 * n)) & 0x000F000Fu) | magic;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// First row and number of new tokens of request b, checked against the arguments.
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

template <int D>
struct RowsSmem {
  static constexpr int kCodes = kTile * D / 2;              // bytes of a tile's key (or value) codes
  static constexpr int kParams = kTile * (D / kKv4Group) * 4;
  static constexpr int kStage = 2 * (kCodes + kParams);
  static constexpr int kWarpRing = kStages * kStage;
  static constexpr int kPitch = D + 4;  // floats a partial output row: lanes of one store hit different banks
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(256, NT == 1 ? 2 : 1) kv4_rows_kernel(const Kv4AttnArgs a, int row_blocks,
                                                                        uint64_t wait_ns) {
  using S = RowsSmem<D>;
  constexpr int NG = D / kKv4Group;
  constexpr int kRows = 8 * NT;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kMagicK = kBf16 ? 0x43004300u : 0x64006400u;
  constexpr float kBaseK = kBf16 ? 128.f : 1024.f;
  constexpr uint32_t kMagicV = 0x43004300u;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[8][kStages];
  __shared__ float stat_m[8][kRows], stat_l[8][kRows];  // of each warp
  __shared__ float part_m[kRows], part_l[kRows];        // of the CTA

  const int warps = blockDim.x >> 5;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int splits = gridDim.x;
  const int rank = blockIdx.x;
  const int rb = blockIdx.y % row_blocks;
  const int kvh = blockIdx.y / row_blocks;
  const int b = blockIdx.z;
  if (lane < kStages) mbar_init(&full[warp][lane], 1);
  fence_mbarrier_init();
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait();

  int start = 0, n = 0;
  bool fine = request_rows(a, b, start, n);
  int len = a.lengths[b];
  fine = fine && len >= 0 && len <= static_cast<int64_t>(a.table_cols) * a.cache.page_size &&
         (len == 0 || a.cache.pages > 0);
  if (!fine) {
    if (threadIdx.x == 0) record_status(QTTS_ERR_SHAPE);
    len = 0;
    if (!request_rows(a, b, start, n)) n = 0;  // rows that cannot be told are not written
  }
  const int share = a.q_heads / a.cache.kv_heads;
  const int rows = n * share;
  const int r0 = rb * kRows;
  // Tokens that any row of this block sees.
  const int last = (min(rows, r0 + kRows) - 1) / share;  // its last new token
  const int first_lim = a.causal ? len - n + r0 / share + 1 : len;  // what its first row sees (may be negative)
  const int kmax = r0 >= rows ? 0 : max(0, a.causal ? len - n + last + 1 : len);
  const int tiles = (kmax + kTile - 1) / kTile;

  // This warp's tiles: every (splits * warps)-th one.
  uint8_t* ring = smem + warp * S::kWarpRing;
  const int step = splits * warps;
  const int t_first = rank * warps + warp;
  const int32_t* table = a.table + b * a.ld_table;
  auto issue = [&](int tile, int stage) {  // lane 0: the tile's rows, in 16-token runs that lie in one page
    uint8_t* dst = ring + stage * S::kStage;
    const int t0 = tile * kTile;
    const int runs = t0 + 16 < kmax ? 2 : 1;
    mbar_arrive_expect_tx(&full[warp][stage], static_cast<uint32_t>(runs * (S::kStage / 2)));
    int64_t row[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      row[h] = 0;
      if (h < runs) {
        const int t = t0 + 16 * h;
        const int col = t / a.cache.page_size;
        int64_t page = table[col];
        if (page < 0 || page >= a.cache.pages) {
          record_status(QTTS_ERR_SHAPE);
          page = 0;
        }
        row[h] = kv4_row(a.cache, page, kvh, t - col * a.cache.page_size);
      }
    }
    const bool joined = runs == 2 && row[1] == row[0] + 16;
    const int copies = joined ? 1 : runs;
    for (int h = 0; h < copies; ++h) {
      const int m = joined ? 2 : 1;
      const int64_t r = row[h];
      bulk_load(dst + h * (S::kCodes / 2), a.cache.k_codes + r * (D / 2), m * S::kCodes / 2, &full[warp][stage]);
      bulk_load(dst + S::kCodes + h * (S::kParams / 2), a.cache.k_params + r * NG, m * S::kParams / 2,
                &full[warp][stage]);
      bulk_load(dst + S::kCodes + S::kParams + h * (S::kCodes / 2), a.cache.v_codes + r * (D / 2), m * S::kCodes / 2,
                &full[warp][stage]);
      bulk_load(dst + 2 * S::kCodes + S::kParams + h * (S::kParams / 2), a.cache.v_params + r * NG,
                m * S::kParams / 2, &full[warp][stage]);
    }
  };
  if (lane == 0) {
    for (int s = 0; s < kStages && t_first + s * step < tiles; ++s) issue(t_first + s * step, s);
  }

  // q as the B operand: row 8 nt + g, channels 32j + 8c .. + 7 as pairs (i, i + 4); and the
  // sums over each group of the rows 8 nt + 2c, + 1, whose scores this lane holds.
  uint32_t qf[NT][NG][4];
  float qsum[NT][NG][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = r0 + 8 * nt + g;
    const T* qr = static_cast<const T*>(a.q) + static_cast<int64_t>(start + r / share) * a.q_token_stride +
                  (kvh * share + r % share) * a.q_head_stride + 8 * c;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows) u = *reinterpret_cast<const uint4*>(qr + 32 * j);
      qf[nt][j][0] = __byte_perm(u.x, u.z, 0x5410);
      qf[nt][j][1] = __byte_perm(u.x, u.z, 0x7632);
      qf[nt][j][2] = __byte_perm(u.y, u.w, 0x5410);
      qf[nt][j][3] = __byte_perm(u.y, u.w, 0x7632);
      const T* e = reinterpret_cast<const T*>(&u);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += to_float(e[i]);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      qsum[nt][j][0] = __shfl_sync(0xffffffffu, sum, (2 * c) * 4);
      qsum[nt][j][1] = __shfl_sync(0xffffffffu, sum, (2 * c + 1) * 4);
    }
  }
  int lim[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = (r0 + 8 * nt + 2 * c + e) / share;
      lim[nt][e] = a.causal ? min(len - n + i + 1, kmax) : len;
    }
  }
  const float to_log2 = a.scale * 1.4426950408889634f;

  float m[NT][2], l[NT][2], zacc[NT][NG][2];
  float acc[NT][NG][2][4];  // [group][channel pair] of out^T, fp32
  float csum[NT][4];        // row j: -136 * sum of the rounded probabilities * scale of group j
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) m[nt][e] = -INFINITY, l[nt][e] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) csum[nt][e] = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) zacc[nt][j][e] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][j][h][e] = 0.f;
      }
    }
  }

  // Token of row slot s of a 16-token operand: s with the last bit turned in every other
  // pair, so that neither the key nor the value loads below hit one bank with more than two rows.
  const int kslot = g ^ ((g >> 1) & 1);
  const int v0 = (2 * c) ^ (c & 1), v1 = (2 * c + 1) ^ (c & 1);

  int it = 0;
  bool tile_failed = false;
  for (int tile = t_first; tile < tiles; tile += step, ++it) {
    const int stage = it % kStages;
    const bool got = mbar_wait_bounded(&full[warp][stage], (it / kStages) & 1, wait_ns);
    if (!__all_sync(0xffffffffu, got)) {
      if (lane == 0) record_status(QTTS_ERR_TIMEOUT);
      tile_failed = true;
      break;
    }
    const uint8_t* kc = ring + stage * S::kStage;
    const uint8_t* kp = kc + S::kCodes;
    const uint8_t* vc = kp + S::kParams;
    const uint8_t* vp = vc + S::kCodes;
    const int t0 = tile * kTile;

    // Scores of 2 x 16 tokens: s[nt][mt][token half][row of the pair].
    float s[NT][2][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      uint32_t kw[2][NG], pw[2][NG];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = 16 * mt + 8 * h + kslot;
        if constexpr (NG == 4) {
          *reinterpret_cast<uint4*>(kw[h]) = *reinterpret_cast<const uint4*>(kc + t * 64 + 16 * c);
          *reinterpret_cast<uint4*>(pw[h]) = *reinterpret_cast<const uint4*>(kp + t * 16);
        } else {
          *reinterpret_cast<uint2*>(kw[h]) = *reinterpret_cast<const uint2*>(kc + t * 32 + 8 * c);
          *reinterpret_cast<uint2*>(pw[h]) = *reinterpret_cast<const uint2*>(kp + t * 8);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][mt][e] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        uint32_t a0[4], a1[4];
        a0[0] = nib_pair(kw[0][j], 0, kMagicK), a0[1] = nib_pair(kw[1][j], 0, kMagicK);
        a0[2] = nib_pair(kw[0][j], 1, kMagicK), a0[3] = nib_pair(kw[1][j], 1, kMagicK);
        a1[0] = nib_pair(kw[0][j], 2, kMagicK), a1[1] = nib_pair(kw[1][j], 2, kMagicK);
        a1[2] = nib_pair(kw[0][j], 3, kMagicK), a1[3] = nib_pair(kw[1][j], 3, kMagicK);
        const float sc0 = kv4_scale(pw[0][j]), sc1 = kv4_scale(pw[1][j]);
        const float z0 = kv4_min(pw[0][j]), z1 = kv4_min(pw[1][j]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float d[4];
          d[0] = d[2] = -kBaseK * qsum[nt][j][0];
          d[1] = d[3] = -kBaseK * qsum[nt][j][1];
          Mma16816<T>::run(d, a0, qf[nt][j][0], qf[nt][j][1]);
          Mma16816<T>::run(d, a1, qf[nt][j][2], qf[nt][j][3]);
          s[nt][mt][0] = fmaf(sc0, d[0], fmaf(z0, qsum[nt][j][0], s[nt][mt][0]));
          s[nt][mt][1] = fmaf(sc0, d[1], fmaf(z0, qsum[nt][j][1], s[nt][mt][1]));
          s[nt][mt][2] = fmaf(sc1, d[2], fmaf(z1, qsum[nt][j][0], s[nt][mt][2]));
          s[nt][mt][3] = fmaf(sc1, d[3], fmaf(z1, qsum[nt][j][1], s[nt][mt][3]));
        }
      }
    }
    const bool masked = t0 + kTile > first_lim;  // some row does not see all of the tile
    if (masked) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = t0 + 16 * mt + 8 * (e >> 1) + kslot;
            if (t >= lim[nt][e & 1]) s[nt][mt][e] = -INFINITY;
          }
        }
      }
    }

    // Running maximum (in units of log2) and sum; p replaces s.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mx[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = fmaxf(fmaxf(s[nt][0][e], s[nt][0][e + 2]), fmaxf(s[nt][1][e], s[nt][1][e + 2]));
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], o));
        mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], o));
      }
      // scale > 0: the largest score stays the largest.
      mx[0] = fmaxf(m[nt][0], mx[0] * to_log2);
      mx[1] = fmaxf(m[nt][1], mx[1] * to_log2);
      const bool moved = mx[0] > m[nt][0] || mx[1] > m[nt][1];
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f = mx[e] > m[nt][e] ? ex2(m[nt][e] - mx[e]) : 1.f;
          m[nt][e] = mx[e];
          l[nt][e] *= f;
          csum[nt][e] *= f;
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            zacc[nt][j][e] *= f;
            acc[nt][j][0][e] *= f, acc[nt][j][0][e + 2] *= f;
            acc[nt][j][1][e] *= f, acc[nt][j][1][e + 2] *= f;
          }
        }
      }
      const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0];
      const float m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt][mt][e] = ex2(fmaf(s[nt][mt][e], to_log2, -((e & 1) ? m1 : m0)));
          l[nt][e & 1] += s[nt][mt][e];
        }
      }
    }

    // Weighted values.
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      uint32_t vw[4][NG / 2], pw[2][NG];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int ta = 16 * mt + 8 * h + v0, tb = 16 * mt + 8 * h + v1, tp = 16 * mt + 8 * h + kslot;
        if constexpr (NG == 4) {
          *reinterpret_cast<uint2*>(vw[2 * h]) = *reinterpret_cast<const uint2*>(vc + ta * 64 + 8 * g);
          *reinterpret_cast<uint2*>(vw[2 * h + 1]) = *reinterpret_cast<const uint2*>(vc + tb * 64 + 8 * g);
          *reinterpret_cast<uint4*>(pw[h]) = *reinterpret_cast<const uint4*>(vp + tp * 16);
        } else {
          vw[2 * h][0] = *reinterpret_cast<const uint32_t*>(vc + ta * 32 + 4 * g);
          vw[2 * h + 1][0] = *reinterpret_cast<const uint32_t*>(vc + tb * 32 + 4 * g);
          *reinterpret_cast<uint2*>(pw[h]) = *reinterpret_cast<const uint2*>(vp + tp * 8);
        }
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        // Tokens (2c, 2c + 1) and (2c + 8, 2c + 9) of group j, interleaved by half-words.
        const uint32_t xa = __byte_perm(vw[0][j / 2], vw[1][j / 2], (j & 1) ? 0x7632 : 0x5410);
        const uint32_t xb = __byte_perm(vw[2][j / 2], vw[3][j / 2], (j & 1) ? 0x7632 : 0x5410);
        uint32_t a0[4], a1[4];
        a0[0] = nib_pair(xa, 0, kMagicV), a0[1] = nib_pair(xa, 1, kMagicV);
        a0[2] = nib_pair(xb, 0, kMagicV), a0[3] = nib_pair(xb, 1, kMagicV);
        a1[0] = nib_pair(xa, 2, kMagicV), a1[1] = nib_pair(xa, 3, kMagicV);
        a1[2] = nib_pair(xb, 2, kMagicV), a1[3] = nib_pair(xb, 3, kMagicV);
        const uint32_t bias = g == j ? 0xC308C308u : 0u;  // (-136, -136)
        const uint32_t ab[4] = {bias, 0u, bias, 0u};
        const float sc0 = kv4_scale(pw[0][j]), sc1 = kv4_scale(pw[1][j]);
        const float z0 = fmaf(8.f, sc0, kv4_min(pw[0][j])), z1 = fmaf(8.f, sc1, kv4_min(pw[1][j]));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float* p = s[nt][mt];
          float w[4] = {p[0] * sc0, p[1] * sc0, p[2] * sc1, p[3] * sc1};
          float y[4] = {p[0] * z0, p[1] * z0, p[2] * z1, p[3] * z1};
          if (masked) {  // what a row does not see stays out even where it is NaN
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[e] = p[e] == 0.f ? 0.f : w[e];
              y[e] = p[e] == 0.f ? 0.f : y[e];
            }
          }
          zacc[nt][j][0] += y[0] + y[2];
          zacc[nt][j][1] += y[1] + y[3];
          const uint32_t b0 = transpose8x8(pack_bf16(w[0], w[1]));
          const uint32_t b1 = transpose8x8(pack_bf16(w[2], w[3]));
          Mma16816<__nv_bfloat16>::run(acc[nt][j][0], a0, b0, b1);
          Mma16816<__nv_bfloat16>::run(acc[nt][j][1], a1, b0, b1);
          Mma16816<__nv_bfloat16>::run(csum[nt], ab, b0, b1);
        }
      }
    }
    __syncwarp();
    if (lane == 0 && tile + kStages * step < tiles) issue(tile + kStages * step, stage);
  }
  if (tile_failed) {  // copies still in flight must land before their memory is used again
    for (int s = 0; s < kStages; ++s) (void)mbar_wait_bounded(&full[warp][(it + s) % kStages], ((it + s) / kStages) & 1, wait_ns);
  }

  // Finish the warp: the rest of the sums over its lanes, then its partial outputs.
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], o);
#pragma unroll
        for (int j = 0; j < NG; ++j) zacc[nt][j][e] += __shfl_xor_sync(0xffffffffu, zacc[nt][j][e], o);
      }
    }
  }
  __syncthreads();  // every warp is done with its ring: the partial outputs take its place
  float* part = reinterpret_cast<float*>(smem) + warp * kRows * S::kPitch;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 8 * nt + 2 * c + e;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const float add = zacc[nt][j][e] + __shfl_sync(0xffffffffu, csum[nt][e], 4 * j + c);
        *reinterpret_cast<float4*>(part + r * S::kPitch + 32 * j + 4 * g) =
            make_float4(acc[nt][j][0][e] + add, acc[nt][j][0][e + 2] + add, acc[nt][j][1][e] + add,
                        acc[nt][j][1][e + 2] + add);
      }
      if (g == 0) stat_m[warp][r] = m[nt][e], stat_l[warp][r] = l[nt][e];
    }
  }
  __syncthreads();

  // The CTA's warps together; with one CTA that is the answer, else it goes to the cluster.
  const bool alone = splits == 1;
  float* whole = reinterpret_cast<float*>(smem);  // [kRows][kPitch], in place of warp 0's
  for (int i = threadIdx.x; i < kRows * (D / 4); i += blockDim.x) {
    const int r = i / (D / 4), ch = 4 * (i % (D / 4));
    float top = -INFINITY;
    for (int w = 0; w < warps; ++w) top = fmaxf(top, stat_m[w][r]);
    const float safe = top == -INFINITY ? 0.f : top;
    float lsum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < warps; ++w) {
      const float f = ex2(stat_m[w][r] - safe);
      const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) +
                                                        (w * kRows + r) * S::kPitch + ch);
      lsum += f * stat_l[w][r];
      o.x = fmaf(f, x.x, o.x), o.y = fmaf(f, x.y, o.y), o.z = fmaf(f, x.z, o.z), o.w = fmaf(f, x.w, o.w);
    }
    if (alone) {
      const int rr = r0 + r;
      if (rr < rows) {
        const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
        T* dst = static_cast<T*>(a.out) + static_cast<int64_t>(start + rr / share) * a.out_token_stride +
                 static_cast<int64_t>(kvh * share + rr % share) * D + ch;
        T v[4] = {from_float<T>(o.x * inv), from_float<T>(o.y * inv), from_float<T>(o.z * inv),
                  from_float<T>(o.w * inv)};
        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(v);
      }
    } else {
      // Each thread reads exactly the elements of every warp's part that it then overwrites.
      *reinterpret_cast<float4*>(whole + r * S::kPitch + ch) = o;
      if (ch == 0) part_m[r] = top, part_l[r] = lsum;
    }
  }
  if (alone) return;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int i = rank * blockDim.x + threadIdx.x; i < kRows * D; i += splits * blockDim.x) {
    const int r = i / D, ch = i % D;
    const int rr = r0 + r;
    if (rr < rows) {
      const uint32_t am = smem_u32(&part_m[r]), al = smem_u32(&part_l[r]), ao = smem_u32(&whole[r * S::kPitch + ch]);
      float top = -INFINITY;
      for (int q = 0; q < splits; ++q) top = fmaxf(top, ld_cluster_f32(mapa_shared(am, q)));
      const float safe = top == -INFINITY ? 0.f : top;
      float lsum = 0.f, o = 0.f;
      for (int q = 0; q < splits; ++q) {
        const float f = ex2(ld_cluster_f32(mapa_shared(am, q)) - safe);
        lsum = fmaf(f, ld_cluster_f32(mapa_shared(al, q)), lsum);
        o = fmaf(f, ld_cluster_f32(mapa_shared(ao, q)), o);
      }
      static_cast<T*>(a.out)[static_cast<int64_t>(start + rr / share) * a.out_token_stride +
                             static_cast<int64_t>(kvh * share + rr % share) * D + ch] =
          from_float<T>(lsum == 0.f ? 0.f : o / lsum);
    }
  }
  // Nobody leaves while a peer may still read its shared memory.
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T, int D, int NT>
int launch_rows(const Kv4AttnArgs& a, bool pdl, cudaStream_t stream) {
  const int share = a.q_heads / a.cache.kv_heads;
  const int64_t rows = static_cast<int64_t>(a.max_q) * share;
  const int64_t row_blocks = (rows + 8 * NT - 1) / (8 * NT);
  const int64_t units = row_blocks * a.cache.kv_heads * a.batch;
  if (row_blocks * a.cache.kv_heads > 65535) return QTTS_ERR_SHAPE;
  // Warps and CTAs for one unit: as many as give each SM some 16 warps in all, at least
  // one tile a warp.
  const int64_t most = static_cast<int64_t>(a.table_cols) * a.cache.page_size;
  const int64_t tiles = (most + kTile - 1) / kTile;
  const int warps = tiles > 4 ? 8 : 4;
  int splits = 1;
  while (splits < 16 && 2 * splits * warps <= tiles && units * splits * warps < 16 * kNumSMs) splits *= 2;
  using S = RowsSmem<D>;
  const size_t ring = static_cast<size_t>(warps) * S::kWarpRing;
  const size_t part = static_cast<size_t>(warps) * 8 * NT * S::kPitch * 4;
  const size_t smem = ring > part ? ring : part;
  auto kern = kv4_rows_kernel<T, D, NT>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess ||
      (splits > 8 && cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)) {
    (void)cudaGetLastError();
    return QTTS_ERR_LAUNCH;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits, static_cast<unsigned>(row_blocks * a.cache.kv_heads), a.batch);
  cfg.blockDim = dim3(32 * warps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, a, static_cast<int>(row_blocks), current_wait_limit_ns()) == cudaSuccess
             ? QTTS_OK
             : QTTS_ERR_LAUNCH;
}

template <typename T, int D>
int launch_ka(const Kv4AttnArgs& a, bool pdl, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.max_q) * (a.q_heads / a.cache.kv_heads);
  return rows <= 8 ? launch_rows<T, D, 1>(a, pdl, stream) : launch_rows<T, D, 2>(a, pdl, stream);
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
  if (!(scale > 0.f) || scale > 3.0e38f) return QTTS_ERR_SHAPE;
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

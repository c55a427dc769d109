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
//     being a (new token, query head) pair that shares the key head. A nibble
//     masked out of a word is an fp16 subnormal as it stands, code * 2^-24 in bits
//     0..3 and code * 2^-20 in bits 4..7, both exact: four masks and one shift
//     make four operand pairs. q is brought to fp16 by a power of two per row
//     (largest magnitude in [2^14, 2^15): exact for bf16 down to 2^-24 of it) and
//     the channels of the higher nibbles by 2^-4 more. The group's scale and
//     minimum enter once per (token, row, group), in fp32;
//   * out^T = V^T P^T: two tokens' half-words are interleaved by bytes, so that a mask
//     leaves two codes of one channel in neighbouring bytes. Read as e4m3 these are
//     code * 2^-9, and one conversion makes them an fp16 pair, one fused multiply-add
//     the value itself, rounded once: code * scale + minimum, in units of a power of two
//     that follows the largest scale or minimum the warp has met (values then reach
//     2^10 and keep their 11 bits down to 2^-14, 2^-24 of the largest). Used as the
//     subnormals that they are, the codes would save the conversions (2 x 131071 tokens
//     75.5 us instead of 79.6, 64 x 4096 tokens 78 instead of 84; no less for 16 rows), but
//     a value would keep no more than 2^-15 of the largest scale in any group and token,
//     too little for groups of unlike size. Scale and minimum of a tile are
//     brought to those units once, a word a lane, through shared memory.
//     Probabilities are fp16 too, times 2^7: up to 2^15 while the running maximum
//     may lag by 2^8, and the small ones normal down to 2^-21;
//   * every warp streams its own tiles of 32 tokens through a ring of asynchronous copies
//     and keeps its own running maximum and sum; the warps of a CTA meet in shared
//     memory, and where there are few (request, head) pairs a cluster of up to 8
//     CTAs splits one of them and meets in distributed shared memory, or, where
//     that is not enough to fill the machine, any number of CTAs through a
//     workspace that a second kernel joins. Sums are in a fixed order.
// 2 requests over 131071 tokens, 32 + 2 x 8 heads of 128 channels: 336 MB of cache in
// 79.6 us, 4.2 TB/s: the nibbles' instructions and the waits
// between them bound it, the copies are ahead. 8 requests over 513 tokens: 7.1 us, a
// launch and the chain lengths -> page -> codes -> scores -> meeting of the CTAs.
#include <type_traits>

#include "kernels.h"
#include "kv4.cuh"

namespace qtts {
namespace {

constexpr int kTile = 32;   // tokens a warp takes at a time
constexpr int kStages = 2;  // tiles in flight a warp
constexpr int kWarps = 4;   // a CTA
constexpr int kMaxCluster = 8;
constexpr int kMaxSplits = 512;  // parts of a row in the workspace
constexpr int kFewSplits = 32;   // up to which one warp joins a row

// Nibbles n and n + 4 (n = 0, 1) of a word as a pair of fp16 subnormals: code * 2^-24 for
// n = 0, code * 2^-20 for n = 1; nibbles n + 2 and n + 6 from the word shifted by eight.
__device__ __forceinline__ uint32_t nib_pair(uint32_t w, int n) { return w & (n ? 0x00F000F0u : 0x000F000Fu); }

// Two 4-bit codes, a byte each, as fp16 numbers code * 2^-9, exactly: read as e4m3 a byte below 16 is
// that many steps of 2^-9 (subnormals, and the first eight normal numbers).
__device__ __forceinline__ uint32_t codes_f16x2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two)));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// D = A x B (no accumulator to be zeroed first), m16n8k16 fp16 -> fp32.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

template <int D>
struct RowsSmem {
  static constexpr int kCodes = kTile * D / 2;              // bytes of a tile's key (or value) codes
  static constexpr int kParams = kTile * (D / kKv4Group) * 4;
  static constexpr int kStage = 2 * (kCodes + kParams);
  static constexpr int kWarpRing = kStages * kStage;
  static constexpr int kPitch = D + 4;  // floats a partial output row: lanes of one store hit different banks
};

template <typename T, int D, int NT, int kCtas>
__global__ void __launch_bounds__(32 * kWarps, kCtas) kv4_rows_kernel(const Kv4AttnArgs a, int row_blocks,
                                                                      int cta_tiles_log2) {
  using S = RowsSmem<D>;
  constexpr int NG = D / kKv4Group;
  constexpr int kRows = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  // Value scales and minima of a tile in fp16: word p * NG + j holds the two tokens of pair p.
  __shared__ __align__(16) uint32_t vscale[kWarps][kTile / 2 * NG], vmin[kWarps][kTile / 2 * NG];
  __shared__ float stat_m[kWarps][kRows], stat_l[kWarps][kRows];  // of each warp
  __shared__ float part_m[kRows], part_l[kRows];        // of the CTA

  constexpr int warps = kWarps;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int rank = blockIdx.x;
  const int kvh = row_blocks == 1 ? blockIdx.y : blockIdx.y / row_blocks;
  const int rb = blockIdx.y - kvh * row_blocks;
  const int b = blockIdx.z;
  pdl_launch_dependents();
  // The first tile's place in the table does not depend on the length: both are fetched at once.
  const int t_first = rank * warps + warp;
  const int per_page = a.per_page;
  const int32_t* table = a.table + b * a.ld_table;
  int at = 2 * t_first;  // number of the tile's first run within the request
  int col = div_by(at, per_page, a.page_inv), off = at - col * per_page;
  const bool whole_tiles = per_page % 2 == 0;
  pdl_wait();
  int page[2];
  page[0] = col < a.table_cols ? table[col] : 0;
  page[1] = !whole_tiles && off + 1 == per_page && col + 1 < a.table_cols ? table[col + 1] : page[0];

  int start = 0, n = 0;
  int len = a.lengths[b];
  bool fine = request_rows(a, b, start, n);
  fine = fine && len >= 0 && len <= static_cast<int64_t>(a.table_cols) * a.cache.page_size &&
         (len == 0 || a.cache.pages > 0);
  if (!fine) {
    if (threadIdx.x == 0) record_status(QTTS_ERR_SHAPE);
    len = 0;
    if (!request_rows(a, b, start, n)) n = 0;  // rows that cannot be told are not written
  }
  const int share = a.share;
  const int rows = n * share;
  const int r0 = rb * kRows;
  // Tokens that any row of this block sees.
  const int last = div_by(max(0, min(rows, r0 + kRows) - 1), share, a.share_inv);  // its last new token
  // What its first row sees (may be negative).
  const int first_lim = a.causal ? len - n + div_by(r0, share, a.share_inv) + 1 : len;
  const int kmax = r0 >= rows ? 0 : max(0, a.causal ? len - n + last + 1 : len);
  if (at * 16 + 16 >= kmax) page[1] = 0;  // what the table holds beyond the tokens is not a page
  const int tiles = (kmax + kTile - 1) / kTile;
  // CTAs that take part in this unit: as many as have 2^cta_tiles_log2 tiles. The others leave (one
  // at least stays, to answer for a unit that sees nothing).
  const int splits = max(1, min(static_cast<int>(gridDim.x), (tiles + (1 << cta_tiles_log2) - 1) >> cta_tiles_log2));
  if (rank >= splits) {
    if (a.parts != nullptr && threadIdx.x < kRows && r0 + threadIdx.x < rows) {  // says that it saw nothing
      const int rr = r0 + threadIdx.x;
      const int token = div_by(rr, share, a.share_inv);
      const int64_t orow = static_cast<int64_t>(start + token) * a.q_heads + kvh * share + rr - token * share;
      a.stats[orow * gridDim.x + rank] = make_float2(-INFINITY, 0.f);
    }
    return;
  }

  // This warp's tiles: every (splits * warps)-th one, 16 bytes a lane and copy into a ring. A
  // tile is two runs of 16 tokens, each within one page. Column and row within the page advance
  // without a division, and the pages of the next tile are fetched one tile ahead.
  uint8_t* ring = smem + warp * S::kWarpRing;
  const int step = splits * warps;
  const int dcol = div_by(2 * step, per_page, a.page_inv), doff = 2 * step - dcol * per_page;
  auto find_pages = [&]() {
    page[0] = at * 16 < kmax ? table[col] : 0;
    if (!whole_tiles) page[1] = off + 1 < per_page ? page[0] : at * 16 + 16 < kmax ? table[col + 1] : 0;
  };
  auto issue = [&](int stage) {
    const uint32_t dst = smem_u32(ring) + stage * S::kStage + 16 * lane;
    if (page[0] < 0 || page[0] >= a.cache.pages) {
      record_status(QTTS_ERR_SHAPE);
      page[0] = 0;
    }
    constexpr int kLanes = S::kParams / 16;  // lanes that copy params: 32 or 16
    const int64_t row = kv4_row(a.cache, page[0], kvh, 16 * off);
    if (whole_tiles) {
      // The tile lies in one page (to its end: what is beyond kmax is there and is masked).
      const uint8_t* k = a.cache.k_codes + row * (D / 2) + 16 * lane;
      const uint8_t* v = a.cache.v_codes + row * (D / 2) + 16 * lane;
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        copy16(dst + 512 * i, k + 512 * i);
        copy16(dst + S::kCodes + S::kParams + 512 * i, v + 512 * i);
      }
      if (lane < kLanes) {
        copy16(dst + S::kCodes, a.cache.k_params + row * NG + 4 * lane);
        copy16(dst + 2 * S::kCodes + S::kParams, a.cache.v_params + row * NG + 4 * lane);
      }
    } else {
      if (page[1] < 0 || page[1] >= a.cache.pages) {
        record_status(QTTS_ERR_SHAPE);
        page[1] = 0;
      }
      const int64_t row1 = off + 1 == per_page ? kv4_row(a.cache, page[1], kvh, 0) : row + 16;
      const bool second = at * 16 + 16 < kmax;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 0 || second) {
          const int64_t r = h ? row1 : row;
#pragma unroll
          for (int i = 0; i < NG / 2; ++i) {  // 16 tokens' codes: NG / 2 copies of 512 bytes
            const int o = 512 * i;
            copy16(dst + (S::kCodes / 2) * h + o, a.cache.k_codes + r * (D / 2) + 16 * lane + o);
            copy16(dst + S::kCodes + S::kParams + (S::kCodes / 2) * h + o,
                   a.cache.v_codes + r * (D / 2) + 16 * lane + o);
          }
        }
      }
      const bool upper = lane >= kLanes / 2;
      if (lane < kLanes && (!upper || second)) {
        const int64_t prow = (upper ? row1 : row) * NG + 4 * (lane - (upper ? kLanes / 2 : 0));
        copy16(dst + S::kCodes, a.cache.k_params + prow);
        copy16(dst + 2 * S::kCodes + S::kParams, a.cache.v_params + prow);
      }
    }
    at += 2 * step, col += dcol, off += doff;
    if (off >= per_page) off -= per_page, ++col;
    find_pages();
  };
  // One group a tile, empty ones too, so that waiting counts tiles.
#pragma unroll 1
  for (int s = 0; s < kStages; ++s) {
    if (t_first + s * step < tiles) issue(s);
    copy_commit();
  }

  // q as the B operand: row 8 nt + g, channels 32j + 8c .. + 7 as pairs (i, i + 4); and the
  // sums over each group of the rows 8 nt + 2c, + 1, whose scores this lane holds, in the
  // same units. to_log2: from those units to the exponent of two.
  uint32_t qf[NT][NG][4];
  float qsum[NT][NG][2], to_log2[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = r0 + 8 * nt + g;
    const int token = div_by(r, share, a.share_inv);
    const T* qr = static_cast<const T*>(a.q) + static_cast<int64_t>(start + token) * a.q_token_stride +
                  (kvh * share + r - token * share) * a.q_head_stride + 8 * c;
    if (r >= rows) qr = static_cast<const T*>(a.q);  // read all the same (not one by one) and cleared
    uint4 u[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) u[j] = *reinterpret_cast<const uint4*>(qr + 32 * j);
    float x[NG][8];
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      if (r >= rows) u[j] = make_uint4(0u, 0u, 0u, 0u);
      const T* e = reinterpret_cast<const T*>(&u[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[j][i] = to_float(e[i]), top = fmaxf(top, fabsf(x[j][i]));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = min(100, max(-100, 14 + 127 - static_cast<int>(__float_as_uint(top) >> 23)));
    const float up = exp2_int(e);
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[j][i] *= up, sum += x[j][i];
      qf[nt][j][0] = pack_f16(x[j][0], x[j][4]);
      qf[nt][j][1] = pack_f16(0.0625f * x[j][1], 0.0625f * x[j][5]);
      qf[nt][j][2] = pack_f16(x[j][2], x[j][6]);
      qf[nt][j][3] = pack_f16(0.0625f * x[j][3], 0.0625f * x[j][7]);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum *= 0x1p-24f;
      qsum[nt][j][0] = __shfl_sync(0xffffffffu, sum, (2 * c) * 4);
      qsum[nt][j][1] = __shfl_sync(0xffffffffu, sum, (2 * c + 1) * 4);
    }
    const float back = a.scale * 1.4426950408889634f * exp2_int(24 - e);
    to_log2[nt][0] = __shfl_sync(0xffffffffu, back, (2 * c) * 4);
    to_log2[nt][1] = __shfl_sync(0xffffffffu, back, (2 * c + 1) * 4);
  }
  int lim[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = div_by(r0 + 8 * nt + 2 * c + e, share, a.share_inv);
      lim[nt][e] = a.causal ? min(len - n + i + 1, kmax) : len;
    }
  }

  float m[NT][2], l[NT][2];
  float acc[NT][NG][2][4];  // [group][channel pair] of out^T, fp32, in units of 2^(vexp - 127 - 5)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) m[nt][e] = -INFINITY, l[nt][e] = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][j][h][e] = 0.f;
      }
    }
  }
  // Unit of the values: 2^(vexp - 127 - 5), vexp the exponent field of the largest value scale
  // so far (or of the largest minimum / 16, where that is more): 15 scale + |minimum| < 2^15 units.
  // What reaches vlimit moves it.
  int vexp = 0;
  float vlimit = 0.f;
  float vs_to = 0.f, vz_to = 0.f;  // 2^9 and 1 in those units

  // Token of row slot s of a 16-token operand: s with the last bit turned in every other
  // pair, so that neither the key nor the value loads below hit one bank with more than two rows.
  const int kslot = g ^ ((g >> 1) & 1);
  const int v0 = (2 * c) ^ (c & 1), v1 = (2 * c + 1) ^ (c & 1);

  auto load_params = [&](const void* p, int t, uint32_t(&w)[NG]) {
    if constexpr (NG == 4) {
      *reinterpret_cast<uint4*>(w) = static_cast<const uint4*>(p)[t];
    } else {
      *reinterpret_cast<uint2*>(w) = static_cast<const uint2*>(p)[t];
    }
  };

  // One tile. kMasked: some row of the block does not see all of it.
  auto attend = [&](const uint8_t* kc, int t0, auto masked) {
    constexpr bool kMasked = decltype(masked)::value;
    const uint8_t* kp = kc + S::kCodes;
    const uint8_t* vc = kp + S::kParams;
    const uint8_t* vp = vc + S::kCodes;

    // This tile's value scales and minima to fp16, NG words a lane.
    float vs[NG], vz[NG];
    float top = 0.f;
    uint32_t bad = 0;  // masked tiles: tokens with a non-finite scale or minimum
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int i = lane + 32 * k;
      uint32_t w = reinterpret_cast<const uint32_t*>(vp)[i];
      if constexpr (kMasked) {  // beyond the request's tokens the cache holds anything
        if (t0 + i / NG >= kmax) w = 0u;
        const bool nf = (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
        const uint32_t who = __ballot_sync(0xffffffffu, nf);
        if (who != 0) {
          for (int t = 0; t < 32 / NG; ++t) {
            if (who >> (t * NG) & ((1u << NG) - 1u)) bad |= 1u << (k * (32 / NG) + t);
          }
        }
      }
      vs[k] = kv4_scale(w), vz[k] = kv4_min(w);
    }
    if constexpr (kMasked) {
      // Rows that do not see such a token must not meet it (0 * NaN): its values become
      // zeros here and its score NaN below, for the rows that do see it.
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        if (bad >> ((lane + 32 * k) / NG) & 1u) vs[k] = vz[k] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < NG; ++k) top = fmaxf(top, fmaxf(vs[k], fabsf(vz[k]) * 0x1p-4f));
    if (__any_sync(0xffffffffu, !(top < vlimit))) {
      float most = 0.f;  // of the finite ones; others reach the output as they are
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        const float x = fmaxf(vs[k], fabsf(vz[k]) * 0x1p-4f);
        most = fmaxf(most, x < INFINITY ? x : 0.f);
      }
      most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
      if (!(most < vlimit)) {
        const int to = min(253, max(16, static_cast<int>(__float_as_uint(most) >> 23)));
        const float f = vlimit == 0.f ? 1.f : exp2_int(max(-126, vexp - to));
        vexp = to;
        vlimit = exp2_int(to - 126);
        vs_to = exp2_int(127 - to) * 0x1p14f;
        vz_to = exp2_int(127 - to) * 0x1p5f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int j = 0; j < NG; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][j][0][e] *= f, acc[nt][j][1][e] *= f;
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int i = lane + 32 * k, t = i / NG;
      // Token t is the first or second of its operand pair as the row slots below have it.
      const int half = 2 * ((t >> 1) * NG + i % NG) + ((t ^ (t >> 1)) & 1);
      reinterpret_cast<__half*>(vscale[warp])[half] = __float2half_rn(vs[k] * vs_to);
      reinterpret_cast<__half*>(vmin[warp])[half] = __float2half_rn(vz[k] * vz_to);
    }

    // Scores of 2 x 16 tokens: s[nt][mt][2 * token half + row of the pair].
    float s[NT][2][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      uint32_t kw[2][NG], pw[2][NG];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = 16 * mt + 8 * h + kslot;
        if constexpr (NG == 4) {
          *reinterpret_cast<uint4*>(kw[h]) = *reinterpret_cast<const uint4*>(kc + t * 64 + 16 * c);
        } else {
          *reinterpret_cast<uint2*>(kw[h]) = *reinterpret_cast<const uint2*>(kc + t * 32 + 8 * c);
        }
        load_params(kp, t, pw[h]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][mt][e] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const uint32_t h0 = kw[0][j] >> 8, h1 = kw[1][j] >> 8;
        const uint32_t a0[4] = {nib_pair(kw[0][j], 0), nib_pair(kw[1][j], 0), nib_pair(kw[0][j], 1),
                                nib_pair(kw[1][j], 1)};
        const uint32_t a1[4] = {nib_pair(h0, 0), nib_pair(h1, 0), nib_pair(h0, 1), nib_pair(h1, 1)};
        const float sc0 = kv4_scale(pw[0][j]), sc1 = kv4_scale(pw[1][j]);
        const float z0 = kv4_min(pw[0][j]), z1 = kv4_min(pw[1][j]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float d[4];
          mma_f16_first(d, a0, qf[nt][j][0], qf[nt][j][1]);
          Mma16816<__half>::run(d, a1, qf[nt][j][2], qf[nt][j][3]);
          s[nt][mt][0] = fmaf(sc0, d[0], fmaf(z0, qsum[nt][j][0], s[nt][mt][0]));
          s[nt][mt][1] = fmaf(sc0, d[1], fmaf(z0, qsum[nt][j][1], s[nt][mt][1]));
          s[nt][mt][2] = fmaf(sc1, d[2], fmaf(z1, qsum[nt][j][0], s[nt][mt][2]));
          s[nt][mt][3] = fmaf(sc1, d[3], fmaf(z1, qsum[nt][j][1], s[nt][mt][3]));
        }
      }
    }
    if constexpr (kMasked) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = t0 + 16 * mt + 8 * (e >> 1) + kslot;
            if (bad >> (t - t0) & 1u) s[nt][mt][e] = NAN;
            if (t >= lim[nt][e & 1]) s[nt][mt][e] = -INFINITY;
          }
        }
      }
    }

    // Running maximum (exponent of two) and sum; p replaces s.
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
      // to_log2 > 0: the largest score stays the largest. The reference m follows the maximum
      // only when that has grown by more than 2^8: probabilities stay below 2^15.
      mx[0] *= to_log2[nt][0];
      mx[1] *= to_log2[nt][1];
      if (__any_sync(0xffffffffu, mx[0] > m[nt][0] + 8.f || mx[1] > m[nt][1] + 8.f)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float to = fmaxf(m[nt][e], mx[e]);
          const float f = to > m[nt][e] ? ex2(m[nt][e] - to) : 1.f;
          m[nt][e] = to;
          l[nt][e] *= f;
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            acc[nt][j][0][e] *= f, acc[nt][j][0][e + 2] *= f;
            acc[nt][j][1][e] *= f, acc[nt][j][1][e + 2] *= f;
          }
        }
      }
      const float m0 = 7.f - (kMasked && m[nt][0] == -INFINITY ? 0.f : m[nt][0]);
      const float m1 = 7.f - (kMasked && m[nt][1] == -INFINITY ? 0.f : m[nt][1]);
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt][mt][e] = ex2(fmaf(s[nt][mt][e], to_log2[nt][e & 1], (e & 1) ? m1 : m0));
          l[nt][e & 1] += s[nt][mt][e];
        }
      }
    }

    // Weighted values.
    __syncwarp();  // vscale, vmin
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      uint32_t vw[4][NG / 2], sw[2][NG], zw[2][NG];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int t = 16 * mt + 8 * (h >> 1) + ((h & 1) ? v1 : v0);
        if constexpr (NG == 4) {
          *reinterpret_cast<uint2*>(vw[h]) = *reinterpret_cast<const uint2*>(vc + t * 64 + 8 * g);
        } else {
          vw[h][0] = *reinterpret_cast<const uint32_t*>(vc + t * 32 + 4 * g);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load_params(vscale[warp], 8 * mt + 4 * h + c, sw[h]);
        load_params(vmin[warp], 8 * mt + 4 * h + c, zw[h]);
      }
      uint32_t b0[NT], b1[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        b0[nt] = transpose8x8(pack_f16(s[nt][mt][0], s[nt][mt][1]));
        b1[nt] = transpose8x8(pack_f16(s[nt][mt][2], s[nt][mt][3]));
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        // Tokens (2c, 2c + 1) and (2c + 8, 2c + 9) of group j, interleaved by bytes.
        const uint32_t xa = __byte_perm(vw[0][j / 2], vw[1][j / 2], (j & 1) ? 0x7362 : 0x5140);
        const uint32_t xb = __byte_perm(vw[2][j / 2], vw[3][j / 2], (j & 1) ? 0x7362 : 0x5140);
        const uint32_t la = xa & 0x0F0F0F0Fu, ha = xa >> 4 & 0x0F0F0F0Fu;
        const uint32_t lb = xb & 0x0F0F0F0Fu, hb = xb >> 4 & 0x0F0F0F0Fu;
        const uint32_t sa = sw[0][j], za = zw[0][j], sb = sw[1][j], zb = zw[1][j];
        const uint32_t a0[4] = {fma_f16x2(codes_f16x2(la), sa, za), fma_f16x2(codes_f16x2(ha), sa, za),
                                fma_f16x2(codes_f16x2(lb), sb, zb), fma_f16x2(codes_f16x2(hb), sb, zb)};
        const uint32_t a1[4] = {fma_f16x2(codes_f16x2(la >> 16), sa, za), fma_f16x2(codes_f16x2(ha >> 16), sa, za),
                                fma_f16x2(codes_f16x2(lb >> 16), sb, zb), fma_f16x2(codes_f16x2(hb >> 16), sb, zb)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          Mma16816<__half>::run(acc[nt][j][0], a0, b0[nt], b1[nt]);
          Mma16816<__half>::run(acc[nt][j][1], a1, b0[nt], b1[nt]);
        }
      }
    }
  };

  int stage = 0;
  for (int tile = t_first; tile < tiles; tile += step) {
    copy_wait<kStages - 1>();
    __syncwarp();
    const int t0 = tile * kTile;
    if (t0 + kTile > first_lim) {
      attend(ring + stage * S::kStage, t0, std::true_type{});
    } else {
      attend(ring + stage * S::kStage, t0, std::false_type{});
    }
    __syncwarp();
    if (tile + kStages * step < tiles) issue(stage);
    copy_commit();
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }

  // Finish the warp: the rest of the sums over its lanes, then its partial outputs.
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], o);
    }
  }
  __syncthreads();  // every warp is done with its ring: the partial outputs take its place
  float* part = reinterpret_cast<float*>(smem) + warp * kRows * S::kPitch;
  const float vref = vlimit == 0.f ? 0.f : exp2_int(vexp - 127) * 0x1p-5f;  // no tile: no values
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 8 * nt + 2 * c + e;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        *reinterpret_cast<float4*>(part + r * S::kPitch + 32 * j + 4 * g) = make_float4(
            acc[nt][j][0][e] * vref, acc[nt][j][0][e + 2] * vref,
            acc[nt][j][1][e] * vref, acc[nt][j][1][e + 2] * vref);
      }
      if (g == 0) stat_m[warp][r] = m[nt][e], stat_l[warp][r] = l[nt][e];
    }
  }
  __syncthreads();

  // The CTA's warps together; with one CTA that is the answer, else its part goes to the
  // cluster or, where more CTAs share a unit than a cluster holds, to the workspace.
  const int mode = a.parts != nullptr ? 2 : splits > 1 ? 1 : 0;
  float* whole = reinterpret_cast<float*>(smem);  // [kRows][kPitch], in place of warp 0's
  for (int i = threadIdx.x; i < kRows * (D / 4); i += 32 * kWarps) {
    const int r = i / (D / 4), ch = 4 * (i % (D / 4));
    const int rr = r0 + r;
    if (rr >= rows) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stat_m[w][r]);
    const float safe = top == -INFINITY ? 0.f : top;
    float lsum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(stat_m[w][r] - safe);
      const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) +
                                                        (w * kRows + r) * S::kPitch + ch);
      lsum += f * stat_l[w][r];
      o.x = fmaf(f, x.x, o.x), o.y = fmaf(f, x.y, o.y), o.z = fmaf(f, x.z, o.z), o.w = fmaf(f, x.w, o.w);
    }
    const int token = div_by(rr, share, a.share_inv);
    const int64_t orow = static_cast<int64_t>(start + token);
    const int head = kvh * share + rr - token * share;
    if (mode == 0) {
      const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
      T v[4] = {from_float<T>(o.x * inv), from_float<T>(o.y * inv), from_float<T>(o.z * inv),
                from_float<T>(o.w * inv)};
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + orow * a.out_token_stride + head * D + ch) =
          *reinterpret_cast<uint2*>(v);
    } else if (mode == 2) {
      const int64_t at_row = (orow * a.q_heads + head) * gridDim.x + rank;
      if (top != -INFINITY) *reinterpret_cast<float4*>(a.parts + at_row * D + ch) = o;
      if (ch == 0) a.stats[at_row] = make_float2(top, lsum);
    } else {
      // Each thread reads exactly the elements of every warp's part that it then overwrites.
      *reinterpret_cast<float4*>(whole + r * S::kPitch + ch) = o;
      if (ch == 0) part_m[r] = top, part_l[r] = lsum;
    }
  }
  if (mode != 1) return;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int i = rank * 32 * kWarps + threadIdx.x; i < kRows * D; i += splits * 32 * kWarps) {
    const int r = i / D, ch = i % D;
    const int rr = r0 + r;
    if (rr < rows) {
      const uint32_t am = smem_u32(&part_m[r]), al = smem_u32(&part_l[r]), ao = smem_u32(&whole[r * S::kPitch + ch]);
      float pm[kMaxCluster], pl[kMaxCluster], po[kMaxCluster];
      float top = -INFINITY;
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q) {
        const int peer = min(q, splits - 1);  // all at once, no branch between them
        pm[q] = ld_cluster_f32(mapa_shared(am, peer));
        pl[q] = ld_cluster_f32(mapa_shared(al, peer));
        po[q] = ld_cluster_f32(mapa_shared(ao, peer));
      }
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q) {
        if (q < splits) top = fmaxf(top, pm[q]);
      }
      const float safe = top == -INFINITY ? 0.f : top;
      float lsum = 0.f, o = 0.f;
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q) {
        if (q < splits) {
          const float f = ex2(pm[q] - safe);
          lsum = fmaf(f, pl[q], lsum);
          o = fmaf(f, po[q], o);
        }
      }
      const int token = div_by(rr, share, a.share_inv);
      static_cast<T*>(a.out)[static_cast<int64_t>(start + token) * a.out_token_stride +
                             static_cast<int64_t>(kvh * share + rr - token * share) * D + ch] =
          from_float<T>(lsum == 0.f ? 0.f : o / lsum);
    }
  }
  // Nobody leaves while a peer may still read its shared memory.
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The parts of a (token, head) row from the workspace, request by request: rows of no request have
// none and are not written. Bound by latency: all statistics are read
// at once, and four parts a warp are in flight. Eight warps a row where there are many parts (one
// long cache: 256 parts in 4 us instead of 28 with one warp), one where there are many rows.
constexpr int kJoinWarps = 8;  // a CTA

template <typename T, int D, int kRowWarps>
__global__ void __launch_bounds__(32 * kJoinWarps) kv4_join_kernel(const Kv4AttnArgs a, int splits) {
  constexpr int kPer = D / 32;  // channels a lane
  constexpr int kRows = kJoinWarps / kRowWarps;
  constexpr int kParts = kRowWarps == 1 ? kFewSplits : kMaxSplits;
  constexpr int kSlots = (kParts + 32 * kRowWarps - 1) / (32 * kRowWarps);
  __shared__ float weight[kRows][kParts];
  __shared__ float red[2][kJoinWarps];
  __shared__ float out[kJoinWarps][D];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = warp / kRowWarps, rw = warp % kRowWarps;
  const int tid = rw * 32 + lane;  // within the row
  int start = 0, n = 0;
  if (!request_rows(a, blockIdx.y, start, n)) n = 0;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows;
  const int64_t rows = static_cast<int64_t>(n) * a.q_heads;  // of this request
  if (first >= rows) return;
  const bool there = first + sub < rows;
  const int64_t row = static_cast<int64_t>(start) * a.q_heads + first + sub;
  const float2* st = a.stats + row * splits;
  float2 s[kSlots];
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < kSlots; ++k) {
    const int q = tid + k * 32 * kRowWarps;
    s[k] = there && q < splits ? st[q] : make_float2(-INFINITY, 0.f);
    top = fmaxf(top, s[k].x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if constexpr (kRowWarps > 1) {
    if (lane == 0) red[0][warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, red[0][sub * kRowWarps + w]);
  }
  const float safe = top == -INFINITY ? 0.f : top;
  float lsum = 0.f;
#pragma unroll
  for (int k = 0; k < kSlots; ++k) {
    const int q = tid + k * 32 * kRowWarps;
    // A part that saw nothing was not written: its weight is exactly 0 and it is passed over.
    const float f = s[k].x == -INFINITY ? 0.f : ex2(s[k].x - safe);
    lsum = fmaf(f, s[k].y, lsum);
    if (q < splits) weight[sub][q] = f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) lsum += __shfl_xor_sync(0xffffffffu, lsum, o);
  if constexpr (kRowWarps > 1) {
    if (lane == 0) red[1][warp] = lsum;
    __syncthreads();
  } else {
    __syncwarp();
  }
  float acc[kPer] = {};
  const float* part = a.parts + row * splits * D + lane * kPer;
#pragma unroll 4
  for (int q = rw; q < splits; q += kRowWarps) {
    const float f = weight[sub][q];
    float x[kPer] = {};
    if (there && f != 0.f) {
      if constexpr (kPer == 4) {
        *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(part + static_cast<int64_t>(q) * D);
      } else {
        *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(part + static_cast<int64_t>(q) * D);
      }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = fmaf(f, x[i], acc[i]);
  }
  T* dst = static_cast<T*>(a.out) + row / a.q_heads * a.out_token_stride + row % a.q_heads * D;
  if constexpr (kRowWarps > 1) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) out[warp][lane * kPer + i] = acc[i];
    __syncthreads();
    if (there && tid < D) {
      float l = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) l += red[1][sub * kRowWarps + w], o += out[sub * kRowWarps + w][tid];
      dst[tid] = from_float<T>(l == 0.f ? 0.f : o / l);
    }
  } else if (there) {
    const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
    T v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = from_float<T>(acc[i] * inv);
    if constexpr (kPer == 4) {
      *reinterpret_cast<uint2*>(dst + lane * kPer) = *reinterpret_cast<uint2*>(v);
    } else {
      *reinterpret_cast<uint32_t*>(dst + lane * kPer) = *reinterpret_cast<uint32_t*>(v);
    }
  }
}

// Which kernel: 16-row blocks that each read the cache (kv4_rows_kernel), or 128-row tiles
// (kv4_prompt.cu), whose time hardly depends on how many of a tile's rows there are. Times
// of the two in microseconds, 16 query and 8 key heads of 128 channels, from a request's
// rows (new tokens x 2; both within 8 % of this since their operands keep more bits):
//                                      32 rows        64 rows        128 rows
//   1 request,   1000 tokens        9.1 |  18.5    10.2 |  18.4    13.1 |  17.5
//   8 requests,  1000 tokens       17.5 |  19.6    19.9 |  19.9    37.6 |  20.5
//   8 requests,  8192 tokens       73.6 | 110.3   144.1 | 112.5   278.8 | 111.6
//   64 requests, 2048 tokens      128.9 | 163.7   224.9 | 164.0   441.5 | 160.5
// So few rows stay here whatever the length, more than one tile's go there, and between
// them the blocks are the faster while their work (blocks x tokens) is well below one wave's.
constexpr int64_t kPromptRows = 64, kTileRows = 128, kWaveTokens = 1 << 17;
bool kv4_takes_prompt(int64_t max_q, int share, int kv_heads, int batch, int64_t tokens) {
  const int64_t rows = max_q * share;
  if (rows < kPromptRows || rows > kTileRows) return rows > kTileRows;
  return (rows + 15) / 16 * kv_heads * batch * tokens > kWaveTokens;
}

// How a call is laid out: rows a CTA, and CTAs that share the tokens of one (request, key
// head, row block).
struct RowsPlan {
  int nt;
  int ctas;  // an SM
  int64_t row_blocks;
  int splits;      // CTAs at most
  int cta_tiles_log2;  // tiles for which another CTA joins in: one a warp, or four
};

// Tiles that a warp of the longest request gets at most, as far as kEvenCtas CTAs (a
// cluster) do it: a long request then holds the others of the call up less. With no
// limit | 8 tiles | 16 tiles, at three CTAs an SM: 64 requests of 17 to 8192 tokens 104 | 61 | 56 us; 64 of 4096
// tokens 87 | 93 | 79 us; 128 of 1000 to 2000 tokens 66 | 80 | 66 us.
constexpr int kEvenTiles = 16, kEvenCtas = 8;

RowsPlan plan_rows(int64_t max_q, int share, int kv_heads, int batch, int64_t most_tokens, int head_dim) {
  RowsPlan p;
  const int64_t rows = max_q * share;
  // Eight rows fill an operand; more share what is made of the cache by pairs of eight
  // (64 x 2048 tokens: 8 rows 50 us, 16 rows 67).
  p.nt = rows <= 8 ? 1 : 2;
  p.row_blocks = (rows + 8 * p.nt - 1) / (8 * p.nt);
  const int64_t units = p.row_blocks * kv_heads * batch;
  // CTAs an SM: two with 16 rows. With 8, three at 168 registers where units are split anyway (8 x 513
  // tokens 7.1 us, four at 128 registers 8.3; 8 x 2048: 10.9, 12.3). Four where there is a unit for
  // every SM and three would not hold two CTAs of each (32 x 2048 tokens: 29.8 us, three 34.0); beyond
  // that the few values that 128 channels spill at 128 registers cost more than the fourth CTA gives
  // (64 x 4096 tokens: 84.4, three 81.4; 64 x 17..8192: 60.8, 57.7; 128 x 1000..2000: 63.3, 62.2), and
  // 64 channels spill none (64 x 2000..4000: 44.8, 48.6).
  const bool four = units > kNumSMs && (head_dim == 64 || units <= 3 * kNumSMs);
  p.ctas = p.nt == 2 ? 2 : four ? 4 : 3;
  // One wave of them, at least one tile a warp, and the limit above. CTAs that a shorter request
  // has no use for leave at once.
  const int64_t wave = static_cast<int64_t>(kNumSMs) * p.ctas;
  const int64_t tiles = (most_tokens + kTile - 1) / kTile;
  const int64_t want = wave / (units > 0 ? units : 1);
  const int64_t can = (tiles + kWarps - 1) / kWarps;
  const int64_t even = (tiles + kEvenTiles * kWarps - 1) / (kEvenTiles * kWarps);
  int64_t s = even < kEvenCtas ? even : kEvenCtas;
  if (s * units > 16 * wave) s = 16 * wave / units;
  static_assert(kWarps == 4, "one tile a warp, or four, as powers of two");
  p.cta_tiles_log2 = s > want ? 4 : 2;
  if (s < want) s = want;
  if (s > can) s = can;
  p.splits = static_cast<int>(s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s);
  return p;
}

template <typename KernT, typename... Args>
int launch(KernT kern, dim3 grid, int threads, size_t smem, int cluster, bool pdl, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? QTTS_OK : QTTS_ERR_LAUNCH;
}

template <typename T, int D, int NT, int kCtas>
int launch_rows(Kv4AttnArgs a, const RowsPlan& p, bool pdl, cudaStream_t stream) {
  using S = RowsSmem<D>;
  constexpr size_t kRing = static_cast<size_t>(kWarps) * S::kWarpRing;
  constexpr size_t kPart = static_cast<size_t>(kWarps) * 8 * NT * S::kPitch * 4;
  constexpr size_t kSmem = kRing > kPart ? kRing : kPart;
  if (kSmem > 48 * 1024 &&
      cudaFuncSetAttribute(kv4_rows_kernel<T, D, NT, kCtas>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(kSmem)) != cudaSuccess) {
    (void)cudaGetLastError();
    return QTTS_ERR_LAUNCH;
  }
  const bool workspace = p.splits > kMaxCluster;
  if (!workspace) a.parts = nullptr, a.stats = nullptr;
  return launch(kv4_rows_kernel<T, D, NT, kCtas>,
                dim3(p.splits, static_cast<unsigned>(p.row_blocks * a.cache.kv_heads), a.batch), 32 * kWarps, kSmem,
                workspace ? 1 : p.splits, pdl, stream, a, static_cast<int>(p.row_blocks),
                p.cta_tiles_log2);
}

template <typename T, int D>
int launch_join(const Kv4AttnArgs& a, int splits, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.max_q) * a.q_heads;  // of a request, at most
  if (splits <= kFewSplits) {
    return launch(kv4_join_kernel<T, D, 1>, dim3(static_cast<unsigned>((rows + kJoinWarps - 1) / kJoinWarps), a.batch),
                  32 * kJoinWarps, 0, 1, true, stream, a, splits);
  }
  return launch(kv4_join_kernel<T, D, kJoinWarps>, dim3(static_cast<unsigned>(rows), a.batch), 32 * kJoinWarps, 0, 1,
                true, stream, a, splits);
}

template <typename T, int D>
int launch_ka(const Kv4AttnArgs& a, int dtype, bool pdl, cudaStream_t stream) {
  const int share = a.share;
  const int64_t tokens = static_cast<int64_t>(a.table_cols) * a.cache.page_size;
  if (kv4_takes_prompt(a.max_q, share, a.cache.kv_heads, a.batch, tokens)) {
    const PromptPlan p = plan_prompt(a.max_q, share, a.cache.kv_heads, a.batch, tokens);
    const int r = launch_kv4_prompt(a, p, dtype, D, pdl, stream);
    return r != QTTS_OK || p.splits == 1 ? r : launch_join<T, D>(a, p.splits, stream);
  }
  const RowsPlan p = plan_rows(a.max_q, share, a.cache.kv_heads, a.batch, tokens, D);
  if (p.row_blocks * a.cache.kv_heads > 65535) return QTTS_ERR_SHAPE;
  const int r = p.ctas == 4   ? launch_rows<T, D, 1, 4>(a, p, pdl, stream)
                : p.ctas == 3 ? launch_rows<T, D, 1, 3>(a, p, pdl, stream)
                              : launch_rows<T, D, 2, 2>(a, p, pdl, stream);
  return r != QTTS_OK || p.splits <= kMaxCluster ? r : launch_join<T, D>(a, p.splits, stream);
}

// CTAs whose parts meet in the workspace; 1 where none do.
int workspace_splits(int64_t max_q, int share, int kv_heads, int batch, int64_t tokens, int head_dim) {
  if (kv4_takes_prompt(max_q, share, kv_heads, batch, tokens)) {
    return plan_prompt(max_q, share, kv_heads, batch, tokens).splits;
  }
  const int s = plan_rows(max_q, share, kv_heads, batch, tokens, head_dim).splits;
  return s > kMaxCluster ? s : 1;
}

}  // namespace

int launch_kv4_attention(const Kv4AttnArgs& a, int dtype, int head_dim, bool pdl, cudaStream_t stream) {
  if (dtype == QTTS_BF16) {
    return head_dim == 128 ? launch_ka<__nv_bfloat16, 128>(a, dtype, pdl, stream)
                           : launch_ka<__nv_bfloat16, 64>(a, dtype, pdl, stream);
  }
  return head_dim == 128 ? launch_ka<__half, 128>(a, dtype, pdl, stream)
                         : launch_ka<__half, 64>(a, dtype, pdl, stream);
}

}  // namespace qtts

extern "C" int64_t qtts_kv4_attention_workspace(int total_q, int max_q, int batch, int q_heads, int kv_heads,
                                                int head_dim, int64_t max_tokens) {
  using namespace qtts;
  if (total_q < 1 || max_q < 1 || batch < 1 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads != 0) return 0;
  const int splits = workspace_splits(max_q, q_heads / kv_heads, kv_heads, batch, max_tokens, head_dim);
  return splits == 1 ? 0 : static_cast<int64_t>(total_q) * q_heads * splits * (head_dim + 2) * 4;
}

extern "C" int qtts_kv4_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype,
                                  const uint8_t* k_codes, const void* k_params, const uint8_t* v_codes,
                                  const void* v_params, int64_t pages, int page_size, const int32_t* block_table,
                                  int64_t ld_table, int table_cols, const int32_t* lengths, const int32_t* q_starts,
                                  int total_q, int max_q, int batch, int q_heads, int kv_heads, int head_dim,
                                  float scale, int causal, void* out, int64_t out_token_stride, void* workspace,
                                  unsigned flags, void* stream) {
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
  if (static_cast<int64_t>(table_cols) * page_size > (1 << 30)) return QTTS_ERR_SHAPE;
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
  const int64_t need = qtts_kv4_attention_workspace(total_q, max_q, batch, q_heads, kv_heads, head_dim,
                                                    static_cast<int64_t>(table_cols) * page_size);
  if (need > 0 && workspace == nullptr) return QTTS_ERR_NULL;
  if (need > 0 && !al(workspace, 16)) return QTTS_ERR_ALIGN;
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
  a.share = q_heads / kv_heads;
  a.per_page = page_size / 16;
  a.share_inv = 0xffffffffu / static_cast<uint32_t>(a.share);
  a.page_inv = 0xffffffffu / static_cast<uint32_t>(a.per_page);
  a.scale = scale;
  a.causal = causal;
  a.out = out;
  a.out_token_stride = out_token_stride;
  if (need > 0) {
    a.parts = static_cast<float*>(workspace);
    a.stats = reinterpret_cast<float2*>(a.parts + need / ((head_dim + 2) * 4) * head_dim);
  }
  return launch_kv4_attention(a, dtype, head_dim, (flags & QTTS_FLAG_PDL) != 0, static_cast<cudaStream_t>(stream));
}

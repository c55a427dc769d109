// Attention over the 4-bit cache for many rows a request (prompts, chunks): the
// 5th-generation tensor cores, 128 rows a tile, a row being a (new token, query
// head) pair that shares the key head; see kv4_attention.cu for the definition.
//
// A CTA takes one or two tiles of rows of one (request, key head) and walks over
// the tokens, 128 at a time:
//   * warps 8-11 turn the tile's codes into fp16 in shared memory, one token a thread, a
//     key or value rounded once (in units of their own, below). Keys and values have the same
//     layout there, 128-byte rows of 64 channels a token, swizzled: the keys are the
//     K-major B operand of S = Q K^T, the values the transposed (N-contiguous) B
//     operand of O += P V. The order of channels within a row is the order in which
//     masks give pairs; q is stored to match, and the outputs are put back in order
//     at the end;
//   * warps 12 and 13 issue the products of a tile each, 64 tokens of S at a time into
//     one of two buffers a tile, so that S(u + 1) is made while the probabilities of
//     S(u) are. P replaces S in tensor memory. The products of one tile run in the
//     order issued, so S(u + 2) may overwrite P(u);
//   * warps 0-3 and 4-7 (a thread a row, no exchange between threads) take the running
//     maximum and sum in fp32 and write P in fp16, rounded to nearest
//     (the sum takes it unrounded). The reference maximum follows only when the
//     maximum has grown by more than 2^8, so O is rescaled rarely (and then waits for
//     the product before); the row's sum divides at the end;
//   * where there are few (request, key head, block) units, up to 64 CTAs share the
//     tokens of one and leave fp32 parts in a workspace, which kv4_join_kernel joins.
// Floor: the two products. 4 prompts of 2048 tokens, 16 + 2 x 8 heads of 128 channels,
// causal: 105 us, 0.65 PFLOP/s in bf16 (fp16 operands in units: 13 us more than bf16 operands
// took, for half the error) and 100 us in fp16, whose q needs no units; not causal, twice
// the work, 184 us. fp16 operands are the choice because the products run at half that
// rate from 32-bit ones, which would need twice the shared memory that two tiles fill
// already; with fp16 activations they make 4e-4 of error (2-norm) where the output's own
// rounding makes 2e-4. What bounds it is latency: some 4000 clocks for 128
// tokens of two tiles, where the tensor cores need 2600 and the exponentials 2050, as
// the chain S -> maximum -> exponentials -> P -> products has only the other tile to
// hide behind (two tiles fill the tensor memory), and 12000 clocks a CTA before its
// first S and after its last P, for cold code and first loads. Rolled loops where they
// are rare and one body for masked and whole steps took 4 us off by fetching less.
#include <type_traits>

#include "kernels.h"
#include "kv4.cuh"
#include "tmem.cuh"

namespace qtts {
namespace {

constexpr int kPmTile = 128;  // rows of a tile, and tokens at a time
constexpr int kPmSub = 64;     // tokens of S at a time
constexpr int kPmStages = 2;
constexpr int kPmDqWarp = 8;   // first of four warps that make the operands
constexpr int kPmMmaWarp = 12;  // one issuing warp a tile
constexpr int kPmThreads = 14 * 32;

template <int D>
struct PromptSmem {
  static constexpr int kTileBytes = kPmTile * D * 2;  // a tile of q, keys or values, 16 bits each
  static constexpr int kQ = 0;
  static constexpr int kK = 2 * kTileBytes;
  static constexpr int kV = kK + kPmStages * kTileBytes;
  static constexpr int kBars = kV + kPmStages * kTileBytes;
  static constexpr int kUnits = kBars + 256;             // [step % 4]: of the keys, of the values, four each
  static constexpr int kBytes = kUnits + 128 + 1024;     // slack to align the base to 1024
};

__device__ __forceinline__ float ex2f(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// The operands are fp16, rounded once from what the codes stand for; sums are fp32. Keys, values and
// bf16 activations reach further than fp16, and their scales further down, so they are brought to
// units of a power of two: q a row (largest magnitude 2^14 to 2^15; fp16 ones stay as they are), keys
// and values every 32 tokens, a warp of those that make them (2^7 to 2^15, in steps of 2^8 so that units
// seldom differ); what is below 2^-21 of the largest of those 32 tokens loses bits. The units of q and
// keys go into the scores' factor, that of the values into P where it is not the output's own, which
// follows the largest. Against 64 bits (2-norm) bf16 operands had 3.2e-3, these have 1.7e-3, the
// output's own rounding; fp16 activations have 3e-4 to 4e-4, of which that is 2e-4. (fp16 activations
// over keys and values as they are: 92 us instead of 100 for 4 x 2048 tokens, but scales below 2^-14
// are subnormals then, and keys with a scale of 2^-18 gave scores off by 2^-8.)
__device__ __forceinline__ uint32_t values(uint32_t w, int n, uint32_t s, uint32_t z) {
  // code * s + z of nibbles n and n + 4 of a word: 1024 + code by a mask, less 1024 (exact), and one
  // rounding in the multiply-add.
  uint32_t x = ((w >> (4 * n)) & 0x000F000Fu) | 0x64006400u;
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0x64006400u));
  asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(x) : "r"(s), "r"(z));
  return x;
}
// The largest finite magnitude that a group's codes can stand for, as ordered bits.
__device__ __forceinline__ uint32_t group_top(uint32_t p) {
  const float z = fabsf(kv4_min(p)), y = fabsf(fmaf(15.f, kv4_scale(p), kv4_min(p)));
  return __float_as_uint(fmaxf(z < INFINITY ? z : 0.f, y < INFINITY ? y : 0.f));
}
// The larger magnitude of a bf16 pair's, as floats.
__device__ __forceinline__ float pair_top(uint32_t w) {
  return fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u)));
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// Byte offset of 16-byte chunk `chunk` (eight channels) of row `row` of a tile.
__device__ __forceinline__ uint32_t tile_offset(int row, int chunk) {
  return static_cast<uint32_t>((chunk >> 3) * (kPmTile * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

template <typename T, int D>
__global__ void __launch_bounds__(kPmThreads, 1)
    kv4_prompt_kernel(const Kv4AttnArgs a, int tiles_a_cta, int max_splits, int split_steps, uint64_t wait_ns) {
  using S = PromptSmem<D>;
  constexpr int NG = D / kKv4Group;
  constexpr int kWords = D / 8;  // 32-bit words of codes a row; chunks of eight channels
  constexpr uint32_t kIdescS = umma_idesc(0u, 0u, kPmTile, kPmSub);
  constexpr uint32_t kIdescO = umma_idesc(0u, 0u, kPmTile, D) | kUmmaBTransposed;
  constexpr uint32_t kColS = 0, kColO = 2 * kPmTile;
  constexpr bool kQUnits = std::is_same_v<T, __nv_bfloat16>;
  constexpr float kLift = 7.f;  // of P: at most 2^15 while the maximum lags by 2^8; normal down to 2^-21
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* kempty = kfull + kPmStages;
  uint64_t* vfull = kempty + kPmStages;
  uint64_t* vempty = vfull + kPmStages;
  uint64_t* sfull = vempty + kPmStages;  // [tile][buffer]: S is there
  uint64_t* pfull = sfull + 4;           // [tile][buffer]: P is there
  uint64_t* odone = pfull + 4;           // [tile]: O has taken one more P
  uint64_t* ofull = odone + 2;           // [tile]: all of O is there
  uint64_t* mdone = ofull + 2;           // [tile]: everything issued is done
  uint64_t* qfull = mdone + 2;           // [tile]: q is there
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(qfull + 2);
  volatile int* units = reinterpret_cast<volatile int*>(smem + S::kUnits);  // as exponents of two

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < kPmStages; ++s) {
      mbar_init(&kfull[s], kPmTile);
      mbar_init(&kempty[s], tiles_a_cta);
      mbar_init(&vfull[s], kPmTile);
      mbar_init(&vempty[s], tiles_a_cta);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], kPmTile);
    }
    for (int i = 0; i < 6; ++i) mbar_init(&odone[i], 1);  // and ofull, mdone
    for (int i = 0; i < 2; ++i) mbar_init(&qfull[i], kPmTile);
    fence_mbarrier_init();
  }
  if (warp == kPmMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  pdl_wait();

  // The longest blocks first, of all requests and heads: with `causal` the last rows see most.
  const int rb = static_cast<int>(gridDim.z - 1 - blockIdx.z);
  const int kvh = max_splits == 1 ? blockIdx.x : blockIdx.x / max_splits;
  const int split = blockIdx.x - kvh * max_splits;
  const int b = blockIdx.y;
  int start = 0, n = 0;
  int len = a.lengths[b];
  bool fine = request_rows(a, b, start, n);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  // Only now that the columns are this CTA's: the next kernel may want some on this SM and, holding
  // them, waits for this one to end.
  pdl_launch_dependents();
  fine = fine && len >= 0 && len <= static_cast<int64_t>(a.table_cols) * a.cache.page_size &&
         (len == 0 || a.cache.pages > 0);
  if (!fine) {
    if (tid == 0) record_status(QTTS_ERR_SHAPE);
    len = 0;
    if (!request_rows(a, b, start, n)) n = 0;  // rows that cannot be told are not written
  }
  const int share = a.share;
  const int rows = n * share;
  const int r0 = rb * tiles_a_cta * kPmTile;
  // Tiles of rows that exist, and the 128-token steps that each of them needs.
  int steps[2];
  int kmax = 0;  // tokens that any row sees
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int first = r0 + i * kPmTile;
    steps[i] = 0;
    if (i < tiles_a_cta && first < rows) {
      const int last = div_by(min(rows, first + kPmTile) - 1, share, a.share_inv);
      const int sees = max(0, a.causal ? len - n + last + 1 : len);
      steps[i] = (sees + kPmTile - 1) / kPmTile;
      kmax = max(kmax, sees);
    }
  }
  // This CTA's share of the steps: `most` from step j0 on, and what each tile needs of them.
  const int all = max(steps[0], steps[1]);
  // CTAs that take part: one for every split_steps steps. The others only say that they saw
  // nothing.
  const int splits = max_splits == 1 ? 1 : max(1, min(max_splits, (all + split_steps - 1) / split_steps));
  const bool idle = split >= splits;
  // At most 2^23 steps by 64 CTAs.
  const int j0 = idle || splits == 1 ? 0 : all * split / splits;
  const int most = idle ? 0 : splits == 1 ? all : all * (split + 1) / splits - j0;
  steps[0] = max(0, min(steps[0] - j0, most));
  steps[1] = max(0, min(steps[1] - j0, most));

  if (warp >= kPmDqWarp && warp < kPmMmaWarp) {
    // ---------------- operands: one token a thread ----------------
    const int t = tid - kPmDqWarp * 32;
    const int per_page = a.per_page;
    const int32_t* table = a.table + b * a.ld_table;
    const int run0 = (j0 * kPmTile + t) / 16;
    int col = div_by(run0, per_page, a.page_inv), off = run0 - col * per_page;
    const int dcol = div_by(kPmTile / 16, per_page, a.page_inv), doff = (kPmTile / 16) - dcol * per_page;
    // What every row of the block sees from here on: below it no row is masked.
    const int first_lim = a.causal ? len - n + div_by(r0, share, a.share_inv) + 1 : len;
    uint4 kc[NG], vc[NG];
    uint32_t kp[NG], vp[NG], vq[NG];  // vq: the next step's vp
    int64_t row = 0;  // of this thread's token of the step being fetched; -1 beyond the tokens
    auto find = [&](int j) {
      row = -1;
      if ((j0 + j) * kPmTile + t < kmax) {
        int64_t page = table[col];
        if (page < 0 || page >= a.cache.pages) {
          record_status(QTTS_ERR_SHAPE);
          page = 0;
        }
        row = kv4_row(a.cache, page, kvh, 16 * off + (t & 15));
      }
      col += dcol, off += doff;
      if (off >= per_page) off -= per_page, ++col;
    };
    auto fetch_params = [&](const uint32_t* params, uint32_t(&p)[NG]) {
#pragma unroll
      for (int i = 0; i < NG; ++i) p[i] = 0u;
      if (row >= 0) {
        const uint2* p2 = reinterpret_cast<const uint2*>(params + row * NG);
#pragma unroll
        for (int i = 0; i < NG / 2; ++i) {
          const uint2 x = __ldg(p2 + i);
          p[2 * i] = x.x, p[2 * i + 1] = x.y;
        }
      }
    };
    auto fetch = [&](const uint8_t* codes, uint4(&c)[NG]) {
#pragma unroll
      for (int i = 0; i < NG; ++i) c[i] = make_uint4(0u, 0u, 0u, 0u);
      if (row >= 0) {
        const uint4* c4 = reinterpret_cast<const uint4*>(codes + row * (D / 2));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) c[i] = __ldg(c4 + i);
      }
    };
    // Scales (z = false) or minima (z = true) of two groups as a pair in fp16.
    const auto pair = [&](uint32_t x, uint32_t y, bool z, float up) {
      return z ? pack_f16x2(kv4_min(x) * up, kv4_min(y) * up) : pack_f16x2(kv4_scale(x) * up, kv4_scale(y) * up);
    };
    if (most > 0) {
      find(0);
      fetch_params(a.cache.k_params, kp);
      fetch_params(a.cache.v_params, vp);
      fetch(a.cache.k_codes, kc);
      fetch(a.cache.v_codes, vc);
    }
    // A wait that runs out ends the loop for the whole warp: its reductions and ballots need all lanes.
    const auto wait = [&](uint64_t* bar, int phase) {
      return __all_sync(0xffffffffu, mbar_wait_bounded(bar, phase & 1, wait_ns));
    };
    bool ok = true;
    for (int j = 0; j < most; ++j) {
      const int s = j % kPmStages;
      if ((j0 + j + 1) * kPmTile > first_lim) {
        // Rows that do not see a token must not meet its NaN or infinity (0 * NaN): a token with
        // one among its values becomes zeros there, and NaN in its key for the rows that see it.
        bool bad = false;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          bad = bad || (vp[i] & 0x7F80u) == 0x7F80u || (vp[i] & 0x7F800000u) == 0x7F800000u;
        }
        if (bad) {
#pragma unroll
          for (int i = 0; i < NG; ++i) vp[i] = 0u, kp[i] = 0x7FC07FC0u;
        }
      }
      uint32_t ktop = 0u, vtop = 0u;
#pragma unroll
      for (int i = 0; i < NG; ++i) ktop = max(ktop, group_top(kp[i])), vtop = max(vtop, group_top(vp[i]));
      const int ke = max(16, static_cast<int>(__reduce_max_sync(0xffffffffu, ktop) >> 23) | 7) - 141;
      const int ve = max(16, static_cast<int>(__reduce_max_sync(0xffffffffu, vtop) >> 23) | 7) - 141;
      const float kup = exp2_int(-ke), vup = exp2_int(-ve);
      // Both tiles have read this slot: vempty of step j - 3 was waited for, and it is handed back
      // after P of that step, which is after what this slot held (step j - 4).
      if (lane == 0) {
        units[(j & 3) * 8 + warp - kPmDqWarp] = ke;
        units[(j & 3) * 8 + 4 + warp - kPmDqWarp] = ve;
      }
      ok = j < kPmStages || wait(&kempty[s], j / kPmStages - 1);
      if (!ok) break;
      const uint32_t kt = smem_u32(smem + S::kK) + s * S::kTileBytes;
      const uint32_t vt = smem_u32(smem + S::kV) + s * S::kTileBytes;
      // Keys: word c * NG + g holds channels 32 g + 8 c .. + 7, one group; chunk 4 g + c.
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t sc = pair(kp[g], kp[g], false, kup), z = pair(kp[g], kp[g], true, kup);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int wi = c * NG + g;
          const uint32_t w = reinterpret_cast<const uint32_t*>(kc)[wi];
          sts128(kt + tile_offset(t, 4 * g + c), values(w, 0, sc, z), values(w, 1, sc, z),
                 values(w, 2, sc, z), values(w, 3, sc, z));
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&kfull[s]);
      if (j + 1 < most) {  // the next keys are on their way while the values are made
        find(j + 1);
        fetch_params(a.cache.k_params, kp);
        fetch_params(a.cache.v_params, vq);
        fetch(a.cache.k_codes, kc);
      }
      ok = j < kPmStages || wait(&vempty[s], j / kPmStages - 1);
      if (!ok) break;
      // Values: word wi holds four channels each of two neighbouring groups in its halves.
#pragma unroll
      for (int h = 0; h < NG / 2; ++h) {
        const uint32_t sc = pair(vp[2 * h], vp[2 * h + 1], false, vup);
        const uint32_t z = pair(vp[2 * h], vp[2 * h + 1], true, vup);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int wi = c * (NG / 2) + h;
          const uint32_t w = reinterpret_cast<const uint32_t*>(vc)[wi];
          sts128(vt + tile_offset(t, wi), values(w, 0, sc, z), values(w, 1, sc, z),
                 values(w, 2, sc, z), values(w, 3, sc, z));
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&vfull[s]);
      if (j + 1 < most) {
        fetch(a.cache.v_codes, vc);
#pragma unroll
        for (int i = 0; i < NG; ++i) vp[i] = vq[i];
      }
    }
    if (!ok && lane == 0) record_status(QTTS_ERR_TIMEOUT);
  } else if (warp >= kPmMmaWarp) {
    // ---------------- the products of tile i ----------------
    // The whole warp runs along, so that operands and branches are uniform; one elected lane issues.
    const int i = warp - kPmMmaWarp;
    if (most > 0 && i < tiles_a_cta) {
      const uint32_t qa = smem_u32(smem + S::kQ) + i * S::kTileBytes;
      const uint32_t ka = smem_u32(smem + S::kK), va = smem_u32(smem + S::kV);
      const uint32_t ts = tmem + kColS + i * kPmTile, to = tmem + kColO + i * D;
      const auto wait = [&](uint64_t* bar, int phase) {
        const bool got = __all_sync(0xffffffffu, mbar_wait_bounded(bar, phase & 1, wait_ns));
        tc_fence_after();
        return got;
      };
      // Sub-step u: tokens 64 u .. + 63, half u % 2 of stage (u / 2) % kPmStages. By the elected lane.
      const auto scores = [&](int u) {
        const uint64_t ad = smem_desc_k_sw128(qa);
        const uint64_t bd = smem_desc_k_sw128(ka + (u / 2 % kPmStages) * S::kTileBytes + (u & 1) * (kPmSub * 128));
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t o = ((ks / 4) * (kPmTile * 128) + (ks % 4) * 32) >> 4;
          umma_f16_ss(ts + (u & 1) * kPmSub, ad + o, bd + o, kIdescS, ks != 0 ? 1u : 0u);
        }
        tc_commit(&sfull[2 * i + (u & 1)]);
      };
      const int mine = steps[i];
      bool ok = wait(&qfull[i], 0) && wait(&kfull[0], 0);
      if (ok && elect_one()) {
        if (mine > 0) {
          scores(0);
          scores(1);
        }
        tc_commit(&kempty[0]);
      }
      // A tile that needs fewer steps than the other goes on handing the stages back, each only
      // once it has seen it filled.
      for (int j = 0; ok && j < most; ++j) {
        const int s = j % kPmStages, s1 = (j + 1) % kPmStages;
        ok = wait(&vfull[s], j / kPmStages) && (j + 1 >= most || wait(&kfull[s1], (j + 1) / kPmStages));
        for (int h = 0; ok && h < 2 && j < mine; ++h) {
          const int u = 2 * j + h;
          ok = wait(&pfull[2 * i + h], j);
          if (ok && elect_one()) {
            const uint64_t vd = smem_desc_mn_sw128(va + s * S::kTileBytes + h * (kPmSub * 128), kPmTile * 128, 1024);
#pragma unroll
            for (int ks = 0; ks < kPmSub / 16; ++ks) {
              umma_f16_ts(to, ts + h * kPmSub + 8 * ks, vd + ks * (2048 >> 4), kIdescO, (u | ks) != 0 ? 1u : 0u);
            }
            tc_commit(&odone[i]);
            if (u + 1 == 2 * mine) tc_commit(&ofull[i]);
            if (j + 1 < mine) scores(u + 2);
          }
          __syncwarp();
        }
        if (ok && elect_one()) {
          tc_commit(&vempty[s]);
          if (j + 1 < most) tc_commit(&kempty[s1]);
        }
        __syncwarp();
      }
      // Nothing issued here may outlive the CTA: its last commit has to arrive.
      if (elect_one()) tc_commit(&mdone[i]);
      if (!wait(&mdone[i], 0)) ok = false;
      if (!ok && lane == 0) record_status(QTTS_ERR_TIMEOUT);
    }
  } else {
    // ---------------- softmax: one row a thread ----------------
    const int i = warp >> 2;
    const int r = r0 + i * kPmTile + (tid & 127);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + kColS + i * kPmTile;
    const uint32_t to = tmem + lanes + kColO + i * D;
    const int token = div_by(r, share, a.share_inv), head = kvh * share + r - token * share;
    // What the row sees, from this CTA's first token on.
    const int lim = r < rows ? (a.causal ? len - n + token + 1 : len) - j0 * kPmTile : 0;
    // Tokens that all rows of this tile see (they are in order).
    const int first_lim = (a.causal ? len - n + div_by(r0 + i * kPmTile, share, a.share_inv) + 1 : len) - j0 * kPmTile;
    const bool whole = r0 + i * kPmTile + kPmTile <= rows;
    float to_log2 = a.scale * 1.4426950408889634f;  // from the units of the row's q
    float m = -INFINITY, l = 0.f;
    int vunit = -1000;  // of O, an exponent of two; none yet
    bool ok = true;

    // Rows of a warp as it moves them: kWords lanes a row, the rows' offsets from their lanes.
    constexpr int kRowsAPass = 32 / kWords, kPasses = 32 / kRowsAPass;
    const int ch = lane % kWords, sub = lane / kWords;
    const int tile_row = (warp & 3) * 32;  // the warp's first row of the tile
    // q, channels of a chunk in the order 0 4 1 5 2 6 3 7, all loads of the warp's rows at once:
    // rows beyond the last read the first and are cleared, since loads under a condition of
    // their own were waited for one by one (4 prompts of 2048 tokens: 108 us, against 94 at that step).
    if (most > 0 && i < tiles_a_cta) {
      const int64_t mine = r < rows ? (start + token) * a.q_token_stride + head * a.q_head_stride : -1;
      uint4 v[kPasses];
      uint32_t keep = 0;
#pragma unroll
      for (int x = 0; x < kPasses; ++x) {
        const int64_t from = __shfl_sync(0xffffffffu, mine, x * kRowsAPass + sub);
        v[x] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (from >= 0 ? from : 0) + 8 * ch);
        keep |= from >= 0 ? 1u << x : 0u;
      }
      const uint32_t qt = smem_u32(smem + S::kQ) + i * S::kTileBytes;
#pragma unroll
      for (int x = 0; x < kPasses; ++x) {
        if (!(keep >> x & 1)) v[x] = make_uint4(0u, 0u, 0u, 0u);
        const uint32_t at = qt + tile_offset(tile_row + x * kRowsAPass + sub, ch);
        if constexpr (kQUnits) {
          sts128(at, v[x].x, v[x].y, v[x].z, v[x].w);
        } else {
          sts128(at, __byte_perm(v[x].x, v[x].z, 0x5410), __byte_perm(v[x].x, v[x].z, 0x7632),
                 __byte_perm(v[x].y, v[x].w, 0x5410), __byte_perm(v[x].y, v[x].w, 0x7632));
        }
      }
      if constexpr (kQUnits) {
        // Each thread brings its own row to its unit.
        __syncwarp();
        float top = 0.f;
#pragma unroll 4
        for (int k = 0; k < kWords; ++k) {
          const uint4 e = lds128(qt + tile_offset(tid & 127, k));
          top = fmaxf(fmaxf(top, fmaxf(pair_top(e.x), pair_top(e.y))), fmaxf(pair_top(e.z), pair_top(e.w)));
        }
        const int e = min(100, max(-100, 141 - static_cast<int>(__float_as_uint(top) >> 23)));
        const float up = exp2_int(e);
        to_log2 *= exp2_int(-e);
#pragma unroll 4
        for (int k = 0; k < kWords; ++k) {
          const uint32_t at = qt + tile_offset(tid & 127, k);
          const uint4 x = lds128(at);
          const auto two = [&](uint32_t p, uint32_t q, bool hi) {
            return pack_f16x2(__uint_as_float(hi ? p & 0xffff0000u : p << 16) * up,
                              __uint_as_float(hi ? q & 0xffff0000u : q << 16) * up);
          };
          sts128(at, two(x.x, x.z, false), two(x.x, x.z, true), two(x.y, x.w, false), two(x.y, x.w, true));
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&qfull[i]);
    }
    auto step = [&](int u, bool masked) {
      const int left = lim - u * kPmSub;  // columns that this row sees
      const uint32_t tb = ts + (u & 1) * kPmSub;
      // Factors of the scores of the two halves, and units of their values.
      const volatile int* un = units + (u >> 1 & 3) * 8 + 2 * (u & 1);
      const float to0 = fminf(fmaxf(to_log2 * exp2_int(un[0]), 1e-37f), 1e37f);
      const float to1 = fminf(fmaxf(to_log2 * exp2_int(un[1]), 1e-37f), 1e37f);
      const int v0 = un[4], v1 = un[5];
      uint32_t s[2][32];
      tmem_ld<32>(tb, s[0]);
      tmem_ld<32>(tb + 32, s[1]);
      tc_wait_ld();
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (masked) {
#pragma unroll
        for (int k = 0; k < kPmSub; ++k) s[k / 32][k % 32] = k >= left ? 0xFF800000u : s[k / 32][k % 32];  // -inf
      }
#pragma unroll
      for (int k = 0; k < kPmSub; ++k) {
        float& top = mx4[2 * (k / 32) + k % 2];
        top = fmaxf(top, __uint_as_float(s[k / 32][k % 32]));
      }
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]) * to0, fmaxf(mx4[2], mx4[3]) * to1);  // scale > 0
      const int vmost = max(v0, v1);
      if (__any_sync(0xffffffffu, mx > m + 8.f) || vmost > vunit) {
        const float up = fmaxf(m, mx);
        float f = up > m ? ex2f(m - up) : 1.f;
        m = up;
        l *= f;
        if (vmost > vunit) {
          if (u > 0) f *= exp2_int(max(-126, vunit - vmost));
          vunit = vmost;
        }
        if (u > 0) {
          // S(u) came after O took P(u - 2); it may be taking P(u - 1).
          ok = ok && __all_sync(0xffffffffu, mbar_wait_bounded(&odone[i], (u - 1) & 1, wait_ns));
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld<16>(to + 16 * c, o);
            tc_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tmem_st_x16(to + 16 * c, o);
          }
        }
      }
      const float off = kLift - (m == -INFINITY ? 0.f : m);
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float x = ex2f(fmaf(__uint_as_float(s[c][k]), c ? to1 : to0, off));
          const float y = ex2f(fmaf(__uint_as_float(s[c][k + 1]), c ? to1 : to0, off));
          sum[k / 2 % 2] += x;
          sum[2 + k / 2 % 2] += y;
          p[k / 2] = pack_f16x2(x, y);
        }
        const int d = vunit - (c ? v1 : v0);
        if (d != 0) {  // 2^-d as an fp16 pair, 0 below 2^-24
          const uint32_t g = (d < 15 ? (15 - d) << 10 : d <= 24 ? 1 << (24 - d) : 0) * 0x10001u;
#pragma unroll
          for (int k = 0; k < 16; ++k) asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(p[k]) : "r"(g));
        }
        tmem_st_x16(tb + 16 * c, p);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&pfull[2 * i + (u & 1)]);
    };
    for (int u = 0; ok && u < 2 * steps[i]; ++u) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&sfull[2 * i + (u & 1)], (u / 2) & 1, wait_ns));
      if (!ok) break;
      tc_fence_after();
      step(u, !whole || (u + 1) * kPmSub > first_lim);
    }
    if (ok && steps[i] > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ofull[i], 0, wait_ns));
      tc_fence_after();
    }
    if (!ok && lane == 0) record_status(QTTS_ERR_TIMEOUT);
    if (i < tiles_a_cta && r0 + i * kPmTile < rows) {
      const float unit = steps[i] > 0 ? exp2_int(vunit) : 1.f;
      const float inv = l == 0.f ? 0.f : unit / l;
      // Column 8 wi + 2 x + e of O is channel 32 (2 (wi % (NG/2)) + e) + 4 (wi / (NG/2)) + x: the
      // columns of NG words together are eight channels of every group. A warp's 32 rows go through
      // shared memory (its part of q's tile, which no product reads any more), so that whole
      // rows are stored; lane and chunk are swizzled as in the operand tiles.
      const uint32_t qt = smem_u32(smem + S::kQ) + i * S::kTileBytes;
      const int row = tid & 127;
      const bool part = max_splits > 1;
      // This thread's row of the output, or of the workspace.
      const int64_t out_row = (static_cast<int64_t>(start) + token) * a.q_heads + head;
      const int64_t part_row = out_row * max_splits + split;
      if (part && r < rows) a.stats[part_row] = make_float2(m, l);
#pragma unroll 1
      for (int c = 0; c < D / (8 * NG); ++c) {
        uint32_t o[8 * NG];
        if (steps[i] > 0) {
          if constexpr (NG == 4) {
            tmem_ld<32>(to + 32 * c, o);
          } else {
            tmem_ld<16>(to + 16 * c, o);
          }
          tc_wait_ld();
        } else {
#pragma unroll
          for (int k = 0; k < 8 * NG; ++k) o[k] = 0u;
        }
        if (part && steps[i] == 0) break;
        if (part) {
          // Unnormalized fp32, to be joined: 16 channels of every group are a row of this layout, so
          // the row goes in two halves.
#pragma unroll
          for (int g = 0; g < NG; ++g) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int k = 8 * (q * (NG / 2) + g / 2) + (g & 1);
              const auto out = [&](uint32_t x) { return __float_as_uint(__uint_as_float(x) * unit); };
              sts128(qt + tile_offset(row, 4 * g + 2 * (c & 1) + q), out(o[k]), out(o[k + 2]), out(o[k + 4]),
                     out(o[k + 6]));
            }
          }
          if (c & 1) {
            __syncwarp();
            static_assert(kWords == 4 * NG, "sixteen of a group's channels are four chunks");
#pragma unroll 4
            for (int x = 0; x < kPasses; ++x) {
              const int wrow = x * kRowsAPass + sub;
              const int64_t to_row = __shfl_sync(0xffffffffu, part_row, wrow);
              if (r0 + i * kPmTile + tile_row + wrow < rows) {
                *reinterpret_cast<uint4*>(a.parts + to_row * D + 32 * (ch / 4) + 8 * (c - 1) + 4 * (ch % 4)) =
                    lds128(qt + tile_offset(tile_row + wrow, ch));
              }
            }
            __syncwarp();
          }
          continue;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          T v[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const int wi = (q / 4) * (NG / 2) + g / 2;
            v[q] = from_float<T>(__uint_as_float(o[8 * wi + 2 * (q % 4) + (g & 1)]) * inv);
          }
          const uint4 u = *reinterpret_cast<uint4*>(v);
          sts128(qt + tile_offset(row, 4 * g + c), u.x, u.y, u.z, u.w);
        }
      }
      __syncwarp();
      if (!part) {
        const int64_t dst = (static_cast<int64_t>(start) + token) * a.out_token_stride + head * D;
#pragma unroll
        for (int x0 = 0; x0 < kPasses; x0 += 8) {
          uint4 v[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = lds128(qt + tile_offset(tile_row + (x0 + x) * kRowsAPass + sub, ch));
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const int wrow = (x0 + x) * kRowsAPass + sub;
            const int64_t to_row = __shfl_sync(0xffffffffu, dst, wrow);
            if (r0 + i * kPmTile + tile_row + wrow < rows) {
              *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + to_row + 8 * ch) = v[x];
            }
          }
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == kPmMmaWarp) tmem_dealloc(tmem, 512);
}

template <typename T, int D>
int launch_pm(const Kv4AttnArgs& a, const PromptPlan& p, bool pdl, cudaStream_t stream) {
  constexpr int kSmem = PromptSmem<D>::kBytes;
  if (cudaFuncSetAttribute(kv4_prompt_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) !=
      cudaSuccess) {
    (void)cudaGetLastError();
    return QTTS_ERR_LAUNCH;
  }
  if (p.blocks > 65535) return QTTS_ERR_SHAPE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.cache.kv_heads * p.splits, a.batch, static_cast<unsigned>(p.blocks));
  cfg.blockDim = dim3(kPmThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kv4_prompt_kernel<T, D>, a, p.tiles, p.splits, p.split_steps,
                            current_wait_limit_ns()) == cudaSuccess
             ? QTTS_OK
             : QTTS_ERR_LAUNCH;
}

}  // namespace

PromptPlan plan_prompt(int64_t max_q, int share, int kv_heads, int batch, int64_t most_tokens) {
  PromptPlan p;
  const int64_t rows = max_q * share;
  // Two tiles a CTA share the operands and hide each other's softmax (4 prompts of 2048 tokens,
  // 16 + 2 x 8 heads of 128 channels: 105 us, one tile a CTA 156).
  p.tiles = rows > kPmTile ? 2 : 1;
  p.blocks = (rows + p.tiles * kPmTile - 1) / (p.tiles * kPmTile);
  const int64_t units = p.blocks * kv_heads * batch;
  const int64_t steps = (most_tokens + kPmTile - 1) / kPmTile;
  // Enough CTAs for three a SM, so that long ones among short ones do not hold the call up, but
  // at least four steps each of the longest request (a shorter one takes fewer CTAs). 193 new
  // tokens over 1500 to 5001 earlier ones, three requests of 32 + 2 x 4 heads of 64 channels: 52 us;
  // measured before its operands had units: 47 us, one CTA an SM 52, at least eight steps 48, two
  // steps 47.
  const int64_t want = units >= 2 * kNumSMs ? 1 : (3 * kNumSMs + units - 1) / (units > 0 ? units : 1);
  const int64_t can = steps / 4;
  const int64_t s = want < can ? want : can;
  p.splits = static_cast<int>(s < 1 ? 1 : s > 64 ? 64 : s);
  p.split_steps = static_cast<int>((steps + p.splits - 1) / p.splits);
  return p;
}

int launch_kv4_prompt(const Kv4AttnArgs& a, const PromptPlan& p, int dtype, int head_dim, bool pdl,
                      cudaStream_t stream) {
  if (dtype == QTTS_BF16) {
    return head_dim == 128 ? launch_pm<__nv_bfloat16, 128>(a, p, pdl, stream)
                           : launch_pm<__nv_bfloat16, 64>(a, p, pdl, stream);
  }
  return head_dim == 128 ? launch_pm<__half, 128>(a, p, pdl, stream) : launch_pm<__half, 64>(a, p, pdl, stream);
}

}  // namespace qtts

// The 4-bit key/value cache: its layout and the arithmetic shared by the kernel
// that writes it (rope_kv4.cu) and the kernels that read it.
//
// A key or value row (one token, one head, D channels) is D / 32 groups of 32
// neighbouring channels. A group holds
//   scale = bf16((max - min) / 15),  minimum = bf16(min),
//   code  = clamp(rne((x - minimum) / scale), 0, 15)   (0 where scale is 0)
// and stands for code * scale + minimum. Scale and minimum are rounded first and
// the codes computed against the rounded pair, so that reading adds no error of
// its own; bf16 because a 16-bit pair a group is what the format affords and
// the range of bf16 holds every scale that bf16 activations can have. A NaN or an
// infinity anywhere in a group makes its scale or minimum non-finite: the group
// reads back as non-finite, it is not lost.
//
// Order of the codes in a row (n = D / 32 groups), chosen so that the attention
// kernels' matrix fragments are single wide loads:
//   keys    channel 32j + 8c + i  = nibble i of 32-bit word c * n + j: the lane
//           that feeds quarter c of every group reads its n words at once;
//   values  channel 32j + 4g + i  = nibble i of 16-bit word g * n + j: the lane
//           that feeds rows 4g.. of every group reads its n half-words at once.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace qtts {

constexpr int kKv4Group = 32;

// Row of (page, head, token in page) in the codes and params arrays.
__device__ __forceinline__ int64_t kv4_row(const Kv4Cache& c, int64_t page, int head, int off) {
  return (page * c.kv_heads + head) * static_cast<int64_t>(c.page_size) + off;
}

__device__ __forceinline__ float kv4_scale(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float kv4_min(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// n / d for 0 <= n < 2^31 by inv = (2^32 - 1) / d, rounded down: n inv / 2^32 falls short of the
// quotient by less than one.
__device__ __forceinline__ int div_by(int n, int d, uint32_t inv) {
  const int q = static_cast<int>(__umulhi(static_cast<uint32_t>(n), inv));
  return q + (n - q * d >= d ? 1 : 0);
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

}  // namespace qtts

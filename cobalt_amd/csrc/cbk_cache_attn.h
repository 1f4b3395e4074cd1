// What the attention kernels over the 4-bit cache share: arguments, the workspace, the end of a row.
#pragma once
#include "cbk_cache.h"

namespace cbk {

struct AttnArgs {
  const void* q;                            // [tokens, ratio * heads, D] fp16 or bf16
  void* out;
  int64_t qt, qh, ot, oh;                   // strides of rows and heads, in elements
  int bf;                                   // 1: bf16
  int ratio;                                // query heads on a cache head
  float scale;                              // times log2 e
  int window, sinks;                        // window 0: none
  int least;                                // units a workgroup takes at least
  uint8_t* ws;                              // nullptr: nothing is cut
};

// A tile of rows that begins in a workgroup and ends in a later one: `count` workgroups have a part of it, the first
// in part `slot` of its own, the others in part 0.  count 0: none.
struct AttnPiece { int count, slot, first, row0, valid, head, pad[2]; };

// rows of a part: D sums, the maximum they stand against, the sum of p, padding to 16 bytes
constexpr int attn_row(int dim) { return dim + 4; }
inline size_t attn_bytes(int grid, int rows, int dim) {
  return ((size_t)grid * sizeof(AttnPiece) + 255) / 256 * 256 + (size_t)grid * 2 * rows * attn_row(dim) * sizeof(float);
}
template <int D>
__device__ inline float* attn_part(uint8_t* ws, int64_t grid, int64_t row) {
  return (float*)(ws + (grid * (int64_t)sizeof(AttnPiece) + 255) / 256 * 256) + row * attn_row(D);
}

// four channels of a row: sums over the sum of p, 0 where the row saw nothing
__device__ inline void store_row4(const AttnArgs& a, int row, int head, int d, const float (&y)[4], float sum) {
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* const p = (uint16_t*)a.out + (int64_t)row * a.ot + (int64_t)head * a.oh + d;
  uint2 v;
  if (a.bf) {
    v.x = (uint32_t)f2bf(y[0] * f) | (uint32_t)f2bf(y[1] * f) << 16;
    v.y = (uint32_t)f2bf(y[2] * f) | (uint32_t)f2bf(y[3] * f) << 16;
  } else {
    v.x = (uint32_t)f2h(y[0] * f) | (uint32_t)f2h(y[1] * f) << 16;
    v.y = (uint32_t)f2h(y[2] * f) | (uint32_t)f2h(y[3] * f) << 16;
  }
  *(uint2*)p = v;
}

}  // namespace cbk

// What the attention kernels over the 4-bit cache share: arguments, the workspace, the end of a row.
#pragma once
#include "cbk_cache.h"

namespace cbk {

constexpr float FLOOR = -3.0e38f;           // running maximum before the first token: below every score that is one
constexpr float P_BITS = 8.f, P_SLACK = 6.f;   // p = 2^(t - M + P_BITS) with t <= M + P_SLACK: at most 2^14

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
inline size_t attn_bytes(int grid, int rows, int slots, int dim) {   // slots: parts a workgroup may leave
  return ((size_t)grid * sizeof(AttnPiece) + 255) / 256 * 256 + (size_t)grid * slots * rows * attn_row(dim) * sizeof(float);
}
template <int D>
__device__ inline float* attn_part(uint8_t* ws, int64_t grid, int64_t row) {
  return (float*)(ws + (grid * (int64_t)sizeof(AttnPiece) + 255) / 256 * 256) + row * attn_row(D);
}

__device__ inline int64_t shift_up(int64_t x, int by, int lane) {   // the value of the lane `by` below, 0 at the start
  const int lo = __shfl_up((int)x, by), hi = __shfl_up((int)(x >> 32), by);
  return lane >= by ? (int64_t)hi << 32 | (uint32_t)lo : 0;
}
__device__ inline int64_t of_lane(int64_t x, int l) {
  return (int64_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, l);
}
__device__ inline int64_t scan64(int64_t x, int lane) {             // sum of the lanes up to this one
#pragma unroll
  for (int o = 1; o < 64; o *= 2) x += shift_up(x, o, lane);
  return x;
}

// A product that stays one when something is added to it: the largest score less the maximum is 0 only if both were
// rounded alike, and where scores pass 2^24 nothing else keeps p in range.
__device__ inline float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// 2^e for the largest magnitude of a bf16 row (as bits), and `down` = 2^-e, which brings the row to [1, 2) (e = 127: to [2, 4), 2^-127
// is no normal number); 1 for a row of zeros and one with an infinity or a NaN.
__device__ inline float row_factor(uint32_t big, float& down) {
  int e = max((int)(big >> 23), 1) - 127;
  if (big == 0 || big >= 0x7f800000u) e = 0;
  e = min(e, 126);
  down = __uint_as_float((uint32_t)(127 - e) << 23);
  return __uint_as_float((uint32_t)(e + 127) << 23);
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

// cbk_cache_prompt.hip: many rows a sequence
struct PromptPlan { int parts; int64_t grid; size_t bytes; };
PromptPlan plan_prompt(const DCache&, const DRows&, int ratio);
int launch_cache_prompt(const PromptPlan&, const DCache&, const DRows&, const AttnArgs&, hipStream_t);
// Joins what the `grid` workgroups of a launch left; tiles of `rows` rows begin in every `every`th of them (cbk_cache_attn.hip)
void launch_cache_join(int dim, const AttnArgs&, int grid, int every, int rows, int slots, hipStream_t);

}  // namespace cbk

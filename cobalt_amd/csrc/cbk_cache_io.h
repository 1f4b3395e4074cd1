// What the kernels share that move keys and values between dense tensors and a cache: the sequence of a row, reductions over
// neighbouring lanes, eight 16-bit numbers in and out.
#pragma once
#include <type_traits>
#include "cbk_cache.h"

namespace cbk {

// The sequence that row t (the same in all lanes) belongs to or would: offsets at or before it, less one
__device__ inline int seq_at(const DRows& r, int t, int lane) {
  if (!r.starts) return t / r.per;
  int n = 0;
  for (int j = 0; j < r.seqs + 1; j += 64) {
    const int s = j + lane <= r.seqs ? r.starts[j + lane] : 0x7fffffff;
    n += __popcll(__ballot(s <= t));
  }
  return n - 1;
}

// over N consecutive lanes (a power of two up to 16) that stand aligned: neighbours, pairs, then mirrored quads and eights
template <int N, class F>
__device__ inline float over_lanes(float x, F f) {
  auto by = [&](float v, auto ctrl) { return __uint_as_float(__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), decltype(ctrl)::value, 0xf, 0xf, true)); };
  if constexpr (N > 1) x = f(x, by(x, std::integral_constant<int, 0xB1>{}));
  if constexpr (N > 2) x = f(x, by(x, std::integral_constant<int, 0x4E>{}));
  if constexpr (N > 4) x = f(x, by(x, std::integral_constant<int, 0x141>{}));
  if constexpr (N > 8) x = f(x, by(x, std::integral_constant<int, 0x140>{}));
  return x;
}

template <int DT>
__device__ inline void unpack8(const v4u q, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = q[i];
    const uint16_t lo = (uint16_t)(w & 0xffffu), hi = (uint16_t)(w >> 16);
    x[2 * i] = DT == CBK_F16 ? h2f(lo) : bf2f(lo);
    x[2 * i + 1] = DT == CBK_F16 ? h2f(hi) : __uint_as_float(w & 0xffff0000u);
  }
}
// any NaN among eight 16-bit numbers
template <int DT>
__device__ inline bool any_nan(const v4u q) {
  typedef uint16_t v2s __attribute__((ext_vector_type(2)));
  v2s top = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = q[i] & 0x7fff7fffu;
    top = __builtin_elementwise_max(top, __builtin_bit_cast(v2s, w));
  }
  constexpr uint16_t inf = DT == CBK_F16 ? 0x7c00 : 0x7f80;
  return top.x > inf || top.y > inf;
}

template <int DT>
__device__ inline void store8(void* p, int64_t i, const float (&x)[8]) {
  if (DT == CBK_F32) {
    *(float4*)((float*)p + i) = make_float4(x[0], x[1], x[2], x[3]);
    *(float4*)((float*)p + i + 4) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    v4u o;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] = DT == CBK_F16 ? (uint32_t)f2h(as_float32(x[2 * j])) | (uint32_t)f2h(as_float32(x[2 * j + 1])) << 16
                           : (uint32_t)f2bf(x[2 * j]) | (uint32_t)f2bf(x[2 * j + 1]) << 16;
    __builtin_nontemporal_store(o, (v4u*)((uint16_t*)p + i));
  }
}

}  // namespace cbk

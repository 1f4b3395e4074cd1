// The 8-bit key/value cache as the kernels see it: what a page holds where, how a scale follows from its block's
// values, and how codes become fp16 operands.
//
// A page holds `page` tokens of `heads` heads; part (p, h) is page p's part of head h, p * heads + h.  Of a part, with D
// channels:
//   keys    codes: token-major, D bytes a token
//   values  codes: by four tokens, dword c (channel c) of tokens 4i .. 4i+3 at (i * D + c) * 4.  A matrix instruction that sums
//           over tokens takes for one channel the codes of several tokens from one lane, and finds them in one dword.
//   scales  float32 pairs (keys, values), one for each `block` tokens
// A code is an e4m3 number, a scale a power of two in [2^-15, 2^7], or 0 before a block's first write: every held value is
// an fp16 number, 448 * 2^7 at most.  Codes of values are never NaN: what a row does not see has a weight of 0, and the product is 0.
#pragma once
#include "cbk_cache.h"

namespace cbk {

constexpr float CACHE8_TOP = 57344.f;       // larger magnitudes are held as this one
constexpr float CACHE8_LEAST = 0x1p-15f;    // the smallest scale: its steps, 2^-9 of it, are those of an fp16 subnormal

struct DCache8 {
  uint8_t *kc, *vc;
  float2* sc;
  int64_t pages;
  int page, shift;                          // tokens a page, a power of two, and its logarithm
  int heads, dim, block_shift, blocks;      // of the tokens of a block; blocks a page
};

// Byte offsets of a page's part of head h, and of its scales
struct Parts8 {
  uint32_t code_page, scale_page;
  uint64_t code_head;
  uint32_t scale_head;
  __device__ Parts8(const DCache8& c, int h, int dim)
      : code_page((uint32_t)c.heads * c.page * dim), scale_page((uint32_t)c.heads * c.blocks), code_head((uint64_t)h * c.page * dim),
        scale_head((uint32_t)h * c.blocks) {}
  __device__ uint64_t code(int page) const { return (uint64_t)(uint32_t)page * code_page + code_head; }
  __device__ uint64_t scale(int page) const { return (uint64_t)(uint32_t)page * scale_page + scale_head; }   // in pairs
};

// The smallest power of two s in range with top <= 448 s = 1.75 * 2^8 s (top at most CACHE8_TOP): the exponent one up if the mantissa
// passes 1.75
__device__ inline float scale8(float top) {
  const int e = (int)((__float_as_uint(top) + 0x1fffffu) >> 23) - 8;
  return fmaxf(__uint_as_float((uint32_t)max(e, 1) << 23), CACHE8_LEAST);
}
__device__ inline float reciprocal8(float s) { return __uint_as_float(0x7f000000u - __float_as_uint(s)); }   // of a power of two

// Four e4m3 codes of four numbers of at most 448 (nearest, ties to even, subnormals kept; a NaN is one)
__device__ inline uint32_t codes8(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
typedef float v2f __attribute__((ext_vector_type(2)));
__device__ inline void floats8(uint32_t w, float (&x)[4]) {
  const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}
// Codes under a scale that has grown by 1 / f
__device__ inline uint32_t rescaled8(uint32_t w, float f) {
  float x[4];
  floats8(w, x);
  return codes8(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
}
// Eight codes as fp16 operands, times their scale (a power of two): exact
__device__ inline v8h octet8(uint32_t lo, uint32_t hi, float s_lo, float s_hi) {
  const v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s_lo, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s_lo, true);
  const v2h c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s_hi, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s_hi, true);
  return v8h{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The first n bytes of a dword (the tokens of a quad that are there), of any n
__device__ inline uint32_t bytes_below(int n) { return n >= 4 ? 0xffffffffu : n > 0 ? (1u << (8 * n)) - 1u : 0u; }

// The scales (keys, values) of the block that token `in` of a page stands in (never written by a kernel that reads them so)
__device__ inline float2 scales8(const DCache8& c, uint64_t part, uint32_t in) {
  const uint64_t two = ((const __attribute__((address_space(4))) uint64_t*)c.sc)[part + (in >> c.block_shift)];
  return make_float2(__uint_as_float((uint32_t)two), __uint_as_float((uint32_t)(two >> 32)));
}

}  // namespace cbk

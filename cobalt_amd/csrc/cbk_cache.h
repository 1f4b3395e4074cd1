// The 4-bit key/value cache as the kernels see it: what a page holds where, whose tokens the rows of a call are,
// and how codes become fp16 operands.
//
// A page holds `page` tokens of `heads` heads; block (p, h) is page p's part of head h, p * heads + h.  Of a block,
// with D channels and groups of G of them:
//   keys    codes: token-major, D/2 bytes a token; a dword holds eight consecutive channels, and the dwords stand in the order
//           of key_dword: the lane that multiplies channels 8h .. 8h+7 of every 32 finds its dwords side by side
//   values  codes: by four tokens, dword n (channels 8n .. 8n+7) of tokens 4i .. 4i+3 side by side: 16 bytes at
//           (i * D/8 + n) * 16.  A matrix instruction that sums over tokens takes for one channel the codes of several
//           tokens from one lane, and finds them in one 16-byte load.
//   both    scale and minimum, fp16 each, in one dword: [D/G][page], so that four tokens of a group are 16 bytes
// Inside a dword channel 8w + 2i is nibble i and 8w + 2i + 1 nibble i + 4: one shift and one mask give the two
// halves of a pair of fp16 operands.
#pragma once
#include "cbk_device.h"

namespace cbk {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr float CACHE_TOP = 65280.f;        // larger magnitudes are held as this one: 15 rounded steps above a rounded minimum stay finite

struct DCache {
  uint8_t *kc, *vc;
  uint32_t *km, *vm;
  int64_t pages;
  int page, shift;                          // tokens a page, a power of two, and its logarithm
  int heads, dim, group, groups;
};

struct DRows {
  const int32_t *table, *lens, *starts;     // starts nullptr: `per` rows each
  int64_t ld;
  int seqs, cols, per, tokens;
  int cap;                                  // tokens that `cols` pages hold
};

struct CacheIo {                            // dense side: rows [tokens, heads, D] with unit stride along D
  void *k, *v;
  int64_t kt, kh, vt, vh;                   // strides of rows and heads, in elements
};

// Where channels 8w .. 8w+7 of a key stand among its dwords
template <int D>
__host__ __device__ constexpr int key_dword(int w) {
  return D == 64 ? 2 * (w % 4) + w / 4 : w / 16 * 16 + 4 * (w % 4) + w % 16 / 4;
}

// The rows of sequence b: [first, first + n) of the call, token positions pos0 .. pos0 + n - 1, and the tokens the table
// has pages for.  Its offsets may name rows in front of the call's or behind them: those that are there keep their positions.  Offsets that are
// not ascending give rows that do not belong together, never rows outside the call.
struct Seq { int first, n, pos0, held; };
__device__ inline Seq seq_from(const DRows& r, int s0, int s1, int len) {   // of its two offsets and its length
  Seq s;
  s0 = min(max(s0, 0), r.tokens);
  s1 = max(s1, s0);
  len = max(len, 0);
  s.first = s0; s.n = min(s1, r.tokens) - s0;
  s.pos0 = max(len - (s1 - s0), -(1 << 30));                        // (further down no row of fewer than 2^30 reaches token 0, and windows fit an int)
  s.held = min(len, r.cap);
  return s;
}
__device__ inline Seq seq_of(const DRows& r, int b) {
  int s0 = b * r.per, s1 = s0 + r.per;
  if (r.starts) { s0 = r.starts[b]; s1 = r.starts[b + 1]; }
  return seq_from(r, s0, s1, r.lens[b]);
}

// page of token `pos` (not negative) of sequence b; -1: the table has none
template <class Pool>
__device__ inline int page_of(const Pool& c, const DRows& r, int b, int pos) {
  const int i = pos >> c.shift;
  if (i >= r.cols) return -1;
  const int p = ((const __attribute__((address_space(4))) int32_t*)r.table)[(int64_t)b * r.ld + i];   // (never written by a kernel that reads it)
  return p >= 0 && p < c.pages ? p : -1;
}

// A float32 result that is rounded again: without the barrier the compiler takes one instruction that rounds the exact value to fp16.
__device__ inline float as_float32(float x) {
  asm("" : "+v"(x));
  return x;
}

// ------------------------------------------------------------------ codes to fp16
// The low four bits of each half of a dword (hi: the next four) under the exponent of 2^10 (2^6) are the numbers 1024 + c
// (64 + c), and the difference is c, exactly.  One instruction masks and sets the exponent if the exponent is in a vector register: a
// constant would be a second scalar operand, which this architecture does not take.
struct Exponents { uint32_t lo, hi; };
__device__ inline Exponents exponents() {
  Exponents e;
  asm("v_mov_b32 %0, 0x64006400" : "=v"(e.lo));
  asm("v_mov_b32 %0, 0x54005400" : "=v"(e.hi));
  return e;
}
template <bool HI>
__device__ inline v2h codes_of(uint32_t w, const Exponents& e) {
  const uint32_t u = HI ? ((w & 0x00f000f0u) | e.hi) : ((w & 0x000f000fu) | e.lo);
  const v2h off = HI ? v2h{(_Float16)64.f, (_Float16)64.f} : v2h{(_Float16)1024.f, (_Float16)1024.f};
  return __builtin_bit_cast(v2h, u) - off;
}
// the eight codes of a dword in the order of their channels
__device__ inline v8h code_octet(uint32_t w, const Exponents& e) {
  const uint32_t u = w >> 8;
  const v2h a = codes_of<false>(w, e), b = codes_of<true>(w, e), c = codes_of<false>(u, e), d = codes_of<true>(u, e);
  return v8h{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

}  // namespace cbk

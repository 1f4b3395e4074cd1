// The 4-bit key/value cache as the kernels see it: what a page holds where, whose tokens the rows of a call are,
// and how codes become fp16 operands.
//
// A page holds `page` tokens of `heads` heads; block (p, h) is page p's part of head h, p * heads + h.  Of a block,
// with D channels and groups of G of them:
//   keys    codes: token-major, D/2 bytes a token; dword w of a token holds channels 8w .. 8w+7
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

// The rows of sequence b: [first, first + n) of the call, token positions pos0 .. pos0 + n - 1, and the tokens the table
// has pages for.  Offsets that are not ascending give rows that do not belong together, never rows outside the call.
struct Seq { int first, n, pos0, held; };
__device__ inline Seq seq_of(const DRows& r, int b) {
  Seq s;
  int s0 = b * r.per, s1 = s0 + r.per;
  if (r.starts) { s0 = r.starts[b]; s1 = r.starts[b + 1]; }
  s0 = min(max(s0, 0), r.tokens);
  s1 = min(max(s1, s0), r.tokens);
  const int len = max(r.lens[b], 0);
  s.first = s0; s.n = s1 - s0; s.pos0 = len - s.n;
  s.held = min(len, r.cap);
  return s;
}

// page of token `pos` (not negative) of sequence b; -1: the table has none
__device__ inline int64_t page_of(const DCache& c, const DRows& r, int b, int pos) {
  const int i = pos >> c.shift;
  if (i >= r.cols) return -1;
  const int p = r.table[(int64_t)b * r.ld + i];
  return p >= 0 && p < c.pages ? p : -1;
}

// ------------------------------------------------------------------ codes to fp16
// m + c s for two codes that stand in the low four bits of each half of w (hi: in the next four), rounded once to
// fp16.  The bits under an exponent of 2^10 (2^6) are the number 1024 + c (64 + c); the difference is exact.
template <bool HI>
__device__ inline v2h code_pair(uint32_t w, v2h s, v2h m) {
  const uint32_t u = HI ? ((w & 0x00f000f0u) | 0x54005400u) : ((w & 0x000f000fu) | 0x64006400u);
  const v2h off = HI ? v2h{(_Float16)64.f, (_Float16)64.f} : v2h{(_Float16)1024.f, (_Float16)1024.f};
  const v2h c = __builtin_bit_cast(v2h, u) - off;
  return __builtin_elementwise_fma(c, s, m);
}
__device__ inline v2h pair_of(_Float16 x) { return v2h{x, x}; }

// dword w of a key: its eight channels in order
__device__ inline v8h key_octet(uint32_t w, uint32_t meta) {
  const v2h sm = __builtin_bit_cast(v2h, meta);
  const v2h s = pair_of(sm.x), m = pair_of(sm.y);
  const uint32_t u = w >> 8;
  const v2h a = code_pair<false>(w, s, m), b = code_pair<true>(w, s, m), c = code_pair<false>(u, s, m), d = code_pair<true>(u, s, m);
  return v8h{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

}  // namespace cbk

// What the attention kernels over the 4-bit cache share: arguments, the workspace, the end of a row.
#pragma once
#include "cbk_cache.h"

namespace cbk {

constexpr float FLOOR = -3.0e38f;           // running maximum before the first token: below every score that is one
// p = 2^((t - M) + P_BITS) with t <= M + P_SLACK.  Where scores are so large that float32 holds multiples of 2, 4, 8 ... only, P_BITS rounds to
// 8 at most and P_SLACK to 4, never both up in steps of 8 and 16: p stays below 2^13 whatever the size of M.
constexpr float P_BITS = 7.5f, P_SLACK = 3.5f;

struct AttnArgs {
  const void* q;                            // [tokens, ratio * heads, D] fp16 or bf16
  void* out;
  int64_t qt, qh, ot, oh;                   // strides of rows and heads, in elements
  int bf;                                   // 1: bf16
  int ratio;                                // query heads on a cache head
  float scale;                              // times log2 e
  int window, sinks;                        // window 0: none
  int whole;                                // 1: a tile of rows is one workgroup's
  uint8_t* ws;                              // nullptr: nothing is cut
};

// A tile of rows that begins in a workgroup and ends in a later one: `count` workgroups have a part of it, the first
// in part `slot` of its own, the others in part 0.  count 0: none.
struct AttnPiece { int count, slot, first, row0, valid, head, pad[2]; };

// rows of a part: D sums, the maximum they stand against, the sum of p, padding to 16 bytes
constexpr int attn_row(int dim) { return dim + 4; }
inline size_t attn_bytes(int grid, int rows, int dim) {            // a workgroup may leave two parts
  return ((size_t)grid * sizeof(AttnPiece) + 255) / 256 * 256 + (size_t)grid * 2 * rows * attn_row(dim) * sizeof(float);
}
template <int D>
__device__ inline float* attn_part(uint8_t* ws, int64_t grid, int64_t row) {
  return (float*)(ws + (grid * (int64_t)sizeof(AttnPiece) + 255) / 256 * 256) + row * attn_row(D);
}

__device__ inline int64_t of_lane(int64_t x, int l) {
  return (int64_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, l);
}
__device__ inline Seq of_lane(const Seq& s, int l) {
  return Seq{__builtin_amdgcn_readlane(s.first, l), __builtin_amdgcn_readlane(s.n, l), __builtin_amdgcn_readlane(s.pos0, l), __builtin_amdgcn_readlane(s.held, l)};
}
// The value of another lane: CTRL says of which, lanes without one and rows (of sixteen lanes) that are not in ROWS get 0
template <int CTRL, int ROWS>
__device__ inline int64_t moved(int64_t x) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
  return (int64_t)hi << 32 | (uint32_t)lo;
}
__device__ inline int64_t scan64(int64_t x) {                       // sum of the lanes up to this one; all 64 are there
  x += moved<0x111, 0xf>(x);                                        // 1, 2, 4, 8 lanes on in the row
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  x += moved<0x142, 0xa>(x);                                        // the last lane of the row before, to the second and fourth
  return x + moved<0x143, 0xc>(x);                                  // the last of the first half, to the second
}

// A quotient of numbers that are not negative and nearly always short: a division of 64-bit numbers takes some 150 instructions
// (256 sequences of 300 tokens 33 us, 37 with 64-bit divisions)
__device__ inline int64_t quotient(int64_t a, int64_t b) { return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b); }

// `total` units in `pieces` shares that differ by one at most, the longer ones first
struct Shares {
  int64_t each, more;
  __device__ Shares(int64_t total, int64_t pieces) : each(quotient(total, pieces)), more(total - each * pieces) {}
  __device__ int64_t begin(int64_t place) const { return place * each + min(place, more); }
  __device__ int64_t end(int64_t place) const { return begin(place) + each + (place < more); }
  __device__ int64_t of(int64_t unit) const {                       // the share that has the unit
    const int64_t longer = more * (each + 1);
    return unit < longer ? quotient(unit, each + 1) : more + quotient(unit - longer, each);
  }
};

// The sequences one behind the other, units(b) units of work each.  Every wavefront looks for its place by itself: a lane adds up `each`
// consecutive sequences, one scan gives where they begin, and a second one, among the sequences of the lane that has the place, the sequence.
// (1024 sequences of 300 tokens 140 us; with a scan for every 64 of them 152.)
struct Index {
  int seqs, each, lane;
  int64_t sum, total;                       // units up to the end of this lane's sequences, of all
  template <class F>
  __device__ Index(int seqs_, int lane_, F units) : seqs(seqs_), each((seqs_ + 63) / 64), lane(lane_), sum(0) {
    const int first = lane * each, last = min(first + each, seqs);
#pragma unroll 4
    for (int b = first; b < last; ++b) sum += units(b);
    sum = scan64(sum);
    total = of_lane(sum, 63);
  }
  // the sequence that unit `at` < total is of, and the unit it begins with
  template <class F>
  __device__ int find(int64_t at, int64_t& base, F units) const {
    const int q = __popcll(__ballot(sum <= at));
    base = q ? of_lane(sum, min(q, 64) - 1) : 0;
    if (each == 1 || q == 64) return min(q, seqs - 1);              // (64: lengths or offsets that change under the call)
    const int last = min((q + 1) * each, seqs);
    for (int j = q * each; j < last; j += 64) {
      const int64_t to = scan64(j + lane < last ? units(j + lane) : 0), here = of_lane(to, 63);
      if (at < base + here) {
        const int l = __popcll(__ballot(base + to <= at));
        if (l) base += of_lane(to, l - 1);
        return j + l;
      }
      base += here;
    }
    return seqs - 1;
  }
};

// A product that stays one when something is added to it: the largest score less the maximum is 0 only if both were
// rounded alike, and where scores pass 2^24 nothing else keeps p in range.
__device__ inline float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// What two rounded numbers leave of e0 and e1, exactly: one instruction each, which the compiler makes three of
__device__ inline v2h rest_of(v2h rounded, float e0, float e1) {
  const uint32_t two = __builtin_bit_cast(uint32_t, rounded);
  float r0, r1;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(two), "v"(e0));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(two), "v"(e1));
  return v2h{(_Float16)r0, (_Float16)r1};
}

// Power of two that a query row is divided by, and `down`, its reciprocal, for a largest magnitude `top`: 1 if the row is an ordinary fp16 row
// without it, from 2^-6 to 2^BITS (8 where sums of 128 of its elements are fp16 too), else one that leaves [2^(BITS - 1), 2^BITS): the larger what is
// left, the smaller the elements beside `top` that an fp16 still holds, to 2^-(24 + BITS) of it.  Also 1 for zeros and NaN.  An infinity makes the whole
// row NaN (`down` is): products that are -inf alone would leave a row without weights, which is a row that saw nothing.
template <int BITS = 8>
__device__ inline float row_factor(float top, float& down) {
  int e = 0;
  if (!(top >= 0x1p-6f && top < (float)(1 << BITS)) && top > 0.f && top < __builtin_inff())
    e = max((int)(__float_as_uint(top) >> 23) - 126 - BITS, -126);
  down = top < __builtin_inff() ? __uint_as_float((uint32_t)(127 - e) << 23) : __builtin_nanf("");
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
__device__ inline float bits_top(const v4u& w, bool bf, float top) {  // the largest magnitude of eight numbers and top; a NaN or infinity gives one
  uint32_t big = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t hi = w[i] & 0x7fff0000u, lo = w[i] << 16 & 0x7fff0000u;
    big = max(big, max(lo, hi));
  }
  const uint16_t b = (uint16_t)(big >> 16);
  const float t = bf ? bf2f(b) : h2f(b);
  return t > top || t != t ? t : top;
}

// The tokens a row sees, of those the table may hold: lo .. lo + n - 1 and those before `first`
struct Sight { int lo; uint32_t n; int first; };
__device__ inline Sight sight_of(int pos, int held, const AttnArgs& a) {
  const int hi = min(pos, held - 1);
  Sight s;
  s.lo = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
  s.n = (uint32_t)max(hi - s.lo + 1, 0);
  s.first = a.window > 0 ? min(a.sinks, hi + 1) : 0;
  return s;
}
__device__ inline bool sees(const Sight& s, int token) { return (uint32_t)(token - s.lo) < s.n || token < s.first; }

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

// ------------------------------------------------------------------ few rows: tiles of 16, units of tokens
constexpr int UNIT = 128;                   // tokens: 32 a wavefront
constexpr int EXTRA = 2;                    // units that a tile of rows counts for by itself: its queries, its end (32 ragged sequences: 0: 53 us, 2: 42.5, 4: 42)

struct Range { int units, head, skip; };    // units of a sequence; the first `head` from token 0, the others `skip` units on
__device__ inline Range range_of(const Seq& s, const AttnArgs& a) {
  Range g{0, 0, 0};
  if (s.n <= 0) return g;
  const int all = max((s.held + UNIT - 1) / UNIT, 1);
  if (a.window > 0) {
    const int lo = min(max(s.pos0 - a.window + 1, 0) / UNIT, all - 1);
    g.head = min((a.sinks + UNIT - 1) / UNIT, lo);
    g.skip = lo - g.head;
  }
  g.units = all - g.skip;
  return g;
}

__device__ inline int64_t units_of(const Seq& s, const AttnArgs& a, int heads, int rows) {
  const int64_t tiles = ((int64_t)s.n * a.ratio + rows - 1) / rows;
  return tiles * heads * (a.whole ? 1 : range_of(s, a).units + EXTRA);
}
// Over the four quarters of the wavefront, without the trip through LDS: neighbouring quarters side by side, then the halves
struct Two { float a, b; };
__device__ inline Two quarters(float x) {
  const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return Two{__uint_as_float(t[0]), __uint_as_float(t[1])};
}
__device__ inline Two halves(float x) {
  const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return Two{__uint_as_float(t[0]), __uint_as_float(t[1])};
}
__device__ inline float across_max(float x) {
  const Two q = quarters(x), h = halves(fmaxf(q.a, q.b));
  return fmaxf(h.a, h.b);
}
__device__ inline float across_sum(float x) {
  const Two q = quarters(x), h = halves(q.a + q.b);
  return h.a + h.b;
}

// ------------------------------------------------------------------ many rows: tiles of 256
constexpr int WAVES = 8, ROWS = 32 * WAVES;
constexpr int CHIP = 256;                   // workgroups that run at once: one a CU

__device__ inline int row_tiles(const Seq& s, int ratio) { return (int)(((int64_t)s.n * ratio + ROWS - 1) / ROWS); }

// What tiles of rows weigh when the list is cut: the tokens they see, times the query heads of a cache head so that no fraction is lost.  Only
// the balance rests on it, not what is computed: a piece of a tile's weight is that piece of its tokens, rounded to tiles.
struct Weights {
  int ratio, window, sinks;
  int64_t own;                               // what a tile of rows weighs by itself
  __device__ int64_t first(const Seq& s) const { return (int64_t)max(s.pos0, 0) * ratio; }
  __device__ int64_t flat() const { return own + ROWS + (int64_t)ratio * ((int64_t)window + sinks); }
  __device__ int64_t of(const Seq& s, int i) const { return window > 0 ? flat() : own + first(s) + (int64_t)(i + 1) * ROWS; }
  __device__ int64_t before(const Seq& s, int i) const { return window > 0 ? i * flat() : i * (own + first(s)) + (int64_t)i * (i + 1) / 2 * ROWS; }
  __device__ int64_t all(const Seq& s) const { return s.n > 0 ? before(s, row_tiles(s, ratio)) : 0; }
};

// cbk_cache_prompt.hip: many rows a sequence
struct PromptPlan { bool cut; int64_t grid; size_t bytes; };
PromptPlan plan_prompt(const DCache&, const DRows&, int ratio);
int launch_cache_prompt(const PromptPlan&, const DCache&, const DRows&, const AttnArgs&, hipStream_t);
// Joins what the `grid` workgroups of a launch left of tiles of `rows` rows, 16, 32 or 256 (cbk_cache_attn.hip)
void launch_cache_join(int dim, const AttnArgs&, int grid, int rows, hipStream_t, bool wide = false);   // wide: few tiles in hundreds of parts

}  // namespace cbk

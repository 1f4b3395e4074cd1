// Attention over the 4-bit cache for many rows a sequence: prompts, and chunks of them behind what the cache holds.
//
// The formulas are those of cbk_cache_attn.hip; here the products bound the time, so the cache's tiles are widened to fp16 once
// per workgroup and read from LDS by all of its wavefronts.  A workgroup has 256 rows (tokens times the query heads on one cache
// head), 32 a wavefront, as the columns of 32 x 32 x 16 products: S^T = K Q^T and O^T = V^T P^T.  The sums of S^T lie in
// the lanes that P^T wants them in, eight registers a product, if its tokens are numbered 4h + r of the first and of the second
// eight; values are stored to LDS in that order, and keys and values both as whole operands (lane after lane, 16 bytes), so that every
// LDS read is a run of 1 KB without bank conflicts.
//
// While the products of a tile run, the next one, whose codes were loaded a tile before, is widened into the other half of
// LDS: four wavefronts take the keys, four the values, 16 tokens of (at most) 128 channels each.  One barrier for a tile's two blocks.
//
// bf16 results: keys m + c s rounded once to fp16, p rounded to fp16 (both far below the result's own step).  fp16 results: keys
// as their codes with one product a group, multiplied by the token's scale in float32, the minima in a product of their own, and p
// with its rest as a second operand.
//
// Work is dealt out in one of two ways (plan_prompt).  Whole: a workgroup per tile of rows, the longest first.  Cut: as many
// workgroups as the chip holds, each with an equal share of the one list of all tiles of rows and their tokens; what a workgroup has
// of a tile that it does not finish is joined by the second launch of cbk_cache_attn.hip.
//
// A 4096-token prompt of 32 query heads on 8, 128 channels, bf16: 170 us, 810 TFLOP/s; 8192 tokens 590 us, 930 (a large library product
// reaches 1210); fp16, with its half more of products, 860 to 1040 us by the group.  64 channels 815 us (bf16) and 1190 (fp16; groups of 32: 1350) for twice the
// heads, whose bound is the vector unit: an exponential and five instructions a score.  Matrix unit busy 36 %, vector unit 46 %; the bare loop
// of products would take 104 of the 170 us, widening 13 to 35 of them, reads from LDS 31 to 35, exponentials 6 to 9.  256 rows
// a workgroup, because widening is shared by all rows; two blocks of 64 tokens a barrier (one: 180 us).  Built and not kept: the two
// halves of the wavefronts a phase apart (200 against 178 us), two workgroups a CU for 64 channels, which spills (1035 against 745).
#include <type_traits>
#include "cbk_cache.h"
#include "cbk_cache_attn.h"

namespace cbk {

constexpr int WAVES = 8, ROWS = 32 * WAVES;
constexpr int OWN = 2;                      // tiles of tokens that a tile of rows counts for by itself: its queries, its start and end (six ragged
                                            // chunks: none 470 us, 1: 445, 2: 433, 4: 431; a prompt of 8192 tokens, cut: 774, 669, 631, 631)
constexpr float REST = 2048.f;              // What the first fp16 leaves of a sum of q is kept this many times as large, and meets minima that many times smaller: with a small
                                            // scale in it the rest has no digits as an fp16 (2^-25 of a minimum of 60000 is 2e-3 of a score; now 2^-36, and 2^-25 of the sum)
constexpr int CHIP = 256;                   // workgroups that run at once: one a CU

template <int D, int G, bool BF>
struct Tile {
  static constexpr int BLOCK = D == 256 ? 32 : 64, NU = 2;          // tokens whose scores are in registers at a time; of those a tile has NU
  static constexpr int KEYS = NU * BLOCK;                           // tokens of a tile
  static constexpr int KT = BLOCK / 32, KS = D / 16, GS = D / G, GP = G / 16;   // 32-token products of a block, products of a row, groups, products of a group
  static constexpr int VS = BLOCK / 16, VT = D / 32;                // products along a block's tokens, 32-channel blocks
  static constexpr int UG = (D < 128 ? D : 128) / G;                // groups of a wavefront's share of the keys
  static constexpr int K_BYTES = KEYS * D * 2, V_BYTES = KEYS * D * 2;
  static constexpr int M_BYTES = BF ? 0 : KEYS / 32 * 1024, S_BYTES = BF ? 0 : GS * KEYS * 4;   // minima as an operand, scales (float)
  static constexpr int BYTES = K_BYTES + V_BYTES + M_BYTES + S_BYTES + 16;   // and a byte for each sixteen: its page is there
};

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

template <int D, int G, bool BF>
__global__ __launch_bounds__(64 * WAVES, 2) void cache_prompt_kernel(DCache c, DRows r, AttnArgs a, int cut) {
  using T = Tile<D, G, BF>;
  __shared__ v4u lds4[2 * T::BYTES / 16];
  uint8_t* const lds = (uint8_t*)lds4;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const Exponents ex = exponents();

  // ---- this workgroup's share: tile `tile` of head h of sequence b, or units [at, end) of the list
  const Weights wt{a.ratio, a.window, a.sinks, (int64_t)OWN * T::KEYS * a.ratio};
  AttnPiece* desc = nullptr;
  int64_t base = 0, at = 0, end = 0, begin = 0, total = 0, pieces = 0, place = 0;
  int h, b, tile = 0;
  bool joined = false;
  if (!cut) {                                                       // heads fastest: an XCD meets few of them; a sequence's last tiles first
    h = blockIdx.x % c.heads;
    const int64_t item = blockIdx.x / c.heads;
    auto units = [&](int b) { return (int64_t)row_tiles(seq_of(r, b), a.ratio); };
    const Index list(r.seqs, lane, units);
    if (item >= list.total) return;
    b = list.find(item, base, units);
    tile = row_tiles(seq_of(r, b), a.ratio) - 1 - (int)(item - base);
  } else {                                                          // workgroups of an XCD are neighbours in the list: a head's tokens stay in its L2
    place = gridDim.x % 8 ? blockIdx.x : (int64_t)(blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
    desc = (AttnPiece*)a.ws + place;
    auto units = [&](int b) { return wt.all(seq_of(r, b)); };
    const Index list(r.seqs, lane, units);
    const int64_t one = list.total;                                 // units of a head
    total = one * c.heads;
    pieces = total ? min((int64_t)gridDim.x, max(total / ((int64_t)T::KEYS * a.ratio), (int64_t)1)) : 0;   // (0: no sequence has a row)
    if (place >= pieces) {
      if (tid == 0) desc->count = 0;
      return;
    }
    const Shares shares(total, pieces);
    begin = at = shares.begin(place);
    end = shares.end(place);
    h = (int)(begin / one);
    b = list.find(begin - h * one, base, units);
    base += h * one;
    const Seq s = seq_of(r, b);                                     // its tile: the last that begins at or before
    int lo = 0, hi = row_tiles(s, a.ratio) - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (base + wt.before(s, mid) <= begin) lo = mid; else hi = mid - 1;
    }
    tile = lo;
  }

  for (;;) {
  const Seq s = seq_of(r, b);
  const int rows = s.n * a.ratio, row0 = tile * ROWS, valid = min(ROWS, rows - row0);
  const int pos_lo = s.pos0 + row0 / a.ratio, pos_hi = s.pos0 + (row0 + valid - 1) / a.ratio;

  // ---- its tiles of tokens: the first `head`, then the others `skip` on; of them t0 .. t1 - 1
  int all = max((min(s.held, pos_hi + 1) + T::KEYS - 1) / T::KEYS, 1), head = 0, skip = 0;
  if (a.window > 0) {
    const int lo = min(max(pos_lo - a.window + 1, 0) / T::KEYS, all - 1);
    head = min((a.sinks + T::KEYS - 1) / T::KEYS, lo);
    skip = lo - head;
    all -= skip;
  }
  int t0 = 0, t1 = all;
  bool whole_tile = true;
  int64_t first_unit = 0, units = 0;
  if (cut) {
    first_unit = base + wt.before(s, tile);
    units = wt.of(s, tile);
    const int64_t x0 = at - first_unit, x1 = min(units, end - first_unit);
    auto tiles_before = [&](int64_t x) { return x == units ? all : min((int)((double)x / (double)units * all), all); };
    t0 = tiles_before(x0);
    t1 = tiles_before(x1);
    whole_tile = x0 == 0 && x1 == units;
  }
  auto token_of = [&](int t) { return (t < head ? t : t + skip) * T::KEYS; };

  // ---- queries
  const int wrow0 = row0 + 32 * wave, wvalid = min(32, rows - wrow0);   // (none: not positive)
  const int wpos_lo = s.pos0 + wrow0 / a.ratio, wpos_hi = s.pos0 + (wrow0 + max(wvalid, 1) - 1) / a.ratio;
  const bool is = col < wvalid;
  const int tok_q = is ? (wrow0 + col) / a.ratio : 0, head_q = h * a.ratio + (is ? (wrow0 + col) % a.ratio : 0);
  const int pos = is ? s.pos0 + tok_q : wpos_hi;
  const uint16_t* const qp = (const uint16_t*)a.q + (int64_t)(s.first + tok_q) * a.qt + (int64_t)head_q * a.qh;
  const Sight sight = sight_of(pos, s.held, a);
  // The scale of the scores is in the queries (bf16) or in the scales and sums that meet them (fp16, unless it would take those
  // out of range); `grow` is what is left to multiply with.
  const float fold = BF || a.scale <= 2.f ? a.scale : 1.f;
  v8h q[T::KS], qm;
  float grow;
  {
    v4u raw[T::KS];
    float top = 0.f, down;
#pragma unroll
    for (int k = 0; k < T::KS; ++k) {
      raw[k] = is ? *(const v4u*)(qp + 16 * k + 8 * half) : v4u{};
      top = bits_top(raw[k], BF, top);
    }
    top = fmaxf(top, __shfl_xor(top, 32));
    const float size = BF && top < __builtin_inff() ? fminf(top * fold, 0x1.fffffep127f) : top;   // (of what `times` leaves)
    grow = row_factor(size, down) * (a.scale / fold);
    const float times = BF ? fold : 1.f;
#pragma unroll
    for (int k = 0; k < T::KS; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t two = raw[k][i];
        const float x0 = BF ? __uint_as_float(two << 16) : h2f((uint16_t)two), x1 = BF ? __uint_as_float(two & 0xffff0000u) : h2f((uint16_t)(two >> 16));
        q[k][2 * i] = (_Float16)(x0 * down * times);
        q[k][2 * i + 1] = (_Float16)(x1 * down * times);
      }
  }
  if constexpr (!BF) {
#pragma unroll
    for (int i = 0; i < 8; ++i) qm[i] = (_Float16)0.f;
#pragma unroll
    for (int g = 0; g < T::GS; ++g) {
      float sum = 0.f;
#pragma unroll
      for (int k = g * T::GP; k < (g + 1) * T::GP; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += (float)q[k][i];
      sum = as_float32((sum + __shfl_xor(sum, 32)) * fold);         // (rounded one way for both: their first halves have to be the same)
      const _Float16 hi = (_Float16)sum;
      if (half == g / 4) { qm[2 * (g % 4)] = hi; qm[2 * (g % 4) + 1] = (_Float16)((sum - (float)hi) * REST); }
    }
  }
  // Scores start from `start`, P_BITS less the running maximum, so that a sum is p's exponent as it leaves the product.  Rows with
  // something left to multiply with, maxima so large that adding to them rounds, and rows that have seen nothing take the steps one by one.
  const bool plain = __ballot(grow != 1.f) == 0;
  bool ready = false;
  float start = 0.f;

  // ---- the share of a tile that this wavefront widens: keys (0 - 3) or values (4 - 7)
  const bool takes_keys = wave < 4;
  const int sub = D == 256 ? wave & 1 : wave & 3, chunk = D == 256 ? wave >> 1 & 1 : 0;
  const int c16 = lane & 15, h4 = lane >> 4, block = (h4 & 1) << 1 | h4 >> 1;   // block: the four tokens of the sixteen whose values the lane takes
  const uint32_t code_page = (uint32_t)c.heads * c.page * (D / 2), meta_page = (uint32_t)c.heads * c.page * (T::GS * 4);
  const uint8_t* const codes = (takes_keys ? c.kc : c.vc) + (int64_t)h * c.page * (D / 2);
  const uint8_t* const metas = (const uint8_t*)(takes_keys ? c.km : c.vm) + (int64_t)h * c.page * (T::GS * 4);
  const int n8 = D == 64 ? c16 & 7 : c16 + 16 * chunk;             // the dword of a value's eight channels
  const uint32_t code_at = takes_keys ? c16 * (D / 2) + 64 * chunk + h4 * (D == 64 ? 8 : 16) : block * (2 * D) + n8 * 16;
  v4u code[T::NU];
  uint32_t meta[T::NU][4];
  int limit[T::NU], page_next[T::NU];                               // limit: tokens of the sixteen that are there
  auto pages_at = [&](int t) {
#pragma unroll
    for (int u = 0; u < T::NU; ++u) {
      const int tok = token_of(t) + 16 * (sub + T::VS * u);
      page_next[u] = tok < s.held ? page_of(c, r, b, tok) : -1;
    }
  };
  auto fetch = [&](int t) {                                         // the pages of t are in page_next
#pragma unroll
    for (int u = 0; u < T::NU; ++u) {
      const int tok = token_of(t) + 16 * (sub + T::VS * u);
      const uint32_t in = tok & (c.page - 1), p = max(page_next[u], 0);
      const uint8_t* cp = codes + ((uint64_t)p * code_page + in * (D / 2)) + code_at;
      const uint8_t* mp = metas + ((uint64_t)p * meta_page + in * 4);
      limit[u] = page_next[u] < 0 ? 0 : s.held - tok;
      if (takes_keys) {
        if constexpr (D == 64) {
          const v2u two = *(const v2u*)cp;
          code[u] = v4u{two.x, two.y, 0, 0};
        } else {
          code[u] = *(const v4u*)cp;
        }
        if constexpr (BF) {
#pragma unroll
          for (int g = 0; g < T::UG; ++g) meta[u][g] = *(const uint32_t*)(mp + 4 * ((T::UG * chunk + g) * c.page + c16));
        } else {
          meta[u][0] = *(const uint32_t*)(mp + 4 * ((T::UG * chunk + min(h4, T::UG - 1)) * c.page + c16));
        }
      } else {
        code[u] = *(const v4u*)cp;
        const v4u four = *(const v4u*)(mp + 4 * ((8 * n8 / G) * c.page + 4 * block));
#pragma unroll
        for (int i = 0; i < 4; ++i) meta[u][i] = four[i];
      }
    }
  };
  auto widen = [&](uint8_t* buf, auto unit) {
    constexpr int u = decltype(unit)::value;
    const int sb = sub + T::VS * u;
    if (takes_keys) {
      if (lane == 0) *(uint8_t*)(buf + T::BYTES - 16 + sb) = limit[u] > 0;
      uint8_t* const to = buf + (sb >> 1) * (T::KS * 1024) + (h4 & 1) * 512 + (16 * (sb & 1) + c16) * 16 + ((h4 >> 1) + 8 * chunk) * 1024;
#pragma unroll
      for (int j = 0; j < (D == 64 ? 2 : 4); ++j) {
        v8h f = code_octet(code[u][j], ex);
        if constexpr (BF) {
          const v2h sm = __builtin_bit_cast(v2h, meta[u][j * 32 / G]);
          const v8h s8 = {sm.x, sm.x, sm.x, sm.x, sm.x, sm.x, sm.x, sm.x}, m8 = {sm.y, sm.y, sm.y, sm.y, sm.y, sm.y, sm.y, sm.y};
          f = __builtin_elementwise_fma(f, s8, m8);
        }
        *(v8h*)(to + 2 * j * 1024) = f;
      }
      if constexpr (!BF)
        if (h4 < T::UG) {
          const int g = T::UG * chunk + h4, key = 16 * sb + c16;
          uint8_t* const mins = buf + T::K_BYTES + T::V_BYTES;
          const _Float16 least = __builtin_bit_cast(v2h, meta[u][0]).y;
          *(v2h*)(mins + (key >> 5) * 1024 + (g >> 2) * 512 + (key & 31) * 16 + (g & 3) * 4) = v2h{least, least * (_Float16)(1.f / REST)};
          *(float*)(mins + T::M_BYTES + (g * T::KEYS + key) * 4) = h2f((uint16_t)meta[u][0]) * fold;
        }
    } else {
      if (limit[u] < 16)
#pragma unroll
        for (int i = 0; i < 4; ++i) meta[u][i] = 4 * block + i < limit[u] ? meta[u][i] : 0;   // whatever stands there: its value is 0
      v2h s2[2], m2[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s2[i] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(meta[u][2 * i + 1], meta[u][2 * i], 0x05040100u));
        m2[i] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(meta[u][2 * i + 1], meta[u][2 * i], 0x07060302u));
      }
      uint8_t* const to = buf + T::K_BYTES + sb * (T::VT * 1024) + (block & 1) * 512 + (block >> 1) * 8;
#pragma unroll
      for (int by = 0; by < 4; ++by) {
        uint32_t pr[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t w0 = D == 64 ? code[u][2 * i] >> (4 * (c16 >> 3)) : code[u][2 * i], w1 = D == 64 ? code[u][2 * i + 1] >> (4 * (c16 >> 3)) : code[u][2 * i + 1];
          pr[i] = __builtin_amdgcn_perm(w1, w0, 0x0c040c00u + by * 0x00010001u);
        }
        auto put = [&](int nibble, v2h x, v2h y) {
          const int at = n8 + (D / 8) * nibble;                     // row of V^T
          typedef _Float16 v4h __attribute__((ext_vector_type(4)));
          *(v4h*)(to + (at >> 5) * 1024 + (at & 31) * 16) = v4h{x.x, x.y, y.x, y.y};
        };
        put(D == 64 ? 2 * by + (c16 >> 3) : 2 * by, __builtin_elementwise_fma(codes_of<false>(pr[0], ex), s2[0], m2[0]),
            __builtin_elementwise_fma(codes_of<false>(pr[1], ex), s2[1], m2[1]));
        if constexpr (D > 64)
          put(2 * by + 1, __builtin_elementwise_fma(codes_of<true>(pr[0], ex), s2[0], m2[0]),
              __builtin_elementwise_fma(codes_of<true>(pr[1], ex), s2[1], m2[1]));
      }
    }
  };

  v16f o[T::VT];
  float m = FLOOR, l = 0.f;
#pragma unroll
  for (int t = 0; t < T::VT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;

  __syncthreads();                                                  // (the reads of the last tile of rows)
  if constexpr (!BF) {                                              // operand slots of groups that are not: 0, not what LDS holds
    for (int i = tid; i < T::M_BYTES / 4; i += 64 * WAVES) {
      *(uint32_t*)(lds + T::K_BYTES + T::V_BYTES + 4 * i) = 0;
      *(uint32_t*)(lds + T::BYTES + T::K_BYTES + T::V_BYTES + 4 * i) = 0;
    }
    __syncthreads();
  }
  if (t0 < t1) {
    pages_at(t0);
    fetch(t0);
    widen(lds, std::integral_constant<int, 0>{});
    widen(lds, std::integral_constant<int, 1>{});
    if (t0 + 1 < t1) {
      pages_at(t0 + 1);
      fetch(t0 + 1);
      pages_at(min(t0 + 2, t1 - 1));
    }
  }
  __syncthreads();

  for (int t = t0; t < t1; ++t) {
    uint8_t* const buf = lds + ((t - t0) & 1) * T::BYTES;
    const v2u flags = *(const v2u*)(buf + T::BYTES - 16);
    auto block = [&](auto which) {
    constexpr int hb = decltype(which)::value;
    const int tok = token_of(t) + hb * T::BLOCK;
    const bool mine = wvalid > 0 && tok <= wpos_hi && (a.window <= 0 || tok + T::BLOCK > wpos_lo - a.window + 1 || tok < a.sinks);
    v16f sc[T::KT];
    if (mine) {
      const uint8_t* const from = buf + lane * 16;
#pragma unroll
      for (int kt = 0; kt < T::KT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[kt][i] = start;
      if constexpr (BF) {
#pragma unroll
        for (int k = 0; k < T::KS; ++k)
#pragma unroll
          for (int kt = 0; kt < T::KT; ++kt)
            sc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const v8h*)(from + ((hb * T::KT + kt) * T::KS + k) * 1024), q[k], sc[kt], 0, 0, 0);
      } else {
        const uint8_t* const mins = buf + T::K_BYTES + T::V_BYTES;
#pragma unroll
        for (int kt = 0; kt < T::KT; ++kt) {
          sc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const v8h*)(mins + (hb * T::KT + kt) * 1024 + lane * 16), qm, sc[kt], 0, 0, 0);
#pragma unroll
          for (int g = 0; g < T::GS; ++g) {
            v16f sum;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[i] = 0.f;
#pragma unroll
            for (int k = g * T::GP; k < (g + 1) * T::GP; ++k)
              sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const v8h*)(from + ((hb * T::KT + kt) * T::KS + k) * 1024), q[k], sum, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const v4f four = *(const v4f*)(mins + T::M_BYTES + (g * T::KEYS + hb * T::BLOCK + 32 * kt + 8 * i + 4 * half) * 4);
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[kt][4 * i + e] = fmaf(four[e], sum[4 * i + e], sc[kt][4 * i + e]);
            }
          }
        }
      }
    }
    if (t + 1 < t1) widen(lds + ((t + 1 - t0) & 1) * T::BYTES, which);
    if (mine) {
      // every row of the wavefront sees all tokens of the tile, and all of them are there
      bool whole = tok + T::BLOCK <= s.held && tok + T::BLOCK - 1 <= wpos_lo && (a.window <= 0 || tok > wpos_hi - a.window || tok + T::BLOCK <= a.sinks);
      uint32_t there = (uint32_t)__builtin_amdgcn_readfirstlane((int)(T::BLOCK == 64 && hb ? flags.y : flags.x));   // a byte a sixteen
      if constexpr (T::BLOCK == 32) there = (hb ? there >> 16 : there & 0xffffu) | 0x01010000u;
      whole = whole && there == 0x01010101u;
      if (!whole) {
#pragma unroll
        for (int kt = 0; kt < T::KT; ++kt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const bool held = there >> (8 * (2 * kt + j)) & 1;
            const uint32_t n = held ? sight.n : 0;
            const int first = held ? sight.first : 0;
#pragma unroll
            for (int i = 8 * j; i < 8 * j + 8; ++i) {
              const int key = tok + 32 * kt + 8 * (i >> 2) + 4 * half + (i & 3);
              sc[kt][i] = sees(Sight{sight.lo, n, first}, key) ? sc[kt][i] : -__builtin_inff();
            }
          }
      }
      float top = -__builtin_inff();
#pragma unroll
      for (int kt = 0; kt < T::KT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[kt][i]);
      top = fmaxf(top, __shfl_xor(top, 32));
      if (!ready || __ballot(top > P_BITS + P_SLACK)) {             // the maximum follows when p would leave its range
        const float g = ready ? 1.f : grow;
        const float up = fmaxf(m, rounded_product(top, g) - start), f = __builtin_amdgcn_exp2f(m - up);
        m = up;
        l *= f;
#pragma unroll
        for (int v = 0; v < T::VT; ++v) o[v] *= f;
        const float less = ready ? (m + start) - P_BITS : m, more = ready ? 0.f : P_BITS;   // (less the maximum first: it may dwarf P_BITS)
#pragma unroll
        for (int kt = 0; kt < T::KT; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[kt][i] = (rounded_product(sc[kt][i], g) - less) + more;
        ready = plain && __ballot(!(fabsf(m) < 0x1p15f)) == 0;
        start = ready ? P_BITS - m : 0.f;
      }
      // p of sixteen tokens while the products of the sixteen before run
      v8h p[2], rest[2];
      auto weights = [&](int st) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e0 = __builtin_amdgcn_exp2f(sc[st >> 1][8 * (st & 1) + 2 * i]), e1 = __builtin_amdgcn_exp2f(sc[st >> 1][8 * (st & 1) + 2 * i + 1]);
          const v2h ph = {(_Float16)e0, (_Float16)e1};
          p[st & 1][2 * i] = ph.x; p[st & 1][2 * i + 1] = ph.y;
          l = __builtin_amdgcn_fdot2(ph, v2h{(_Float16)1.f, (_Float16)1.f}, l, false);
          if constexpr (!BF) {
            const v2h pl = rest_of(ph, e0, e1);
            rest[st & 1][2 * i] = pl.x; rest[st & 1][2 * i + 1] = pl.y;
            l = __builtin_amdgcn_fdot2(pl, v2h{(_Float16)1.f, (_Float16)1.f}, l, false);
          }
        }
      };
      weights(0);
#pragma unroll
      for (int st = 0; st < T::VS; ++st) {
        const uint8_t* const from = buf + T::K_BYTES + (hb * T::VS + st) * (T::VT * 1024) + lane * 16;
        if (st + 1 < T::VS) weights(st + 1);
#pragma unroll
        for (int v = 0; v < T::VT; ++v) {
          const v8h f = *(const v8h*)(from + v * 1024);
          o[v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, p[st & 1], o[v], 0, 0, 0);
          if constexpr (!BF) o[v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, rest[st & 1], o[v], 0, 0, 0);
        }
      }
    }
    };
    block(std::integral_constant<int, 0>{});
    block(std::integral_constant<int, 1>{});
    if (t + 2 < t1) {
      fetch(t + 2);
      pages_at(min(t + 3, t1 - 1));
    }
    __syncthreads();
  }

  // ---- the ends of the rows
  l += __shfl_xor(l, 32);
  const int slot = at == begin ? 0 : 1;
  if (!whole_tile && at == first_unit) {                            // this workgroup begins the tile: it is joined from here
    joined = true;
    if (tid == 0) {
      desc->first = s.first; desc->row0 = row0; desc->valid = valid; desc->head = h; desc->slot = slot;
      desc->count = (int)(Shares(total, pieces).of(first_unit + units - 1) - place + 1);
    }
  }
  if (is) {
    float* const out = whole_tile ? nullptr : attn_part<D>(a.ws, gridDim.x, (place * 2 + slot) * ROWS + 32 * wave + col);
    const float f = l == 0.f ? 0.f : 1.f / l;
    constexpr int NS = D / 16;                                      // eights of channels a lane holds
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int rr = i & 3, aa = i >> 2, n = 8 * aa + 4 * half + rr;
      float x[8];
#pragma unroll
      for (int ch = 0; ch < 8; ++ch) {
        const int j = ch / 2 + 4 * (ch & 1);                        // the nibble of channel 8n + ch
        x[ch] = D == 64 ? o[j >> 2][4 * (j & 3) + rr] : D == 128 ? o[j >> 1][4 * (aa + 2 * (j & 1)) + rr] : o[j % T::VT][4 * aa + rr];
      }
      if (!whole_tile) {
        *(float4*)(out + 8 * n) = make_float4(x[0], x[1], x[2], x[3]);
        *(float4*)(out + 8 * n + 4) = make_float4(x[4], x[5], x[6], x[7]);
      } else {
        uint16_t* const p = (uint16_t*)a.out + (int64_t)(s.first + tok_q) * a.ot + (int64_t)head_q * a.oh + 8 * n;
        v4u y;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          y[j] = BF ? (uint32_t)f2bf(x[2 * j] * f) | (uint32_t)f2bf(x[2 * j + 1] * f) << 16
                    : (uint32_t)f2h(x[2 * j] * f) | (uint32_t)f2h(x[2 * j + 1] * f) << 16;
        *(v4u*)p = y;
      }
    }
    if (!whole_tile && half == 0) { out[D] = m; out[D + 1] = l; }
  }
  if (!cut) return;

  // ---- the next tile of the list
  at = min(end, first_unit + units);
  if (at >= end) break;
  if (tile + 1 < row_tiles(s, a.ratio)) {
    ++tile;
  } else {
    base += wt.all(s);
    tile = 0;
    do {
      if (++b == r.seqs) { b = 0; ++h; }
    } while (h < c.heads && seq_of(r, b).n <= 0);
    if (h == c.heads) break;                                        // (there is one, unless lengths change under the call)
  }
  }
  if (!joined && tid == 0) desc->count = 0;
}

// ------------------------------------------------------------------ launch
PromptPlan plan_prompt(const DCache& c, const DRows& r, int ratio) {
  PromptPlan p;
  // Whole tiles where there are enough of them or where they are prompts, whose tiles are of all lengths and fill the chip one behind the
  // other; equal shares where a few tiles stand behind long histories.  128 channels, 8 cache heads of 4 query heads, bf16, whole against cut:
  // prompts of 1024 tokens 45 and 56 us, of 2048 80 and 88, of 4096 172 and 199; the last 512 of 2048 tokens 73 and 55, of 16384 512 and 173;
  // the last 1024 of 4096 139 and 103; six ragged chunks (590 tiles) 515 and 507 (64 channels, fp16, 3 query heads: 444 and 380); 8 x 1000 of
  // 6000 (1060 tiles) 825 and 833.
  const int64_t tiles = ((int64_t)r.tokens * ratio / ROWS + r.seqs) * c.heads;   // at most
  const bool prompts = 2 * (int64_t)r.tokens > (int64_t)r.cap * r.seqs;          // most of what the table can hold is new
  p.cut = !prompts && tiles < 3 * CHIP;
  p.grid = p.cut ? CHIP : tiles;
  p.bytes = p.cut ? attn_bytes((int)p.grid, ROWS, c.dim) : 0;
  return p;
}

template <int D, int G, bool BF>
static int prompt3(const PromptPlan& p, const DCache& c, const DRows& r, const AttnArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((cache_prompt_kernel<D, G, BF>), dim3((unsigned)p.grid), dim3(64 * WAVES), 0, st, c, r, a, (int)p.cut);
  return CBK_OK;
}
template <int D, int G>
static int prompt2(const PromptPlan& p, const DCache& c, const DRows& r, const AttnArgs& a, hipStream_t st) {
  return a.bf ? prompt3<D, G, true>(p, c, r, a, st) : prompt3<D, G, false>(p, c, r, a, st);
}
template <int D>
static int prompt1(const PromptPlan& p, const DCache& c, const DRows& r, const AttnArgs& a, hipStream_t st) {
  if (c.group == 32) return prompt2<D, 32>(p, c, r, a, st);
  if (c.group == 64) return prompt2<D, 64>(p, c, r, a, st);
  if constexpr (D > 64) return prompt2<D, 128>(p, c, r, a, st);
  return CBK_ERR_LAYOUT;
}
int launch_cache_prompt(const PromptPlan& p, const DCache& c, const DRows& r, const AttnArgs& a, hipStream_t st) {
  const int rc = c.dim == 64 ? prompt1<64>(p, c, r, a, st) : c.dim == 128 ? prompt1<128>(p, c, r, a, st) : prompt1<256>(p, c, r, a, st);
  if (rc) return rc;
  if (p.cut) launch_cache_join(c.dim, a, (int)p.grid, ROWS, st);
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

}  // namespace cbk

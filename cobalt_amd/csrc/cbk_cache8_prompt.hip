// Attention over the 8-bit cache for many rows a sequence: prompts, and chunks of them behind what the cache holds.
//
// The formulas are those of cbk_cache8_attn.hip; here the products bound the time, so the cache's tiles are widened to fp16 once
// per workgroup (exactly: held values are fp16 numbers) and read from LDS by all of its wavefronts.  A workgroup has 256 rows (tokens times the
// query heads on one cache head), 32 a wavefront, as the columns of 32 x 32 x 16 products: S^T = K Q^T and O^T = V^T P^T.  The sums of S^T lie in
// the lanes that P^T wants them in, eight registers a product, if its tokens are numbered 4h + r of the first and of the second
// eight; values are stored to LDS in that order, and keys and values both as whole operands (lane after lane, 16 bytes), so that every
// LDS read is a run of 1 KB without bank conflicts.  Which channels a block of V^T has is free: those whose stores by neighbouring lanes lie
// side by side.
//
// While the products of a tile run, the next one, whose codes were loaded before, is widened into the other half of LDS: four
// wavefronts take the keys, four the values, 16 tokens of (at most) 128 channels each, half a tile at a time.  A SIMD has one of either.  Keys
// are widened in front of a block, values behind it, so that one wavefront multiplies while the other one does not; products go first
// (s_setprio).  (Both behind the scores' products: 168 us for the 4096-token prompt below, apart 160, with priorities 157.)  One barrier for a tile's two blocks.
//
// bf16 results: queries with the scale of the scores in them and p rounded once to fp16 (an eighth of the result's own step).  fp16 results: queries as
// they are, and p with its rest as a second operand.
//
// Work is dealt out in one of two ways (chosen in cbk_cache8_attn.hip).  Whole: a workgroup per tile of rows, the longest first.  Cut: as many
// workgroups as the chip holds, each with an equal share of the one list of all tiles of rows and their tokens; what a workgroup has
// of a tile that it does not finish is joined by the second launch (cbk_cache_attn.hip).
//
// A 4096-token prompt of 32 query heads on 8, 128 channels: bf16 155 us, 890 TFLOP/s (a large library product reaches 1200), fp16 230 us with its half more
// products; of 8192 tokens and 64 channels 366 and 555 us, where an exponential and five instructions a score bound it; 4096 tokens of 16 heads on
// 4, 256 channels, 242 and 316 us.
#include <type_traits>
#include "cbk_cache8.h"
#include "cbk_cache_attn.h"
#include "cbk_cache8_attn.h"

namespace cbk {

constexpr int OWN8 = 2;                     // tiles of tokens that a tile of rows counts for by itself: its queries, its start and end

// The larger of a lane's number and that of the lane 32 on (not through LDS, which the stores of the next tile keep busy)
__device__ inline float halves_max(float x) {
  const Two h = halves(x);
  return fmaxf(h.a, h.b);
}

template <int D>
struct Tile8 {
  static constexpr int BLOCK = D == 256 ? 32 : 64, NU = 2;          // tokens whose scores are in registers at a time; of those a tile has NU
  static constexpr int KEYS = NU * BLOCK;                           // tokens of a tile
  static constexpr int KT = BLOCK / 32, KS = D / 16;                // 32-token products of a block, products of a row
  static constexpr int VS = BLOCK / 16, VT = D / 32;                // products along a block's tokens, 32-channel blocks
  static constexpr int PIECES = (D < 128 ? D : 128) / 64;           // 16-byte loads of a wavefront's share
  static constexpr int K_BYTES = KEYS * D * 2, V_BYTES = KEYS * D * 2;
  static constexpr int BYTES = K_BYTES + V_BYTES + 16;              // and a byte for each sixteen: its page is there
};

template <int D, bool BF>
__global__ __launch_bounds__(64 * WAVES, 2) void cache8_prompt_kernel(DCache8 c, DRows r, AttnArgs a, int cut) {
  using T = Tile8<D>;
  __shared__ v4u lds4[2 * T::BYTES / 16];
  uint8_t* const lds = (uint8_t*)lds4;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;

  // ---- this workgroup's share: tile `tile` of head h of sequence b, or units [at, end) of the list
  const Weights wt{a.ratio, a.window, a.sinks, (int64_t)OWN8 * T::KEYS * a.ratio};
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

  // ---- the share of a tile that this wavefront widens: keys (0 - 3) or values (4 - 7), a sixteen of a block, of 256 channels a half
  const bool takes_keys = wave < 4;
  const int sub = D == 256 ? wave & 1 : wave & 3, chunk = D == 256 ? wave >> 1 & 1 : 0;
  const int c16 = lane & 15, h4 = lane >> 4, four = (h4 & 1) << 1 | h4 >> 1;   // four: the tokens of the sixteen whose values the lane takes
  const Parts8 part(c, h, D);
  const uint8_t* const codes = takes_keys ? c.kc : c.vc;
  const uint32_t code_at = takes_keys ? c16 * D + 128 * chunk + h4 * 16 : (four * D + 32 * (4 * chunk)) * 4 + c16 * 16;
  v4u code[T::NU][T::PIECES];
  float scale[T::NU];
  int page_first[T::NU], page_next[T::NU];
  int limit[T::NU];                                                 // tokens of the sixteen that are there
  auto pages_at = [&](int t, int (&page)[T::NU]) {
#pragma unroll
    for (int u = 0; u < T::NU; ++u) {
      const int tok = token_of(t) + 16 * (sub + T::VS * u);
      page[u] = tok < s.held ? page_of(c, r, b, tok) : -1;
    }
  };
  auto fetch = [&](int t, const int (&page)[T::NU]) {
#pragma unroll
    for (int u = 0; u < T::NU; ++u) {
      const int tok = token_of(t) + 16 * (sub + T::VS * u);
      const uint32_t in = tok & (c.page - 1);
      const int p = max(page[u], 0);
      const uint8_t* const cp = codes + (part.code(p) + in * D) + code_at;
      const float2 two = scales8(c, part.scale(p), in);
      scale[u] = takes_keys ? two.x : two.y;
      limit[u] = page[u] < 0 ? 0 : s.held - tok;
#pragma unroll
      for (int j = 0; j < T::PIECES; ++j) code[u][j] = *(const v4u*)(cp + (takes_keys ? 64 : 256) * j);
    }
  };
  // The first codes are on their way while the queries are made ready (behind one another: 157.9 against 156.4 us for the 4096-token prompt)
  if (t0 < t1) {
    pages_at(t0, page_first);
    pages_at(min(t0 + 1, t1 - 1), page_next);
  }

  // ---- queries
  const int wrow0 = row0 + 32 * wave, wvalid = min(32, rows - wrow0);   // (none: not positive)
  const int wpos_lo = s.pos0 + wrow0 / a.ratio, wpos_hi = s.pos0 + (wrow0 + max(wvalid, 1) - 1) / a.ratio;
  const bool is = col < wvalid;
  const int tok_q = is ? (wrow0 + col) / a.ratio : 0, head_q = h * a.ratio + (is ? (wrow0 + col) % a.ratio : 0);
  const int pos = is ? s.pos0 + tok_q : wpos_hi;
  const uint16_t* const qp = (const uint16_t*)a.q + (int64_t)(s.first + tok_q) * a.qt + (int64_t)head_q * a.qh;
  const Sight sight = sight_of(pos, s.held, a);
  // The scale of the scores is in the queries (bf16), or meets the scores (fp16) in `grow`, which also has what the queries were divided by.
  v8h q[T::KS];
  float grow;
  {
    v4u raw[T::KS];
    float top = 0.f, down;
#pragma unroll
    for (int k = 0; k < T::KS; ++k) raw[k] = is ? *(const v4u*)(qp + 16 * k + 8 * half) : v4u{};
    if (t0 < t1) fetch(t0, page_first);
#pragma unroll
    for (int k = 0; k < T::KS; ++k) top = bits_top(raw[k], BF, top);
    top = fmaxf(top, __shfl_xor(top, 32));
    const float times = BF ? a.scale : 1.f;
    const float size = BF && top < __builtin_inff() ? fminf(top * times, 0x1.fffffep127f) : top;   // (of what `times` leaves)
    grow = row_factor8<BF>(size, down) * (BF ? 1.f : a.scale);
    if (!BF) grow = fminf(fmaxf(grow, 1e-30f), 0x1.fffffep127f);    // (a smaller one has every score at 0, a larger one every difference past any weight)
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
  // bf16: scores start from `start`, P_BITS less the running maximum, so that a sum is p's exponent as it leaves the product; fp16: one
  // instruction a score multiplies and adds.  Rows with something left to multiply with (bf16), maxima so large that adding to them rounds, and rows
  // that have seen nothing take the steps one by one.
  [[maybe_unused]] const bool plain = __ballot(grow != 1.f) == 0;
  bool ready = false;
  float start = 0.f;

  auto widen = [&](uint8_t* buf, auto unit) {
    constexpr int u = decltype(unit)::value;
    const int sb = sub + T::VS * u;
    if (takes_keys) {                                               // 16 channels a piece: both eights of product 4 j + h4
      if (lane == 0) *(uint8_t*)(buf + T::BYTES - 16 + sb) = limit[u] > 0;
      uint8_t* const to = buf + (sb >> 1) * (T::KS * 1024) + (8 * chunk + h4) * 1024 + (16 * (sb & 1) + c16) * 16;
#pragma unroll
      for (int j = 0; j < T::PIECES; ++j) {
        *(v8h*)(to + 4 * j * 1024) = octet8(code[u][j][0], code[u][j][1], scale[u], scale[u]);
        *(v8h*)(to + 4 * j * 1024 + 512) = octet8(code[u][j][2], code[u][j][3], scale[u], scale[u]);
      }
    } else {                                                        // four tokens of channels 64 j + 4 n + i: row 16 (i & 1) + n of block 2 j + (i >> 1)
      if (limit[u] < 16)
#pragma unroll
        for (int j = 0; j < T::PIECES; ++j) code[u][j] &= bytes_below(limit[u] - 4 * four);   // whatever stands there: its value is 0
      uint8_t* const to = buf + T::K_BYTES + sb * (T::VT * 1024) + 4 * chunk * 1024 + (four & 1) * 512 + (four >> 1) * 8 + c16 * 16;
#pragma unroll
      for (int j = 0; j < T::PIECES; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          typedef _Float16 v4h __attribute__((ext_vector_type(4)));
          const v2h x = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(code[u][j][i], scale[u], false);
          const v2h y = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(code[u][j][i], scale[u], true);
          *(v4h*)(to + (2 * j + (i >> 1)) * 1024 + (i & 1) * 256) = v4h{x.x, x.y, y.x, y.y};
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
  if (t0 < t1) {
    widen(lds, std::integral_constant<int, 0>{});
    widen(lds, std::integral_constant<int, 1>{});
    if (t0 + 1 < t1) {
      fetch(t0 + 1, page_next);
      pages_at(min(t0 + 2, t1 - 1), page_next);
    }
  }
  __syncthreads();

  for (int t = t0; t < t1; ++t) {
    uint8_t* const buf = lds + ((t - t0) & 1) * T::BYTES;
    uint8_t* const next = lds + ((t + 1 - t0) & 1) * T::BYTES;
    const v2u flags = *(const v2u*)(buf + T::BYTES - 16);
    auto block = [&](auto which) {
    constexpr int hb = decltype(which)::value;
    const int tok = token_of(t) + hb * T::BLOCK;
    const bool mine = wvalid > 0 && tok <= wpos_hi && (a.window <= 0 || tok + T::BLOCK > wpos_lo - a.window + 1 || tok < a.sinks);
    v16f sc[T::KT];
    if (takes_keys && t + 1 < t1) {                                 // in front of the block: the other wavefront of the SIMD multiplies meanwhile
      widen(next, which);
      if (hb == 1 && t + 2 < t1) {
        fetch(t + 2, page_next);
        pages_at(min(t + 3, t1 - 1), page_next);
      }
    }
    if (mine) {
      __builtin_amdgcn_s_setprio(1);
      const uint8_t* const from = buf + lane * 16;
#pragma unroll
      for (int kt = 0; kt < T::KT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[kt][i] = BF ? start : 0.f;
#pragma unroll
      for (int k = 0; k < T::KS; ++k)
#pragma unroll
        for (int kt = 0; kt < T::KT; ++kt)
          sc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const v8h*)(from + ((hb * T::KT + kt) * T::KS + k) * 1024), q[k], sc[kt], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(0);
      asm volatile("s_nop 3");                                      // (the scores are looked at next: on every path as far behind the products as the build wants it)
    }
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
      top = halves_max(top);
      if constexpr (BF) {
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
      } else {
        const float high = rounded_product(top, grow);
        if (!ready || __ballot(high > m + P_SLACK)) {
          const float up = fmaxf(m, high), f = __builtin_amdgcn_exp2f(m - up);
          m = up;
          l *= f;
#pragma unroll
          for (int v = 0; v < T::VT; ++v) o[v] *= f;
          ready = __ballot(!(fabsf(m) < 0x1p15f)) == 0;
          start = P_BITS - m;
        }
#pragma unroll
        for (int kt = 0; kt < T::KT; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[kt][i] = ready ? fmaf(sc[kt][i], grow, start) : (rounded_product(sc[kt][i], grow) - m) + P_BITS;
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
      __builtin_amdgcn_s_setprio(1);
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
      __builtin_amdgcn_s_setprio(0);
    }
    if (!takes_keys && t + 1 < t1) {                                // behind it
      widen(next, which);
      if (hb == 1 && t + 2 < t1) {
        fetch(t + 2, page_next);
        pages_at(min(t + 3, t1 - 1), page_next);
      }
    }
    };
    block(std::integral_constant<int, 0>{});
    block(std::integral_constant<int, 1>{});
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
#pragma unroll
    for (int j = 0; j < D / 64; ++j)
#pragma unroll
      for (int hi = 0; hi < 2; ++hi)
#pragma unroll
        for (int rr = 0; rr < 4; rr += 2) {                         // n = 8 hi + 4 half + rr and the next: channels 64 j + 4 n ..
          const int d = 64 * j + 32 * hi + 16 * half + 4 * rr;
          float x[8];
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) x[ch] = o[2 * j + (ch >> 1 & 1)][4 * (2 * (ch & 1) + hi) + rr + (ch >> 2)];
          if (!whole_tile) {
            *(float4*)(out + d) = make_float4(x[0], x[1], x[2], x[3]);
            *(float4*)(out + d + 4) = make_float4(x[4], x[5], x[6], x[7]);
          } else {
            uint16_t* const p = (uint16_t*)a.out + (int64_t)(s.first + tok_q) * a.ot + (int64_t)head_q * a.oh + d;
            v4u y;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              y[i] = BF ? (uint32_t)f2bf(x[2 * i] * f) | (uint32_t)f2bf(x[2 * i + 1] * f) << 16
                        : (uint32_t)f2h(x[2 * i] * f) | (uint32_t)f2h(x[2 * i + 1] * f) << 16;
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
PromptPlan plan_prompt8(const DCache8& c, const DRows& r, int ratio, bool cut) {
  PromptPlan p;
  const int64_t tiles = ((int64_t)r.tokens * ratio / ROWS + r.seqs) * c.heads;   // at most
  p.cut = cut;
  p.grid = cut ? CHIP : tiles;
  p.bytes = cut ? attn_bytes((int)p.grid, ROWS, c.dim) : 0;
  return p;
}

template <int D>
static void prompt(const PromptPlan& p, const DCache8& c, const DRows& r, const AttnArgs& a, hipStream_t st) {
  if (a.bf) hipLaunchKernelGGL((cache8_prompt_kernel<D, true>), dim3((unsigned)p.grid), dim3(64 * WAVES), 0, st, c, r, a, (int)p.cut);
  else hipLaunchKernelGGL((cache8_prompt_kernel<D, false>), dim3((unsigned)p.grid), dim3(64 * WAVES), 0, st, c, r, a, (int)p.cut);
}
int launch_cache8_prompt(const PromptPlan& p, const DCache8& c, const DRows& r, const AttnArgs& a, hipStream_t st) {
  if (c.dim == 64) prompt<64>(p, c, r, a, st);
  else if (c.dim == 128) prompt<128>(p, c, r, a, st);
  else prompt<256>(p, c, r, a, st);
  if (p.cut) launch_cache_join(c.dim, a, (int)p.grid, ROWS, st);
  return hipGetLastError() == hipSuccess ? CBK_OK : CBK_ERR_HIP;
}

}  // namespace cbk
